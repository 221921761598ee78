"""Pages with several holders (q4_gpu_pages_fork, _release) and pools that are cut (q4_gpu_pages_compact) against a plain restatement on lists; the rows that the
requests hold through it all; edges; what is refused."""
import ctypes
import random

import pytest
import torch

import q4gpu
from gpu_util import lib

pytestmark = pytest.mark.gpu
KINDS = {"q8_0": q4gpu.KIND_Q8, "f16": q4gpu.KIND_F16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Plain:
    """the pool on lists; every page's rows are the numbers that were appended to it"""

    def __init__(self, n_pages, page, n_req, stride):
        self.page, self.n_pages, self.stride = page, n_pages, stride
        self.free = list(range(n_pages - 1, -1, -1))
        self.shares = [0] * n_pages
        self.table = [[-1] * stride for _ in range(n_req)]
        self.rows = [0] * n_req
        self.data = {}                                                   # (page, row in it) -> number

    def pages(self, rows):
        return -(-rows // self.page)

    def add(self, r, numbers):
        for x in numbers:
            if self.rows[r] % self.page == 0:
                self.table[r][self.rows[r] // self.page] = self.free.pop()
            self.data[self.table[r][self.rows[r] // self.page], self.rows[r] % self.page] = x
            self.rows[r] += 1

    def held(self, r):
        return [self.data[self.table[r][p // self.page], p % self.page] for p in range(self.rows[r])]

    def fork(self, src, dst, length):
        rows, table, bits, full, named = list(self.rows), [list(t) for t in self.table], 0, False, set()
        for s, d, n in zip(src, dst, length):
            first = d not in named
            if 0 <= d < len(rows):
                named.add(d)
            if not (0 <= s < len(rows) and 0 <= d < len(rows) and first and 0 <= n <= max(rows[s], 0) and rows[s] <= self.stride * self.page and rows[d] <= 0):
                bits |= 4
                continue
            if full or (n % self.page and not self.free):
                full, bits = True, bits | 8
                continue
            for i in range(n // self.page):
                self.table[d][i] = table[s][i]
                if 0 <= table[s][i] < self.n_pages:
                    self.shares[table[s][i]] += 1
                else:
                    bits |= 4
            if n % self.page:
                old, new = table[s][n // self.page], self.free.pop()
                self.table[d][n // self.page] = new
                if not 0 <= old < self.n_pages:
                    bits |= 4
                for i in range(min(self.page, -(-(n % self.page) // 16) * 16)):
                    if (old, i) in self.data:
                        self.data[new, i] = self.data[old, i]
            self.rows[d] = n
        return bits

    def release(self, keep):
        bits, given, after = 0, [], list(self.rows)
        for r, (h, k) in enumerate(zip(self.rows, keep)):
            k = max(k, 0)
            if h > self.stride * self.page:
                bits |= 4
            elif 0 < h and k < h:
                p = self.table[r][k // self.page] if k % self.page else -1
                if 0 <= p < self.n_pages and self.shares[p] > 0:
                    bits |= 4
                    continue
                given += self.table[r][self.pages(k): self.pages(h)]
                after[r] = k
        if any(not 0 <= p < self.n_pages or given.count(p) > self.shares[p] + 1 for p in given):
            return bits | 4
        gone, shares = [], list(self.shares)
        for i, p in enumerate(given):
            if shares[p] == 0:
                gone.append(p)
            else:
                shares[p] -= 1
        if len(self.free) + len(gone) > self.n_pages:
            return bits | 4
        self.free += gone[::-1]
        self.shares, self.rows = shares, after
        return bits

    def compact(self):
        live, free = self.n_pages - len(self.free), set(self.free)
        if len(free) != len(self.free) or any(not 0 <= p < self.n_pages for p in free):
            return list(range(self.n_pages)), 4
        number = [-1 if p in free else p for p in range(self.n_pages)]
        for hole, p in zip([p for p in range(live) if p in free], [p for p in range(live, self.n_pages) if p not in free]):
            number[p] = hole
            self.shares[hole], self.shares[p] = self.shares[p], 0
            for i in range(self.page):
                if (p, i) in self.data:
                    self.data[hole, i] = self.data[p, i]
        bits = 0
        for r, h in enumerate(self.rows):
            for i in range(self.pages(h)):
                p = self.table[r][i]
                if 0 <= p < self.n_pages and number[p] >= 0:
                    self.table[r][i] = number[p]
                else:
                    bits = 4
        self.free = list(range(self.n_pages - 1, live - 1, -1))
        return number, bits


class Both:
    """the same on the GPU"""

    def __init__(self, n_pages=40, page=16, n_req=12, stride=20, layers=2, n_kvh=2, hd=64, kind="q8_0"):
        self.p = Plain(n_pages, page, n_req, stride)
        self.pool = q4gpu.PagePool(layers, n_kvh, hd, n_pages, page, KINDS[kind])
        self.pool.mem.fill_(0xff)
        self.table, self.rows = ints(self.p.table), ints(self.p.rows)
        self.layers, self.width, self.count, self.kind = layers, n_kvh * hd, 0, kind
        lib().q4_gpu_last_error()

    def values(self, numbers, layer):
        """K and V of rows that stand for numbers, exact in a pool of q8_0 (all of a block alike: code 127, and a step that fp16 holds)"""
        x = torch.tensor(numbers, dtype=torch.float32, device="cuda")[:, None].expand(-1, self.width)
        return ((x + layer * 7) % 1024 * 127 * 2.0**-10).contiguous(), (-(x * 3 + layer) % 1024 * 127 * 2.0**-10).contiguous()

    def add(self, add):
        """a step: new rows for every request"""
        n = sum(add)
        if not n:
            return
        start = torch.zeros(len(add) + 1, dtype=torch.int32, device="cuda")
        slot, pos, req = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
        self.pool.plan(self.rows, ints(add), self.table, start, slot, pos, req)
        numbers = list(range(self.count, self.count + n))
        for layer in range(self.layers):
            self.pool.append(layer, *self.values(numbers, layer), slot)
        at = 0
        for r, k in enumerate(add):
            self.p.add(r, numbers[at: at + k])
            at += k
        self.count += n
        self.rows += ints(add)
        assert lib().q4_gpu_last_error() == 0

    def fork(self, src, dst, length):
        bits = self.p.fork(src, dst, length)
        self.pool.fork(self.rows, ints(src), ints(dst), ints(length), self.table)
        assert lib().q4_gpu_last_error() == bits
        return self.check()

    def release(self, keep):
        bits = self.p.release(keep)
        self.pool.release(self.rows, ints(keep), self.table)
        assert lib().q4_gpu_last_error() == bits
        return self.check()

    def compact(self):
        number, bits = self.p.compact()
        got = torch.full((self.pool.n_pages,), -9, dtype=torch.int32, device="cuda")
        self.pool.compact(self.rows, self.table, got)
        assert lib().q4_gpu_last_error() == bits
        assert got.tolist() == number
        return self.check()

    def check(self):
        assert self.rows.tolist() == self.p.rows
        assert self.table.tolist() == self.p.table
        assert self.pool.free[: int(self.pool.n_free[0])].tolist() == self.p.free
        n = self.pool.n_pages
        assert self.pool.shares.tolist() == self.p.shares + [0] * (2 * n)
        return self

    def check_rows(self):
        slots, numbers = [], []
        for r, h in enumerate(self.p.rows):
            slots += [self.p.table[r][i // self.p.page] * self.p.page + i % self.p.page for i in range(h)]
            numbers += self.p.held(r)
        if slots:
            for layer in range(self.layers):
                k, v = torch.empty(2, len(slots), self.width, device="cuda")
                self.pool.gather(layer, ints(slots), k, v)
                want = self.values(numbers, layer)
                if self.kind == "f16":                                   # 127 k 2^-10 has more bits than fp16: rows are rounded as they are appended, to numbers that still differ
                    want = [x.half().float() for x in want]
                assert torch.equal(k, want[0]) and torch.equal(v, want[1])
        return self


@pytest.mark.parametrize("kind,page,hd,n_kvh,layers", [("q8_0", 16, 64, 2, 2), ("f16", 16, 64, 1, 3), ("q8_0", 64, 128, 2, 1), ("f16", 32, 256, 1, 2), ("q8_0", 128, 256, 3, 1), ("f16", 256, 128, 2, 1)])
@pytest.mark.parametrize("seed", range(3))
def test_a_long_run(kind, page, hd, n_kvh, layers, seed):
    """requests come, fork, grow, are rewound and go, and the pool is compacted now and then"""
    rng = random.Random(seed)
    n_req = 14
    b = Both(n_pages=60, page=page, n_req=n_req, stride=9, layers=layers, n_kvh=n_kvh, hd=hd, kind=kind)
    for step in range(60):
        what = rng.choice(["add", "add", "fork", "fork", "release", "compact"])
        rows = list(b.p.rows)
        if what == "add":
            left, add = len(b.p.free), [0] * n_req
            for r in rng.sample(range(n_req), 6):
                n = rng.choice([1, 3, page, rng.randint(1, 2 * page)])
                if (rows[r] == 0 and rng.random() < 0.5) or rows[r] + n > 9 * page:
                    continue
                need = b.p.pages(rows[r] + n) - b.p.pages(rows[r])
                if need <= left:
                    add[r] = n
                    left -= need
            b.add(add)
        elif what == "fork":
            src = [r for r in range(n_req) if rows[r]]
            dst = [r for r in range(n_req) if not rows[r]]
            n = min(len(dst), rng.randint(1, 4)) if src else 0
            if n:
                s = [rng.choice(src) for _ in range(n)]
                b.fork(s, rng.sample(dst, n), [rng.choice([rows[r], rng.randint(0, rows[r]), rows[r] // page * page]) for r in s])
        elif what == "release":
            b.release([rng.choice([h, h, h, 0, rng.randint(0, h), h // page * page, -3]) for h in rows])
        else:
            b.compact()
        if step % 6 == 5:
            b.check_rows()
    b.release([0] * n_req)
    assert sorted(b.p.free) == list(range(60)) and not any(b.p.shares)


def test_forks_of_whole_pages_and_of_parts():
    b = Both()
    b.add([100, 0, 0, 32] + [0] * 8)
    b.fork([0, 0, 3, 0, 3], [1, 2, 4, 5, 6], [100, 96, 32, 5, 0]).check_rows()
    assert b.p.shares[b.p.table[0][0]] == 2


def test_a_fork_s_page_keeps_what_the_parent_writes_later_apart():
    b = Both()
    b.add([20] + [0] * 11)
    b.fork([0], [1], [20])
    b.add([5, 7] + [0] * 10)
    b.check_rows()


def test_forks_that_cannot_be():
    b = Both()
    b.add([50, 10] + [0] * 10)
    b.fork([0, 0, 0, -1, 12, 0, 0, 0, 2, 0, 0], [0, 1, 2, 3, 4, 12, -1, 2, 5, 6, 7], [50, 50, 17, 5, 5, 5, 5, 3, 1, 51, -1])
    assert b.p.rows == [50, 10, 17] + [0] * 9
    # the place of a fork that cannot be is not free for a later one of the call
    b.fork([1, 0], [8, 8], [11, 3])
    assert b.p.rows[8] == 0
    b.check_rows()


def test_forks_up_to_the_first_without_a_page():
    b = Both(n_pages=6, n_req=8)
    b.add([40, 0, 0, 0, 0, 0, 0, 0])            # three pages, three left
    b.fork([0] * 6, [1, 2, 3, 4, 5, 6], [40, 16, 33, 40, 40, 32])
    assert b.p.rows == [40, 40, 16, 33, 40, 0, 0, 0]
    b.check_rows()
    b.release([0] * 8)


def test_a_fork_of_a_place_that_is_filled_in_the_same_call():
    b = Both()
    b.add([30] + [0] * 11)
    b.fork([0, 1, 1], [1, 2, 3], [30, 0, 10])   # request 1 holds nothing before the call
    assert b.p.rows[:4] == [30, 30, 0, 0]


def test_a_source_with_an_entry_that_is_no_page():
    b = Both()
    b.add([70] + [0] * 11)
    for r, c, x in ((0, 1, -1), (0, 4, 77)):
        b.p.table[r][c] = x
        b.table[r, c] = x
    b.fork([0, 0], [1, 2], [64, 70])
    assert b.p.rows[:3] == [70, 64, 70]


def test_rows_that_pass_the_table():
    b = Both(stride=3)
    b.add([48] + [0] * 11)
    b.p.rows[0] = 49
    b.rows[0] = 49
    b.fork([0], [1], [5])
    b.release([0] * 12)
    number = torch.empty(b.pool.n_pages, dtype=torch.int32, device="cuda")
    b.pool.compact(b.rows, b.table, number)
    assert lib().q4_gpu_last_error() == 4


@pytest.mark.parametrize("keep", [[0, 100, 100], [100, 0, 100], [0, 0, 100], [100, 0, 0], [0, 0, 0], [48, 48, 100], [48, 0, 0], [100, 96, 0]])
def test_pages_go_back_with_their_last_holder(keep):
    b = Both()
    b.add([100] + [0] * 11)
    b.fork([0, 0], [1, 2], [100, 100])
    b.release(keep + [0] * 9).check_rows()
    b.release([0] * 12)
    assert sorted(b.p.free) == list(range(40))


def test_part_of_a_shared_page_cannot_be_kept():
    b = Both()
    b.add([64, 20] + [0] * 10)
    b.fork([0], [2], [64])
    b.release([50, 3, 10] + [0] * 9).check_rows()          # 0 and 2 stay as they are, 1 is rewound
    assert b.p.rows[:3] == [64, 3, 64]
    b.fork([0], [3], [50])                                 # the way that is documented
    b.release([0, 3, 64, 50] + [0] * 8).check_rows()
    b.release([64, 3, 50, 50] + [0] * 8)                   # its other holder has gone, but for whole pages that 3 has too
    assert b.p.rows[:4] == [0, 3, 50, 50]


def test_pages_given_back_too_often():
    b = Both()
    b.add([40, 40] + [0] * 10)
    b.fork([0], [2], [40])
    for r in (3, 4):                                       # two requests that name pages without holding them
        b.p.table[r][:3] = b.p.table[0][:3]
        b.table[r, :3] = b.table[0, :3]
        b.p.rows[r] = 40
        b.rows[r] = 40
    b.release([0, 40, 0, 0, 40] + [0] * 7)                 # three times the pages of two holders
    assert b.p.rows[:5] == [40, 40, 40, 40, 40]
    b.table[1, 1] = -1
    b.p.table[1][1] = -1
    b.release([40, 0, 40, 40, 40] + [0] * 7)               # no page of the pool


def test_a_pool_without_forks_is_released_as_it_is_trimmed():
    b, c = Both(), Both()
    for x in (b, c):
        x.add([70, 0, 33, 200] + [0] * 8)
    keep = [16, 0, 40, 17] + [0] * 8
    b.release(keep)
    c.pool.trim(c.rows, ints(keep), c.table)
    assert torch.equal(b.pool.free[: int(b.pool.n_free[0])], c.pool.free[: int(c.pool.n_free[0])])


@pytest.mark.parametrize("n_req,stride,page", [(8192, 4, 16), (3000, 60, 16), (1, 20000, 16), (700, 300, 32)])
def test_many_requests(n_req, stride, page):
    """shared prefixes among thousands of requests, against torch's own counting"""
    g = torch.Generator(device="cuda").manual_seed(n_req)
    per = max(1, min(stride - 1, 120000 // n_req))
    n_pages = n_req * per + n_req + 7
    pool = q4gpu.PagePool(1, 1, 64, n_pages, page, q4gpu.KIND_Q8)
    half = n_req // 2
    table = torch.full((n_req, stride), -1, dtype=torch.int32, device="cuda")
    owners = n_req - half
    table[:owners, :per] = pool.free[n_pages - owners * per:].flip(0).view(owners, per)
    pool.n_free.fill_(n_pages - owners * per)
    rows = torch.zeros(n_req, dtype=torch.int32, device="cuda")
    rows[:owners] = torch.randint(max(1, per * page - page + 1), per * page + 1, (owners,), generator=g, device="cuda", dtype=torch.int32)
    L = lib()
    L.q4_gpu_last_error()
    if half:
        src = torch.randint(0, owners, (half,), generator=g, device="cuda", dtype=torch.int32)
        dst = owners + torch.randperm(half, generator=g, device="cuda").int()
        length = (torch.rand(half, generator=g, device="cuda") * (rows[src.long()] + 1)).int()
        top = int(pool.n_free[0])
        pool.fork(rows, src, dst, length, table)
        assert L.q4_gpu_last_error() == 0
        part = length % page > 0
        assert int(pool.n_free[0]) == top - int(part.sum())
        assert torch.equal(rows[dst.long()], length)
        col = torch.arange(stride, device="cuda")
        whole = col[None] < (length // page)[:, None]
        assert torch.equal(table[dst.long()][whole], table[src.long()][whole])
        new = table[dst.long()].gather(1, (length // page).clamp(max=stride - 1)[:, None].long())[:, 0][part]
        assert torch.equal(new, pool.free[top - int(part.sum()): top].flip(0))
        want = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        want.index_add_(0, table[src.long()][whole].long(), torch.ones(int(whole.sum()), dtype=torch.int32, device="cuda"))
        assert torch.equal(pool.shares[:n_pages], want)
    for keep in (rows.clone() // page // 2 * page, torch.zeros_like(rows)):
        before = pool.shares.clone()
        held = (rows + page - 1) // page
        col = torch.arange(stride, device="cuda")
        given = (col[None] >= ((keep + page - 1) // page)[:, None]) & (col[None] < held[:, None])
        named = table[given].long()
        times = torch.bincount(named, minlength=n_pages).int()
        order = torch.arange(named.numel(), device="cuda")
        last = torch.full((n_pages,), -1, device="cuda").scatter_reduce_(0, named, order, "amax")
        gone = named[(last[named] == order) & (times[named] == before[:n_pages][named] + 1)]
        top = int(pool.n_free[0])
        pool.release(rows, keep, table)
        assert L.q4_gpu_last_error() == 0
        assert int(pool.n_free[0]) == top + gone.numel()
        assert torch.equal(pool.free[top: top + gone.numel()], gone.flip(0).int())
        assert torch.equal(rows, keep)
        assert not pool.shares[n_pages:].any()
    assert not pool.shares.any() and int(pool.n_free[0]) == n_pages
    assert torch.equal(pool.free.sort().values, torch.arange(n_pages, dtype=torch.int32, device="cuda"))


def test_compact_of_all_and_of_nothing():
    b = Both()
    b.compact()                                            # empty
    b.add([20] * 12)
    b.compact().check_rows()
    b.release([0, 20, 0, 20, 0, 20, 0, 20, 0, 20, 0, 20])
    b.compact().check_rows()
    b.compact().check_rows()                               # nothing is left to move
    b = Both(n_pages=24, n_req=12)
    b.add([32] * 12)                                       # full
    b.compact().check_rows()


def test_compact_without_tables_tells_where_the_pages_are():
    b = Both()
    b.add([40] * 8 + [0] * 4)
    b.release([0, 40] * 4 + [0] * 4)
    number = torch.full((40,), -9, dtype=torch.int32, device="cuda")
    b.pool.compact(None, None, number)
    assert lib().q4_gpu_last_error() == 0
    want, _ = b.p.compact()
    assert number.tolist() == want
    old = b.table.clone()
    held = torch.arange(20, device="cuda")[None] < ((b.rows + 15) // 16)[:, None]
    b.table[held] = number[old[held].long()]
    b.check().check_rows()


@pytest.mark.parametrize("wrong", ["twice", "below", "beyond", "height", "negative"])
def test_a_stack_that_is_none_moves_nothing(wrong):
    b = Both()
    b.add([40] * 8 + [0] * 4)
    b.release([0, 40] * 4 + [0] * 4)
    free = b.pool.free
    if wrong == "twice":
        free[3] = free[5]
    elif wrong == "below":
        free[0] = -1
    elif wrong == "beyond":
        free[1] = 40
    elif wrong == "height":
        b.pool.n_free.fill_(41)
    else:
        b.pool.n_free.fill_(-1)
    mem, table, before = b.pool.mem.clone(), b.table.clone(), free.clone()
    number = torch.full((40,), -9, dtype=torch.int32, device="cuda")
    b.pool.compact(b.rows, b.table, number)
    assert lib().q4_gpu_last_error() == 4
    assert torch.equal(b.pool.mem, mem) and torch.equal(b.table, table) and torch.equal(free, before)
    assert number.tolist() == list(range(40))


def test_entries_that_are_no_pages_in_use_stay():
    b = Both()
    b.add([40] * 8 + [0] * 4)
    b.release([0, 40] * 4 + [0] * 4)
    b.p.table[1][1] = -1
    b.p.table[3][0] = b.p.free[0]
    b.table[1, 1], b.table[3, 0] = -1, b.p.free[0]
    b.compact()


@pytest.mark.parametrize("n_pages", [1_310_719, 1_310_720, 1_310_721, 1_400_037])
def test_a_pool_of_more_pages_than_are_marked_at_once(n_pages):
    g = torch.Generator(device="cuda").manual_seed(1)
    pool = q4gpu.PagePool(1, 1, 64, n_pages, 16, q4gpu.KIND_Q8)
    words = pool.mem.view(torch.int64).view(n_pages, -1)
    words[:, 0] = words[:, -1] = torch.arange(n_pages, device="cuda")
    used = torch.rand(n_pages, generator=g, device="cuda") < 0.3
    used[-1] = True
    free = torch.nonzero(~used).flatten().int()
    pool.free[: free.numel()] = free[torch.randperm(free.numel(), generator=g, device="cuda")]
    pool.n_free.fill_(free.numel())
    live = n_pages - free.numel()
    number = torch.empty(n_pages, dtype=torch.int32, device="cuda")
    lib().q4_gpu_last_error()
    pool.compact(None, None, number)
    assert lib().q4_gpu_last_error() == 0
    old = torch.nonzero(used).flatten()
    assert (number[~used] == -1).all()
    new = number[old].long()
    assert torch.equal(new.sort().values, torch.arange(live, device="cuda"))
    low = old < live
    assert torch.equal(new[low], old[low]) and (new[~low].diff() > 0).all()
    assert torch.equal(words[new, 0], old) and torch.equal(words[new, -1], old)
    assert torch.equal(pool.free[: free.numel()], torch.arange(n_pages - 1, live - 1, -1, device="cuda", dtype=torch.int32))


def test_captured_and_replayed():
    """one graph of a fork, a release and a compaction, replayed on other lengths"""
    b = Both(n_pages=60)
    b.add([100, 50] + [0] * 10)
    src, dst, length, keep = ints([0, 1]), ints([2, 3]), ints([100, 40]), ints([90, 2**31 - 1] + [2**31 - 1] * 10)
    number = torch.empty(60, dtype=torch.int32, device="cuda")
    L = lib()
    b.pool.compact(b.rows, b.table, number)                # the scratch is there
    b.p.compact()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    L.q4_gpu_set_stream(s.cuda_stream)
    try:
        assert L.q4_hip_graph_begin()
        b.pool.fork(b.rows, src, dst, length, b.table)
        b.pool.release(b.rows, keep, b.table)
        b.pool.compact(b.rows, b.table, number)
        graph = L.q4_hip_graph_end()
        assert graph
        for s_, d_, n_, k_ in (([0, 1], [2, 3], [100, 40], [90] + [2**31 - 1] * 11), ([2, 3], [4, 5], [64, 33], [90, 0, 2**31 - 1] + [2**31 - 1] * 9),
                               ([4, 4], [6, 6], [10, 10], [0] * 3 + [2**31 - 1] * 9)):
            for t, v in ((src, s_), (dst, d_), (length, n_), (keep, k_)):
                t.copy_(ints(v))
            torch.cuda.synchronize()
            assert L.q4_hip_graph_launch(ctypes.c_void_p(graph))
            bits = b.p.fork(s_, d_, n_) | b.p.release(k_) | b.p.compact()[1]
            assert L.q4_gpu_last_error() == bits
            b.check().check_rows()
        L.q4_hip_graph_free(ctypes.c_void_p(graph))
    finally:
        q4gpu.use_torch_stream()


def test_refusals():
    b = Both()
    L, p = lib(), lambda t: t.data_ptr()  # noqa: E731
    src = ints([0])
    L.q4_gpu_last_error()
    fork = dict(pg=b.pool.p, shares=b.pool.shared, rows=p(b.rows), n=12, src=p(src), dst=p(src), len=p(src), m=1, table=p(b.table), stride=20)
    release = dict(pg=b.pool.p, shares=b.pool.shared, rows=p(b.rows), keep=p(b.rows), n=12, table=p(b.table), stride=20)
    compact = dict(pg=b.pool.p, shares=b.pool.shared, rows=p(b.rows), n=12, table=p(b.table), stride=20, map=p(b.table))
    no_stack = q4gpu.PagePool(1, 1, 64, 4, 16, q4gpu.KIND_Q8, mem=b.pool.mem)
    for fn, args, ok in ((L.q4_gpu_pages_fork, fork, ()), (L.q4_gpu_pages_release, release, ()), (L.q4_gpu_pages_compact, compact, ("shares",))):
        for name in args:
            if name in ok:
                continue
            other = no_stack.p if name == "pg" else None if name not in ("n", "m", "stride") else 8193 if name != "stride" else 2**31
            if fn is L.q4_gpu_pages_compact and name == "n":
                continue
            assert not fn(*{**args, name: other}.values()), name
            assert L.q4_gpu_last_error() == 1
        if "m" in args:
            assert not fn(*{**args, "m": 0}.values()) and L.q4_gpu_last_error() == 1
    bare = q4gpu.PagePool(1, 1, 64, 4, 16, q4gpu.KIND_Q8, mem=b.pool.mem, free=ints([0, 1, 2, 3]), n_free=ints([4]))
    with pytest.raises(RuntimeError):                      # a pool that was made without counts
        bare.release(ints([0]), ints([0]), ints([[0, 0]]))
    L.q4_gpu_last_error()
    b.check()


def test_lengths_that_are_what_the_requests_hold():
    """rows given as the lengths too: all forks see them as they were, those that a thread comes to later among them"""
    n_req, n = 1300, 600
    pool = q4gpu.PagePool(1, 1, 64, 40, 16)
    table = torch.full((n_req, 8), -1, dtype=torch.int32, device="cuda")
    rows, add = torch.zeros(2, n_req, dtype=torch.int32, device="cuda").unbind(0)
    add[0] = 64
    start, slot, pos, req = torch.zeros(n_req + 1, dtype=torch.int32, device="cuda"), *torch.zeros(3, 64, dtype=torch.int32, device="cuda").unbind(0)
    lib().q4_gpu_last_error()
    pool.plan(rows, add, table, start, slot, pos, req)
    rows += add
    dst = torch.arange(512, 512 + n, dtype=torch.int32, device="cuda")      # the first fork's place is the one whose rows are the 512th's length
    pool.fork(rows, torch.zeros_like(dst), dst, rows[:n], table)
    assert lib().q4_gpu_last_error() == 0
    want = torch.zeros(n_req, dtype=torch.int32)
    want[0] = want[512] = 64
    assert torch.equal(rows.cpu(), want)
    assert table[512, :4].tolist() == table[0, :4].tolist() and int((table != -1).sum()) == 8
    assert int(pool.shares.sum()) == 4
