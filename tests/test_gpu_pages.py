"""The paged KV cache (q4_gpu_pages_*): the planning of a step against a plain restatement on lists, appended rows against the
store's quantiser, attention against softmax(q k) v in 64 bits."""
import numpy as np
import pytest
import torch

import q4gpu
from gpu_util import lib

pytestmark = pytest.mark.gpu
KINDS = {"q8_0": q4gpu.KIND_Q8, "f16": q4gpu.KIND_F16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def plan_plain(rows, add, table, free, page, max_tok):
    """the definition, request by request: (table, free, start, slot, pos, req, status bits)"""
    table, free = [list(t) for t in table], list(free)
    start, slot, pos, req, bits, full = [0], [], [], [], 0, False
    for r, (h, n) in enumerate(zip(rows, add)):
        n = max(n, 0)
        if n and (h < 0 or h + n > len(table[r]) * page):
            n, bits = 0, bits | 4
        need = -(-(h + n) // page) - -(-h // page) if n else 0
        if full or need > len(free) or len(slot) + n > max_tok:
            if not full:
                full, bits = True, bits | 8
            n = need = 0
        for i in range(need):
            table[r][-(-h // page) + i] = free.pop()
        for j in range(n):
            p = h + j
            slot.append(table[r][p // page] * page + p % page)
            pos.append(p)
            req.append(r)
        start.append(start[-1] + n)
    for v in (slot, pos, req):
        v.extend([-1] * (max_tok - len(v)))
    return table, free, start, slot, pos, req, bits


class Step:
    """requests with the given lengths on a pool, their pages in a random order"""

    def __init__(self, rows, add, page=16, n_pages=None, stride=None, max_tok=None, seed=0, **pool):
        rng = np.random.default_rng(seed)
        self.rows, self.add, self.page = rows, add, page
        held = [-(-max(h, 0) // page) for h in rows]
        need = sum(-(-max(max(h, 0) + max(n, 0), 0) // page) - c for h, n, c in zip(rows, add, held))
        n_pages = sum(held) + need + 3 if n_pages is None else n_pages
        self.stride = max(1, max(-(-(max(h, 0) + max(n, 0)) // page) for h, n in zip(rows, add))) + 1 if stride is None else stride
        order = [int(x) for x in rng.permutation(n_pages)]
        self.table = []
        for c in held:
            self.table.append([order.pop() for _ in range(c)] + [-1] * (self.stride - c))
        self.free = order
        self.max_tok = sum(max(n, 0) for n in add) + 5 if max_tok is None else max_tok
        kw = dict(n_layers=1, n_kvh=1, hd=64, kind=q4gpu.KIND_Q8)
        kw.update(pool)
        size = lib().q4_gpu_pages_bytes(kw["n_layers"], kw["n_kvh"], kw["hd"], n_pages, page, kw["kind"])
        mem = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")   # every unwritten number is NaN
        self.pool = q4gpu.PagePool(kw["n_layers"], kw["n_kvh"], kw["hd"], n_pages, page, kw["kind"], mem=mem,
                                   free=ints(self.free + [-7] * (n_pages - len(self.free))), n_free=ints([len(self.free)]))
        self.d_rows, self.d_add, self.d_table = ints(rows), ints(add), ints(self.table)
        self.start = torch.full((len(rows) + 1,), -9, dtype=torch.int32, device="cuda")
        self.slot, self.pos, self.req = (torch.full((max(1, self.max_tok),), -9, dtype=torch.int32, device="cuda") for _ in range(3))

    def plan(self):
        self.pool.plan(self.d_rows, self.d_add, self.d_table, self.start, self.slot, self.pos, self.req)
        return self

    def free_now(self):
        return self.pool.free[: int(self.pool.n_free[0])].tolist()


@pytest.mark.parametrize("rows,add,page", [
    ([0], [1], 16), ([15], [1], 16), ([16], [1], 16), ([0], [16], 16), ([0], [17], 16), ([5], [0], 16),
    ([3, 0, 40, 16], [1, 33, 8, 1], 16), ([0, 7, 0, 0, 300], [0, 0, 5, 0, 260], 32), ([255, 256, 257], [1, 1, 1], 256),
    (list(range(0, 1500, 3)), [(7 * i) % 5 for i in range(500)], 64),
    ([(13 * i) % 97 for i in range(1300)], [(i * i) % 4 for i in range(1300)], 16),
    ([0] * 8192, [1] * 8192, 16), ([100, 50], [3000, 5000], 16), ([9, -1, 4], [2, 0, 3], 16)])
def test_plan_and_trim(rows, add, page):
    s = Step(rows, add, page)
    want = plan_plain(rows, add, s.table, s.free, page, s.max_tok)
    L = lib()
    L.q4_gpu_last_error()
    s.plan()
    assert L.q4_gpu_last_error() == want[6] == 0
    assert s.d_table.tolist() == want[0]
    assert s.free_now() == want[1]
    assert (s.start.tolist(), s.slot.tolist(), s.pos.tolist(), s.req.tolist()) == tuple(want[2:6])
    # taken back: the stack is what it was
    s.pool.trim(ints([max(h, 0) + max(n, 0) for h, n in zip(rows, add)]), ints(rows), s.d_table)
    assert L.q4_gpu_last_error() == 0
    assert s.free_now() == s.free
    # and all of it: every page is free
    s.pool.trim(ints(rows), ints([0] * len(rows)), s.d_table)
    assert L.q4_gpu_last_error() == 0
    assert sorted(s.free_now()) == list(range(s.pool.n_pages))


@pytest.mark.parametrize("rows,add,kw", [
    ([0, 0, 0], [20, 40, 3], dict(n_pages=4)),                  # the second does not fit; the third would, but waits too
    ([0, 0, 0], [20, 4, 3], dict(n_pages=2)),
    ([10, 10], [30, 3], dict(max_tok=20)), ([10, 10], [5, 3], dict(max_tok=7)), ([0], [1], dict(n_pages=1, max_tok=1)),
    ([0, 33, 0], [5, 40, 6], dict(stride=4)),                   # the second would pass its table's row: the third is served
    ([0, -5, 3], [5, 2, 6], {}), ([0, 0], [2**31 - 1, 1], dict(stride=2, max_tok=9, n_pages=5)),
    ([2**31 - 1, 0], [2**31 - 1, 1], dict(stride=2, max_tok=9, n_pages=5, held0=True))])
def test_plan_without_room(rows, add, kw):
    kw = dict(kw)
    if kw.pop("held0", False):
        s = Step([0, 0], [1, 1], **kw)
        s.rows, s.d_rows, s.add, s.d_add = rows, ints(rows), add, ints(add)
    else:
        s = Step(rows, add, **kw) if max(add) < 2**30 else Step([0, 0], [1, 1], **kw)
        s.add, s.d_add = add, ints(add)
    want = plan_plain(rows, add, s.table, s.free, s.page, s.max_tok)
    L = lib()
    L.q4_gpu_last_error()
    s.plan()
    assert L.q4_gpu_last_error() == want[6] != 0 or (want[6] == 0 and len(rows) == 1)
    assert s.d_table.tolist() == want[0]
    assert s.free_now() == want[1]
    assert (s.start.tolist(), s.slot.tolist(), s.pos.tolist(), s.req.tolist()) == tuple(want[2:6])


def test_trim_refuses_pages_given_back_twice():
    s = Step([40, 20], [0, 0])
    L = lib()
    s.pool.trim(s.d_rows, ints([0, 0]), s.d_table)
    assert L.q4_gpu_last_error() == 0
    free = s.free_now()
    s.pool.trim(s.d_rows, ints([0, 0]), s.d_table)
    assert L.q4_gpu_last_error() == 4
    assert s.free_now() == free


def test_trim_keeps_and_hands_out_in_the_same_order():
    s = Step([70, 0, 33, 200], [0, 0, 0, 0])
    s.pool.trim(s.d_rows, ints([16, 0, 40, 17]), s.d_table)
    given = s.table[0][1:5] + s.table[3][2:13]
    assert s.free_now() == s.free + given[::-1]


def quantised(x):
    b = x.reshape(-1, 32).astype(np.float32)
    d = np.abs(b).max(1, keepdims=True) / np.float32(127)
    with np.errstate(divide="ignore"):
        inv = np.where(d > 0, np.float32(1) / d, np.float32(0))
    return (np.clip(np.rint(b * inv), -127, 127) * d.astype(np.float16).astype(np.float32)).reshape(x.shape)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("n_kvh,hd,n_tok,page", [(2, 128, 1, 16), (1, 64, 37, 16), (3, 256, 100, 64), (8, 128, 333, 128), (5, 64, 7, 256)])
def test_append_and_gather(kind, n_kvh, hd, n_tok, page):
    rng = np.random.default_rng(n_tok)
    k, v = rng.standard_normal((2, n_tok, n_kvh * hd)).astype(np.float32) * 3
    k[0, :32] = 0
    v[-1, 32:64] = 1e-7
    s = Step([9] * 3, [n_tok // 3, n_tok - 2 * (n_tok // 3), n_tok // 3], page, n_layers=2, n_kvh=n_kvh, hd=hd, kind=KINDS[kind]).plan()
    slot = s.slot[:n_tok].clone()
    slot[n_tok // 2] = -1 if n_tok > 2 else slot[n_tok // 2]
    L = lib()
    before = s.pool.mem[: s.pool.mem.numel() // 2].clone()
    s.pool.append(1, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), slot)
    ko, vo = torch.full((2, n_tok, n_kvh * hd), 7.0, device="cuda")
    s.pool.gather(1, slot, ko, vo)
    assert L.q4_gpu_last_error() == 0
    assert torch.equal(s.pool.mem[: s.pool.mem.numel() // 2], before)   # the other layer
    for x, got in ((k, ko), (v, vo)):
        want = quantised(x) if kind == "q8_0" else x.astype(np.float16).astype(np.float32)
        if n_tok > 2:
            want[n_tok // 2] = 0
        assert np.array_equal(got.cpu().numpy(), want)
    only = torch.empty_like(vo)
    s.pool.gather(1, slot, None, only)
    assert torch.equal(only, vo)
    slot[0] = s.pool.n_pages * page
    s.pool.append(1, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), slot)
    assert L.q4_gpu_last_error() == 4


def test_append_is_the_store_s_quantiser():
    rng = np.random.default_rng(5)
    n, n_kvh, hd = 50, 2, 128
    k, v = (torch.from_numpy(x).cuda() for x in rng.standard_normal((2, n, n_kvh * hd)).astype(np.float32))
    s = Step([0], [n], n_kvh=n_kvh, hd=hd).plan()
    s.pool.append(0, k, v, s.slot[:n])
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    s.pool.gather(0, s.slot[:n], ko, vo)
    st = q4gpu.KVStore(1, n_kvh, hd, n, q4gpu.KIND_Q8)
    st.append(0, k, v, 0, n)
    for which, got in ((0, ko), (1, vo)):
        raw = torch.empty(n * st.token_bytes, dtype=torch.uint8, device="cuda")
        st.export(0, which, 0, n, raw)
        blocks = raw.cpu().numpy().reshape(-1, 34)
        want = blocks[:, 2:].view(np.int8).astype(np.float32) * blocks[:, :2].copy().view(np.float16).astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want.reshape(n, -1))


def attend_exact(q, k, v, gate, held, scale):
    """one request in 64 bits: q [n][n_head][hd], k and v [rows][n_kvh][hd]"""
    n, n_head, hd = q.shape
    k, v = (x.double().repeat_interleave(n_head // x.shape[1], 1) for x in (k, v))
    w = torch.einsum("thd,phd->htp", q.double(), k) * scale
    p, j = torch.arange(k.shape[0], device=q.device), torch.arange(n, device=q.device)
    w = w.masked_fill(p[None, :] > held + j[:, None], -np.inf)
    o = torch.einsum("htp,phd->thd", torch.softmax(w, -1), v)
    return o * torch.sigmoid(gate.double()) if gate is not None else o


def run_attend(rows, add, n_head, n_kvh, hd, kind, page=16, gate=False, q_bf16=True, out_bf16=False, max_add=0, seed=0, q_scale=1.0):
    s = Step(rows, add, page, n_layers=2, n_kvh=n_kvh, hd=hd, kind=KINDS[kind], seed=seed)
    L = lib()
    L.q4_gpu_last_error()
    g = torch.Generator(device="cuda").manual_seed(seed)
    # the rows that are held, then the step's
    k, v = torch.randn(2, max(1, sum(rows)), n_kvh * hd, generator=g, device="cuda")
    slot = [s.table[r][p // page] * page + p % page for r, h in enumerate(rows) for p in range(h)]
    if slot:
        s.pool.append(1, k, v, ints(slot))
    s.plan()
    n_tok = sum(add)
    kn, vn = torch.randn(2, n_tok, n_kvh * hd, generator=g, device="cuda")
    s.pool.append(1, kn, vn, s.slot[:n_tok])
    q = torch.randn(n_tok, n_head, hd, generator=g, device="cuda") * q_scale
    q = q.to(torch.bfloat16) if q_bf16 else q
    gt = torch.randn(n_tok, n_head, hd, generator=g, device="cuda") if gate else None
    out = torch.full((n_tok + 1, n_head, hd), 77.0, device="cuda", dtype=torch.bfloat16 if out_bf16 else torch.float32)
    scale = float(1 / np.sqrt(hd))
    s.pool.attend(1, q, out[:n_tok], s.d_rows, s.start, s.d_table, n_head, scale, gate=gt, max_add=max_add)
    assert L.q4_gpu_last_error() == 0
    assert (out[n_tok] == 77).all()
    # rows as the pool holds them
    table = s.d_table.tolist()
    at = 0
    for r, (h, n) in enumerate(zip(rows, add)):
        if not n:
            continue
        sl = ints([table[r][p // page] * page + p % page for p in range(h + n)])
        kr, vr = torch.empty(2, h + n, n_kvh * hd, device="cuda")
        s.pool.gather(1, sl, kr, vr)
        want = attend_exact(q[at: at + n], kr.view(-1, n_kvh, hd), vr.view(-1, n_kvh, hd), gt[at: at + n] if gate else None, h, scale)
        got = out[at: at + n].double()
        # queries, weights and K and V values are rounded to fp16 (2^-11 each, against sums of squares of the order of the output):
        # 2e-3 + 1e-3 |o| is the attention's stated tolerance; a bf16 output is 2^-8 of its value away at most
        # larger queries: K as fp16(code x scale) moves a score by 2e-4 of its size (one sigma); five of them, on values 2 apart
        tol = 2e-3 + (1e-3 + (2.0**-8 if out_bf16 else 0.0)) * want.abs() + (2e-3 * q_scale if q_scale > 1 and kind == "q8_0" else 0.0)
        bad = (got - want).abs() - tol
        assert bad.max() <= 0, "request %d: %.3e over the bound" % (r, bad.max())
        at += n
    return s, out


SHAPES = [(16, 2, 128), (24, 2, 256), (8, 4, 64), (32, 2, 64), (4, 4, 128), (12, 1, 128), (6, 2, 256)]


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("n_head,n_kvh,hd", SHAPES)
def test_attend_decode(kind, n_head, n_kvh, hd):
    run_attend([0, 1, 15, 16, 17, 127, 128, 300, 1111], [1] * 9, n_head, n_kvh, hd, kind, gate=True, max_add=1)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("n_head,n_kvh,hd", SHAPES)
@pytest.mark.parametrize("max_add", [0, 200])
def test_attend_mixed(kind, n_head, n_kvh, hd, max_add):
    run_attend([0, 33, 500, 64, 0, 129, 0], [5, 1, 7, 0, 200, 64, 1], n_head, n_kvh, hd, kind, page=32, max_add=max_add, out_bf16=True)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 9, 33])
def test_attend_tokens_of_a_request(page, n):
    run_attend([77], [n], 16, 2, 128, "q8_0", page=page, gate=True, max_add=n)
    run_attend([0], [n], 16, 2, 128, "f16", page=page, max_add=n, q_bf16=False)


def test_attend_long():
    run_attend([20011], [1], 16, 2, 128, "q8_0", page=64, max_add=1)
    run_attend([5003, 9], [3, 1], 16, 2, 128, "f16", page=16, max_add=3)
    run_attend([3001], [300], 16, 2, 128, "q8_0", page=128, gate=True, max_add=300)


def test_attend_large_scores():
    """scores far apart: the running maximum moves all the time, and most weights vanish"""
    run_attend([700, 90], [1, 40], 16, 2, 128, "f16", q_scale=30.0)
    run_attend([700, 90], [1, 40], 16, 2, 128, "q8_0", q_scale=30.0)


def test_attend_many_requests():
    rows = [(37 * i) % 211 for i in range(700)]
    run_attend(rows, [1 if i % 3 else 2 for i in range(700)], 8, 4, 64, "f16", max_add=2)


def test_attend_pages_that_are_not_the_pool_s():
    L = lib()
    s, out = run_attend([100, 50], [1, 1], 16, 2, 128, "q8_0")
    q = torch.randn(2, 16, 128, device="cuda")
    o = torch.empty(2, 16, 128, device="cuda")
    scale = float(128 ** -0.5)
    s.pool.attend(1, q, o, s.d_rows, s.start, s.d_table, 16, scale)
    good = o.clone()
    assert L.q4_gpu_last_error() == 0
    bad = s.d_table.clone()
    bad[0, 2], bad[0, 3] = s.pool.n_pages, -1
    s.pool.attend(1, q, o, s.d_rows, s.start, bad, 16, scale)
    assert L.q4_gpu_last_error() == 4
    assert torch.equal(o[1], good[1]) and torch.isfinite(o).all() and not torch.equal(o[0], good[0])
    bad[0] = -1   # nothing is left: zeros
    s.pool.attend(1, q, o, s.d_rows, s.start, bad, 16, scale)
    assert L.q4_gpu_last_error() == 4
    assert (o[0] == 0).all() and torch.equal(o[1], good[1])
    rows = s.d_rows.clone()
    rows[0] = 10000   # passes its table's row: left out
    o.fill_(5)
    s.pool.attend(1, q, o, rows, s.start, s.d_table, 16, scale)
    assert L.q4_gpu_last_error() == 4
    assert (o[0] == 5).all() and torch.equal(o[1], good[1])


def test_refusals():
    L = lib()
    L.q4_gpu_last_error()
    for bad in (dict(hd=32), dict(hd=96), dict(page_rows=8), dict(page_rows=48), dict(page_rows=512), dict(kind=0), dict(kind=3), dict(n_kvh=0), dict(n_pages=1 << 27)):
        a = dict(n_layers=1, n_kvh=2, hd=128, n_pages=64, page_rows=16, kind=2)
        a.update(bad)
        assert L.q4_gpu_pages_bytes(a["n_layers"], a["n_kvh"], a["hd"], a["n_pages"], a["page_rows"], a["kind"]) == 0
        with pytest.raises(RuntimeError):
            q4gpu.PagePool(**a)
    s = Step([5, 6], [1, 1], n_kvh=2, hd=128)
    s.plan()
    p, i = s.pool.p, lambda t: t.data_ptr()
    plan = lambda **kw: L.q4_gpu_pages_plan(*dict(dict(a=p, b=i(s.d_rows), c=i(s.d_add), d=2, e=i(s.d_table), f=s.stride, g=i(s.start), h=i(s.slot), j=i(s.pos), k=i(s.req), m=7), **kw).values())  # noqa: E731
    for kw in ("a", "b", "c", "d", "e", "f", "g", "h", "j", "k", "m"):
        assert not plan(**{kw: 0 if kw in "dfm" else None}), kw
        assert L.q4_gpu_last_error() == 1
    assert not plan(d=8193)
    assert L.q4_gpu_last_error() == 1
    x = torch.zeros(4 * 16 * 128 + 8, device="cuda")
    for args in ((None, 0, i(x), i(x), i(s.slot), 2), (p, 1, i(x), i(x), i(s.slot), 2), (p, 0, None, i(x), i(s.slot), 2), (p, 0, i(x) + 4, i(x), i(s.slot), 2),
                 (p, 0, i(x), i(x), None, 2), (p, 0, i(x), i(x), i(s.slot), 0)):
        assert not L.q4_gpu_pages_append(*args)
        assert L.q4_gpu_last_error() == 1
    assert not L.q4_gpu_pages_gather(p, 0, i(s.slot), 2, None, None)
    assert not L.q4_gpu_pages_trim(p, i(s.d_rows), None, 2, i(s.d_table), s.stride)
    L.q4_gpu_last_error()
    base = dict(a=p, layer=0, q=i(x), qb=0, gate=None, out=i(x), ob=0, n_head=16, rows=i(s.d_rows), start=i(s.start), n_req=2, n_tok=2, table=i(s.d_table), stride=s.stride, max_add=1, scale=0.1)
    for kw in (dict(a=None), dict(layer=1), dict(q=None), dict(out=None), dict(n_head=0), dict(n_head=15), dict(n_head=34), dict(rows=None), dict(start=None), dict(n_req=0),
               dict(n_tok=0), dict(table=None), dict(stride=0), dict(scale=0.0), dict(scale=-1.0), dict(q=i(x) + 4), dict(out=i(x) + 8), dict(gate=i(x) + 4)):
        assert not L.q4_gpu_pages_attend(*dict(base, **kw).values()), kw
        assert L.q4_gpu_last_error() == 1
    desc = q4gpu.PagesDesc(i(s.pool.mem), None, None, 1, 2, 128, s.pool.n_pages, 16, 2)
    import ctypes
    assert not plan(a=ctypes.addressof(desc))
    assert L.q4_gpu_last_error() == 1
