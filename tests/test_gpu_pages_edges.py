"""The paged KV cache (q4_gpu_pages_*) where it can go wrong: numbers that are not finite in masked places, units shared out over many
blocks, pages shared by tables, steps captured in graphs whose lengths then change, another stream, hints that are wrong."""
import numpy as np
import pytest
import torch

import q4gpu
from gpu_util import lib
from test_gpu_pages import KINDS, Step, attend_exact, ints, run_attend

pytestmark = pytest.mark.gpu


def step_of(rows, add, kind, n_kvh, hd, page=16, seed=0, n_pages=None):
    """requests whose rows are normal numbers, the step's own k and v not appended yet: (step, k, v)"""
    s = Step(rows, add, page, n_pages, n_kvh=n_kvh, hd=hd, kind=KINDS[kind], seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    slot = [s.table[r][p // page] * page + p % page for r, h in enumerate(rows) for p in range(h)]
    if slot:
        k, v = torch.randn(2, len(slot), n_kvh * hd, generator=g, device="cuda")
        s.pool.append(0, k, v, ints(slot))
    s.plan()
    kn, vn = torch.randn(2, sum(add), n_kvh * hd, generator=g, device="cuda")
    return s, kn, vn


BAD = [float("inf"), -float("inf"), float("nan"), 1e6]


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("n_head,n_kvh,hd", [(16, 2, 128), (12, 2, 64), (24, 2, 256), (4, 2, 256)])
@pytest.mark.parametrize("held,n,at", [(37, 3, 1), (0, 3, 2), (120, 70, 9), (0, 200, 128), (1000, 40, 39), (6007, 150, 1), (31, 4, 3), (100, 1500, 700)])
def test_new_rows_that_are_not_finite_stay_with_the_tokens_that_attend_them(kind, n_head, n_kvh, hd, held, n, at):
    """a weight of 0 times a V that is not finite is no 0.  Tokens before `at` have to come out bit by bit as without it"""
    s, k, v = step_of([held, 50], [n, 2], kind, n_kvh, hd)
    q = torch.randn(n + 2, n_head, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    scale = float(hd ** -0.5)

    def attend(k, v):
        s.pool.append(0, k, v, s.slot[: n + 2])
        out = torch.full((n + 2, n_head, hd), 77.0, device="cuda")
        s.pool.attend(0, q, out, s.d_rows, s.start, s.d_table, n_head, scale, max_add=n)
        return out.view(n + 2, n_kvh, n_head // n_kvh, hd)

    clean = attend(k, v)
    assert torch.isfinite(clean).all()
    for x in BAD if kind == "f16" else (BAD[0], BAD[3], 7e4):
        for dim in (0, hd - 1):
            v2 = v.clone()
            v2[at, hd + dim] = x                       # of the second kv head
            got = attend(k, v2)
            assert torch.equal(got[:at], clean[:at]) and torch.equal(got[n:], clean[n:]) and torch.equal(got[:, 0], clean[:, 0])
            assert not torch.isfinite(got[at:n, 1, :, dim]).any()
    if kind == "f16":
        k2 = k.clone()
        k2[at, 5] = float("nan")                       # a score of NaN: of those that have it
        got = attend(k2, v)
        assert torch.equal(got[:at], clean[:at]) and torch.equal(got[n:], clean[n:]) and torch.equal(got[:, 1], clean[:, 1])
        assert torch.isnan(got[at:n, 0]).all()
    assert torch.equal(attend(k, v), clean)
    assert lib().q4_gpu_last_error() == 0


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
def test_a_held_row_that_is_not_finite_reaches_every_token(kind):
    s, k, v = step_of([300, 40], [30, 1], kind, 2, 128)
    bad = torch.zeros(1, 256, device="cuda")
    bad[0, 3] = float("inf")
    s.pool.append(0, torch.zeros_like(bad), bad, ints([s.table[0][7] * 16 + 5]))
    s.pool.append(0, k, v, s.slot[:31])
    q = torch.randn(31, 16, 128, device="cuda")
    out = torch.empty_like(q)
    s.pool.attend(0, q, out, s.d_rows, s.start, s.d_table, 16, 0.1)
    o = out.view(31, 2, 8, 128)
    assert not torch.isfinite(o[:30, 0, :, 3]).any() and torch.isfinite(o[:30, 1]).all() and torch.isfinite(o[30]).all()
    assert lib().q4_gpu_last_error() == 0


# units in one block, in two or three, in up to sixteen, in more, with one and with many blocks behind the last whole one
@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("n_head,n_kvh,hd", [(16, 2, 128), (8, 4, 64), (4, 4, 256), (16, 1, 256)])
@pytest.mark.parametrize("rows", [[129], [257], [385, 3], [1500], [9001], [40000], [30011, 5, 12000], [1200] * 40, [4000, 300] * 20])
def test_one_token_each(kind, n_head, n_kvh, hd, rows):
    run_attend(rows, [1] * len(rows), n_head, n_kvh, hd, kind, page=32, max_add=1)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("n_head,n_kvh,hd", [(16, 2, 128), (8, 4, 64), (24, 2, 256), (32, 2, 128)])
@pytest.mark.parametrize("rows,add", [([15000], [70]), ([700, 9000, 40], [5, 5, 5]), ([0], [900]), ([20000, 0, 0, 33], [1, 300, 1, 130]), ([11, 4000] * 9, [7, 3] * 9),
                                      ([5000], [17]), ([0, 128, 127, 1], [128, 128, 1, 127])])
def test_several_tokens(kind, n_head, n_kvh, hd, rows, add):
    run_attend(rows, add, n_head, n_kvh, hd, kind, page=64, gate=True, max_add=max(add))


# many tokens over q8_0: rows are read from a copy in fp16
@pytest.mark.parametrize("n_head,n_kvh,hd", [(16, 2, 128), (32, 2, 64), (24, 2, 256), (16, 1, 256)])
@pytest.mark.parametrize("rows,add", [([300], [1500]), ([0, 77, 1000], [1300, 1999, 900]), ([33, 0, 5, 128], [1200, 0, 1, 2600])])
def test_many_tokens(n_head, n_kvh, hd, rows, add):
    run_attend(rows, add, n_head, n_kvh, hd, "q8_0", page=32, max_add=max(add))


def test_many_tokens_with_pages_that_are_not_the_pool_s():
    L = lib()
    n_head, n_kvh, hd = 16, 2, 128
    s, k, v = step_of([200, 64], [2200, 1], "q8_0", n_kvh, hd, page=16)
    s.pool.append(0, k, v, s.slot[:2201])
    q = torch.randn(2201, n_head, hd, device="cuda")
    out, short = torch.empty_like(q), torch.empty_like(q)
    scale = float(hd ** -0.5)
    bad = s.d_table.clone()
    bad[0, 3], bad[0, 140] = -1, s.pool.n_pages        # positions 48 to 63 and 2240 to 2255
    s.pool.attend(0, q, out, s.d_rows, s.start, bad, n_head, scale)
    assert L.q4_gpu_last_error() == 4
    s.pool.attend(0, q[:2200], short[:2200], s.d_rows, ints([0, 0, 0]), bad, n_head, scale)   # no tokens: nothing
    assert L.q4_gpu_last_error() == 0
    table = s.d_table[0].tolist()
    kr, vr = torch.empty(2, 2400, n_kvh * hd, device="cuda")
    s.pool.gather(0, ints([table[p // 16] * 16 + p % 16 for p in range(2400)]), kr, vr)
    keep = torch.ones(2400, dtype=torch.bool, device="cuda")
    keep[48:64] = keep[2240:2256] = False
    kr, vr = (x.view(-1, n_kvh, hd).double().repeat_interleave(n_head // n_kvh, 1) for x in (kr, vr))
    for j in (0, 700, 2039, 2040, 2199):
        p = torch.arange(2400, device="cuda")
        w = torch.einsum("hd,phd->hp", q[j].double(), kr) * scale
        w = w.masked_fill((p > 200 + j) | ~keep, -torch.inf)
        want = torch.einsum("hp,phd->hd", torch.softmax(w, -1), vr)
        assert ((out[j].double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()


def test_many_tokens_that_the_copy_has_no_room_for():
    """a table wide enough for more rows than the copy may hold: used where the step's rows fit, and not where they do not"""
    L = lib()
    n_head, n_kvh, hd, page, wide = 16, 8, 256, 256, 400   # 2 MB of copy per page: 256 of them at most
    s = Step([0], [1100], page, n_pages=300, stride=wide, n_kvh=n_kvh, hd=hd, kind=q4gpu.KIND_Q8)
    g = torch.Generator(device="cuda").manual_seed(3)
    s.plan()
    k, v = torch.randn(2, 1100, n_kvh * hd, device="cuda", generator=g)
    s.pool.append(0, k, v, s.slot[:1100])
    q = torch.randn(1100, n_head, hd, device="cuda", generator=g)
    out = torch.empty(1100, n_head, hd, device="cuda")
    scale = float(hd ** -0.5)
    s.pool.attend(0, q, out, s.d_rows, s.start, s.d_table, n_head, scale, max_add=1100)
    kr, vr = torch.empty(2, 1100, n_kvh * hd, device="cuda")
    s.pool.gather(0, s.slot[:1100], kr, vr)
    want = attend_exact(q, kr.view(-1, n_kvh, hd), vr.view(-1, n_kvh, hd), None, 0, scale)
    assert ((out.double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()
    # 290 pages before the same tokens: all of the first 286 the same page, whose rows are zeros but for V
    s.pool.append(0, torch.zeros(256, n_kvh * hd, device="cuda"), torch.ones(256, n_kvh * hd, device="cuda"), torch.arange(256, dtype=torch.int32, device="cuda") + s.free_now()[0] * page)
    table = torch.full_like(s.d_table, -1)
    table[0, :286] = s.free_now()[0]
    table[0, 286:291] = s.d_table[0, :5]
    s.pool.attend(0, q, out, ints([286 * 256]), s.start, table, n_head, scale, max_add=1100)
    assert L.q4_gpu_last_error() == 0
    # 73 216 weights of exp(0) on ones beside the tokens' own
    kr, vr = (x.view(-1, n_kvh, hd).double().repeat_interleave(2, 1) for x in (kr, vr))
    for j in (0, 500, 1099):
        w = torch.einsum("hd,phd->hp", q[j].double(), kr[: j + 1]) * scale
        e = torch.exp(w)
        want = (286 * 256 + torch.einsum("hp,phd->hd", e, vr[: j + 1])) / (286 * 256 + e.sum(-1, keepdim=True))
        assert ((out[j].double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()


@pytest.mark.parametrize("hint", [0, 1, 2, 5, 100000])
def test_any_hint_is_right(hint):
    run_attend([400, 0, 90, 2000], [1, 45, 3, 130], 16, 2, 128, "q8_0", max_add=hint)
    run_attend([400], [77], 8, 2, 256, "f16", max_add=hint)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("add", [1, 33])
def test_requests_that_share_pages(kind, add):
    """a prefix of whole pages named by three tables"""
    page, prefix, n_head, n_kvh, hd = 16, 160, 16, 2, 128
    s, k, v = step_of([prefix + 7, prefix + 30, prefix], [add] * 3, kind, n_kvh, hd)
    shared = s.d_table[0, : prefix // page].clone()
    own = s.d_table.clone()
    s.d_table[1:, : prefix // page] = shared
    s.pool.append(0, k, v, s.slot[: 3 * add])
    q = torch.randn(3 * add, n_head, hd, device="cuda").to(torch.bfloat16)
    out = torch.empty(3 * add, n_head, hd, device="cuda")
    s.pool.attend(0, q, out, s.d_rows, s.start, s.d_table, n_head, float(hd ** -0.5), max_add=add)
    assert lib().q4_gpu_last_error() == 0 and not torch.equal(own, s.d_table)
    for r, h in enumerate(s.rows):
        table = s.d_table[r].tolist()
        kr, vr = torch.empty(2, h + add, n_kvh * hd, device="cuda")
        s.pool.gather(0, ints([table[p // page] * page + p % page for p in range(h + add)]), kr, vr)
        at = r * add
        want = attend_exact(q[at: at + add], kr.view(-1, n_kvh, hd), vr.view(-1, n_kvh, hd), None, h, float(hd ** -0.5))
        assert ((out[at: at + add].double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()


@pytest.mark.parametrize("kind,n_pages", [("f16", 2600), ("q8_0", 4700)])
@pytest.mark.parametrize("add", [[1, 1, 1], [3, 70, 1], [1, 1, 1200]])
def test_a_pool_of_more_than_4_gb(kind, n_pages, add):
    """pages of 2 and 1.1 MB anywhere in it"""
    n_head, n_kvh, hd, page, rows = 64, 8, 256, 256, [3000, 700, 5]
    s, k, v = step_of(rows, add, kind, n_kvh, hd, page, n_pages=n_pages)
    n = sum(add)
    assert s.pool.mem.numel() > 1 << 32 and int(s.d_table.max()) * (s.pool.mem.numel() // n_pages) > 1 << 32
    s.pool.append(0, k, v, s.slot[:n])
    q = torch.randn(n, n_head, hd, device="cuda").to(torch.bfloat16)
    out = torch.empty(n, n_head, hd, device="cuda")
    s.pool.attend(0, q, out, s.d_rows, s.start, s.d_table, n_head, float(hd ** -0.5))
    assert lib().q4_gpu_last_error() == 0
    at = 0
    for r, (h, m) in enumerate(zip(rows, add)):
        table = s.d_table[r].tolist()
        kr, vr = torch.empty(2, h + m, n_kvh * hd, device="cuda")
        s.pool.gather(0, ints([table[p // page] * page + p % page for p in range(h + m)]), kr, vr)
        assert torch.isfinite(kr).all() and (kr[h:] - k[at: at + m]).abs().max() < 4 / 127     # where append put them
        want = attend_exact(q[at: at + m], kr.view(-1, n_kvh, hd), vr.view(-1, n_kvh, hd), None, h, float(hd ** -0.5))
        assert ((out[at: at + m].double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()
        at += m


def test_rows_behind_the_step_s_tokens_are_left_alone():
    for n_head, n_kvh, hd, add in ((16, 2, 128, [2, 1]), (24, 2, 256, [50, 1])):
        s, k, v = step_of([20, 300], add, "q8_0", n_kvh, hd)
        n = sum(add)
        s.pool.append(0, k, v, s.slot[:n])
        q = torch.randn(n + 40, n_head, hd, device="cuda")
        q[n:] = float("nan")
        out = torch.full_like(q, 5.0)
        s.pool.attend(0, q, out, s.d_rows, s.start, s.d_table, n_head, 0.1)
        assert torch.isfinite(out[:n]).all() and (out[n:] == 5).all() and not (out[:n] == 5).all()
        assert lib().q4_gpu_last_error() == 0


class Session:
    """two kinds of step, whose inputs stay where they are while their contents change"""

    def __init__(self, max_tok, n_pages=400, n_head=16, n_kvh=2, hd=128, page=16):
        self.n_head, self.n_kvh, self.hd, self.page = n_head, n_kvh, hd, page
        self.pool = q4gpu.PagePool(1, n_kvh, hd, n_pages, page, q4gpu.KIND_Q8)
        self.n_pages = n_pages
        self.rows, self.add, self.after = ints([0] * 3), ints([0] * 3), ints([0] * 3)
        self.table = torch.full((3, 200), -1, dtype=torch.int32, device="cuda")
        self.start = ints([0] * 4)
        self.slot, self.pos, self.req = (ints([0] * max_tok) for _ in range(3))
        self.k, self.v = torch.randn(2, max_tok, n_kvh * hd, device="cuda")
        self.q = torch.randn(max_tok, n_head, hd, device="cuda").to(torch.bfloat16)
        self.out = torch.zeros(max_tok, n_head, hd, device="cuda")
        self.history = [[] for _ in range(3)]

    def launch(self, max_add):
        p = self.pool
        p.plan(self.rows, self.add, self.table, self.start, self.slot, self.pos, self.req)
        p.append(0, self.k, self.v, self.slot)
        p.attend(0, self.q, self.out, self.rows, self.start, self.table, self.n_head, float(self.hd ** -0.5), max_add=max_add)

    def new(self, rows, add, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rows.copy_(ints(rows))
        self.add.copy_(ints(add))
        for t in (self.k, self.v, self.q):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        self.out.fill_(9.0)

    def check(self, rows, add):
        at, table = 0, self.table.tolist()
        for r, (h, n) in enumerate(zip(rows, add)):
            kr, vr = torch.empty(2, h + n, self.n_kvh * self.hd, device="cuda")
            self.pool.gather(0, ints([table[r][p // self.page] * self.page + p % self.page for p in range(h + n)]), kr, vr)
            self.history[r] = self.history[r][:h] + [row for row in self.k[at: at + n].cpu()]
            assert (kr.cpu() - torch.stack(self.history[r])).abs().max() < 4 / 127      # codes: half a step of at most 5 / 127
            want = attend_exact(self.q[at: at + n], kr.view(-1, self.n_kvh, self.hd), vr.view(-1, self.n_kvh, self.hd), None, h, float(self.hd ** -0.5))
            assert ((self.out[at: at + n].double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()
            at += n
        assert (self.out[at:] == 9).all()
        assert int(self.pool.n_free[0]) == self.n_pages - sum(-(-(h + n) // self.page) for h, n in zip(rows, add))


@pytest.mark.parametrize("max_add,steps", [(1, [[1, 1, 1]] * 4 + [[1, 0, 1], [0, 0, 1], [1, 1, 1]]), (0, [[40, 1, 200], [3, 1, 1], [1, 130, 77], [0, 9, 0], [1, 1, 1]])])
def test_a_captured_step_is_replayed_while_its_lengths_change(max_add, steps):
    L = lib()
    L.q4_gpu_last_error()
    assert L.q4_gpu_set_stream(None)              # captures need a created stream
    try:
        with torch.cuda.stream(torch.cuda.ExternalStream(L.q4_gpu_stream())):
            s = Session(250)
            first = [30, 500, 200] if max_add else [300, 60, 0]
            s.new([0, 0, 0], [min(n, 200) if max_add == 0 else 0 for n in first], 1)
            rows = [0, 0, 0]
            if max_add:                           # a prompt each, in chunks
                while any(h < n for h, n in zip(rows, first)):
                    add = [min(80, n - h) for h, n in zip(rows, first)]
                    s.new(rows, add, sum(rows))
                    s.launch(0)
                    s.check(rows, add)
                    rows = [h + n for h, n in zip(rows, add)]
            s.new(rows, [0, 0, 0], 2)
            s.launch(max_add)                     # its scratch is made outside the capture
            assert L.q4_hip_graph_begin()
            s.launch(max_add)
            graph = L.q4_hip_graph_end()
            assert graph
            for i, add in enumerate(steps):
                s.new(rows, add, 100 + i)
                assert L.q4_hip_graph_launch(graph)
                s.check(rows, add)
                rows = [h + n for h, n in zip(rows, add)]
            L.q4_hip_graph_free(graph)
            s.after.copy_(ints(rows))
            s.pool.trim(s.after, ints([0, 0, 0]), s.table)
            assert sorted(s.pool.free.tolist()) == list(range(s.n_pages)) and int(s.pool.n_free[0]) == s.n_pages
            assert L.q4_gpu_last_error() == 0
    finally:
        lib()


def test_another_stream():
    """the step on a stream of the caller's, behind and before work of that stream"""
    L = lib()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        q4gpu.use_torch_stream()
        try:
            s = Session(40)
            rows = [0, 0, 0]
            for i in range(4):
                big = torch.randn(4096, 4096, device="cuda")
                s.new(rows, [5 + i, 1, 20], i)
                s.q += (big @ big).sum().to(torch.bfloat16) * 0     # ready late
                s.launch(20)
                s.check(rows, [5 + i, 1, 20])
                rows = [h + n for h, n in zip(rows, [5 + i, 1, 20])]
        finally:
            st.synchronize()
    assert lib() and L.q4_gpu_last_error() == 0


def test_scratch_does_not_grow_inside_a_capture():
    L = lib()
    L.q4_gpu_set_stream(None)
    L.q4_hip_shutdown()                           # gives back what other tests made it reserve
    L = q4gpu.init()
    try:
        with torch.cuda.stream(torch.cuda.ExternalStream(L.q4_gpu_stream())):
            s = Session(100)
            s.new([0, 0, 0], [10, 1, 60], 0)
            torch.cuda.synchronize()
            assert L.q4_hip_graph_begin()
            with pytest.raises(RuntimeError, match="0x8"):
                s.launch(0)
            graph = L.q4_hip_graph_end()
            if graph:
                L.q4_hip_graph_free(graph)
            s.launch(0)                           # outside it does
            s.check([0, 0, 0], [10, 1, 60])
    finally:
        lib()
    assert L.q4_gpu_last_error() == 0


def test_dense_tensors_only():
    s = Step([5, 6], [1, 1], n_kvh=2, hd=128).plan()
    q = torch.zeros(2, 32, 128, device="cuda")
    out = torch.zeros(2, 16, 128, device="cuda")
    k = torch.zeros(2, 512, device="cuda")
    with pytest.raises(RuntimeError, match="dense"):
        s.pool.attend(0, q[:, ::2], out, s.d_rows, s.start, s.d_table, 16, 0.1)
    with pytest.raises(RuntimeError, match="dense"):
        s.pool.append(0, k[:, :256], k[:, 256:], s.slot[:2])
    with pytest.raises(RuntimeError, match="dense"):
        s.pool.plan(s.d_rows, s.d_add, s.d_table.t(), s.start, s.slot, s.pos, s.req)
    with pytest.raises(RuntimeError, match="dense"):
        s.pool.trim(s.d_rows, s.d_rows, s.d_table[:, ::2])
    for q2, out2, rows in ((q[:, :16].half().contiguous(), out, s.d_rows), (q[:, :16].contiguous(), out.double(), s.d_rows), (q[:, :16].contiguous(), out, s.d_rows.long())):
        with pytest.raises(RuntimeError, match="dense tensor of"):
            s.pool.attend(0, q2, out2, rows, s.start, s.d_table, 16, 0.1)
    with pytest.raises(RuntimeError, match="dense tensor of"):
        s.pool.append(0, k[:, :256].to(torch.bfloat16).contiguous(), k[:, :256].contiguous(), s.slot[:2])
    assert lib().q4_gpu_last_error() == 0
