"""Norm, rotation and append of a step's rows (q4_gpu_pages_prep) against the formulas in 64 bits, over the head sizes, layouts and types; what it
leaves out; what it refuses."""
import ctypes

import numpy as np
import pytest
import torch

import q4gpu
from gpu_util import lib

pytestmark = pytest.mark.gpu
KINDS = {"q8_0": q4gpu.KIND_Q8, "f16": q4gpu.KIND_F16}
EPS = 1e-6


def turned(x, pos, n_rot, base, half, mag):
    """rows [token][head][hd] in 64 bits, and for every number the size of what it is summed from"""
    n = n_rot // 2
    y, size = x.clone(), x.abs()
    f = base ** (-2.0 * torch.arange(n, dtype=torch.float64, device=x.device) / max(n_rot, 1))
    angle = (pos.double()[:, None] * f)[:, None]
    a, b = (slice(0, n), slice(n, n_rot)) if half else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    xa, xb = x[..., a].clone(), x[..., b].clone()
    y[..., a] = mag * (xa * torch.cos(angle) - xb * torch.sin(angle))
    y[..., b] = mag * (xa * torch.sin(angle) + xb * torch.cos(angle))
    both = mag * (xa.abs() + xb.abs())
    size[..., a], size[..., b] = both, both
    return y, size


def normed(x, w, eps):
    if eps is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        x = x * w.double() if w is not None else x
    return x


class Case:
    def __init__(self, n_head, n_kvh, hd, kind, n_tok, n_rot, half=False, gate=True, bf16=False, out_bf16=True, fused=False, page=16, layers=2, mag=1.0, base=1e6, eps=EPS,
                 weights=True, far=262144, seed=0, idle=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        on = dict(device="cuda", generator=g)
        dtype = torch.bfloat16 if bf16 else torch.float32
        self.n_head, self.n_kvh, self.hd, self.n_tok, self.half, self.n_rot, self.mag, self.base, self.eps, self.out_bf16 = n_head, n_kvh, hd, n_tok, half, n_rot, mag, base, eps, out_bf16
        self.page = page
        widths = [n_head * hd * (2 if gate else 1), n_kvh * hd, n_kvh * hd]
        rows = (torch.randn(n_tok, sum(widths) + (16 if fused else 0), **on) * torch.exp(2 * torch.randn(n_tok, 1, **on))).to(dtype)
        parts = rows[:, 16 if fused else 0:].split(widths, 1)
        self.q, self.k, self.v = parts if fused else [x.contiguous() for x in parts]
        self.wq, self.wk = (1 + 0.3 * torch.randn(2, hd, **on)).unbind(0) if weights else (None, None)
        self.pos = torch.randint(0, far, (n_tok,), dtype=torch.int32, **on)
        n_pages = n_tok // page + 3
        self.pool = q4gpu.PagePool(layers, n_kvh, hd, n_pages, page, KINDS[kind], mem=torch.full((lib().q4_gpu_pages_bytes(layers, n_kvh, hd, n_pages, page, KINDS[kind]),), 0xff, dtype=torch.uint8, device="cuda"))
        self.slot = torch.randperm(n_pages * page, **on)[:n_tok].int()
        if idle:
            self.pos[n_tok - idle:] = -1
            self.slot[n_tok - idle:] = -1
        self.rope = q4gpu.Rope(n_rot, base, half=half, mag=mag)
        self.q_out = torch.full((n_tok, n_head, hd), 7.0, dtype=torch.bfloat16 if out_bf16 else torch.float32, device="cuda")
        self.gate = torch.full((n_tok, n_head, hd), 7.0, device="cuda") if gate else None
        self.kind = kind

    def run(self, layer=1):
        lib().q4_gpu_last_error()
        self.pool.prep(layer, self.q, self.k, self.v, self.q_out, self.pos, self.slot, self.rope, wq=self.wq, wk=self.wk, eps=self.eps, gate=self.gate)
        return self

    def rows(self, layer=1):
        k, v = torch.empty(2, self.n_tok, self.n_kvh * self.hd, device="cuda")
        self.pool.gather(layer, self.slot, k, v)
        return k.view(self.n_tok, self.n_kvh, self.hd), v.view(self.n_tok, self.n_kvh, self.hd)

    def check(self, live=None):
        live = torch.ones(self.n_tok, dtype=torch.bool, device="cuda") if live is None else live
        q = self.q.double().unflatten(1, (self.n_head, -1))
        if self.gate is not None:
            assert torch.equal(self.gate[live], q[..., self.hd:].float()[live])
            assert (self.gate[~live] == 7).all()
        # the sum of squares is 10 roundings deep at most, its root, the quotient and two products 4, half of the sum's error goes into the root: 10; the angle is off by
        # 2^-26 turns and sine and cosine by 2 units: 4.5 x 2^-24; mag, two products and a sum: 3.  Together below 20 x 2^-24 of the two numbers' sizes
        step = 20 * 2.0**-24
        want, size = turned(normed(q[..., : self.hd], self.wq, self.eps), self.pos, self.n_rot, self.base, self.half, self.mag)
        off = (self.q_out.double() - want).abs() - step * size - (2.0**-8 * want.abs() if self.out_bf16 else 0)
        assert off[live].max() <= 0
        assert (self.q_out[~live] == 7).all()
        k, v = self.rows()
        want, size = turned(normed(self.k.double().unflatten(1, (self.n_kvh, -1)), self.wk, self.eps), self.pos, self.n_rot, self.base, self.half, self.mag)
        for got, want, size in ((k, want, size), (v, self.v.double().unflatten(1, (self.n_kvh, -1)), 0 * size)):
            if self.kind == "q8_0":
                # a code is half a step off, or as much more as the value is, over the step amax / 127, which fp16 rounds by 2^-11 (half its smallest number for small ones)
                amax = want.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
                d = amax / 127 * (1 + 2.0**-20)
                tol = (d * 0.5 * (1 + 2.0**-10) + amax * 2.0**-11 + 127 * 2.0**-25).expand(-1, -1, -1, 32).flatten(-2) + 3 * step * size
            else:
                tol = want.abs() * 2.0**-11 + 2.0**-25 + 1.01 * step * size
            assert ((got.double() - want).abs() - tol)[live].max() <= 0
        assert lib().q4_gpu_last_error() == 0
        return self


SHAPES = [(16, 2, 128), (24, 2, 256), (8, 4, 64), (5, 5, 64), (3, 1, 128), (32, 8, 128), (1, 1, 256)]


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n_tok,gate,bf16,fused", [(1, True, False, False), (37, False, True, True), (200, True, True, False), (701, True, False, True)])
def test_rows(kind, half, shape, n_tok, gate, bf16, fused):
    Case(*shape, kind, n_tok, shape[2], half=half, gate=gate, bf16=bf16, fused=fused, out_bf16=n_tok % 2 == 1, seed=n_tok).run().check()


@pytest.mark.parametrize("shape,n_rot,half", [((24, 2, 256), 64, False), ((24, 2, 256), 64, True), ((24, 2, 256), 136, True), ((24, 2, 256), 2, False), ((24, 2, 256), 130, False), ((16, 2, 128), 32, True),
                                              ((16, 2, 128), 8, True), ((16, 2, 128), 6, False), ((16, 2, 128), 72, True), ((8, 4, 64), 16, True), ((8, 4, 64), 40, True), ((8, 4, 64), 24, False),
                                              ((16, 2, 128), 0, False), ((16, 2, 128), 0, True)])
@pytest.mark.parametrize("n_tok", [3, 640])
def test_part_of_the_head(shape, n_rot, half, n_tok):
    Case(*shape, "f16", n_tok, n_rot, half=half, out_bf16=False, mag=1.3).run().check()


@pytest.mark.parametrize("eps,weights", [(None, True), (0.0, True), (1e-5, False), (10.0, True)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_norms(eps, weights, hd):
    Case(4, 2, hd, "f16", 50, hd, out_bf16=False, eps=eps, weights=weights).run().check()


def test_a_row_of_zeros_has_no_nan():
    c = Case(4, 2, 128, "q8_0", 5, 128, out_bf16=False)
    c.q[2], c.k[2], c.v[2] = 0, 0, 0
    c.run().check()
    assert (c.q_out[2] == 0).all() and all((x[2] == 0).all() for x in c.rows())


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("n_tok", [2, 1000])
def test_positions_up_to_the_last(page, n_tok):
    c = Case(6, 2, 128, "f16", n_tok, 128, half=True, page=page, out_bf16=False, far=2**31 - 1)
    c.pos[0], c.pos[1] = 0, 2**31 - 1
    c.run()
    # the definition's angle in 64 bits is itself off by 2^-53 of pos there: 2^31 x 2^-53 radians, beside which 20 x 2^-24 is large
    c.check()


def test_idle_places_are_left_alone():
    c = Case(16, 2, 128, "q8_0", 70, 128, idle=6, out_bf16=False)
    before = c.pool.mem.clone()
    c.run()
    live = c.pos >= 0
    c.check(live)
    touched = c.pool.mem.view(2, -1, 2, 16, 272)[1].ne(before.view(2, -1, 2, 16, 272)[1]).any(-1).any(1).sum()
    assert touched <= 64
    assert torch.equal(c.pool.mem.view(2, -1)[0], before.view(2, -1)[0])     # the other layer


def test_rows_without_a_slot_keep_their_queries():
    c = Case(16, 2, 128, "f16", 9, 128, out_bf16=False)
    want = c.run().q_out.clone()
    before = c.pool.mem.clone()
    c.slot.fill_(-1)
    c.q_out.zero_()
    c.run()
    assert torch.equal(c.q_out, want) and torch.equal(c.pool.mem, before)
    assert lib().q4_gpu_last_error() == 0
    c.slot[4] = c.pool.n_pages * c.page
    c.run()
    assert torch.equal(c.pool.mem, before)
    assert lib().q4_gpu_last_error() == 4


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
def test_what_is_not_finite_stays_in_its_row(kind):
    c = Case(4, 2, 64, kind, 20, 64, out_bf16=False)
    q, k = c.run().q_out.clone(), c.rows()
    c.q[7, 64 * 2 + 5] = float("inf")           # head 1 of token 7
    c.k[8, 3], c.v[9, 64 + 40] = float("nan"), float("inf")
    c.run()
    same = torch.ones(20, 4, dtype=torch.bool, device="cuda")
    same[7, 1] = False
    assert torch.equal(c.q_out[same], q[same])
    same = torch.ones(20, 2, dtype=torch.bool, device="cuda")
    same[8, 0] = same[9, 1] = False
    for got, want in zip(c.rows(), k):
        assert torch.equal(got[same], want[same])


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_are_those_of_append(kind, hd):
    c = Case(4, 2, hd, kind, 66, hd).run()
    _, got = c.rows()
    c.pool.append(0, c.k, c.v, c.slot)
    _, want = c.rows(0)
    assert torch.equal(got, want)


def test_as_the_single_session_s_prep():
    n_head, n_kvh, hd, n_rot, n = 24, 2, 256, 64, 33
    c = Case(n_head, n_kvh, hd, "f16", n, n_rot, base=1e7, out_bf16=False)
    c.pos.copy_(torch.arange(100, 100 + n))
    c.run()
    L = lib()
    q, g, k = torch.empty(n, n_head, hd, device="cuda"), torch.empty(n, n_head, hd, device="cuda"), c.k.clone()
    assert L.q4_hip_qsa_q_prep_n(c.q.data_ptr(), c.wq.data_ptr(), q.data_ptr(), g.data_ptr(), n_head, hd, n_rot, 100, 1e7, EPS, n)
    assert L.q4_hip_qsa_k_prep_n(k.data_ptr(), c.wk.data_ptr(), n_kvh, hd, n_rot, 100, 1e7, EPS, n)
    assert torch.equal(c.gate, g)
    # the angle there is in fp32: off by 2^-24 of up to 132 radians and of its frequency (powf: 2 units), 4e-5 of sizes up to 8
    assert (c.q_out - q).abs().max() < 132 * 6 * 2.0**-24 * c.q_out.abs().max()
    got, _ = c.rows()
    assert (got - k.view(n, n_kvh, hd)).abs().max() < 2.0**-11 * k.abs().max() + 132 * 6 * 2.0**-24 * k.abs().max()


def test_captured_and_replayed_with_other_positions():
    c = Case(16, 2, 128, "q8_0", 40, 128, out_bf16=False)
    L = lib()
    c.run().check()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    L.q4_gpu_set_stream(s.cuda_stream)
    try:
        assert L.q4_hip_graph_begin()
        c.pool.prep(1, c.q, c.k, c.v, c.q_out, c.pos, c.slot, c.rope, wq=c.wq, wk=c.wk, eps=c.eps, gate=c.gate)
        graph = L.q4_hip_graph_end()
        assert graph
        c.rope.turn[1] = 0                       # the call has taken the descriptor along
        for seed in (1, 2):
            c.pos.copy_(torch.randint(0, 100000, (40,), generator=torch.Generator().manual_seed(seed)))
            c.k.mul_(-0.5)
            torch.cuda.synchronize()
            assert L.q4_hip_graph_launch(ctypes.c_void_p(graph))
            L.q4_hip_stream_sync()
            c.check()
        L.q4_hip_graph_free(ctypes.c_void_p(graph))
    finally:
        q4gpu.use_torch_stream()


def test_refusals():
    c = Case(4, 2, 128, "q8_0", 6, 128)
    L, p = lib(), lambda t: None if t is None else t.data_ptr()  # noqa: E731
    before = c.pool.mem.clone()

    def call(**other):
        a = dict(pg=c.pool.p, layer=0, q=p(c.q), k=p(c.k), v=p(c.v), bf16=0, qs=c.q.stride(0), ks=c.k.stride(0), n_head=4, wq=p(c.wq), wk=p(c.wk), eps=EPS, rope=c.rope.p, pos=p(c.pos), slot=p(c.slot),
                 n_tok=6, q_out=p(c.q_out), out_bf16=1, gate=p(c.gate))
        a.update(other)
        return L.q4_gpu_pages_prep(*a.values())

    L.q4_gpu_last_error()
    wide = q4gpu.Rope(256, 1e4)
    for other in (dict(pg=None), dict(layer=2), dict(q=None), dict(k=None), dict(v=None), dict(rope=None), dict(pos=None), dict(slot=None), dict(q_out=None), dict(n_tok=0), dict(n_head=0),
                  dict(qs=c.q.stride(0) - 4), dict(ks=2), dict(ks=c.k.stride(0) + 2), dict(q=p(c.q) + 4), dict(gate=p(c.gate) + 8), dict(wq=p(c.wq) + 4), dict(eps=float("nan")), dict(rope=wide.p),
                  dict(n_tok=2**31), dict(q_out=p(c.q_out) + 2)):
        assert not call(**other)
        assert L.q4_gpu_last_error() == 1, other
    torch.cuda.synchronize()
    assert torch.equal(c.pool.mem, before) and (c.q_out == 7).all()
    assert call() and L.q4_gpu_last_error() == 0
    with pytest.raises(RuntimeError):
        c.pool.prep(0, c.q, c.k, c.v.double(), c.q_out, c.pos, c.slot, c.rope, gate=c.gate)
    with pytest.raises(RuntimeError):
        c.pool.prep(0, c.q, c.k, c.v[:, :-4], c.q_out, c.pos, c.slot, c.rope, gate=c.gate)
    with pytest.raises(RuntimeError):
        c.pool.prep(0, c.q, c.k, torch.empty(6, 300, device="cuda")[:, :256], c.q_out, c.pos, c.slot, c.rope, gate=c.gate)
    assert np.isfinite(c.q_out.float().cpu().numpy()).all()
