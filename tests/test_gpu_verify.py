"""Drafts held against the target's distributions (q4_gpu_verify) against the definition in 64 bits, request by request; edges of the vocabulary, masks,
temperatures, what is no distribution; the distribution that comes out; captured; refusals."""
import ctypes
import math

import pytest
import torch

import q4gpu
from gpu_util import lib

pytestmark = pytest.mark.gpu
INF = float("inf")


def softmax(x, t):
    z = (x.double() - x.double().max()) / t
    return z.exp() / z.exp().sum()


def plain(c):
    """accepted, next, logp by request, and whether any of them has no distribution"""
    accepted, nexts, logp, bad = [], [], torch.zeros(c.n_tok, dtype=torch.float64), False
    start, token = c.start.tolist(), c.token.tolist()
    for r in range(c.n_req):
        a, b = start[r], start[r + 1]
        t = float(c.temp[r]) if c.temp is not None else 1.0
        if a == b:
            accepted.append(0)
            nexts.append(-1)
            continue
        at, n = a, -1
        while True:
            x = c.logits[at]
            q = c.draft[at] if c.draft is not None and at + 1 < b and t != 0 else None
            rows = [x] + ([q] if q is not None else [])
            if not (0 <= t < INF) or any(not (float(y.max()) < INF) or float(y.max()) == -INF or bool(y.isnan().any()) for y in rows):
                bad = True
                break
            last, d = at + 1 == b, token[at + 1] if at + 1 < b else None
            inside = d is not None and 0 <= d < c.vocab
            bad |= d is not None and not inside
            if t == 0:
                n = int(torch.nonzero(x == x.max())[0])
                if not last and d == n:
                    at, n = at + 1, -1
                    continue
                break
            p = softmax(x, t)
            if last:
                w = p
            else:
                q = softmax(q, t) if q is not None else torch.nn.functional.one_hot(torch.tensor(d if inside else 0, device=x.device), c.vocab).double() * inside
                if inside and float(c.u_accept[at]) * float(q[d]) < float(p[d]):
                    logp[at] = math.log(float(p[d]))
                    at += 1
                    continue
                w = (p - q).clamp(min=0)
                if float(w.sum()) == 0:
                    w = p
            s = w.cumsum(0)
            above = torch.nonzero(s > float(c.u_next[r]) * float(s[-1]))
            n = int(above[0]) if len(above) else int(torch.nonzero(w > 0)[-1])
            logp[at] = math.log(float(p[n]))
            break
        accepted.append(at - a)
        nexts.append(n)
    return accepted, nexts, logp, bad


class Case:
    def __init__(self, drafts, vocab, bf16=False, draft="logits", temp=None, ld=None, seed=0, sharp=2.0, idle=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        on = dict(device="cuda", generator=g)
        self.vocab, self.n_req = vocab, len(drafts)
        add = [n + 1 if n is not None else 0 for n in drafts]          # None: a request without tokens
        start = [0]
        for n in add:
            start.append(start[-1] + n)
        self.live, self.n_tok = start[-1], start[-1] + idle
        ld = vocab if ld is None else ld
        dtype = torch.bfloat16 if bf16 else torch.float32
        x = torch.randn(self.n_tok, ld, **on) * sharp
        y = x + torch.randn(self.n_tok, ld, **on) * (0.4 * sharp)
        self.logits = x.to(dtype)[:, :vocab]
        self.draft = y.to(dtype)[:, :vocab] if draft == "logits" else None
        token = torch.multinomial(torch.softmax(y[:, :vocab], 1), 1, generator=g)[:, 0] if vocab < 2**20 else y[:, :vocab].argmax(1)
        self.token = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), token.int()[:-1]]) if self.n_tok else token.int()
        self.start = torch.tensor(start, dtype=torch.int32, device="cuda")
        self.temp = None if temp is None else torch.tensor([temp[i % len(temp)] for i in range(self.n_req)], device="cuda")
        self.u_accept, self.u_next = torch.rand(self.n_tok, **on), torch.rand(self.n_req, **on)
        self.rows = torch.randint(0, 1000, (self.n_req,), dtype=torch.int32, **on)
        word = dict(dtype=torch.int32, device="cuda")
        self.accepted, self.next, self.keep = (torch.full((self.n_req,), -7, **word) for _ in range(3))
        self.logp = torch.full((self.n_tok,), 5.0, device="cuda")

    def run(self, **kw):
        lib().q4_gpu_last_error()
        a = dict(draft=self.draft, temp=self.temp, logp=self.logp, rows=self.rows, keep=self.keep)
        a.update(kw)
        q4gpu.verify(self.logits, self.token, self.start, self.u_accept, self.u_next, self.accepted, self.next, **a)
        return self

    def check(self):
        accepted, nexts, logp, bad = plain(self)
        assert lib().q4_gpu_last_error() == (4 if bad else 0)
        assert self.accepted.tolist() == accepted
        assert self.next.tolist() == nexts
        tokens = (self.start[1:] - self.start[:-1]).tolist()
        assert self.keep.tolist() == [h + (k + 1 if n else 0) for h, k, n in zip(self.rows.tolist(), accepted, tokens)]
        got = self.logp.cpu().double()
        # rounded to fp32 once.  log p = (x - M) / T - log S: S is off by 5e-9 of itself at most, which is by how much its logarithm is: its terms' exponents by
        # 2.25 x 2^-25 steps of ln 2 / 32 = 1.5e-9, the last factor of each, e^q - 1 < 0.0109, by 1.5 x 2^-25 of that = 5e-10 and by its series' fourth term,
        # q^4 / 24 = 6e-10, up to eight of these added in 32 bits by 7 x 2^-25 x 0.0109 = 2.3e-9; all else is in 64 bits
        assert ((got - logp).abs() <= 2.0**-24 * logp.abs() * (1 + 1e-6) + 5e-9)[: self.live].all()
        assert (got[self.live:] == 5).all()
        return self


VOCABS = [1, 2, 31, 255, 8191, 8192, 8193, 50001]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("draft", ["logits", "none"])
def test_drafts(vocab, bf16, draft):
    Case([3, 0, 5, 1, 8, 2, 4], vocab, bf16, draft, temp=[0.7, 1.0, 1.3, 0.0], seed=vocab).run().check()


@pytest.mark.parametrize("drafts", [[0], [1], [7], [8], [9], [40], [0] * 70, [None, 3, None, None, 2, None], [None], [2] * 33, [1, None] * 40, [5, 17, 16, 0]])
@pytest.mark.parametrize("draft", ["logits", "none"])
def test_numbers_of_drafts(drafts, draft):
    idle = 3 if drafts != [None] else 1
    c = Case(drafts, 500, False, draft, seed=len(drafts), idle=idle, sharp=0.7)
    if draft == "none":       # certain drafts that are likely
        c.logits[torch.arange(c.n_tok - 1), c.token[1:].long()] += 8.0
    c.run().check()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("ld", [1003, 1008, 4001])
def test_rows_apart(bf16, ld):
    Case([2, 3, 0], 1001, bf16, ld=ld, seed=ld).run().check()


def test_large_vocabulary_and_many_requests():
    Case([4] * 20, 200003, True, seed=3, sharp=3.0).run().check()
    Case([0] * 300, 32003, False, seed=4, temp=[0.9, 0.0, 0.5]).run().check()


@pytest.mark.parametrize("vocab", [32768 - 3, 32768 + 1, 6 * 32768 + 1, 600001])
@pytest.mark.parametrize("draft", ["logits", "none"])
def test_vocabularies_around_a_lane_s_share_of_chunks(vocab, draft):
    c = Case([2, 0, 1, 3], vocab, draft=draft, temp=[1.0, 3.0, 0.8, 0.0], seed=vocab, sharp=1.5)
    for u in (0.0, 0.3, 0.9999):
        c.u_next.fill_(u)
        c.run().check()


@pytest.mark.parametrize("sharp", [0.0, 0.01, 30.0])
def test_flat_and_sharp(sharp):
    for seed in range(4):
        Case([2, 0, 3, 4], 30011, seed=seed, sharp=sharp).run().check()


@pytest.mark.parametrize("draft", ["logits", "none"])
def test_masked_tokens_are_never_drawn(draft):
    c = Case([3] * 40, 9001, draft=draft, seed=5)
    keep = torch.rand(c.n_tok, c.vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.01
    keep[:, 8999] = True
    c.logits.masked_fill_(~keep, -INF)
    c.u_next[:20] = 0.0
    c.u_accept[: c.n_tok // 2] = 0.0
    c.run().check()
    start = c.start.tolist()
    for r, (k, n) in enumerate(zip(c.accepted.tolist(), c.next.tolist())):
        assert bool(keep[start[r] + k, n])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("draft", ["logits", "none"])
def test_tokens_masked_by_the_type_s_lowest_value(bf16, draft):
    """finite, so that they count where there is nothing else: a row of them alone is flat"""
    c = Case([2, 0, 3, 1] * 3, 5003, bf16=bf16, draft=draft, seed=20)
    keep = torch.rand(c.n_tok, c.vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) < 0.02
    keep[5] = False
    c.logits.masked_fill_(~keep, torch.finfo(c.logits.dtype).min)
    c.run().check()


@pytest.mark.parametrize("temp", [1e-30, 1e-37, 1e-38, 1e-45])
def test_temperatures_near_nothing(temp):
    """the largest logits share everything between them; with a largest of 0 their sizes in steps stay small"""
    c = Case([1, 0, 2], 5003, temp=[temp] * 3, seed=4)
    g = torch.Generator(device="cuda").manual_seed(5)
    for x in (c.logits, c.draft):
        x.clamp_(max=-0.01)
        x[torch.rand(x.shape, device="cuda", generator=g) < 0.01] = 0.0
    c.run().check()


def test_sizes_that_change_along_a_row():
    """chunks whose logits lie a thousand powers of two and more above or below those before them"""
    for seed in range(3):
        c = Case([1, 0, 2], 40000, seed=seed, sharp=1.0, temp=[1.0, 0.05, 20.0])
        for x in (c.logits, c.draft):
            x[:, 3000:6000] -= 3000.0
            x[:, 9000:9100] += 5.0
            x[:, :1500] -= 900.0
            x[1, 20000:] += 1500.0
            x[2, 39999] = 60000.0
        c.run().check()


def test_one_token_left_of_a_row():
    c = Case([2] * 9, 8200, seed=6)
    c.logits.fill_(-INF)
    c.logits[:, 8195] = -1e30
    c.token.fill_(8195)
    c.draft[:, 8195] = 50.0
    c.run().check()
    assert (c.next == 8195).all()


@pytest.mark.parametrize("u", [0.0, 1e-30, 0.5, 1 - 2.0**-24, 1.0, 2.0, float("nan")])
def test_ends_of_the_random_numbers(u):
    c = Case([2, 0, 1] * 5, 8300, seed=7, temp=[1.0, 0.3])
    c.u_next.fill_(u)
    if u <= 1:
        c.u_accept.fill_(u)
    c.run()
    if u == u:
        c.check()
    else:
        assert (c.next >= 0).all() and (c.next < c.vocab).all()


def test_draft_and_target_alike():
    c = Case([6] * 12, 20000, seed=8)
    c.draft.copy_(c.logits)
    c.run().check()
    assert (c.accepted == 6).all()
    c.u_accept.fill_(1.0)                    # u q < p does not hold: nothing of p is over q, so that p itself is drawn from
    c.run().check()
    assert (c.accepted == 0).all()


@pytest.mark.parametrize("scale", [1e-30, 1.0, 1e3, 3e38])
def test_sizes_of_logits(scale):
    c = Case([1, 2, 0], 8500, seed=9, sharp=1.0)
    for x in (c.logits, c.draft):
        x.div_(x.abs().amax()).mul_(scale)
    c.run().check()


def test_temperatures_from_tiny_to_large():
    Case([2, 1, 0, 3, 2, 2], 8200, seed=10, temp=[1e-38, 1e-3, 1e3, 3e38, 1e-45, 0.25]).run().check()


def test_greedy_takes_the_first_of_equals():
    c = Case([4, 0, 3, 20], 20000, temp=[0.0], seed=11)
    c.logits[:, 12345] = c.logits[:, 77] = 1e4
    c.token.fill_(77)
    c.token[2] = 12345
    c.run().check()
    assert (c.next == 77).all()
    assert (c.logp[: c.live] == 0).all()


@pytest.mark.parametrize("what", [float("nan"), INF])
@pytest.mark.parametrize("where", ["target", "draft", "last", "behind", "all of it"])
@pytest.mark.parametrize("greedy", [False, True])
def test_what_is_no_distribution(what, where, greedy):
    c = Case([3, 3, 3, 0], 8300, seed=12, temp=[0.0 if greedy else 1.0])
    # request 1's rows are 4 to 7: all its drafts would be kept
    best = c.logits[4:7].argmax(1).int()
    c.token[5:8] = best
    c.u_accept[4:7] = 0.0
    if where == "target":
        c.logits[5, 8299] = what
    elif where == "draft":
        c.draft[5, 100] = what
    elif where == "last":
        c.logits[7, 0] = what
    elif where == "behind":                  # a row behind the one that decides is not needed
        c.token[6] = -1 if greedy else c.vocab
        c.logits[6, 5] = what
    else:
        c.logits[4].fill_(-INF)
    c.run().check()
    first = {"target": 1, "draft": 3 if greedy else 1, "last": 3, "behind": 1, "all of it": 0}[where]
    assert int(c.accepted[1]) == first
    assert (int(c.next[1]) == -1) == (where != "behind" and not (where == "draft" and greedy))


@pytest.mark.parametrize("t", [-1.0, float("nan"), INF, -0.0])
def test_temperatures_that_are_none(t):
    c = Case([2, 2, 1], 700, seed=13, temp=[1.0, t, 0.5])
    c.run().check()
    assert (int(c.next[1]) == -1) == (t != 0)


def test_drafts_outside_the_vocabulary():
    for draft in ("logits", "none"):
        c = Case([2, 2, 2], 900, draft=draft, seed=14, temp=[1.0, 0.0])
        c.token[1], c.token[4], c.token[8] = 900, -5, 2**31 - 1
        c.run().check()


def test_what_may_be_left_out():
    c = Case([2, 0, 3], 3000, seed=15)
    c.run().check()
    want = c.next.tolist(), c.accepted.tolist()
    c.logp.fill_(5.0)
    c.keep.fill_(-7)
    c.run(logp=None, rows=None, keep=None)
    assert (c.next.tolist(), c.accepted.tolist()) == want
    assert (c.logp == 5).all() and (c.keep == -7).all()


@pytest.mark.parametrize("draft", ["logits", "none"])
def test_what_comes_out_is_the_target_s_distribution(draft):
    """all pairs of random numbers on a grid: the first token that is kept or drawn has the target's probabilities, whatever the draft's"""
    n, vocab = 64, 6
    c = Case([1] * (n * n), vocab, draft=draft, seed=16)
    p, q = torch.randn(vocab, device="cuda"), torch.randn(vocab, device="cuda")
    c.logits.copy_(p.expand(c.n_tok, -1))
    if draft == "logits":
        c.draft.copy_(q.expand(c.n_tok, -1))
    grid = (torch.arange(n, device="cuda") + 0.5) / n
    c.u_accept[0::2] = grid.repeat_interleave(n)
    c.u_next.copy_(grid.repeat(n))
    p, q = softmax(p, 1.0).cpu(), softmax(q, 1.0).cpu()
    got = torch.zeros(vocab, dtype=torch.float64)
    for d in range(vocab):
        c.token[1::2] = d
        c.run()
        assert lib().q4_gpu_last_error() == 0
        kept = c.accepted.cpu() == 1
        first = torch.where(kept, d, c.next.cpu())
        of_d = torch.bincount(first, minlength=vocab).double() / (n * n)
        if draft == "logits":
            got += float(q[d]) * of_d
        else:
            assert (of_d - p).abs().max() <= 2.0 / n + 1e-9          # certain drafts: each of them alone
    if draft == "logits":
        assert (got - p).abs().max() <= 2.0 / n                       # each of the two grids is off by one step


def test_the_same_again_and_captured():
    c = Case([3, 5, 0, 1] * 6, 12000, seed=17, idle=4)
    L = lib()
    c.run().check()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    L.q4_gpu_set_stream(s.cuda_stream)
    try:
        assert L.q4_hip_graph_begin()
        q4gpu.verify(c.logits, c.token, c.start, c.u_accept, c.u_next, c.accepted, c.next, draft=c.draft, logp=c.logp, rows=c.rows, keep=c.keep)
        graph = L.q4_hip_graph_end()
        assert graph
        for seed in range(3):
            g = torch.Generator(device="cuda").manual_seed(seed)
            c.u_accept.copy_(torch.rand(c.n_tok, generator=g, device="cuda"))
            c.u_next.copy_(torch.rand(c.n_req, generator=g, device="cuda"))
            if seed == 2:                    # other numbers of drafts in the same rows
                c.start.copy_(torch.tensor([0] + sorted(torch.randint(0, c.live, (c.n_req - 1,), generator=torch.Generator().manual_seed(3)).tolist()) + [c.live], dtype=torch.int32))
            torch.cuda.synchronize()
            for _ in range(2):
                assert L.q4_hip_graph_launch(ctypes.c_void_p(graph))
            L.q4_hip_stream_sync()
            c.check()
        L.q4_hip_graph_free(ctypes.c_void_p(graph))
    finally:
        q4gpu.use_torch_stream()


def test_starts_that_are_none_touch_nothing():
    c = Case([2, 2, 2], 600, seed=18)
    c.start.copy_(torch.tensor([0, 9999, -5, 9], dtype=torch.int32))
    c.run()
    assert lib().q4_gpu_last_error() == 4
    assert c.next.tolist()[:2] == [-1, -1]


def test_refusals():
    c = Case([2, 2], 600, seed=19, ld=601)
    L, p = lib(), lambda t: None if t is None else t.data_ptr()  # noqa: E731

    def call(**other):
        a = dict(logits=p(c.logits), bf16=0, ld=601, draft=p(c.draft), dld=601, vocab=600, token=p(c.token), start=p(c.start), n_req=2, n_tok=6, temp=None, ua=p(c.u_accept), un=p(c.u_next),
                 accepted=p(c.accepted), next=p(c.next), logp=p(c.logp), rows=p(c.rows), keep=p(c.keep))
        a.update(other)
        return L.q4_gpu_verify(*a.values())

    L.q4_gpu_last_error()
    for other in (dict(logits=None), dict(ld=599), dict(dld=10), dict(vocab=0), dict(token=None), dict(start=None), dict(n_req=0), dict(n_req=8193), dict(n_tok=0), dict(ua=None), dict(un=None),
                  dict(accepted=None), dict(next=None), dict(rows=None), dict(keep=None), dict(logits=p(c.logits) + 2), dict(bf16=1, draft=p(c.draft) + 1), dict(vocab=2**31, ld=2**32, dld=2**32)):
        assert not call(**other)
        assert L.q4_gpu_last_error() == 1, other
    torch.cuda.synchronize()
    assert (c.next == -7).all()
    assert call() and L.q4_gpu_last_error() == 0
    for bad in (dict(draft=c.draft.double()), dict(draft=c.draft[:, :599]), dict(temp=torch.ones(1, device="cuda")), dict(logp=torch.ones(6))):
        with pytest.raises(RuntimeError):
            c.run(**bad)


# ---- so many rows that those behind refused drafts are left out
@pytest.mark.parametrize("n_req,draft", [(110, "logits"), (200, "none")])
def test_many_rows(n_req, draft):
    c = Case([8] * (n_req - 2) + [None, 7], 50001, bf16=True, draft=draft, temp=[1.0, 0.0, 0.7, 1.2], seed=31, idle=3)
    if draft == "none":                                                     # half of the drafts are likely
        c.logits.scatter_add_(1, c.token.roll(-1).long()[:, None], 20 * (torch.arange(c.n_tok, device="cuda") % 2).to(c.logits.dtype)[:, None])
    c.run().check()
    first = [t.clone() for t in (c.accepted, c.next, c.keep, c.logp)]
    c.run()
    assert all(torch.equal(a, b) for a, b in zip(first, (c.accepted, c.next, c.keep, c.logp)))


class Many(Case):
    """a case whose requests can be taken by parts, in which nothing is left out"""
    def __init__(self, draft):
        gen = torch.Generator().manual_seed(8)
        drafts = torch.randint(-1, 9, (5000,), generator=gen).tolist()
        super().__init__([None if n < 0 else n for n in drafts], 300, draft=draft, temp=[1.0, 0.8, 0.0, 1.0, 0.6, -1.0, 1.1], seed=32, idle=9)
        kept = torch.rand(self.n_tok, device="cuda") < 0.5
        self.logits.scatter_add_(1, self.token.roll(-1).long()[:, None], 6 * kept.float()[:, None])
        self.logits[torch.rand(self.n_tok, device="cuda") < 0.03, 7] = float("nan")
        self.token[torch.rand(self.n_tok, device="cuda") < 0.03] = 300
        self.parts = 500

    def by_parts(self):
        out = [torch.full_like(t, x) for t, x in ((self.accepted, -7), (self.next, -7), (self.keep, -7), (self.logp, 5.0))]
        for r in range(0, self.n_req, self.parts):
            n, a, b = self.parts, int(self.start[r]), int(self.start[r + self.parts])
            q4gpu.verify(self.logits[a:b], self.token[a:b], self.start[r:r + n + 1] - a, self.u_accept[a:b], self.u_next[r:r + n], out[0][r:r + n], out[1][r:r + n],
                         draft=None if self.draft is None else self.draft[a:b], temp=self.temp[r:r + n], logp=out[3][a:b], rows=self.rows[r:r + n], keep=out[2][r:r + n])
        return out

    def results(self):
        return self.accepted, self.next, self.keep, self.logp


@pytest.mark.parametrize("draft", ["logits", "none"])
def test_many_requests_are_their_parts(draft):
    c = Many(draft)
    want = c.by_parts()
    assert lib().q4_gpu_last_error() == 4
    for _ in range(2):
        c.logp.fill_(5.0)
        c.run()
        assert lib().q4_gpu_last_error() == 4
        assert all(torch.equal(a, b) for a, b in zip(c.results(), want))
    # rows behind a first one count: of 5000 requests with 0 to 8 drafts, certain ones kept with 0.3 to 0.4 each, some keep 3 and more (not all 8: 0.35^8 of 500 is 0.1)
    assert int(c.accepted.max()) >= 3


def test_many_rows_with_starts_that_are_none():
    """they are told, and leave nothing behind for the next call"""
    c = Many("logits")
    want = c.by_parts()
    good = c.start.clone()
    for at, to in ((17, -5), (18, 2**31 - 1), (400, 0), (2000, c.n_tok + 1), (4990, 3)):
        c.start[at] = to
    c.run()
    assert lib().q4_gpu_last_error() == 4
    c.start.copy_(good)
    c.logp.fill_(5.0)
    c.run()
    assert all(torch.equal(a, b) for a, b in zip(c.results(), want))
    assert lib().q4_gpu_last_error() == 4                                   # rows that are none, as in the parts


# ---- what blocks share
@pytest.mark.parametrize("draft", ["logits", "none"])
def test_what_other_kernels_left_in_shared_memory(draft):
    """a launch over 8192 requests that hold nothing leaves zeros on every SM: the decision's table is not read before it is there"""
    n = 8192
    pool = q4gpu.PagePool(1, 1, 64, 64, 16)
    rows, keep = torch.zeros(2, n, dtype=torch.int32, device="cuda").unbind(0)
    table = torch.zeros(n, 20, dtype=torch.int32, device="cuda")
    c = Case([7, 3, 5, 9] * 60, 300, draft=draft, seed=33, sharp=0.7)
    if draft == "none":
        c.logits[torch.arange(c.n_tok - 1), c.token[1:].long()] += 8.0
    c.run().check()
    want = [t.clone() for t in (c.accepted, c.next, c.keep, c.logp)]
    for _ in range(30):
        pool.release(rows, keep, table)
        c.run()
        assert all(torch.equal(a, b) for a, b in zip((c.accepted, c.next, c.keep, c.logp), want))


# ---- tokens that are next to impossible
def far_below(base, bf16):
    """five requests whose rows are -inf but for some tokens 2^-1010 to 2^-1040 below the largest, all of them ahead of what else there is; one token of every row takes nearly all"""
    c = Case([0] * 5, 9000, bf16=bf16, draft="none", seed=34)
    c.logits.fill_(-INF)
    c.logits[:, 8000] = base
    c.logits[0, 600:1024] = base - 704.0     # 2^-1015.6; the first half of the chunk holds nothing
    c.logits[1, 1023] = base - 720.0
    c.logits[2, 3000] = base - 704.0
    c.logits[2, 5000] = base - 672.0         # 2^-969.5: counts
    c.logits[3, :700] = base - 704.0
    c.logits[3, 700:900] = base - 688.0      # 2^-992.6
    return c


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("base", [0.0, 256.0, 131072.0])
def test_a_draw_of_the_first_token_that_can_be(base, bf16):
    """a probability below 2^-1000 of the row's largest is none; 131 072 is beyond the steps of the fast exponential (there bf16 has no such differences)"""
    if bf16 and base:
        base = -512.0
    c = far_below(base, bf16)
    want = [int((c.logits[r].float() >= base - 1000 * math.log(2)).nonzero()[0]) for r in range(5)]
    c.u_next.fill_(0.0)
    c.run()
    assert lib().q4_gpu_last_error() == 0
    assert c.next.tolist() == want
    for u in (2.0**-24, 0.5, 1 - 2.0**-24):
        c.u_next.fill_(u)
        c.run()
        assert c.next.tolist() == [8000] * 5 and lib().q4_gpu_last_error() == 0


def test_a_draw_behind_a_refused_draft_that_was_all_there_is_ahead():
    c = Case([1] * 3, 9000, draft="none", seed=35)
    c.logits.fill_(-INF)
    c.logits[:, 8000] = 0.0
    c.logits[:, 40] = -650.0                 # the draft: 2^-938
    c.logits[:, 2000:2040] = -705.0          # 2^-1017: within 100 powers of two of what its warp saw first, and none
    c.token.fill_(40)
    c.u_accept.fill_(0.5)
    c.u_next.fill_(0.0)
    c.run()
    assert lib().q4_gpu_last_error() == 0
    assert c.accepted.tolist() == [0] * 3 and c.next.tolist() == [8000] * 3


@pytest.mark.parametrize("vocab", [1, 2, 5000, 40000])
@pytest.mark.parametrize("u", [1.0, 2.0, float("nan")])
def test_a_refused_draft_that_is_all_there_is(vocab, u):
    """max(p - q, 0) is 0 throughout, so that p is drawn from: random numbers that refuse what cannot be"""
    c = Case([1, 2, 1], vocab, draft="none", seed=36)
    d = vocab * 3 // 4
    c.logits.fill_(-INF)
    c.logits[:, d] = 3.0
    c.token.fill_(d)
    c.u_accept.fill_(u)
    c.run()
    assert lib().q4_gpu_last_error() == 0
    # at u = 1 either is right: u S < w with S = w (1 + x), |x| <= 7e-9 as the row's sum is off, holds where x is below 0
    assert u == 1 or c.accepted.tolist() == [0] * 3
    assert c.next.tolist() == [d] * 3
    assert (c.logp[c.start[:-1].long()].abs() <= 7e-9).all()              # log p = 0, by a sum that is off by so much of itself


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("limit", [5400.0, 43300.0])
def test_sums_at_the_largest_sizes_of_the_fast_exponential(limit, bf16):
    """rows of equal logits, one or many of them, |x / T| up to 2e6 steps of 1/32 of a power of two, where the rest of a step is largest"""
    n_req, vocab = 600, 2100
    g = torch.Generator(device="cuda").manual_seed(37)
    temp = 0.5 + 1.5 * torch.rand(n_req, device="cuda", generator=g)
    c = Case([0] * n_req, vocab, bf16=bf16, draft="none", seed=37)
    c.temp = temp
    sign = torch.where(torch.rand(n_req, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    x = (temp * limit * sign * (0.9 + 0.1 * torch.rand(n_req, device="cuda", generator=g))).to(c.logits.dtype)
    x = torch.where((x.float() / temp).abs() > limit, (x.float() * 0.99).to(x.dtype), x)
    assert float((x.float() / temp).abs().max()) <= limit * 1.002
    many = torch.tensor([1, 2, 8, 64, vocab], device="cuda")[torch.arange(n_req, device="cuda") % 5]
    c.logits.copy_(torch.where(torch.arange(vocab, device="cuda")[None] < many[:, None], x.float()[:, None], -INF))
    c.u_next.copy_((torch.arange(n_req, device="cuda") // 5 % 8 + 0.5) / 8)
    c.run()
    assert lib().q4_gpu_last_error() == 0
    # token k of n equal ones has 1 / n: borders at k / n.  Of 64, u = (2 j + 1) / 16 is the one at 4 (2 j + 1): sums that are off by 7e-9 put it on either side
    at = [u * n for u, n in zip(c.u_next.tolist(), many.tolist())]
    assert all(got == int(k) or (n == 64 and got == k - 1) for got, k, n in zip(c.next.tolist(), at, many.tolist()))
    # log p = -log n: its own rounding to fp32, the sum's 7e-9, and the exponent of x over the row's step in 64 bits (2e6 x 2^-53 x ln 2 / 32 and less)
    want = -many.double().log()
    assert ((c.logp.double() - want).abs() <= 2.0**-24 * want.abs() * (1 + 1e-6) + 7e-9).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("vocab", [700, 9001, 140001])
@pytest.mark.parametrize("shift", [14.9, 37.3])
def test_what_p_has_over_a_q_that_is_nearly_the_same(vocab, bf16, shift):
    """a token has nearly all of both; what p has over q is 1e-10 and less, far below what their sums may be off by.  Drafts that cannot be are refused"""
    n_req = 64
    c = Case([1] * n_req, vocab, bf16=bf16, seed=38, ld=vocab + 3)
    g = torch.Generator(device="cuda").manual_seed(38)
    other = shift + torch.linspace(0, 9, c.n_tok, device="cuda")[:, None].to(c.logits.dtype).float()      # softmax knows no shift, but the sums of exponentials are rounded otherwise
    for x, m in ((c.logits, shift), (c.draft, other[:, 0])):
        x.fill_(-INF)
        x[:, vocab // 3] = m
    over = torch.randint(vocab // 2, vocab, (c.n_tok, 5), device="cuda", generator=g)
    c.logits.scatter_(1, over, (shift - 24 - 3 * torch.rand(c.n_tok, 5, device="cuda", generator=g)).to(c.logits.dtype))       # 4e-11 and less
    c.draft.scatter_(1, over[:, :2], (other - 28 - 3 * torch.rand(c.n_tok, 2, device="cuda", generator=g)).to(c.logits.dtype))
    c.draft[:, 1] = other[:, 0] - 30
    c.token.fill_(1)
    c.u_next.copy_((torch.arange(n_req, device="cuda") + 0.5) / n_req)
    c.run()
    assert lib().q4_gpu_last_error() == 0 and c.accepted.tolist() == [0] * n_req
    accepted, nexts, logp, bad = plain(c)
    # in the definition's own 64 bits what is over is 2^-52 / 1e-11 off at most; of 64 x 6 borders some lie that near a random number by 2^-10 at most
    for r, (got, want) in enumerate(zip(c.next.tolist(), nexts)):
        x = softmax(c.logits[2 * r], 1.0) - softmax(c.draft[2 * r], 1.0)
        s = x.clamp(min=0).cumsum(0) / x.clamp(min=0).sum()
        assert got == want or min(abs(float(s[k]) - float(c.u_next[r])) for k in over[2 * r].tolist()) < 1e-4, (r, got, want)
