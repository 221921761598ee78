"""A whole step with drafts as one graph: plan, per layer prep and attend, verify, release, replayed while the tokens, the random numbers and the lengths change, against the
same calls one by one."""
import ctypes

import pytest
import torch

import q4gpu
from gpu_util import lib

pytestmark = pytest.mark.gpu
N_HEAD, N_KVH, HD, VOCAB, LAYERS, DRAFTS = 8, 2, 128, 1500, 2, 3


class Step:
    def __init__(self, kind, n_req=7, idle=5, seed=0):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        on, word = dict(device="cuda", generator=g), dict(dtype=torch.int32, device="cuda")
        self.n_req, self.max_tok = n_req, n_req * (DRAFTS + 1) + idle
        self.pool = q4gpu.PagePool(LAYERS, N_KVH, HD, 120, 16, kind)
        self.rope = q4gpu.Rope(64, 1e6, half=True)
        self.table = torch.full((n_req, 14), -1, **word)
        self.rows, self.keep, self.accepted, self.next, self.diff = (torch.zeros(n_req, **word) for _ in range(5))
        self.start = torch.zeros(n_req + 1, **word)
        self.add = torch.full((n_req,), DRAFTS + 1, **word)
        self.slot, self.pos, self.req, self.token = (torch.zeros(self.max_tok, **word) for _ in range(4))
        self.x = torch.randn(LAYERS, self.max_tok, (2 * N_HEAD + 2 * N_KVH) * HD, **on)
        self.wq, self.wk = (1 + 0.1 * torch.randn(2, HD, **on)).unbind(0)
        self.q = torch.zeros(self.max_tok, N_HEAD, HD, dtype=torch.bfloat16, device="cuda")
        self.gate, self.out = torch.zeros(self.max_tok, N_HEAD, HD, device="cuda"), torch.zeros(LAYERS, self.max_tok, N_HEAD, HD, dtype=torch.bfloat16, device="cuda")
        self.logits, self.draft = torch.randn(2, self.max_tok, VOCAB, **on).unbind(0)
        self.u_accept, self.u_next, self.logp = torch.rand(self.max_tok, **on), torch.rand(n_req, **on), torch.zeros(self.max_tok, device="cuda")
        self.temp = torch.full((n_req,), 0.9, device="cuda")

    def again(self, add):
        """other numbers, in the same places"""
        self.add.copy_(torch.tensor(add, dtype=torch.int32))
        self.x.normal_(generator=self.g)
        self.logits.normal_(generator=self.g)
        self.draft.copy_(self.logits).add_(torch.randn(self.draft.shape, generator=self.g, device="cuda"), alpha=0.4)
        self.token.copy_(self.draft.argmax(1).roll(1))
        self.u_accept.uniform_(generator=self.g)
        self.u_next.uniform_(generator=self.g)

    def run(self):
        p, n = self.pool, self.max_tok
        p.plan(self.rows, self.add, self.table, self.start, self.slot, self.pos, self.req)
        for layer in range(LAYERS):
            q, k, v = self.x[layer].split([2 * N_HEAD * HD, N_KVH * HD, N_KVH * HD], 1)
            p.prep(layer, q, k, v, self.q, self.pos, self.slot, self.rope, wq=self.wq, wk=self.wk, gate=self.gate)
            p.attend(layer, self.q, self.out[layer], self.rows, self.start, self.table, N_HEAD, HD**-0.5, gate=self.gate, max_add=DRAFTS + 1)
        q4gpu.verify(self.logits[:n], self.token, self.start, self.u_accept, self.u_next, self.accepted, self.next, draft=self.draft, temp=self.temp, logp=self.logp, rows=self.rows, keep=self.keep)
        torch.sub(self.start[1:], self.start[:-1], out=self.diff)
        self.rows.add_(self.diff)
        p.release(self.rows, self.keep, self.table)

    def state(self):
        return dict(mem=self.pool.mem, free=self.pool.free, n_free=self.pool.n_free, shares=self.pool.shares, table=self.table, rows=self.rows, start=self.start, slot=self.slot, pos=self.pos, q=self.q,
                    gate=self.gate, out=self.out, accepted=self.accepted, next=self.next, logp=self.logp, keep=self.keep)


@pytest.mark.parametrize("kind", [q4gpu.KIND_Q8, q4gpu.KIND_F16])
def test_a_step_replayed_is_the_step_itself(kind):
    s = Step(kind)
    L = lib()
    L.q4_gpu_last_error()
    s.again([DRAFTS + 1] * s.n_req)
    s.run()                                                     # the scratch is there
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        q4gpu.use_torch_stream()
        try:
            assert L.q4_hip_graph_begin()
            s.run()
            graph = L.q4_hip_graph_end()
            assert graph
            kept = 0
            for add in ([4] * 7, [1, 4, 2, 0, 4, 3, 4], [4, 0, 4, 4, 0, 1, 4], [0] * 6 + [4], [4] * 7, [2] * 7):
                s.again(add)
                before = {k: t.clone() for k, t in s.state().items()}
                s.run()
                assert L.q4_gpu_last_error() == 0
                want = {k: t.clone() for k, t in s.state().items()}
                for k, t in s.state().items():
                    t.copy_(before[k])
                assert L.q4_hip_graph_launch(ctypes.c_void_p(graph))
                assert L.q4_gpu_last_error() == 0
                for k, t in s.state().items():
                    assert torch.equal(t.view(torch.uint8), want[k].view(torch.uint8)), k
                kept += int(s.accepted.sum())
            assert kept > 0
            L.q4_hip_graph_free(ctypes.c_void_p(graph))
        finally:
            stream.synchronize()
    q4gpu.use_torch_stream()
    s.pool.release(s.rows, torch.zeros_like(s.rows), s.table)
    assert int(s.pool.n_free[0]) == 120 and L.q4_gpu_last_error() == 0


def test_drafts_beside_a_chunk_of_a_prompt():
    """verify over the rows that the host gathers: drafts and the token before them, of a chunk its last token; what it says to keep is what release takes"""
    s = Step(q4gpu.KIND_Q8, n_req=3, idle=20)
    L = lib()
    L.q4_gpu_last_error()
    p, held = s.pool, [37, 16, 90]
    for add in (held, [DRAFTS + 1, 20, 1]):
        s.add.copy_(torch.tensor(add, dtype=torch.int32))
        n = sum(add)
        slot, pos, req = torch.zeros(3, n, dtype=torch.int32, device="cuda").unbind(0)
        p.plan(s.rows, s.add, s.table, s.start, slot, pos, req)
        before = s.rows.clone()
        s.rows.add_(s.start.diff())
    gathered = torch.tensor([0, 1, 2, 3, DRAFTS + 20, DRAFTS + 21], device="cuda")         # of the step's 25 tokens
    start = torch.tensor([0, DRAFTS + 1, DRAFTS + 2, DRAFTS + 3], dtype=torch.int32, device="cuda")
    s.draft.copy_(s.logits)                                     # drafts that are as likely to both: kept
    token = s.token[:25][gathered].contiguous()
    token[1:DRAFTS + 1] = s.logits[gathered[:DRAFTS]].argmax(1)
    rows = before + torch.tensor([0, 19, 0], dtype=torch.int32, device="cuda")
    u, logits = s.u_accept[:6] * 0.9, s.logits[gathered]
    q4gpu.verify(logits, token, start, u, s.u_next, s.accepted, s.next, draft=logits.clone(), temp=s.temp, logp=s.logp, rows=rows, keep=s.keep)
    assert s.accepted.tolist() == [DRAFTS, 0, 0] and all(0 <= x < VOCAB for x in s.next.tolist())
    assert s.keep.tolist() == [37 + DRAFTS + 1, 36, 91]
    p.release(s.rows, s.keep, s.table)
    assert s.rows.tolist() == s.keep.tolist() and L.q4_gpu_last_error() == 0
    token[2] = (token[2] + 1) % VOCAB                           # a draft that is refused, and its rows' place given back
    u.fill_(1.0)
    q4gpu.verify(logits, token, start, u, s.u_next, s.accepted, s.next, temp=s.temp, rows=rows, keep=s.keep)
    p.release(s.rows, s.keep, s.table)
    assert s.rows.tolist() == [37 + int(s.accepted[0]) + 1, 36, 91] and L.q4_gpu_last_error() == 0
