"""Serving with drafts on the paged KV cache: chats that begin with the same instructions share the pages that hold them, every step brings each chat's last token and
some drafts, and what the target does not keep of these is given back.

    python examples/paged_drafts.py [--layers 3] [--chats 8] [--drafts 4] [--steps 30] [--kind q8_0] [--temp 0.8]

A chat's place is filled by a fork of the place that holds the instructions.  A step is
    plan; per layer prep, attend; verify; release
and every so often the pool is compacted, as if its end were to be handed on.

There is no model here: projections and logits are random, made from the token and its place so that a chat that is asked again gives the same.  Every --check
steps what the pool holds is compared with the rows that the kept tokens stand for, the last layer's attention with softmax(q k) v in 64 bits over them, and the
kept tokens with the definition in 64 bits.  Prints the tokens served, the share of drafts that were kept, and the time of a step.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "suzuqu-engine-4exp_b200"))
import q4gpu  # noqa: E402

N_HEAD, N_KVH, HD, N_ROT, EPS = 8, 2, 128, 64, 1e-6


class Loop:
    def __init__(self, layers, chats, drafts, kind, temp, vocab=2000, page_rows=16, prefix=75, seed=0):
        q4gpu.init()
        q4gpu.use_torch_stream()
        on = dict(device="cuda")
        self.layers, self.chats, self.drafts, self.vocab, self.page_rows, self.prefix, self.temp = layers, chats, drafts, vocab, page_rows, prefix, temp
        self.most = 400                                                    # rows of a chat
        self.places = chats + 1                                            # place 0 holds the instructions
        n_pages = self.places * (self.most // page_rows + 1) + 8
        self.pool = q4gpu.PagePool(layers, N_KVH, HD, n_pages, page_rows, kind)
        self.rope = q4gpu.Rope(N_ROT, 1e6, half=True, scaling="ramp", factor=4.0, orig=128, mag=1.1)
        g = self.gen = torch.Generator(device="cuda").manual_seed(seed)
        # "the model": a projection per token of the vocabulary, logits from the last token
        self.proj = torch.randn(layers, vocab, (N_HEAD + 2 * N_KVH) * HD, generator=g, **on)
        self.head = 3 * torch.randn(vocab, vocab, generator=g, **on)
        self.draft_head = self.head + torch.randn(vocab, vocab, generator=g, **on)
        self.wq, self.wk = (1 + 0.1 * torch.randn(2, HD, generator=g, **on)).unbind(0)
        word = dict(dtype=torch.int32, **on)
        self.table = torch.full((self.places, self.most // page_rows + 2), -1, **word)
        self.rows = torch.zeros(self.places, **word)                       # what the places hold: fork and release keep it up to date
        self.start = torch.zeros(self.places + 1, **word)
        self.max_tok = max(prefix, chats * (drafts + 1))
        self.slot, self.pos, self.req = (torch.zeros(self.max_tok, **word) for _ in range(3))
        self.accepted, self.next, self.keep = (torch.zeros(self.places, **word) for _ in range(3))
        self.number = torch.zeros(n_pages, **word)
        self.text = [[] for _ in range(self.places)]                       # tokens whose rows a place holds
        self.last = [0] * self.places                                      # a chat's newest token, which has no row yet
        self.token = torch.randint(0, vocab, (prefix,), generator=g, **word)
        self.step_of(self.token, [prefix] + [0] * chats)                   # the instructions, once
        self.rows += self.start.diff()
        self.text[0] = self.token.tolist()

    def step_of(self, token, add):
        """plan, and prep and attend layer by layer, for these tokens; the last layer's queries and outputs"""
        n = token.numel()
        self.pool.plan(self.rows, torch.tensor(add, dtype=torch.int32).cuda(), self.table, self.start, self.slot, self.pos, self.req)
        for layer in range(self.layers):
            row = self.proj[layer][token.long()]
            q, k, v = row.split([N_HEAD * HD, N_KVH * HD, N_KVH * HD], 1)
            q_out = torch.empty(n, N_HEAD, HD, dtype=torch.bfloat16, device="cuda")
            out = torch.empty_like(q_out)
            self.pool.prep(layer, q, k, v, q_out, self.pos[:n], self.slot[:n], self.rope, wq=self.wq, wk=self.wk, eps=EPS)
            self.pool.attend(layer, q_out, out, self.rows, self.start, self.table, N_HEAD, HD**-0.5, max_add=max(add))
        return q_out, out

    def step(self, check=False):
        free = [r for r in range(1, self.places) if not self.text[r]]
        over = [r for r in range(1, self.places) if len(self.text[r]) > self.most - self.drafts - 2]
        if free:                                                           # new chats begin with the instructions
            ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()     # noqa: E731
            self.pool.fork(self.rows, ints([0] * len(free)), ints(free), ints([self.prefix] * len(free)), self.table)
            for r in free:
                self.text[r] = list(self.text[0])
                self.last[r] = int(torch.randint(0, self.vocab, (1,)))
        # the newest token of each chat, and drafts behind it
        ids, draft_rows = [], []
        for r in range(1, self.places):
            t = [self.last[r]]
            for _ in range(self.drafts):
                p = torch.softmax(self.draft_head[t[-1]] / (self.temp or 0.1), 0)
                t.append(int(torch.multinomial(p, 1, generator=self.gen)))
            ids += t
            draft_rows += t
        token = torch.tensor(ids, dtype=torch.int32).cuda()
        n, add = token.numel(), [0] + [self.drafts + 1] * self.chats
        q, out = self.step_of(token, add)
        logits, draft = self.head[token.long()], self.draft_head[torch.tensor(draft_rows).cuda()]
        u_accept, u_next = torch.rand(n, generator=self.gen, device="cuda"), torch.rand(self.places, generator=self.gen, device="cuda")
        temp = torch.full((self.places,), self.temp, device="cuda")
        q4gpu.verify(logits, token, self.start, u_accept, u_next, self.accepted, self.next, draft=draft, temp=temp, rows=self.rows, keep=self.keep)
        held = self.rows
        self.rows = held + self.start.diff()
        if check:
            self.check(held, q, out, token, logits, draft, u_accept, u_next)
        keep = self.keep.clone()
        keep[over] = 0                                                     # a chat that is over gives all of it back
        self.pool.release(self.rows, keep, self.table)
        got, new = self.accepted.tolist(), self.next.tolist()
        for i, r in enumerate(range(1, self.places)):
            self.text[r] += ids[i * (self.drafts + 1): i * (self.drafts + 1) + got[r] + 1]
            self.last[r] = new[r]
            if r in over:
                self.text[r] = []
        status = q4gpu.load().q4_gpu_last_error()
        if status:
            raise RuntimeError("a step's status is 0x%x" % status)
        return sum(got) + self.chats, sum(got)

    def compact(self):
        self.pool.compact(self.rows, self.table, self.number)

    def row(self, layer, token, pos, part):
        """a head's rows from the definition, in 64 bits"""
        x = self.proj[layer][token].double().split([N_HEAD * HD, N_KVH * HD, N_KVH * HD], 1)[part].unflatten(1, (-1, HD))
        if part == 2:
            return x
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (self.wq if part == 0 else self.wk).double()
        turn = torch.tensor([t / 2**64 for t in self.rope.turn[: N_ROT // 2]], dtype=torch.float64, device="cuda")
        angle = (pos.double()[:, None] * turn % 1.0 * 2 * torch.pi)[:, None]
        a, b = x[..., : N_ROT // 2], x[..., N_ROT // 2: N_ROT]
        cos, sin = self.rope.mag * torch.cos(angle), self.rope.mag * torch.sin(angle)
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., N_ROT:]], -1)

    def check(self, held, q, out, token, logits, draft, u_accept, u_next):
        start, held, table, layer = self.start.tolist(), held.tolist(), self.table.tolist(), self.layers - 1
        for r in range(1, self.places):
            a, b = start[r], start[r + 1]
            mine = torch.tensor(self.text[r] + token[a:b].tolist(), device="cuda")
            at = torch.arange(mine.numel(), device="cuda")
            slot = torch.tensor([table[r][p // self.page_rows] * self.page_rows + p % self.page_rows for p in at.tolist()], dtype=torch.int32, device="cuda")
            k, v = torch.empty(2, mine.numel(), N_KVH * HD, device="cuda")
            self.pool.gather(layer, slot, k, v)
            for got, part in ((k, 1), (v, 2)):
                want = self.row(layer, mine, at, part)
                step = want.unflatten(-1, (-1, 32)).abs().amax(-1).amax() / 127
                assert (got.view(want.shape).double() - want).abs().max() <= 0.6 * step, "rows of place %d" % r
            k, v = (x.double().view(-1, N_KVH, HD).repeat_interleave(N_HEAD // N_KVH, 1) for x in (k, v))
            w = torch.einsum("thd,phd->htp", q[a:b].double(), k) * HD**-0.5
            w = w.masked_fill(at[None, None] > held[r] + torch.arange(b - a, device="cuda")[None, :, None], -torch.inf)
            o = torch.einsum("htp,phd->thd", torch.softmax(w, -1), v)
            assert ((out[a:b].double() - o).abs() <= 4e-3 + (1e-3 + 2.0**-8) * o.abs()).all(), "attention of place %d" % r
            j = 0
            while True:                                                    # the drafts, from the definition
                p = torch.softmax(logits[a + j].double() / (self.temp or 1), 0)
                if a + j + 1 == b:
                    w = p
                    break
                d, q_row = int(token[a + j + 1]), torch.softmax(draft[a + j].double() / (self.temp or 1), 0)
                if float(u_accept[a + j]) * float(q_row[d]) < float(p[d]) if self.temp else d == int(logits[a + j].argmax()):
                    j += 1
                    continue
                w = (p - q_row).clamp(min=0)
                break
            s = w.cumsum(0)
            new = int((s > float(u_next[r]) * float(s[-1])).float().argmax()) if self.temp else int(logits[a + j].argmax())
            assert (int(self.accepted[r]), int(self.next[r])) == (j, new), "drafts of place %d" % r


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=3)
    ap.add_argument("--chats", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--check", type=int, default=5)
    ap.add_argument("--kind", choices=("q8_0", "f16"), default="q8_0")
    ap.add_argument("--temp", type=float, default=0.8)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    loop = Loop(a.layers, a.chats, a.drafts, {"q8_0": q4gpu.KIND_Q8, "f16": q4gpu.KIND_F16}[a.kind], a.temp)
    served = kept = checks = 0
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for i in range(a.steps):
        check = a.check and i % a.check == a.check - 1
        n, k = loop.step(check)
        served, kept, checks = served + n, kept + k, checks + bool(check)
        if i % 7 == 6:
            loop.compact()
    end.record()
    loop.pool.release(loop.rows, torch.zeros_like(loop.rows), loop.table)
    status = q4gpu.load().q4_gpu_last_error()
    back = int(loop.pool.n_free[0]) == loop.pool.n_pages and not bool(loop.pool.shares.any())
    print("%d tokens served, %.0f %% of the drafts kept, %.2f ms a step with the host's part; %d steps checked; status %d; pages back: %s"
          % (served, 100.0 * kept / max(1, a.steps * a.chats * a.drafts), begin.elapsed_time(end) / a.steps, checks, status, back))
    return 0 if status == 0 and back else 1


if __name__ == "__main__":
    sys.exit(main())
