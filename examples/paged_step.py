"""A serving loop on the paged KV cache: chats come and go, and every step takes the next piece of each prompt and one token of each
chat that answers, in one plan, and one append and one attention per layer.

    python examples/paged_step.py [--layers 4] [--chats 12] [--steps 40] [--pages 512] [--kind q8_0]

A plan serves the chats up to the first one that does not fit: a chat has as many rows more as `start` says that it was served, and where
pages ran out the last chat that holds any gives them back and begins again.

Queries, keys and values are random, as there is no model here; every --check steps the rows that the pool holds are compared with the ones
that each chat was given, and a layer's outputs with softmax(q k) v in 64 bits over them.  Prints the tokens served and the time of a step.
"""
import argparse
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "suzuqu-engine-4exp_b200"))
import q4gpu  # noqa: E402


class Loop:
    def __init__(self, layers, places, n_head=16, n_kvh=2, hd=128, page_rows=64, n_pages=512, kind=q4gpu.KIND_Q8, max_tok=512, chunk=128, seed=0):
        q4gpu.init()
        q4gpu.use_torch_stream()
        self.layers, self.places, self.n_head, self.n_kvh, self.hd, self.page_rows, self.max_tok, self.chunk = layers, places, n_head, n_kvh, hd, page_rows, max_tok, chunk
        self.pool = q4gpu.PagePool(layers, n_kvh, hd, n_pages, page_rows, kind)
        self.rng, self.gen = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
        word = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((places, max(n_pages // 4, -(-640 // page_rows))), -1, **word)
        self.start = torch.zeros(places + 1, **word)
        self.slot, self.pos, self.req = (torch.zeros(max_tok, **word) for _ in range(3))
        self.held, self.prompt, self.answer = [0] * places, [0] * places, [0] * places    # rows in the pool; tokens still to come
        self.given = [[] for _ in range(places)]                                          # the last layer's K and V of the rows in the pool
        self.again = 0                                                                    # chats that had to begin again

    def words(self, values):
        return torch.tensor(values, dtype=torch.int32).pin_memory().to("cuda", non_blocking=True)

    def step(self, check=False):
        """one step of all chats; returns the tokens it served"""
        for r in range(self.places):
            if self.prompt[r] + self.answer[r] == 0 and self.rng.random() < 0.5:                # a new chat takes the place
                self.prompt[r], self.answer[r] = self.rng.randint(1, 600), self.rng.randint(1, 30)
        add = [min(p, self.chunk) if p else min(a, 1) for p, a in zip(self.prompt, self.answer)]
        left = self.max_tok
        for r in range(self.places):
            add[r] = min(add[r], left)
            left -= add[r]
        rows, n_tok = self.words(self.held), sum(add)
        if n_tok == 0:
            return 0
        self.pool.plan(rows, self.words(add), self.table, self.start, self.slot, self.pos, self.req)
        for layer in range(self.layers):
            k, v = torch.randn(2, n_tok, self.n_kvh * self.hd, device="cuda", generator=self.gen)
            q = torch.randn(n_tok, self.n_head, self.hd, device="cuda", generator=self.gen).to(torch.bfloat16)
            out = torch.empty_like(q)
            self.pool.append(layer, k, v, self.slot[:n_tok])
            self.pool.attend(layer, q, out, rows, self.start, self.table, self.n_head, self.hd**-0.5, max_add=max(add))
        start = self.start.tolist()                                                              # a host waits here for the new tokens in any case
        status = q4gpu.load().q4_gpu_last_error()
        if status & ~8:                                                                          # 8: not all were served
            raise RuntimeError("a step's status is 0x%x" % status)
        got = [b - a for a, b in zip(start, start[1:])]
        for r, n in enumerate(got):
            if n:
                self.given[r].append((k[start[r]: start[r + 1]], v[start[r]: start[r + 1]]))
        if check:
            self.check(q, out, start)
        rows = self.held = [h + n for h, n in zip(self.held, got)]
        for r, n in enumerate(got):
            if self.prompt[r]:
                self.prompt[r] -= n
            else:
                self.answer[r] -= n
        keep = [h if p + a else 0 for h, p, a in zip(rows, self.prompt, self.answer)]            # a chat that is over gives its pages back
        if status & 8 and keep == rows:
            last = max(r for r, h in enumerate(rows) if h)
            self.prompt[last], keep[last] = self.prompt[last] + rows[last], 0
            self.again += 1
        if keep != rows:
            self.pool.trim(self.words(rows), self.words(keep), self.table)
            self.given = [g if h else [] for g, h in zip(self.given, keep)]
            self.held = keep
        return start[-1]

    def check(self, q, out, start):
        """the last layer's rows and outputs, request by request"""
        for r, h in enumerate(self.held):
            at, n = start[r], start[r + 1] - start[r]
            if n == 0:
                continue
            p = torch.arange(h + n, device="cuda")
            slot = (self.table[r].long()[p // self.page_rows] * self.page_rows + p % self.page_rows).int()
            k, v = torch.empty(2, h + n, self.n_kvh * self.hd, device="cuda")
            self.pool.gather(self.layers - 1, slot, k, v)
            for x, mine in zip((k, v), zip(*self.given[r])):
                mine = torch.cat(mine)
                # codes are half of amax / 127 off, their scale 2^-11 of itself (127 codes of it: 0.06)
                assert ((x - mine).abs() <= 0.6 / 127 * mine.abs().max()).all(), "rows of request %d" % r
            k, v = (x.view(-1, self.n_kvh, self.hd).double().repeat_interleave(self.n_head // self.n_kvh, 1) for x in (k, v))
            w = torch.einsum("thd,phd->htp", q[at: at + n].double(), k) * self.hd**-0.5
            w = w.masked_fill(p > h + torch.arange(n, device="cuda")[:, None], -torch.inf)
            want = torch.einsum("htp,phd->thd", torch.softmax(w, -1), v)
            # 2e-3 + 1e-3 |o| of the attention, 2^-8 of a bf16 output
            assert ((out[at: at + n].double() - want).abs() <= 2e-3 + (1e-3 + 2.0**-8) * want.abs()).all(), "request %d" % r

    def end(self):
        """all chats end; whether every page came back once"""
        self.pool.trim(self.words(self.held), self.words([0] * self.places), self.table)
        self.held = [0] * self.places
        return torch.equal(self.pool.free.sort().values, torch.arange(self.pool.n_pages, dtype=torch.int32, device="cuda")) and int(self.pool.n_free[0]) == self.pool.n_pages


def main(argv=None):
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--layers", type=int, default=4)
    a.add_argument("--chats", type=int, default=12)
    a.add_argument("--steps", type=int, default=40)
    a.add_argument("--check", type=int, default=5, metavar="N")
    a.add_argument("--pages", type=int, default=512, help="of 64 rows; a chat alone takes up to 10")
    a.add_argument("--kind", choices=("q8_0", "f16"), default="q8_0")
    a = a.parse_args(argv)
    loop = Loop(a.layers, a.chats, n_pages=a.pages, kind=q4gpu.KIND_Q8 if a.kind == "q8_0" else q4gpu.KIND_F16)
    times, tokens, checked = [], 0, 0
    for i in range(a.steps):
        begin, end = torch.cuda.Event(True), torch.cuda.Event(True)
        check = a.check > 0 and i % a.check == 0
        begin.record()
        tokens += loop.step(check)
        end.record()
        checked += check
        if not check:
            times.append((begin, end))
    torch.cuda.synchronize()
    ms = sorted(b.elapsed_time(e) for b, e in times)
    status = q4gpu.load().q4_gpu_last_error()
    back = loop.end()
    print("%d tokens in %d steps of %d layers, %.3f ms per step (median); %d steps checked; status %d; pages back: %s; begun again: %d"
          % (tokens, a.steps, a.layers, ms[len(ms) // 2] if ms else 0.0, checked, status, back, loop.again))
    return 0 if back and status == 0 else 1


if __name__ == "__main__":
    sys.exit(main())
