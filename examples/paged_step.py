"""A serving loop on the paged KV cache: chats come and go, and every step takes the next piece of each prompt and one token of each
chat that answers, in one plan, and one append and one attention per layer.

    python examples/paged_step.py [--layers 4] [--chats 12] [--steps 40] [--kind q8_0]

Queries, keys and values are random, as there is no model here; every --check steps a layer's outputs are compared with softmax(q k) v
in 64 bits over the rows that the pool holds.  Prints the tokens served and the time of a step.
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
        self.table = torch.full((places, n_pages // 4), -1, **word)
        self.start = torch.zeros(places + 1, **word)
        self.slot, self.pos, self.req = (torch.zeros(max_tok, **word) for _ in range(3))
        self.held, self.prompt, self.answer = [0] * places, [0] * places, [0] * places    # rows in the pool; tokens still to come

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
        if check:
            self.check(q, out, add)
        self.held = [h + n for h, n in zip(self.held, add)]
        keep = []
        for r, n in enumerate(add):
            if self.prompt[r]:
                self.prompt[r] -= n
            else:
                self.answer[r] -= n
            keep.append(self.held[r] if self.prompt[r] + self.answer[r] else 0)                  # a chat that is over gives its pages back
        if keep != self.held:
            self.pool.trim(self.words(self.held), self.words(keep), self.table)
            self.held = keep
        return n_tok

    def check(self, q, out, add):
        """the last layer's outputs, request by request"""
        at = 0
        for r, (h, n) in enumerate(zip(self.held, add)):
            if n == 0:
                continue
            p = torch.arange(h + n, device="cuda")
            slot = (self.table[r].long()[p // self.page_rows] * self.page_rows + p % self.page_rows).int()
            k, v = torch.empty(2, h + n, self.n_kvh * self.hd, device="cuda")
            self.pool.gather(self.layers - 1, slot, k, v)
            k, v = (x.view(-1, self.n_kvh, self.hd).double().repeat_interleave(self.n_head // self.n_kvh, 1) for x in (k, v))
            w = torch.einsum("thd,phd->htp", q[at: at + n].double(), k) * self.hd**-0.5
            w = w.masked_fill(p > h + torch.arange(n, device="cuda")[:, None], -torch.inf)
            want = torch.einsum("htp,phd->thd", torch.softmax(w, -1), v)
            # 2e-3 + 1e-3 |o| of the attention, 2^-8 of a bf16 output
            assert ((out[at: at + n].double() - want).abs() <= 2e-3 + (1e-3 + 2.0**-8) * want.abs()).all(), "request %d" % r
            at += n

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
    a.add_argument("--kind", choices=("q8_0", "f16"), default="q8_0")
    a = a.parse_args(argv)
    loop = Loop(a.layers, a.chats, kind=q4gpu.KIND_Q8 if a.kind == "q8_0" else q4gpu.KIND_F16)
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
    print("%d tokens in %d steps of %d layers, %.3f ms per step (median); %d steps checked; status %d; pages back: %s"
          % (tokens, a.steps, a.layers, ms[len(ms) // 2] if ms else 0.0, checked, status, back))
    return 0 if back and status == 0 else 1


if __name__ == "__main__":
    sys.exit(main())
