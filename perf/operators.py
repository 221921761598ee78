"""The operators of a paged KV cache, as cases that can be timed and compared.

A serving host keeps the rows of all requests in one pool of pages and takes steps in which every request brings some new
tokens: one (decoding), a few (drafts to be verified) or many (a chunk of prompt).  Per step it plans once and then, layer by
layer, appends the new K / V rows and attends:

  plan     from the requests' lengths: pages off the free list into the block tables, and for every new token its slot, its
           position and its request; then the pages back again (the step is taken back), so that a pass can be repeated
  append   new K / V rows into the slots of their tokens (quantised or rounded), and read back from there
  attend   attention of the new tokens of all requests over their pages, causal inside a chunk

Shapes are those of this repository's benchmark (16 query / 2 kv heads, head size 128), of the engine's own model
(24 / 2 / 256), and generic ones.  Memory of a pool, as documented with the entry points:
[layer][page][kv head][tile of 16 rows]; a q8_0 tile is 16 records {K codes | V codes | K scales | V scales}, padded to 16
bytes; an f16 tile is K then V, each hd / 64 blocks of 16 rows x 128 bytes with the 16-byte chunk c of row r at c ^ (r & 7).
"""
import math
import os
import random
import sys

import torch

own = False

SMALL = {"n_head": 16, "n_kvh": 2, "hd": 128}     # the benchmark's shape
MODEL = {"n_head": 24, "n_kvh": 2, "hd": 256}     # the engine's model
WIDE = {"n_head": 32, "n_kvh": 8, "hd": 128}      # more kv heads, fewer query heads on each
NARROW = {"n_head": 8, "n_kvh": 4, "hd": 64}      # a small model's heads


def attend(shape, n_req, rows, add, one=0, kind="q8_0", page=64, gate=False, lens=1):
    """n_req requests that hold rows[0] .. rows[1] rows and bring add[0] .. add[1] new tokens; the first `one` of them bring one."""
    return dict(op="attend", n_req=n_req, rows_lo=rows[0], rows_hi=rows[1], add_lo=add[0], add_hi=add[1], one=one, kind=kind, page=page,
                gate=gate, lens=lens, **shape)


def plan(n_req, rows, add, page=64, lens=1):
    return dict(op="plan", n_req=n_req, rows_lo=rows[0], rows_hi=rows[1], add_lo=add[0], add_hi=add[1], one=0, page=page, lens=lens)


def append(n_tok, n_kvh, hd, kind, page=64):
    return dict(op="append", n_tok=n_tok, n_kvh=n_kvh, hd=hd, kind=kind, page=page)


def listed():
    return [
        # a decode step of a few sessions: nearly every page is there already
        dict(plan(16, (0, 4096), (1, 1), page=16), name="plan_16_decode"),
        # many requests at once, chunks of prompt among them
        dict(plan(1000, (0, 8000), (1, 512)), name="plan_1000_chunks"),
        # one layer's new rows of 64 decoding sessions
        dict(append(64, 2, 128, "q8_0"), name="append_64_q8"),
        # one layer's new rows of long prompts in a 16-bit pool
        dict(append(16001, 8, 128, "f16", page=32), name="append_16001_f16"),
        # a token of four short chats with a small model
        dict(attend(NARROW, 4, (30, 1500), (1, 1), kind="f16", page=16, gate=True), name="decode_4_f16_64"),
        # a token at the largest context
        dict(attend(SMALL, 1, (262143, 262143), (1, 1)), name="decode_1_262144"),
        # 64 sessions of very different lengths decode together
        dict(attend(SMALL, 64, (1024, 32768), (1, 1), gate=True), name="decode_64_32768"),
        # five drafted tokens per session are verified, engine's model
        dict(attend(MODEL, 13, (700, 9000), (5, 5), page=32), name="draft_13x5_256"),
        # a 512-token slice of a prompt behind a prefix, gated
        dict(attend(SMALL, 1, (16001, 16001), (512, 512), gate=True), name="chunk_512_16001"),
        # a server's mixed step: sessions that decode beside chunks of prompt, odd lengths everywhere
        dict(attend(WIDE, 24, (0, 6000), (100, 700), one=18, kind="f16"), name="mixed_24_f16"),
        # prompts of the engine's model from their first token
        dict(attend(MODEL, 3, (0, 0), (500, 2048)), name="prompts_3_256"),
        # the benchmark's chunked prefill: a long chunk behind a long prefix
        dict(attend(SMALL, 1, (16384, 16384), (8192, 8192)), name="chunk_8192_16384"),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["plan", "append", "attend", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 64, 128])
    lens = rng.randrange(1 << 20)
    if op == "plan":
        return plan(log(1, 2000), (0, log(16, 8192)), (1, log(1, 512)), page=page, lens=lens)
    kind = rng.choice(["q8_0", "q8_0", "f16"])
    shape = rng.choice([SMALL, SMALL, MODEL, WIDE, NARROW])
    if op == "append":
        return append(log(1, 16000), shape["n_kvh"], shape["hd"], kind, page=page)
    form = rng.choice(["decode", "decode", "draft", "chunk", "mixed"])
    n_req = rng.choice([1, log(2, 64)])
    if form == "decode":
        add = (1, 1)
    elif form == "draft":
        k = rng.randint(2, 8)
        add = (rng.choice([1, k]), k)
    else:
        n_req = rng.choice([1, 1, log(2, 12)])
        hi = log(20, 4096 if n_req == 1 else 1024)
        add = (hi if n_req == 1 else max(1, hi // rng.choice([1, 2, 8])), hi)
    one = rng.randint(0, 3 * n_req) if form == "mixed" else 0
    n_req += one
    # rows of all requests and scores of all heads, together, stay below those of the largest listed cases
    most = int(min(5e8 / (n_req * shape["n_kvh"] * shape["hd"]), 2.5e9 / max(1, shape["hd"] / 128) / (n_req * add[1] * shape["n_head"]))) - add[1]
    hi = log(16, max(32, min(262143 if n_req == 1 else 32768, most)))
    return attend(shape, n_req, (rng.choice([0, hi // 16, hi]), hi), add, one=one, kind=kind, page=page, gate=rng.random() < 0.5, lens=lens)


# ------------------------------------------------------------------------------------------- sizes
def lengths(case):
    """rows held and new tokens of every request: of the case alone, so that its work is known"""
    r = random.Random(case["lens"])
    rows = [r.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["n_req"])]
    add = [r.randint(case["add_lo"], case["add_hi"]) for _ in range(case["n_req"])]
    return rows, [1 if i < case["one"] else n for i, n in enumerate(add)]


def pages_of(rows, page):
    return -(-rows // page)


def row_bytes(kind, hd):
    """K and V of one position and kv head in a pool"""
    return -(-(2 * hd + hd // 8) // 16) * 16 if kind == "q8_0" else 4 * hd


def tile_bytes(kind, hd):
    return 16 * row_bytes(kind, hd)


def work(case):
    if case["op"] == "append":
        kvw, n = case["n_kvh"] * case["hd"], case["n_tok"]
        # rows in, pages written and read, rows out
        return {"bytes": n * (2 * 8 * kvw + 2 * case["n_kvh"] * row_bytes(case["kind"], case["hd"]) + 8), "flops": 0}
    rows, add = lengths(case)
    if case["op"] == "plan":
        new = sum(pages_of(h + n, case["page"]) - pages_of(h, case["page"]) for h, n in zip(rows, add))
        # lengths twice, starts, three words per token, new pages out of the list into the tables and back
        return {"bytes": 16 * case["n_req"] + 4 * (case["n_req"] + 1) + 12 * sum(add) + 16 * new, "flops": 0}
    per_row = case["n_kvh"] * row_bytes(case["kind"], case["hd"])
    token = case["n_head"] * case["hd"] * (2 + 2 + (4 if case["gate"] else 0))
    attended = sum(n * h + n * (n + 1) // 2 for h, n in zip(rows, add))
    return {"bytes": sum(h + n for h, n in zip(rows, add)) * per_row + sum(add) * token,
            "flops": 4 * case["n_head"] * case["hd"] * attended}


# ------------------------------------------------------------------------------------------- inputs
def swizzle(device):
    """[row][place] -> the 16-byte chunk that lies there; its own inverse"""
    return torch.arange(8, device=device)[None, :] ^ (torch.arange(16, device=device) & 7)[:, None]


def quantised(x):
    """q8_0: fp32 rows [..., hd] -> codes int8 [..., hd], scales fp16 [..., hd / 32]"""
    b = x.unflatten(-1, (-1, 32))
    d = b.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    return (b * inv).round().clamp(-127, 127).to(torch.int8).flatten(-2), d.squeeze(-1).to(torch.float16)


def packed(x, kind, live=None):
    """rows [..., 16, 2, hd] fp32 (K, V) of whole tiles -> bytes [..., tile bytes]; rows that are not live hold NaN"""
    hd = x.shape[-1]
    if kind == "q8_0":
        codes, scales = quantised(x)
        if live is not None:
            scales = torch.where(live[..., None, None], scales, float("nan"))
        rec = torch.cat([codes.flatten(-2).view(torch.uint8), scales.flatten(-2).view(torch.uint8)], -1)
        return torch.nn.functional.pad(rec, (0, row_bytes(kind, hd) - rec.shape[-1])).flatten(-2)
    h = x.to(torch.float16)
    if live is not None:
        h = torch.where(live[..., None, None], h, float("nan"))
    t = h.unflatten(-1, (hd // 64, 8, 8)).movedim(-5, -3)   # [..., K or V, block, row, chunk, 8]
    t = t[..., torch.arange(16, device=x.device)[:, None], swizzle(x.device), :]
    return t.flatten(-5).view(torch.uint8)


def unpacked(tiles, kind, hd):
    """bytes [..., tile bytes] -> K, V as fp32 [..., 16, hd]"""
    if kind == "q8_0":
        rec = tiles.unflatten(-1, (16, -1))
        codes = rec[..., : 2 * hd].view(torch.int8).float().unflatten(-1, (2, hd // 32, 32))
        scales = rec[..., 2 * hd: 2 * hd + hd // 8].contiguous().view(torch.float16).float().unflatten(-1, (2, hd // 32))
        kv = (codes * scales[..., None]).flatten(-2)
        return kv[..., 0, :], kv[..., 1, :]
    t = tiles.view(torch.float16).unflatten(-1, (2, hd // 64, 16, 8, 8))
    t = t[..., torch.arange(16, device=tiles.device)[:, None], swizzle(tiles.device), :].float()
    kv = t.movedim(-3, -5).flatten(-3).movedim(-2, -3)      # [..., K or V, row, hd]
    return kv[..., 0, :, :], kv[..., 1, :, :]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    on = dict(device="cuda")
    if case["op"] == "append":
        n, page, n_kvh, hd = case["n_tok"], case["page"], case["n_kvh"], case["hd"]
        n_pages = pages_of(n, page) * 2 + 1
        mem = torch.zeros(1, n_pages, n_kvh, page // 16, tile_bytes(case["kind"], hd), dtype=torch.uint8, **on)
        k, v = torch.randn(2, n, n_kvh * hd, generator=g, **on).unbind(0)
        if n < 200:   # a token of each of many sessions: its page is its own
            slot = torch.randperm(n_pages, generator=g, **on)[:n] * page + torch.randint(page, (n,), generator=g, **on) if n <= n_pages else torch.randperm(n_pages * page, generator=g, **on)[:n]
        else:         # prompts: whole pages in any order
            slot = (torch.randperm(n_pages, generator=g, **on)[:, None] * page + torch.arange(page, **on)).flatten()[:n]
        return dict(case=case, mem=mem, k=k, v=v, slot=slot.to(torch.int32), k_out=torch.empty_like(k), v_out=torch.empty_like(v))
    rows, add = lengths(case)
    order = torch.randperm(case["n_req"], generator=torch.Generator().manual_seed(seed)).tolist()
    rows, add = [rows[i] for i in order], [add[i] for i in order]
    page = case["page"]
    held = [pages_of(h if case["op"] == "plan" else h + n, page) for h, n in zip(rows, add)]
    total = sum(add)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, **on)  # noqa: E731
    stride = max(max(pages_of(h + n, page) for h, n in zip(rows, add)), 1) + 1
    new = sum(pages_of(h + n, page) for h, n in zip(rows, add)) - sum(held)
    n_pages = sum(held) + new + max(1, (sum(held) + new) // 16)
    pages = torch.randperm(n_pages, generator=g, **on).to(torch.int32)
    # block tables of the pages that the requests hold
    col = torch.arange(stride, **on)
    has = col[None, :] < ints(held)[:, None]
    table = torch.full((case["n_req"], stride), -1, dtype=torch.int32, **on)
    table[has] = pages[: sum(held)]
    s = dict(case=case, rows=ints(rows), add=ints(add), table=table, n_tok=total, max_add=max(add), max_rows=max(h + n for h, n in zip(rows, add)))
    if case["op"] == "plan":
        n_tok = total + total // 8   # a step's arrays have room for more tokens
        s |= dict(after=s["rows"] + s["add"], max_tok=n_tok, new=new, start=torch.empty(case["n_req"] + 1, dtype=torch.int32, **on),
                  **{k: torch.empty(n_tok, dtype=torch.int32, **on) for k in ("slot", "pos", "req")})
        s["free"] = torch.cat([pages[sum(held):], pages[: sum(held)]])   # a stack of n_free pages; what lies above it has no meaning
        s["n_free"] = ints([n_pages - sum(held)])
        return s
    n_kvh, hd = case["n_kvh"], case["hd"]
    live = torch.zeros(n_pages, page, dtype=torch.bool, **on)
    live[pages[: sum(held)].long()] = (torch.arange(stride * page, **on)[None, :] < (s["rows"] + s["add"])[:, None]).unflatten(1, (stride, page))[has]
    live = live.unflatten(1, (page // 16, 16))
    mem = torch.empty(1, n_pages, n_kvh, page // 16, tile_bytes(case["kind"], hd), dtype=torch.uint8, **on)
    step = max(1, (1 << 28) // (n_kvh * page * 2 * hd))
    for a in range(0, n_pages, step):
        b = min(n_pages, a + step)
        x = torch.randn(b - a, n_kvh, page // 16, 16, 2, hd, generator=g, **on)
        mem[0, a:b] = packed(x, case["kind"], live[a:b, None].expand(-1, n_kvh, -1, -1))
    start = [0]
    for n in add:
        start.append(start[-1] + n)
    s |= dict(mem=mem, start=ints(start), q=torch.randn(total, case["n_head"], hd, generator=g, **on).to(torch.bfloat16),
              gate=torch.randn(total, case["n_head"], hd, generator=g, **on) if case["gate"] else None,
              out=torch.empty(total, case["n_head"], hd, dtype=torch.bfloat16, **on))
    return s


# ------------------------------------------------------------------------------------------- one pass
def pool(s):
    """the handle that a user's program keeps beside the pool's memory"""
    if "pool" not in s:
        at = os.path.join(os.getcwd(), "suzuqu-engine-4exp_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import q4gpu
        q4gpu.init()
        q4gpu.use_torch_stream()
        c = s["case"]
        kind = {"q8_0": q4gpu.KIND_Q8, "f16": q4gpu.KIND_F16}[c.get("kind", "q8_0")]
        if c["op"] == "plan":   # the free list alone
            s["pool"] = q4gpu.PagePool(1, 1, 64, s["free"].numel(), c["page"], kind, free=s["free"], n_free=s["n_free"])
        else:
            s["pool"] = q4gpu.PagePool(1, c["n_kvh"], c["hd"], s["mem"].shape[1], c["page"], kind, mem=s["mem"])
    return s["pool"]


def run(s):
    op = s["case"]["op"]
    if op == "plan":
        if own:
            p = pool(s)
            p.plan(s["rows"], s["add"], s["table"], s["start"], s["slot"], s["pos"], s["req"])
            p.trim(s["after"], s["rows"], s["table"])
        else:
            plain_plan(s)
            plain_trim(s)
        return {k: s[k] for k in ("table", "start", "slot", "pos", "req", "free", "n_free")}
    if op == "append":
        if own:
            p = pool(s)
            p.append(0, s["k"], s["v"], s["slot"])
            p.gather(0, s["slot"], s["k_out"], s["v_out"])
            return {"k": s["k_out"], "v": s["v_out"]}
        return plain_append(s)
    if own:
        c = s["case"]
        pool(s).attend(0, s["q"], s["out"], s["rows"], s["start"], s["table"], c["n_head"], 1.0 / math.sqrt(c["hd"]), gate=s["gate"], max_add=s["max_add"])
        return s["out"]
    return plain_attend(s)


# ------------------------------------------------------------------------------------------- the plain forms
def plain_plan(s):
    page, table = s["case"]["page"], s["table"]
    stride = table.shape[1]
    h, n = s["rows"].long(), s["add"].long().clamp(min=0)
    n = torch.where((h < 0) | (h + n > stride * page), 0, n)
    first = (h + page - 1) // page
    need = torch.where(n > 0, (h + n + page - 1) // page - first, 0)
    fits = (need.cumsum(0) <= s["n_free"]) & (n.cumsum(0) <= s["max_tok"])
    n, need = n * fits, need * fits
    ends, page_ends = n.cumsum(0), need.cumsum(0)
    s["start"][0] = 0
    s["start"][1:] = ends
    # the pages, in the order of the requests, from the top of the stack
    i = torch.arange(s["new"], device=table.device)
    r = torch.searchsorted(page_ends, i, right=True)
    at = r * stride + first[r] + i - (page_ends - need)[r]
    table.view(-1)[at] = s["free"][s["n_free"] - 1 - i]
    s["n_free"] -= page_ends[-1:].int()
    # the tokens
    t = torch.arange(s["max_tok"], device=table.device)
    r = torch.searchsorted(ends, t, right=True)
    live = t < ends[-1]
    r = torch.where(live, r, 0)
    pos = h[r] + t - (ends - n)[r]
    slot = table[r, torch.where(live, pos // page, 0)] * page + pos % page
    for name, x in (("slot", slot), ("pos", pos), ("req", r)):
        s[name].copy_(torch.where(live, x, -1))


def plain_trim(s):
    page, table = s["case"]["page"], s["table"]
    first, last = (s["rows"].long() + page - 1) // page, (s["after"].long() + page - 1) // page
    ends = (last - first).cumsum(0)
    i = torch.arange(s["new"], device=table.device)
    r = torch.searchsorted(ends, i, right=True)
    s["free"][s["n_free"] + ends[-1:] - 1 - i] = table[r, first[r] + i - (ends - (last - first))[r]]
    s["n_free"] += ends[-1:].int()


def plain_append(s):
    c = s["case"]
    n_kvh, hd, page, kind = c["n_kvh"], c["hd"], c["page"], c["kind"]
    slot = s["slot"].long()
    at, row = slot // page, slot % page
    x = torch.stack([s["k"].view(-1, n_kvh, hd), s["v"].view(-1, n_kvh, hd)], 2)   # [token, kv head, K or V, hd]
    if kind == "q8_0":
        codes, scales = quantised(x)
        rec = torch.cat([codes.flatten(-2).view(torch.uint8), scales.flatten(-2).view(torch.uint8)], -1)
        mem = s["mem"][0].view(s["mem"].shape[1], n_kvh, page, -1)
        mem[at, :, row, : rec.shape[-1]] = rec
        got = mem[at, :, row]
        codes = got[..., : 2 * hd].contiguous().view(torch.int8).float().unflatten(-1, (2, hd // 32, 32))
        scales = got[..., 2 * hd: 2 * hd + hd // 8].contiguous().view(torch.float16).float().unflatten(-1, (2, hd // 32, 1))
        kv = (codes * scales).flatten(-2)
    else:
        # [page, kv head, tile, K or V, block, row, place, 8]
        mem = s["mem"][0].view(torch.float16).view(s["mem"].shape[1], n_kvh, page // 16, 2, hd // 64, 16, 8, 8)
        chunks = swizzle(slot.device)[row % 16][:, None, None, None, :, None].expand(-1, n_kvh, 2, hd // 64, 8, 8)
        mem[at, :, row // 16, :, :, row % 16] = x.to(torch.float16).unflatten(-1, (hd // 64, 8, 8)).gather(-2, chunks)
        kv = mem[at, :, row // 16, :, :, row % 16].gather(-2, chunks).flatten(-3).float()
    return {"k": kv[:, :, 0].flatten(1), "v": kv[:, :, 1].flatten(1)}


def plain_attend(s):
    c = s["case"]
    n_req, n_kvh, hd, page = c["n_req"], c["n_kvh"], c["hd"], c["page"]
    group, most = c["n_head"] // n_kvh, s["max_add"]
    used = pages_of(s["max_rows"], page)
    tiles = s["mem"][0][s["table"][:, :used].clamp(min=0).long()]           # [request, page, kv head, tile, bytes]
    k, v = unpacked(tiles.transpose(1, 2).flatten(2, 3), c["kind"], hd)     # [request, kv head, tile, 16, hd]
    k, v = k.flatten(2, 3), v.flatten(2, 3)
    p = torch.arange(used * page, device=k.device)
    v = torch.where((p[None, :] < (s["rows"] + s["add"])[:, None])[:, None, :, None], v, 0.0)
    # the requests' tokens, padded to the longest
    j = torch.arange(most, device=k.device)
    live = j[None, :] < s["add"][:, None]
    tok = torch.where(live, s["start"][:-1, None] + j[None, :], 0).long()
    q = s["q"][tok].float().unflatten(2, (n_kvh, group)).transpose(1, 2).flatten(2, 3)   # [request, kv head, token x head, hd]
    w = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    seen = p[None, None, :] <= (s["rows"][:, None] + j[None, :])[:, :, None]             # [request, token, position]
    w = w.unflatten(2, (most, group)).masked_fill_(~seen[:, None, :, None, :], float("-inf")).flatten(2, 3)
    w = (w - w.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    o = o.unflatten(2, (most, group)).transpose(1, 2).flatten(2, 3)[live]                # [token, head, hd]
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"]))
    return o.to(torch.bfloat16)


# ------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """From the definitions, request by request and head by head, in 64 bits."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    n_kvh, hd, page = case["n_kvh"], case["hd"], case["page"]
    if case["op"] == "append":
        res = {}
        for name in ("k", "v"):
            x = s[name].double()
            if case["kind"] == "q8_0":
                b = x.view(x.shape[0], -1, 32)
                step = b.abs().max(2, keepdim=True).values / 127
                x = (torch.round(b / step).nan_to_num(0.0) * step.half().double()).view_as(x)
            else:
                x = x.half().double()
            res[name] = x
        return res
    rows, add, start, table = s["rows"].tolist(), s["add"].tolist(), s["start"].tolist(), s["table"].long()
    out = torch.zeros(s["n_tok"], case["n_head"], hd, dtype=torch.float64, device="cuda")
    group = case["n_head"] // n_kvh
    for r, (held, new) in enumerate(zip(rows, add)):
        n = held + new
        raw = s["mem"][0, table[r, : pages_of(n, page)]]                    # [page, kv head, tile, bytes]
        for kh in range(n_kvh):
            tiles = raw[:, kh].reshape(-1, raw.shape[-1])
            if case["kind"] == "q8_0":
                rec = tiles.view(-1, row_bytes("q8_0", hd))[:n]
                num = rec[:, : 2 * hd].contiguous().view(torch.int8).double()
                num *= rec[:, 2 * hd: 2 * hd + hd // 8].contiguous().view(torch.float16).double().repeat_interleave(32, 1)
                k, v = num[:, :hd], num[:, hd:]
            else:
                h = tiles.view(torch.float16).view(-1, 2, hd // 64, 16, 64)
                parts = []
                for i in range(16):   # row i of every tile
                    places = torch.tensor([(d // 8 ^ (i & 7)) * 8 + d % 8 for d in range(64)], device="cuda")
                    parts.append(h[:, :, :, i][..., places].reshape(-1, 2, hd))
                kv = torch.stack(parts, 1).reshape(-1, 2, hd)[:n].double()
                k, v = kv[:, 0], kv[:, 1]
            for head in range(kh * group, (kh + 1) * group):
                for a in range(0, new, 2048):   # tokens of the chunk
                    b = min(new, a + 2048)
                    q = s["q"][start[r] + a: start[r] + b, head].double()
                    z = q @ k.T / math.sqrt(hd)
                    late = torch.arange(n, device="cuda")[None, :] > held + torch.arange(a, b, device="cuda")[:, None]
                    z[late] = -math.inf
                    out[start[r] + a: start[r] + b, head] = torch.softmax(z, 1) @ v
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out
