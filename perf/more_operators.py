"""What a step over the paged KV cache does around its attention, as cases that can be timed and compared.

A serving host plans a step and attends with it; before, between and behind that it

  prep     takes the projections' rows of the step's tokens: norm of every query and key head, rotation by the token's own position,
           the gate split off, keys and values into the pages (q8_0 or fp16)
  verify   holds drafted tokens against the target's distributions, given random numbers, and draws the token behind the last one
           that is kept; without drafts it draws a token per request
  fork     lets requests share the pages of a common prefix and copies the page that it ends in; release gives up a request's pages, which go
           back to the stack with their last holder
  compact  moves the pages in use to the low end of the pool and renames them in the tables

Shapes are those of this repository's benchmark (16 query / 2 kv heads of 128), of the engine's own model (24 / 2 / 256, 64 of the dims
rotated), and generic ones.  Memory of a pool, as documented with the entry points: [layer][page][kv head][tile of 16 rows]; a q8_0 tile is 16
records {K codes | V codes | K scales | V scales}, padded to 16 bytes; an f16 tile is K then V, each hd / 64 blocks of 16 rows x 128
bytes with the 16-byte chunk c of row r at c ^ (r & 7).
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
EPS = 1e-6
ORIG = 8192                                       # the context that scaled frequencies were made for


def prep(shape, n_tok, n_rot, kind="q8_0", page=64, gate=True, half=False, scaling="none", fused=False, bf16=False, chunk=1, idle=0):
    """n_tok tokens in runs of `chunk` positions (1: a token of each of many requests); `idle` more places without a token behind them"""
    return dict(op="prep", n_tok=n_tok, n_rot=n_rot, kind=kind, page=page, gate=gate, half=half, scaling=scaling, fused=fused, bf16=bf16, chunk=chunk, idle=idle, **shape)


def verify(n_req, drafts, vocab, bf16=False, draft="logits", greedy=0.0, sharp=2.5, lens=1):
    """n_req requests with drafts[0] .. drafts[1] drafted tokens; draft: logits, or none where drafts are certain (looked up); a share of greedy requests"""
    return dict(op="verify", n_req=n_req, drafts_lo=drafts[0], drafts_hi=drafts[1], vocab=vocab, bf16=bf16, draft=draft, greedy=greedy, sharp=sharp, lens=lens)


def fork(n_par, children, rows, layers, shape, kind="q8_0", page=64, lens=1):
    """n_par requests of rows[0] .. rows[1] rows, each with so many children"""
    return dict(op="fork", n_par=n_par, children=children, rows_lo=rows[0], rows_hi=rows[1], layers=layers, n_kvh=shape["n_kvh"], hd=shape["hd"], kind=kind, page=page, lens=lens)


def compact(n_pages, used, layers, shape, kind="q8_0", page=64, shared=4):
    """a pool of which the share `used` is in use, by requests of 40 pages; `shared` requests each begin with the same 10"""
    return dict(op="compact", n_pages=n_pages, used=used, layers=layers, n_kvh=shape["n_kvh"], hd=shape["hd"], kind=kind, page=page, shared=shared)


def listed():
    return [
        # a token of one session of the engine's model
        dict(prep(MODEL, 1, 64), name="prep_1_256"),
        # one layer's rows of 64 decoding sessions, four places of the captured step idle
        dict(prep(SMALL, 64, 128, idle=4), name="prep_64_q8"),
        # chunks of prompt of the engine's model
        dict(prep(MODEL, 4096, 64, chunk=512), name="prep_4096_256"),
        # long prompts out of a fused 16-bit projection into a 16-bit pool, far positions
        dict(prep(WIDE, 16001, 128, kind="f16", page=32, gate=False, half=True, scaling="ramp", fused=True, bf16=True, chunk=4000), name="prep_16001_fused"),
        # a single session's five drafts
        dict(verify(1, (5, 5), 131072), name="verify_1x5"),
        # a token is drawn for each of many sessions
        dict(verify(256, (0, 0), 32003, greedy=0.25), name="draw_256"),
        # a batch of sessions whose drafts differ in number, looked up instead of drawn, 16-bit logits of an odd vocabulary
        dict(verify(64, (1, 8), 50001, bf16=True, draft="none", greedy=0.1), name="verify_64_lookup"),
        # a batch of sessions with five drafts each over a large vocabulary
        dict(verify(48, (5, 5), 131072), name="verify_48x5"),
        # four beams of a chat
        dict(fork(1, 4, (700, 700), 2, SMALL), name="fork_4_beams"),
        # parallel answers to many long prompts
        dict(fork(64, 4, (1000, 16000), 12, SMALL), name="fork_256"),
        # a small pool, a few chats
        dict(compact(300, 0.5, 2, SMALL), name="compact_300"),
        # a server's pool after its load went down
        dict(compact(4096, 0.45, 12, SMALL), name="compact_4096"),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["prep", "prep", "verify", "verify", "fork", "compact"])
    page = rng.choice([16, 32, 64, 64, 128])
    kind = rng.choice(["q8_0", "q8_0", "f16"])
    shape = rng.choice([SMALL, SMALL, MODEL, WIDE, NARROW])
    lens = rng.randrange(1 << 20)
    if op == "prep":
        n_tok = log(1, 3500)
        n_rot = rng.choice([shape["hd"], shape["hd"], shape["hd"] // 2, shape["hd"] // 4, 16])
        return prep(shape, n_tok, n_rot, kind=kind, page=page, gate=rng.random() < 0.5, half=rng.random() < 0.5, scaling=rng.choice(["none", "none", "linear", "ramp", "smooth"]),
                    fused=rng.random() < 0.5, bf16=rng.random() < 0.5, chunk=rng.choice([1, 1, log(2, 1024)]), idle=rng.choice([0, 0, log(1, 20)]))
    if op == "verify":
        vocab, most = log(1000, 160000), rng.choice([0, 4, 8])
        n_req = log(1, max(2, min(512, int(6e7 / vocab / (2 * most + 1)))))
        return verify(n_req, (rng.randint(0, most), most), vocab, bf16=rng.random() < 0.5, draft=rng.choice(["logits", "logits", "none"]), greedy=rng.choice([0.0, 0.0, 0.3, 1.0]),
                      sharp=rng.uniform(0.5, 4.0), lens=lens)
    row = shape["n_kvh"] * row_bytes(kind, shape["hd"])
    if op == "fork":
        children, layers = rng.randint(1, 5), log(1, 12)
        n_par = log(1, max(2, min(64, int(6e8 / ((children + 1) * page * layers * row)))))
        hi = log(40, max(41, min(20000, int(1.2e9 / (n_par * layers * row)))))
        return fork(n_par, children, (rng.choice([0, hi // 8, hi]), hi), layers, shape, kind=kind, page=page, lens=lens)
    layers = log(1, 12)
    return compact(log(64, max(65, min(20000, int(1.2e9 / (layers * page * row))))), rng.uniform(0.05, 0.95), layers, shape, kind=kind, page=page, shared=rng.randint(1, 8))


# ------------------------------------------------------------------------------------------- sizes
def pages_of(rows, page):
    return -(-rows // page)


def row_bytes(kind, hd):
    """K and V of one position and kv head in a pool"""
    return -(-(2 * hd + hd // 8) // 16) * 16 if kind == "q8_0" else 4 * hd


def counts(case):
    """of the case alone, so that its work is known: drafts of every request, or rows of every parent"""
    r = random.Random(case["lens"])
    if case["op"] == "verify":
        return [r.randint(case["drafts_lo"], case["drafts_hi"]) for _ in range(case["n_req"])]
    return [r.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["n_par"])]


def moved(case):
    """pages in use, and those of them that a compaction moves, as many as fall behind the used part by chance"""
    live = max(1, int(case["n_pages"] * case["used"]))
    return live, int(live * (1 - live / case["n_pages"]))


def work(case):
    if case["op"] == "prep":
        n, hd = case["n_tok"], case["hd"]
        read = (case["n_head"] * (2 if case["gate"] else 1) + 2 * case["n_kvh"]) * hd * (2 if case["bf16"] else 4)
        write = case["n_head"] * hd * (2 + (4 if case["gate"] else 0)) + case["n_kvh"] * row_bytes(case["kind"], hd)
        return {"bytes": n * (read + write + 8), "flops": 0}
    if case["op"] == "verify":
        k = counts(case)
        rows = sum(k) + case["n_req"] + (sum(k) if case["draft"] == "logits" else 0)
        return {"bytes": rows * case["vocab"] * (2 if case["bf16"] else 4), "flops": 0}
    per_row = case["layers"] * case["n_kvh"] * row_bytes(case["kind"], case["hd"])
    if case["op"] == "fork":
        # the children's last pages and table rows, the parents' in return; shares counted up and down
        rows, page = counts(case), case["page"]
        times = case["children"] + 1
        return {"bytes": times * sum(2 * (r % page) * per_row + (r // page) * 24 + 16 for r in rows), "flops": 0}
    live, m = moved(case)
    return {"bytes": 2 * m * case["page"] * per_row + 12 * case["n_pages"] + 8 * live, "flops": 0}


# ------------------------------------------------------------------------------------------- inputs
def frequencies(case):
    """radians per position of every pair, in 64 bits, and the factor on the rotated part"""
    n_rot, base = case["n_rot"], 1e7 if case["hd"] == 256 else 1e6
    f = [base ** (-2 * i / n_rot) for i in range(n_rot // 2)]
    factor, scaling, mag = 8.0, case["scaling"], 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "ramp":     # pairs that turn less than once over the original context are slowed down, those that turn 32 times kept
        at = lambda turns: n_rot / 2 * math.log(ORIG / (turns * 2 * math.pi)) / math.log(base)  # noqa: E731
        lo, hi = max(0, math.floor(at(32.0))), min(n_rot // 2 - 1, math.ceil(at(1.0)))
        slow = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(n_rot // 2)]
        f = [x * (1 - s) + x / factor * s for x, s in zip(f, slow)]
        mag = 0.1 * math.log(factor) + 1
    elif scaling == "smooth":   # the same with a ramp over the turns themselves, from 1 to 4
        keep = [min(1.0, max(0.0, (x * ORIG / (2 * math.pi) - 1) / 3)) for x in f]
        f = [x * k + x / factor * (1 - k) for x, k in zip(f, keep)]
    return f, mag


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    on = dict(device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, **on)  # noqa: E731
    host = torch.Generator().manual_seed(seed)
    if case["op"] == "prep":
        n, page, n_kvh, hd, n_head = case["n_tok"], case["page"], case["n_kvh"], case["hd"], case["n_head"]
        kind = torch.bfloat16 if case["bf16"] else torch.float32
        wide = n + case["idle"]
        heads = [n_head * (2 if case["gate"] else 1), n_kvh, n_kvh]
        rows = torch.randn(wide, sum(heads) * hd, generator=g, **on)
        rows = (rows * torch.exp(torch.randn(wide, 1, generator=g, **on))).to(kind)
        parts = rows.split([h * hd for h in heads], 1)
        q, k, v = parts if case["fused"] else [x.contiguous() for x in parts]
        runs = -(-n // case["chunk"])
        first = torch.randint(0, 262144 - case["chunk"], (runs, 1), generator=g, **on)
        pos = (first + torch.arange(case["chunk"], **on)).flatten()[:n]
        n_pages = runs * pages_of(case["chunk"] + page, page) + 3
        order = torch.randperm(n_pages, generator=g, **on)
        if case["chunk"] == 1:   # a page of its own for every token
            slot = order[:n] * page + pos % page
        else:                    # a run's rows lie in whole pages, in any order
            slot = (order[: runs * pages_of(case["chunk"], page)].view(runs, -1, 1) * page + torch.arange(page, **on)).flatten(1)[:, : case["chunk"]].flatten()[:n]
        none = torch.full((case["idle"],), -1, dtype=torch.int32, **on)
        f, mag = frequencies(case)
        mem = torch.zeros(1, n_pages, n_kvh, page // 16, 16 * row_bytes(case["kind"], hd), dtype=torch.uint8, **on)
        s = dict(case=case, q=q, k=k, v=v, pos=torch.cat([pos.int(), none]), slot=torch.cat([slot.int(), none]), f=torch.tensor(f, dtype=torch.float64, **on), mag=mag, mem=mem,
                 wq=1 + 0.2 * torch.randn(hd, generator=g, **on), wk=1 + 0.2 * torch.randn(hd, generator=g, **on),
                 q_out=torch.zeros(wide, n_head, hd, dtype=torch.bfloat16, **on), gate=torch.zeros(wide, n_head, hd, **on) if case["gate"] else None)
        if case["kind"] == "q8_0":
            s |= dict(k_out=torch.empty(wide, n_kvh * hd, **on), v_out=torch.empty(wide, n_kvh * hd, **on))
        return s
    if case["op"] == "verify":
        n_req, vocab = case["n_req"], case["vocab"]
        k = [counts(case)[i] for i in torch.randperm(n_req, generator=host).tolist()]
        add = torch.tensor([x + 1 for x in k])
        start = torch.cat([torch.zeros(1, dtype=torch.long), add.cumsum(0)])
        n_tok = int(start[-1])
        kind = torch.bfloat16 if case["bf16"] else torch.float32
        target = torch.randn(n_tok, vocab, generator=g, **on) * case["sharp"]
        drafted = (target + torch.randn(n_tok, vocab, generator=g, **on) * (0.4 * case["sharp"])).to(kind)
        # temperatures; a share of the requests is greedy
        temp = 0.6 + 0.8 * torch.rand(n_req, generator=g, **on)
        temp[: int(n_req * case["greedy"])] = 0.0
        temp = temp[torch.randperm(n_req, generator=g, **on)]
        req = torch.repeat_interleave(torch.arange(n_req), add).cuda()
        z = drafted.float() / torch.where(temp > 0, temp, 0.05)[req, None]
        z -= torch.log(-torch.log(torch.rand(n_tok, vocab, generator=g, **on).clamp_(1e-20)).clamp_(1e-20))   # drawn from the draft's distribution
        drawn = z.argmax(1, keepdim=True)
        token = torch.empty(n_tok + 1, dtype=torch.int32, **on)
        token[0], token[1:] = 1, drawn[:, 0]
        if case["draft"] == "none":   # what was found in the text so far is likely to come again
            target.scatter_add_(1, drawn, 5 * case["sharp"] * torch.rand(n_tok, 1, generator=g, **on))
        target = target.to(kind)
        del z
        return dict(case=case, target=target, draft=drafted if case["draft"] == "logits" else None, token=token[:n_tok].contiguous(), start=start.int().cuda(), req=req, n_tok=n_tok, temp=temp,
                    rows=torch.randint(0, 5000, (n_req,), generator=g, dtype=torch.int32, **on), u_accept=torch.rand(n_tok, generator=g, **on), u_draw=torch.rand(n_req, generator=g, **on),
                    accepted=torch.empty(n_req, dtype=torch.int32, **on), next=torch.empty(n_req, dtype=torch.int32, **on), keep=torch.empty(n_req, dtype=torch.int32, **on),
                    logp=torch.empty(n_tok, **on))
    page, per_page = case["page"], case["page"] * case["n_kvh"] * row_bytes(case["kind"], case["hd"])
    if case["op"] == "fork":
        rows = [counts(case)[i] for i in torch.randperm(case["n_par"], generator=host).tolist()]
        n_par, c = case["n_par"], case["children"]
        held = torch.tensor([pages_of(r, page) for r in rows])
        n_pages = int(held.sum()) + n_par * c + max(4, int(held.sum()) // 8)
        stride = int(held.max()) + 2
        pages = torch.randperm(n_pages, generator=g, **on).int()
        n_req = n_par * (1 + c)
        places = torch.randperm(n_req, generator=host)      # parents and children lie among one another
        par, kids = places[:n_par].sort().values, places[n_par:].view(n_par, c)
        dst, by = kids.flatten().sort()                     # in the order of the places: forks that are taken back leave the stack as it was
        table = torch.full((n_req, stride), -1, dtype=torch.int32, **on)
        has = torch.arange(stride)[None, :] < held[:, None]
        table[par.cuda()[:, None].expand(-1, stride)[has.cuda()], torch.arange(stride).expand(n_par, -1)[has].cuda()] = pages[: int(held.sum())]
        at = torch.zeros(n_req, dtype=torch.int32)
        at[par] = torch.tensor(rows, dtype=torch.int32)
        stay = torch.full((n_req,), 2**31 - 1, dtype=torch.int32)
        no_parent, no_child = stay.clone(), stay.clone()
        no_parent[par] = 0
        no_child[kids.flatten()] = 0
        mem = torch.empty(case["layers"], n_pages, per_page // 8, dtype=torch.int64, **on).random_(generator=g)
        length = ints(rows)
        return dict(case=case, mem=mem, table=table, rows=at.cuda(), free=torch.cat([pages[int(held.sum()):], pages[: int(held.sum())]]), n_free=ints([n_pages - int(held.sum())]),
                    shares=torch.zeros(3 * n_pages, dtype=torch.int32, **on), seen=torch.zeros(3 * n_pages, dtype=torch.int32, **on), n_pages=n_pages,
                    src=par.repeat_interleave(c)[by].int().cuda(), dst=dst.int().cuda(), length=length.repeat_interleave(c)[by.cuda()], back=kids[:, 0].int().cuda().contiguous(), par=par.int().cuda(),
                    par_length=length, no_parent=no_parent.cuda(), no_child=no_child.cuda(), most=max(rows))
    n_pages, (live, m) = case["n_pages"], moved(case)
    low, high = torch.randperm(live, generator=g, **on)[: live - m], live + torch.randperm(n_pages - live, generator=g, **on)[:m]
    used = torch.cat([low, high])[torch.randperm(live, generator=g, **on)].int()
    each, common = 40, 10
    own_pages = each - common
    n_req = max(1, live // (own_pages + common / case["shared"]).__ceil__())
    groups = -(-n_req // case["shared"])
    table = torch.full((n_req, each + 3), 2**30, dtype=torch.int32, **on)     # behind a request's rows lies anything
    shares = torch.zeros(3 * n_pages, dtype=torch.int32, **on)
    shared_pages = used[: groups * common].view(groups, -1) if groups * common <= live // 2 else used[:0].view(0, 0)
    rest = used[shared_pages.numel():]
    rows = torch.zeros(n_req, dtype=torch.int32)
    at, with_shared = 0, shared_pages.numel() > 0
    for r in range(n_req):      # what is left goes to the last one that has room
        n = min(own_pages, rest.numel() - at) if with_shared else min(each, rest.numel() - at)
        head = shared_pages[r // case["shared"]] if with_shared else used[:0]
        row = torch.cat([head, rest[at: at + n]])
        table[r, : row.numel()] = row
        at += n
        rows[r] = row.numel() * page - (r % page if n else 0)
    left = rest[at:]            # held by requests of one row of the table each
    if left.numel():
        extra = -(-left.numel() // each)
        more = torch.full((extra, each + 3), 2**30, dtype=torch.int32, **on)
        more[:, :each].view(extra, each)[torch.arange(extra * each, **on).view(extra, each) < left.numel()] = left
        table = torch.cat([table, more])
        rows = torch.cat([rows, torch.tensor([min(each, left.numel() - i * each) * page for i in range(extra)], dtype=torch.int32)])
    if with_shared:
        holders = torch.tensor([min(case["shared"], n_req - i * case["shared"]) for i in range(groups)], dtype=torch.int32, **on)
        shares[shared_pages.long()] = (holders - 1)[:, None].expand(-1, common).contiguous()
    is_used = torch.zeros(n_pages, dtype=torch.bool, **on)
    is_used[used.long()] = True
    empty = torch.nonzero(~is_used).flatten().int()
    free = torch.cat([empty[torch.randperm(empty.numel(), generator=g, **on)], used])   # a stack of n_free pages; what lies above it has no meaning
    mem = torch.empty(case["layers"], n_pages, per_page // 8, dtype=torch.int64, **on).random_(generator=g)
    s = dict(case=case, mem=mem, rows=rows.cuda(), table0=table, shares0=shares, free0=free, n_free=ints([empty.numel()]), live=live)
    return s | dict(table=table.clone(), shares=shares.clone(), free=free.clone(), map=torch.empty(n_pages, dtype=torch.int32, **on))


# ------------------------------------------------------------------------------------------- one pass
def package():
    at = os.path.join(os.getcwd(), "suzuqu-engine-4exp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import q4gpu
    q4gpu.init()
    q4gpu.use_torch_stream()
    return q4gpu


def pool(s):
    """the handle that a user's program keeps beside the pool's memory"""
    if "pool" not in s:
        q4gpu = package()
        c = s["case"]
        kind = {"q8_0": q4gpu.KIND_Q8, "f16": q4gpu.KIND_F16}[c["kind"]]
        stack = dict(free=s["free"], n_free=s["n_free"], shares=s["shares"]) if "free" in s else {}
        s["pool"] = q4gpu.PagePool(c.get("layers", 1), c["n_kvh"], c["hd"], s["mem"].shape[1], c["page"], kind, mem=s["mem"], **stack)
        if c["op"] == "prep":
            scaled = {} if c["scaling"] == "none" else dict(scaling=c["scaling"], factor=8.0, orig=ORIG)
            if c["scaling"] == "ramp":
                scaled |= dict(fast=32.0, slow=1.0, mag=s["mag"])
            elif c["scaling"] == "smooth":
                scaled |= dict(fast=4.0, slow=1.0)
            s["rope"] = q4gpu.Rope(c["n_rot"], 1e7 if c["hd"] == 256 else 1e6, half=c["half"], **scaled)
    return s["pool"]


def run(s):
    op = s["case"]["op"]
    if op == "prep":
        if own:
            p = pool(s)
            p.prep(0, s["q"], s["k"], s["v"], s["q_out"], s["pos"], s["slot"], s["rope"], wq=s["wq"], wk=s["wk"], eps=EPS, gate=s["gate"])
            if "k_out" in s:
                p.gather(0, s["slot"], s["k_out"], s["v_out"])
        else:
            plain_prep(s)
        if "k_out" in s:   # what the codes stand for; in a 16-bit pool the numbers as they lie there
            pages = (s["k_out"].half(), s["v_out"].half())
        else:
            pages = s["mem"].view(torch.float16)
        return {"q": s["q_out"], "gate": s["gate"], "pages": pages} if s["gate"] is not None else {"q": s["q_out"], "pages": pages}
    if op == "verify":
        if own:
            if "package" not in s:
                s["package"] = package()
            s["package"].verify(s["target"], s["token"], s["start"], s["u_accept"], s["u_draw"], s["accepted"], s["next"], draft=s["draft"], temp=s["temp"], logp=s["logp"],
                                rows=s["rows"], keep=s["keep"])
        else:
            plain_verify(s)
        return {k: s[k] for k in ("accepted", "next", "keep", "logp")}
    if op == "fork":
        if own:
            p = pool(s)
            p.fork(s["rows"], s["src"], s["dst"], s["length"], s["table"])
            s["seen"].copy_(s["shares"])
            p.release(s["rows"], s["no_parent"], s["table"])
            p.fork(s["rows"], s["back"], s["par"], s["par_length"], s["table"])
            p.release(s["rows"], s["no_child"], s["table"])
        else:
            plain_fork(s, s["src"], s["dst"], s["length"])
            s["seen"].copy_(s["shares"])
            plain_release(s, s["no_parent"])
            plain_fork(s, s["back"], s["par"], s["par_length"])
            plain_release(s, s["no_child"])
        return {k: s[k] for k in ("mem", "table", "rows", "free", "n_free", "shares", "seen")}
    # the pool as it was before it was compacted: its pages still lie there
    s["table"].copy_(s["table0"])
    s["shares"].copy_(s["shares0"])
    s["free"].copy_(s["free0"])
    if own:
        pool(s).compact(s["rows"], s["table"], s["map"])
    else:
        plain_compact(s)
    return {k: s[k] for k in ("mem", "table", "free", "n_free", "shares", "map")}


# ------------------------------------------------------------------------------------------- the plain forms
def swizzle(device):
    """[row][place] -> the 16-byte chunk that lies there; its own inverse"""
    return torch.arange(8, device=device)[None, :] ^ (torch.arange(16, device=device) & 7)[:, None]


def quantised(x):
    """q8_0: fp32 rows [..., hd] -> codes int8 [..., hd], scales fp16 [..., hd / 32]"""
    b = x.unflatten(-1, (-1, 32))
    d = b.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    return (b * inv).round().clamp(-127, 127).to(torch.int8).flatten(-2), d.squeeze(-1).to(torch.float16)


def turned(x, s, angle):
    """norm and rotation of heads [token][head][hd]; angle [token][pair]"""
    c = s["case"]
    n_rot = c["n_rot"]
    cos, sin = (s["mag"] * torch.cos(angle)).float()[:, None], (s["mag"] * torch.sin(angle)).float()[:, None]
    r, rest = x[..., :n_rot], x[..., n_rot:]
    a, b = (r[..., : n_rot // 2], r[..., n_rot // 2:]) if c["half"] else (r[..., 0::2], r[..., 1::2])
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.cat([u, v], -1) if c["half"] else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([r, rest], -1)


def plain_prep(s):
    c = s["case"]
    n, n_head, n_kvh, hd, page = c["n_tok"], c["n_head"], c["n_kvh"], c["hd"], c["page"]
    heads = lambda x, h: x[:n].float().unflatten(1, (h, -1))  # noqa: E731
    normed = lambda x, w: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    q, k, v = heads(s["q"], n_head), heads(s["k"], n_kvh), heads(s["v"], n_kvh)
    if s["gate"] is not None:
        s["gate"][:n] = q[..., hd:]
        q = q[..., :hd]
    angle = s["pos"][:n, None].double() * s["f"]
    s["q_out"][:n] = turned(normed(q, s["wq"]), s, angle).to(torch.bfloat16)
    k = turned(normed(k, s["wk"]), s, angle)
    slot = s["slot"][:n].long()
    at, row = slot // page, slot % page
    x = torch.stack([k, v], 2)                                         # [token, kv head, K or V, hd]
    if c["kind"] == "q8_0":
        codes, scales = quantised(x)
        rec = torch.cat([codes.flatten(-2).view(torch.uint8), scales.flatten(-2).view(torch.uint8)], -1)
        mem = s["mem"][0].view(s["mem"].shape[1], n_kvh, page, -1)
        mem[at, :, row, : rec.shape[-1]] = rec
        got = mem[at, :, row]
        codes = got[..., : 2 * hd].contiguous().view(torch.int8).float().unflatten(-1, (2, hd // 32, 32))
        scales = got[..., 2 * hd: 2 * hd + hd // 8].contiguous().view(torch.float16).float().unflatten(-1, (2, hd // 32, 1))
        kv = (codes * scales).flatten(-2)
        for name, i in (("k_out", 0), ("v_out", 1)):
            s[name].zero_()
            s[name][:n] = kv[:, :, i].flatten(1)
    else:
        # [page, kv head, tile, K or V, block, row, place, 8]
        mem = s["mem"][0].view(torch.float16).view(s["mem"].shape[1], n_kvh, page // 16, 2, hd // 64, 16, 8, 8)
        chunks = swizzle(slot.device)[row % 16][:, None, None, None, :, None].expand(-1, n_kvh, 2, hd // 64, 8, 8)
        mem[at, :, row // 16, :, :, row % 16] = x.to(torch.float16).unflatten(-1, (hd // 64, 8, 8)).gather(-2, chunks)


def probabilities(logits, temp):
    """softmax in 64 bits: borders between tokens are compared with"""
    z = logits.double() / temp[:, None]
    z = (z - z.amax(1, keepdim=True)).exp_()
    return z.div_(z.sum(1, keepdim=True))


def plain_verify(s):
    target, token, req, start = s["target"], s["token"].long(), s["req"], s["start"].long()
    n_tok, n_req, dev = s["n_tok"], start.numel() - 1, target.device
    greedy = s["temp"] == 0
    temp = torch.where(greedy, 1.0, s["temp"]).double()
    j = torch.arange(n_tok, device=dev) - start[req]                  # row of its request
    last = j == (start[1:] - start[:-1])[req] - 1
    drafted = torch.cat([token[1:], token[:1]])                       # the token that a row's draft is
    p = probabilities(target, temp[req])
    best = target.argmax(1)
    pd = p.gather(1, drafted[:, None])[:, 0]
    if s["draft"] is None:
        qd = torch.ones_like(pd)
    else:
        q = probabilities(s["draft"], temp[req])
        qd = q.gather(1, drafted[:, None])[:, 0]
    taken = torch.where(greedy[req], drafted == best, s["u_accept"].double() * qd < pd) & ~last
    # the first row of every request that keeps no draft
    stop = torch.full((n_req,), n_tok, device=dev).scatter_reduce_(0, req, torch.where(taken, n_tok, torch.arange(n_tok, device=dev)), "amin")
    refused = ~last[stop]
    w = p[stop]
    if s["draft"] is None:
        w.scatter_(1, drafted[stop][:, None], torch.where(refused, 0.0, w.gather(1, drafted[stop][:, None])[:, 0])[:, None])
    else:
        w = torch.where(refused[:, None], (w - q[stop]).clamp_(min=0), w)
    w = w.cumsum_(1)
    drawn = (w > s["u_draw"].double()[:, None] * w[:, -1:]).to(torch.int8).argmax(1)
    drawn = torch.where(greedy, best[stop], drawn)
    s["accepted"].copy_(stop - start[:-1])
    s["next"].copy_(drawn)
    s["keep"].copy_(s["rows"] + s["accepted"] + 1)
    chosen = torch.where(j == (stop - start[:-1])[req], drawn[req], drafted)
    logp = p.gather(1, chosen[:, None])[:, 0].log()
    s["logp"].copy_(torch.where(greedy[req] | (j > (stop - start[:-1])[req]), 0.0, logp))


def plain_fork(s, src, dst, length):
    page, table = s["case"]["page"], s["table"]
    src, dst, length = src.long(), dst.long(), length.long()
    col = torch.arange(table.shape[1], device=table.device)
    whole = col[None, :] < (length // page)[:, None]
    partial = length % page > 0
    # whole pages get another holder
    named = table[src]
    s["shares"].index_add_(0, torch.where(whole, named, 0).flatten().long(), whole.flatten().int())
    table[dst] = torch.where(whole, named, table[dst])
    # the pages that prefixes end in: the tiles of 16 rows that hold any of them
    n = partial.cumsum(0)
    new = s["free"][(s["n_free"] - n).clamp(min=0)]
    old = named.gather(1, (length // page).clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    tiles = (length % page + 15) // 16
    m = s["mem"].view(s["mem"].shape[0], s["mem"].shape[1], s["case"]["n_kvh"], page // 16, -1)
    here = torch.arange(page // 16, device=table.device)[None, :] < tiles[:, None]
    f, t = torch.nonzero(here, as_tuple=True)
    m[:, new[f].long(), :, t] = m[:, old[f].long(), :, t]
    at = torch.where(partial, length // page, table.shape[1] - 1)[:, None]
    table[dst] = torch.where(partial[:, None] & (col[None, :] == at), new[:, None], table[dst])
    s["n_free"] -= n[-1:].int()
    s["rows"][dst] = length.int()


def plain_release(s, keep):
    page, table = s["case"]["page"], s["table"]
    rows = s["rows"]
    first, last = (keep.clamp(min=0).long() + page - 1) // page, (rows.long() + page - 1) // page
    col = torch.arange(table.shape[1], device=table.device)
    given = (col[None, :] >= first[:, None]) & (col[None, :] < last[:, None])
    named = table[given].long()                                       # in the order of the requests
    times = torch.zeros(s["n_pages"], dtype=torch.int32, device=table.device).index_add_(0, named, torch.ones_like(named, dtype=torch.int32))
    order = torch.arange(named.numel(), device=table.device)
    final = torch.full((s["n_pages"],), -1, device=table.device).scatter_reduce_(0, named, order, "amax")
    shares = s["shares"][: s["n_pages"]]
    back = (final[named] == order) & (times[named] == shares[named] + 1)
    gone = named[back]
    n = gone.numel()
    shares -= times
    shares[gone] = 0
    s["free"][s["n_free"].long() + n - 1 - torch.arange(n, device=table.device)] = gone.int()
    s["n_free"] += n
    rows.copy_(torch.minimum(rows, keep.clamp(min=0)))


def plain_compact(s):
    n_pages, dev, live, page = s["case"]["n_pages"], s["table"].device, s["live"], s["case"]["page"]
    n_free = n_pages - live
    used = torch.ones(n_pages, dtype=torch.bool, device=dev)
    used[s["free"][:n_free].long()] = False
    number = torch.arange(n_pages, device=dev, dtype=torch.int32)
    low = number < live
    holes, move = torch.nonzero(low & ~used).flatten(), torch.nonzero(~low & used).flatten()
    new = torch.where(used, number, -1)
    new[move] = holes.int()
    s["map"].copy_(new)
    s["mem"][:, holes] = s["mem"][:, move]
    s["shares"][holes] = s["shares"][move]
    s["shares"][move] = 0
    col = torch.arange(s["table"].shape[1], device=dev)
    held = col[None, :] < ((s["rows"].long() + page - 1) // page)[:, None]
    s["table"].copy_(torch.where(held, new[torch.where(held, s["table"], 0).long()], s["table"]))
    s["free"][:n_free] = torch.arange(n_pages - 1, live - 1, -1, device=dev, dtype=torch.int32)


# ------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """From the definitions, in 64 bits: heads by head and pair by pair, requests one by one."""
    if case["op"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    if case["op"] == "verify":
        return exact_verify(s)
    n, hd, n_rot, page, n_kvh = case["n_tok"], case["hd"], case["n_rot"], case["page"], case["n_kvh"]
    f, mag = frequencies(case)
    pos = s["pos"][:n].double()

    def head(x, w):
        y = x.double()
        y = y / torch.sqrt((y**2).sum(1, keepdim=True) / hd + EPS) * w.double()
        z = y.clone()
        for i in range(n_rot // 2):
            a, b = (i, i + n_rot // 2) if case["half"] else (2 * i, 2 * i + 1)
            turn = torch.polar(torch.full_like(pos, mag), pos * f[i])
            t = torch.complex(y[:, a], y[:, b]) * turn
            z[:, a], z[:, b] = t.real, t.imag
        return z

    per = 2 * hd if case["gate"] else hd
    q = torch.zeros(s["q_out"].shape, dtype=torch.float64, device="cuda")
    for h in range(case["n_head"]):
        q[:n, h] = head(s["q"][:n, h * per: h * per + hd], s["wq"])
    res = {"q": q}
    if case["gate"]:
        g = torch.zeros_like(q)
        for h in range(case["n_head"]):
            g[:n, h] = s["q"][:n, h * per + hd: (h + 1) * per].double()
        res["gate"] = g
    k = torch.stack([head(s["k"][:n, h * hd: (h + 1) * hd], s["wk"]) for h in range(n_kvh)], 1)
    v = s["v"][:n].double().view(n, n_kvh, hd)
    if case["kind"] == "q8_0":
        both = []
        for x in (k, v):
            b = x.reshape(-1, 32)
            step = b.abs().max(1, keepdim=True).values / 127
            b = torch.round(b / step).nan_to_num(0.0) * step.half().double()
            whole = torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda")
            whole[:n] = b.view(n, -1)
            both.append(whole)
        return res | {"pages": tuple(both)}
    flat = torch.zeros(s["mem"].numel() // 2, dtype=torch.float64, device="cuda")
    slot = s["slot"][:n].long()
    tile, row = slot // 16, slot % 16
    tile = (tile // (page // 16) * n_kvh)[:, None] * (page // 16) + torch.arange(n_kvh, device="cuda") * (page // 16) + (tile % (page // 16))[:, None]
    d = torch.arange(hd, device="cuda")
    for i, x in enumerate((k, v)):
        place = (d // 64) * 1024 + row[:, None] * 64 + ((d % 64 // 8) ^ (row[:, None] & 7)) * 8 + d % 8
        flat[(tile[:, :, None] * 32 * hd + i * 16 * hd + place[:, None, :]).flatten()] = x.half().double().flatten()
    return res | {"pages": flat.view(s["mem"].view(torch.float16).shape)}


def exact_verify(s):
    start, temp, token = s["start"].tolist(), s["temp"].tolist(), s["token"].tolist()
    accepted, nexts, keep = [], [], []
    logp = torch.zeros(s["n_tok"], dtype=torch.float64, device="cuda")
    u_accept, u_draw, rows = s["u_accept"].tolist(), s["u_draw"].tolist(), s["rows"].tolist()
    for r, t in enumerate(temp):
        a, b = start[r], start[r + 1]
        at = a
        if t == 0.0:
            while True:
                x = s["target"][at].double()
                best = int(torch.nonzero(x == x.max())[0])
                if at + 1 == b or token[at + 1] != best:
                    break
                at += 1
            accepted.append(at - a)
            nexts.append(best)
        else:
            log_of = lambda x: x.double() / t - torch.logsumexp(x.double() / t, 0)  # noqa: E731
            while True:
                lp = log_of(s["target"][at])
                if at + 1 == b:
                    w = lp.exp()
                    break
                d = token[at + 1]
                lq = log_of(s["draft"][at]) if s["draft"] is not None else None
                if u_accept[at] * (math.exp(float(lq[d])) if lq is not None else 1.0) < math.exp(float(lp[d])):
                    logp[at] = lp[d]
                    at += 1
                    continue
                w = lp.exp()
                if lq is None:
                    w[d] = 0.0
                else:
                    w = torch.clamp(w - lq.exp(), min=0.0)
                break
            c = torch.cumsum(w, 0)
            n = int(torch.searchsorted(c, u_draw[r] * c[-1], right=True))
            logp[at] = lp[n]
            accepted.append(at - a)
            nexts.append(n)
        keep.append(rows[r] + at - a + 1)
    return {"accepted": torch.tensor(accepted), "next": torch.tensor(nexts), "keep": torch.tensor(keep), "logp": logp}
