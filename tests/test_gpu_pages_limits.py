"""The paged KV cache (q4_gpu_pages_*) at its limits: tables whose entries are no pages, statuses, places without tokens, scratch that is
not to be had."""
import pytest
import torch

import q4gpu
from gpu_util import lib
from test_gpu_pages import KINDS, Step, attend_exact, ints, plan_plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [-1, -2**31, "n_pages", 2**31 - 1])
@pytest.mark.parametrize("rows,keep,at", [([70, 33], [0, 0], (1, 2)), ([70, 33], [17, 40], (0, 4)), ([16 * 300] + [5] * 2000, [0] * 2001, (0, 299)),
                                          ([16 * 300] + [5] * 2000, [0] * 2001, (2000, 0))])
def test_trim_refuses_entries_that_are_no_pages(rows, keep, at, bad):
    """nothing goes back, whatever the other entries are; a plan behind it gets pages of the pool only"""
    s = Step(rows, [0] * len(rows))
    bad = s.pool.n_pages if bad == "n_pages" else bad
    free = s.free_now()
    L = lib()
    L.q4_gpu_last_error()
    table = s.d_table.clone()
    table[at] = bad
    s.pool.trim(s.d_rows, ints(keep), table)
    assert L.q4_gpu_last_error() == 4
    assert s.free_now() == free
    s.pool.trim(s.d_rows, ints(keep), s.d_table)          # the right table: all of them, and each once
    assert L.q4_gpu_last_error() == 0
    held = sum(-(-max(k, 0) // 16) if k < h else -(-h // 16) for h, k in zip(rows, keep))
    now = s.free_now()
    assert len(now) == s.pool.n_pages - held and len(set(now)) == len(now) and min(now) >= 0 and max(now) < s.pool.n_pages


def test_trim_does_not_look_at_entries_that_stay():
    s = Step([70, 33], [0, 0])
    table = s.d_table.clone()
    table[0, 0], table[1, 2] = -1, -1                     # page 0 of the first is kept, as all of the second's are
    lib().q4_gpu_last_error()
    s.pool.trim(s.d_rows, ints([5, 33]), table)
    assert lib().q4_gpu_last_error() == 0
    assert s.free_now() == s.free + s.table[0][1:5][::-1]


def test_tensors_on_the_host_and_ones_too_small_reach_no_kernel():
    s = Step([5, 6], [1, 1], n_kvh=2, hd=128).plan()
    p, before = s.pool, s.free_now()
    q = torch.zeros(2, 16, 128, device="cuda")
    k = torch.zeros(2, 256, device="cuda")
    calls = [lambda: p.plan(s.d_rows.cpu(), s.d_add, s.d_table, s.start, s.slot, s.pos, s.req), lambda: p.plan(s.d_rows, s.d_add, s.d_table, s.start[:2], s.slot, s.pos, s.req),
             lambda: p.plan(s.d_rows, s.d_add[:1], s.d_table, s.start, s.slot, s.pos, s.req), lambda: p.plan(s.d_rows, s.d_add, s.d_table, s.start, s.slot, s.pos[:3], s.req),
             lambda: p.trim(s.d_rows, s.d_rows[:1], s.d_table), lambda: p.append(0, k[:1], k, s.slot[:2]), lambda: p.append(0, k, k.cpu(), s.slot[:2]),
             lambda: p.gather(0, s.slot[:2], k, k[:1]), lambda: p.attend(0, q, q[:1].clone(), s.d_rows, s.start, s.d_table, 16, 0.1),
             lambda: p.attend(0, q, q.clone(), s.d_rows, s.start, s.d_table.cpu(), 16, 0.1), lambda: p.attend(0, q, q.clone(), s.d_rows, s.start, s.d_table, 16, 0.1, gate=q[:1]),
             lambda: p.attend(0, q, q.clone(), s.d_rows, s.start, s.d_table, 0, 0.1),
             lambda: q4gpu.PagePool(1, 2, 128, p.n_pages, 16, q4gpu.KIND_Q8, mem=p.mem, free=p.free[:2], n_free=p.n_free),
             lambda: q4gpu.PagePool(1, 2, 128, p.n_pages, 16, q4gpu.KIND_Q8, mem=p.mem.cpu())]
    for i, call in enumerate(calls):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("call %d was taken" % i)
    assert lib().q4_gpu_last_error() == 0 and s.free_now() == before


@pytest.mark.parametrize("rows,add,kw", [([0], [1], dict(n_pages=1, max_tok=1)), ([0], [17], dict(n_pages=1)), ([5], [12], dict(max_tok=12)), ([5], [12], dict(max_tok=11)),
                                         ([-3], [1], {}), ([60], [5], dict(stride=4)), ([60], [4], dict(stride=4))])
def test_status_of_a_plan_of_one_request(rows, add, kw):
    s = Step(rows, add, **kw)
    want = plan_plain(rows, add, s.table, s.free, s.page, s.max_tok)
    L = lib()
    L.q4_gpu_last_error()
    s.plan()
    assert L.q4_gpu_last_error() == want[6]
    assert (s.d_table.tolist(), s.free_now(), s.start.tolist(), s.slot.tolist()) == (want[0], want[1], want[2], want[3])


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("idle", [40, 1000, 3000])
@pytest.mark.parametrize("add", [[1, 1, 1], [1, 90, 3], [200, 1, 70]])
def test_many_places_without_tokens(kind, idle, add):
    """requests that bring tokens far apart among places that bring none, held rows or not"""
    n_head, n_kvh, hd, page = 16, 2, 128, 16
    n, at = 2 * idle + 3, [0, idle + 1, 2 * idle + 2]
    rows, adds = [(r % 3) * 8 for r in range(n)], [0] * n
    for r, h, a in zip(at, (700, 0, 333), add):
        rows[r], adds[r] = h, a
    s = Step(rows, adds, page, n_kvh=n_kvh, hd=hd, kind=KINDS[kind])
    g = torch.Generator(device="cuda").manual_seed(idle)
    slot = [s.table[r][p // page] * page + p % page for r in at for p in range(rows[r])]
    k, v = torch.randn(2, len(slot), n_kvh * hd, generator=g, device="cuda")
    s.pool.append(0, k, v, ints(slot))
    s.plan()
    total = sum(add)
    k, v = torch.randn(2, total, n_kvh * hd, generator=g, device="cuda")
    s.pool.append(0, k, v, s.slot[:total])
    q = torch.randn(total, n_head, hd, generator=g, device="cuda").to(torch.bfloat16)
    out = torch.empty(total, n_head, hd, device="cuda")
    s.pool.attend(0, q, out, s.d_rows, s.start, s.d_table, n_head, float(hd ** -0.5))
    assert lib().q4_gpu_last_error() == 0
    first = 0
    for r, m in zip(at, add):
        table = s.d_table[r].tolist()
        kr, vr = torch.empty(2, rows[r] + m, n_kvh * hd, device="cuda")
        s.pool.gather(0, ints([table[p // page] * page + p % page for p in range(rows[r] + m)]), kr, vr)
        want = attend_exact(q[first: first + m], kr.view(-1, n_kvh, hd), vr.view(-1, n_kvh, hd), None, rows[r], float(hd ** -0.5))
        assert ((out[first: first + m].double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()
        first += m


def test_many_tokens_over_q8_0_without_scratch_for_their_copy():
    """a capture for which only a short chunk's scratch is there: the pages are read as they are"""
    L = lib()
    L.q4_gpu_set_stream(None)
    L.q4_hip_shutdown()                                   # gives back what other tests made it reserve
    L = q4gpu.init()
    n_head, n_kvh, hd, page, held, n = 16, 2, 128, 16, 77, 1300
    scale = float(hd ** -0.5)
    try:
        with torch.cuda.stream(torch.cuda.ExternalStream(L.q4_gpu_stream())):
            pool = q4gpu.PagePool(1, n_kvh, hd, 200, page, q4gpu.KIND_Q8)
            table = torch.full((1, 16384), -1, dtype=torch.int32, device="cuda")     # a context of 262 144
            start, maps = ints([0, 0]), [torch.empty(held + n, dtype=torch.int32, device="cuda") for _ in range(3)]
            k, v = torch.randn(2, held + n, n_kvh * hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
            q = torch.randn(held + n, n_head, hd, device="cuda").to(torch.bfloat16)
            out = torch.empty(held + n, n_head, hd, device="cuda")
            pool.plan(ints([0]), ints([held]), table, start, *maps)
            pool.append(0, k[:held], v[:held], maps[0][:held])
            pool.attend(0, q[:held], out[:held], ints([0]), start, table, n_head, scale, max_add=held)
            rows, add = ints([held]), ints([n])
            torch.cuda.synchronize()
            assert L.q4_hip_graph_begin()
            pool.plan(rows, add, table, start, *maps)
            pool.append(0, k[held:], v[held:], maps[0][:n])
            pool.attend(0, q[held:], out[held:], rows, start, table, n_head, scale, max_add=n)
            graph = L.q4_hip_graph_end()
            assert graph and L.q4_gpu_last_error() == 0
            assert L.q4_hip_graph_launch(graph)
            captured = out[held:].clone()
            pool.attend(0, q[held:], out[held:], rows, start, table, n_head, scale, max_add=n)   # outside: by the copy
            p = torch.arange(held + n, device="cuda")
            kr, vr = torch.empty(2, held + n, n_kvh * hd, device="cuda")
            pool.gather(0, (table[0].long()[p // page] * page + p % page).int(), kr, vr)
            want = attend_exact(q[held:], kr.view(-1, n_kvh, hd), vr.view(-1, n_kvh, hd), None, held, scale)
            for got in (captured, out[held:]):
                assert ((got.double() - want).abs() <= 2e-3 + 1e-3 * want.abs()).all()
            L.q4_hip_graph_free(graph)
    finally:
        lib()
    assert L.q4_gpu_last_error() == 0
