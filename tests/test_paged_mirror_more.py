"""What q4gpu refuses on the host in the calls around a step's attention (PagePool.prep, fork, release, compact and q4gpu.verify): tensors that are not on the library's
GPU, of another type, not dense, or too small for the call.  The library and the tensors are stand-ins, so that no address reaches a kernel whatever
is let through."""
import pytest
import torch

import q4gpu
from test_paged_mirror import HD, N_HEAD, N_KVH, N_PAGES, N_REQ, N_TOK, PAGE, SIZE, STRIDE, Library, Stub

F, I, B = torch.float32, torch.int32, torch.bfloat16
N_FORK, VOCAB = 2, 50
WIDTH = N_KVH * HD


class Rows(Stub):
    """rows whose stride may be larger than their width"""

    def __init__(self, *shape, dtype=F, device=0, dense=True, apart=None):
        super().__init__(*shape, dtype=dtype, device=device, dense=dense)
        self.apart = shape[-1] if apart is None else apart

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        s = [1] * len(self.shape)
        for k in range(len(self.shape) - 2, -1, -1):
            s[k] = s[k + 1] * self.shape[k + 1]
        if len(s) == 2:
            s[0] = self.apart
        if not self.dense:
            s[-1] = 2
        return s if i is None else s[i]


# tensors by name: shape, type, whether they may be rows of something wider
CALLS = {
    "prep": dict(q=((N_TOK, 2 * N_HEAD * HD), F, True), k=((N_TOK, WIDTH), F, True), v=((N_TOK, WIDTH), F, True), q_out=((N_TOK, N_HEAD, HD), B, False), pos=((N_TOK,), I, False),
                 slot=((N_TOK,), I, False), wq=((HD,), F, False), wk=((HD,), F, False), gate=((N_TOK, N_HEAD, HD), F, False)),
    "fork": dict(rows=((N_REQ,), I, False), src=((N_FORK,), I, False), dst=((N_FORK,), I, False), length=((N_FORK,), I, False), table=((N_REQ, STRIDE), I, False)),
    "release": dict(rows=((N_REQ,), I, False), keep=((N_REQ,), I, False), table=((N_REQ, STRIDE), I, False)),
    "compact": dict(rows=((N_REQ,), I, False), table=((N_REQ, STRIDE), I, False), number=((N_PAGES,), I, False)),
    "verify": dict(logits=((N_TOK, VOCAB), F, True), token=((N_TOK,), I, False), start=((N_REQ + 1,), I, False), u_accept=((N_TOK,), F, False), u_next=((N_REQ,), F, False),
                   accepted=((N_REQ,), I, False), next=((N_REQ,), I, False), draft=((N_TOK, VOCAB), F, True), temp=((N_REQ,), F, False), logp=((N_TOK,), F, False), rows=((N_REQ,), I, False),
                   keep=((N_REQ,), I, False)),
}
SETS_THE_SIZE = {("prep", "pos"), ("prep", "q_out"), ("fork", "src"), ("fork", "table"), ("release", "table"), ("compact", "table"), ("verify", "logits"), ("verify", "start")}
MAY_BE_NONE = {"prep": ("wq", "wk"), "compact": (), "verify": ("draft", "temp", "logp")}


@pytest.fixture
def library(monkeypatch):
    L = Library()
    monkeypatch.setattr(q4gpu, "init", lambda: L)
    monkeypatch.setattr(q4gpu, "load", lambda: L)
    return L


class NoRope:
    p = 4096


def make_pool(**other):
    t = dict(mem=Stub(SIZE, dtype=torch.uint8), free=Stub(N_PAGES), n_free=Stub(1), shares=Stub(3 * N_PAGES))
    t.update(other)
    return q4gpu.PagePool(1, N_KVH, HD, N_PAGES, PAGE, q4gpu.KIND_Q8, **t)


def call(pool, op, **other):
    t = {name: Rows(*shape, dtype=d) for name, (shape, d, _) in CALLS[op].items()}
    t.update(other)
    if op == "verify":
        q4gpu.verify(**t)
        return
    if op == "prep":
        t.update(layer=0, rope=NoRope())
    getattr(pool, op)(**t)


def name_of(op):
    return "q4_gpu_verify" if op == "verify" else "q4_gpu_pages_" + op


@pytest.mark.parametrize("op", CALLS)
def test_right_tensors_are_taken(library, op):
    call(make_pool(), op)
    assert library.called == [name_of(op)]


@pytest.mark.parametrize("op,name", [(op, n) for op in CALLS for n in CALLS[op] if CALLS[op][n][2]])
def test_rows_of_something_wider_are_taken(library, op, name):
    shape, dtype, _ = CALLS[op][name]
    both = ("k", "v") if name in ("k", "v") else (name,)
    call(make_pool(), op, **{n: Rows(*shape, dtype=dtype, apart=shape[1] + 24) for n in both})
    assert library.called == [name_of(op)]


@pytest.mark.parametrize("op,name", [(op, name) for op in CALLS for name in CALLS[op]])
@pytest.mark.parametrize("wrong", ["on the host", "on another GPU", "of another type", "not dense", "too small"])
def test_wrong_tensors_are_refused(library, op, name, wrong):
    shape, dtype, _ = CALLS[op][name]
    if wrong == "too small":
        if (op, name) in SETS_THE_SIZE:
            pytest.skip("the call's size comes from it")
        bad = Rows(*(shape[:-1] + (shape[-1] - 1,)), dtype=dtype)
    elif wrong == "of another type":
        bad = Rows(*shape, dtype=torch.float64)
    else:
        bad = Rows(*shape, dtype=dtype, device=-1 if wrong == "on the host" else 1 if wrong == "on another GPU" else 0, dense=wrong != "not dense")
    pool = make_pool()
    with pytest.raises(RuntimeError):
        call(pool, op, **{name: bad})
    assert not library.called


@pytest.mark.parametrize("op,name", [(op, n) for op, names in MAY_BE_NONE.items() for n in names])
def test_what_may_be_left_out(library, op, name):
    call(make_pool(), op, **{name: None})
    assert library.called == [name_of(op)]


def test_queries_without_gates_are_half_as_wide(library):
    call(make_pool(), "prep", gate=None, q=Rows(N_TOK, N_HEAD * HD))
    assert library.called == ["q4_gpu_pages_prep"]


def test_fewer_rows_than_tokens(library):
    pool = make_pool()
    for op, name in (("prep", "q"), ("prep", "k"), ("verify", "draft")):
        shape, dtype, _ = CALLS[op][name]
        with pytest.raises(RuntimeError):
            call(pool, op, **{name: Rows(shape[0] - 1, shape[1], dtype=dtype)})
    with pytest.raises(RuntimeError):
        call(pool, "prep", v=Rows(N_TOK, WIDTH, apart=WIDTH + 4))       # not at k's stride
    with pytest.raises(RuntimeError):
        call(pool, "prep", q_out=Rows(N_TOK, N_HEAD, HD // 2, dtype=B))
    with pytest.raises(RuntimeError):
        call(pool, "compact", rows=None)
    assert not library.called


def test_tables_may_be_the_host_s_to_rename(library):
    call(make_pool(), "compact", rows=None, table=None)
    assert library.called == ["q4_gpu_pages_compact"]


@pytest.mark.parametrize("wrong", ["on the host", "on another GPU", "of another type", "not dense", "too small"])
def test_wrong_counts_are_refused(library, wrong):
    bad = Stub(3 * N_PAGES - (wrong == "too small"), dtype=torch.float64 if wrong == "of another type" else I, device=-1 if wrong == "on the host" else 1 if wrong == "on another GPU" else 0,
               dense=wrong != "not dense")
    with pytest.raises(RuntimeError):
        make_pool(shares=bad)

