"""What q4gpu.PagePool refuses on the host: tensors that are not on the pool's GPU, of another type, not dense, or too small for the call.
The library and the tensors are stand-ins, so that no address reaches a kernel whatever is let through."""
import pytest
import torch

import q4gpu

N_REQ, STRIDE, MAX_TOK, N_KVH, HD, N_HEAD, N_TOK, N_PAGES, PAGE = 3, 7, 40, 2, 64, 8, 11, 20, 16
SIZE = 1000


class Stub:
    """as much of a tensor as the mirror looks at"""

    def __init__(self, *shape, dtype=torch.int32, device=0, dense=True):
        self.shape, self.dtype, self.where, self.dense, self.is_cuda = shape, dtype, device, dense, device >= 0
        self.device = torch.device("cuda", device) if device >= 0 else torch.device("cpu")

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def stride(self):
        return (1,)

    def element_size(self):
        return 1 if self.dtype is torch.uint8 else 4

    def get_device(self):
        return self.where

    def is_contiguous(self):
        return self.dense

    def data_ptr(self):
        return 4096


class Library:
    def __init__(self):
        self.called = []

    def __getattr__(self, name):
        def call(*args):
            self.called.append(name)
            return True
        return {"q4_gpu_pages_bytes": lambda *args: SIZE, "q4_gpu_device": lambda: 0}.get(name, call)


@pytest.fixture
def library(monkeypatch):
    L = Library()
    monkeypatch.setattr(q4gpu, "init", lambda: L)
    return L


POOL = dict(mem=(SIZE, torch.uint8), free=(N_PAGES, torch.int32), n_free=(1, torch.int32))
F = torch.float32
CALLS = {   # tensors by name: shape, type
    "plan": dict(rows=((N_REQ,), torch.int32), add=((N_REQ,), torch.int32), table=((N_REQ, STRIDE), torch.int32), start=((N_REQ + 1,), torch.int32),
                 slot=((MAX_TOK,), torch.int32), pos=((MAX_TOK,), torch.int32), req=((MAX_TOK,), torch.int32)),
    "trim": dict(rows=((N_REQ,), torch.int32), keep=((N_REQ,), torch.int32), table=((N_REQ, STRIDE), torch.int32)),
    "append": dict(k=((N_TOK, N_KVH * HD), F), v=((N_TOK, N_KVH * HD), F), slot=((N_TOK,), torch.int32)),
    "gather": dict(slot=((N_TOK,), torch.int32), k=((N_TOK, N_KVH * HD), F), v=((N_TOK, N_KVH * HD), F)),
    "attend": dict(q=((N_TOK, N_HEAD, HD), torch.bfloat16), out=((N_TOK, N_HEAD, HD), F), rows=((N_REQ,), torch.int32), start=((N_REQ + 1,), torch.int32),
                   table=((N_REQ, STRIDE), torch.int32), gate=((N_TOK, N_HEAD, HD), F)),
}
SETS_THE_SIZE = {("plan", "table"), ("plan", "slot"), ("trim", "table"), ("append", "slot"), ("gather", "slot"), ("attend", "table")}   # a smaller one is a smaller call


def make_pool(**other):
    t = {name: Stub(n, dtype=d) for name, (n, d) in POOL.items()}
    t.update(other)
    return q4gpu.PagePool(1, N_KVH, HD, N_PAGES, PAGE, q4gpu.KIND_Q8, **t)


def call(pool, op, **other):
    t = {name: Stub(*shape, dtype=d) for name, (shape, d) in CALLS[op].items()}
    t.update(other)
    if op in ("append", "gather"):
        t["layer"] = 0
    if op == "attend":
        t.update(layer=0, n_head=N_HEAD, scale=0.1)
    getattr(pool, op)(**t)


@pytest.mark.parametrize("op", CALLS)
def test_right_tensors_are_taken(library, op):
    call(make_pool(), op)
    assert library.called == ["q4_gpu_pages_" + op]


@pytest.mark.parametrize("op,name", [(op, name) for op in CALLS for name in CALLS[op]])
@pytest.mark.parametrize("wrong", ["on the host", "on another GPU", "of another type", "not dense", "too small"])
def test_wrong_tensors_are_refused(library, op, name, wrong):
    shape, dtype = CALLS[op][name]
    if wrong == "too small":
        if (op, name) in SETS_THE_SIZE:
            pytest.skip("the call's size comes from it")
        bad = Stub(*(shape[:-1] + (shape[-1] - 1,)), dtype=dtype)
    elif wrong == "of another type":
        bad = Stub(*shape, dtype=torch.float64)
    else:
        bad = Stub(*shape, dtype=dtype, device=-1 if wrong == "on the host" else 1 if wrong == "on another GPU" else 0, dense=wrong != "not dense")
    pool = make_pool()
    with pytest.raises(RuntimeError):
        call(pool, op, **{name: bad})
    assert not library.called


@pytest.mark.parametrize("name", ["k", "v", "gate"])
def test_what_may_be_left_out(library, name):
    call(make_pool(), "attend" if name == "gate" else "gather", **{name: None})
    assert len(library.called) == 1


@pytest.mark.parametrize("name", POOL)
@pytest.mark.parametrize("wrong", ["on the host", "on another GPU", "of another type", "not dense", "too small", "missing"])
def test_wrong_memory_for_a_pool_is_refused(library, name, wrong):
    n, dtype = POOL[name]
    if name == "mem" and wrong in ("of another type", "missing"):
        pytest.skip("any type will do; a pool may be its stack alone")
    bad = None if wrong == "missing" else Stub(n - (wrong == "too small"), dtype=torch.float64 if wrong == "of another type" else dtype,
                                               device=-1 if wrong == "on the host" else 1 if wrong == "on another GPU" else 0, dense=wrong != "not dense")
    with pytest.raises(RuntimeError):
        make_pool(**{name: bad})


def test_heads_that_do_not_divide_the_queries(library):
    pool = make_pool()
    for n_head in (0, 3, -1):
        with pytest.raises(RuntimeError):
            pool.attend(0, *(Stub(*CALLS["attend"][x][0], dtype=CALLS["attend"][x][1]) for x in ("q", "out", "rows", "start", "table")), n_head, 0.1)
    assert not library.called
