"""Arguments that the calls on branching histories refuse, before they touch a device: -1, a reason,
and states and outputs as they were. Runs without a GPU."""
import ctypes as C

import numpy as np
import pytest

import trees
from kvl_mla import inputs, lib
from trees import State, f32p, fn, ints

L = lib.load()
KINDS = ["f32", "bf16", "q8"]


def refused(rc, *words):
    assert rc == -1
    why = lib.last_error()
    assert why and all(w in why for w in words), why


def state(kind, cap, n, dims=trees.LAB):
    st = State(kind, inputs.config(**dims), cap)
    st.s.len = n
    return st


@pytest.fixture(scope="module")
def model():
    cfg = inputs.config(**trees.LAB)
    return cfg, inputs.make_layer(cfg, 0x71)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_arguments(kind, model):
    cfg, layer = model
    w, st = layer.struct(), state(kind, 70, 4)
    call = fn("decode_compressed_%stree_bf16", kind)
    x = np.ones((65, cfg.hidden_size), np.float32)
    out = np.full_like(x, 3.0)

    def go(parents, count=None, start=4, o=out, i=x, c=cfg, ww=w, s=st):
        return call(f32p(o) if o is not None else None, f32p(i) if i is not None else None,
                    ints(parents) if parents is not None else None, len(parents or []) if count is None else count, start,
                    C.byref(c) if c is not None else None, C.byref(ww) if ww is not None else None, s.ref() if s else None)

    refused(go([-1, 1]), "parent")        # its own parent
    refused(go([-1, 2, 1]), "parent")     # a later node
    refused(go([0]), "parent")
    refused(go([-1, -2]), "parent")
    refused(go([-1] * 65), "64")
    refused(go([], 0), "64")
    refused(go([-1], -3), "64")
    refused(go([-1], start=3), "invalid")
    refused(go(None, 1), "invalid")
    refused(go([-1], o=None), "invalid")
    refused(go([-1], i=None), "invalid")
    refused(go([-1], c=None), "invalid")
    refused(go([-1], ww=None), "invalid")
    refused(go([-1], s=None), "invalid")
    st.s.len = 68
    refused(go([-1, -1, -1], start=68), "capacity")
    st.s.len = 4
    other = inputs.config(**dict(trees.LAB, kv_lora_rank=16))
    refused(go([-1], c=other), "dims")
    bad = layer.struct()
    bad.o_proj = None
    refused(go([-1], ww=bad), "invalid")
    assert st.s.len == 4 and np.all(out == 3.0)
    st.free()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_batch_arguments(kind, model):
    cfg, layer = model
    w, a, b = layer.struct(), state(kind, 20, 4), state(kind, 20, 19)
    call = fn("decode_compressed_%stree_batch_device", kind)
    arr, same = trees.pointers([a, b]), trees.pointers([a, a])
    d = C.c_void_p(4096)  # never read: every call below ends in its checks

    def go(counts, parents, batch=2, states=arr, flags=0, o=d):
        return call(o, d, ints(counts) if counts is not None else None, ints(parents) if parents is not None else None, batch,
                    C.byref(cfg), C.byref(w), states, flags)

    refused(go([1, 2], [-1, -1, -1]), "sequence 1", "capacity")
    refused(go([2, 1], [-1, 1, -1]), "sequence 0", "parent")
    refused(go([1, 0], [-1]), "sequence 1")
    refused(go([1, 1], [-1, -1], states=same), "twice")
    refused(go([1, 1], [-1, -1], flags=4), "flags")
    refused(go([1, 1], [-1, -1], batch=0), "invalid")
    refused(go(None, [-1, -1]), "invalid")
    refused(go([1, 1], None), "invalid")
    refused(go([1, 1], [-1, -1], states=None), "invalid")
    refused(go([1, 1], [-1, -1], o=None), "invalid")
    n1 = np.zeros(cfg.hidden_size, np.uint16)
    layer_call = fn("attention_layer_%stree_device", kind)
    args = (ints([1, 1]), ints([-1, -1]), 2, C.byref(cfg), C.byref(w), trees.abi.ptr(n1, C.c_uint16), trees.abi.ptr(n1, C.c_uint16))
    e = C.c_void_p(8192)
    refused(layer_call(d, d, *args, arr, 0), "invalid")          # n2 on h
    refused(layer_call(d, e, *args, arr, lib.RESIDUAL), "flags")
    refused(layer_call(d, e, *args, same, 0), "twice")
    refused(layer_call(d, e, *args[:5], None, args[6], arr, 0), "invalid")
    assert a.s.len == 4 and b.s.len == 19
    for s in (a, b):
        s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_fork_arguments(kind):
    a, b, small = state(kind, 20, 12), state(kind, 30, 5), state(kind, 8, 0)
    odd = state(kind, 20, 12, dict(trees.LAB, kv_lora_rank=16))
    one = fn("compressed_%sstate_fork", kind)
    refused(one(b.ref(), a.ref(), 0, 13), "rows")        # beyond the source
    refused(one(b.ref(), a.ref(), 6, 10), "rows")        # a gap behind the destination's rows
    refused(one(b.ref(), a.ref(), 4, 3), "rows")
    refused(one(b.ref(), a.ref(), -1, 3), "rows")
    refused(one(small.ref(), a.ref(), 0, 9), "rows")     # beyond the destination's capacity
    refused(one(a.ref(), a.ref(), 0, 3), "destination")
    refused(one(odd.ref(), a.ref(), 0, 3), "dims")
    refused(one(None, a.ref(), 0, 3), "pair 0")
    batch = fn("compressed_%sstate_fork_batch_device", kind)
    P = trees.pointers
    refused(batch(P([b, b]), P([a, a]), ints([0, 0]), ints([3, 3]), 2), "twice")
    refused(batch(P([b, small]), P([a, b]), ints([0, 0]), ints([3, 3]), 2), "destination")
    refused(batch(P([b, odd]), P([a, odd]), ints([0, 0]), ints([3, 3]), 2), "dims")
    refused(batch(P([b]), P([a]), ints([0]), ints([3]), 0), "invalid")
    refused(batch(P([b]), P([a]), None, ints([3]), 1), "invalid")
    assert (a.s.len, b.s.len, small.s.len, odd.s.len) == (12, 5, 0, 12)
    for s in (a, b, small, odd):
        s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_accept_arguments(kind):
    a, b = state(kind, 200, 100), state(kind, 20, 6)
    one = fn("compressed_%sstate_accept", kind)
    refused(one(a.ref(), 95, ints([0, 5]), 2), "path")    # node 5 of a tree of 5 rows
    refused(one(a.ref(), 10, ints([0, 64]), 2), "path")   # beyond the nodes of a tree
    refused(one(a.ref(), 95, ints([1, 1]), 2), "path")
    refused(one(a.ref(), 95, ints([2, 1]), 2), "path")
    refused(one(a.ref(), 95, ints([-1]), 1), "path")
    refused(one(a.ref(), 101, ints([0]), 1), "accepted")
    refused(one(a.ref(), -1, ints([0]), 1), "accepted")
    refused(one(a.ref(), 10, ints(list(range(65))), 65), "accepted")
    refused(one(a.ref(), 10, ints([0]), -1), "accepted")
    refused(one(a.ref(), 10, None, 1), "accepted")
    refused(one(None, 0, ints([0]), 1), "state 0")
    batch = fn("compressed_%sstate_accept_batch_device", kind)
    P = trees.pointers
    refused(batch(P([a, a]), ints([95, 95]), ints([1, 1]), ints([0, 0]), 2), "twice")
    refused(batch(P([a, b]), ints([95, 4]), ints([1, 1]), ints([0, 2]), 2), "state 1", "path")
    refused(batch(P([a]), ints([95]), ints([1]), ints([0]), 0), "invalid")
    refused(batch(None, ints([95]), ints([1]), ints([0]), 1), "invalid")
    assert (a.s.len, b.s.len) == (100, 6)
    for s in (a, b):
        s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_device_rows_arguments(kind):
    a = state(kind, 20, 12)
    call = fn("compressed_%sstate_device_rows", kind)
    p = [C.c_void_p() for _ in range(3 if kind == "q8" else 2)]
    refs = [C.byref(q) for q in p]
    refused(call(None, *refs), "invalid")
    for k in range(len(p)):
        refused(call(a.ref(), *[None if i == k else r for i, r in enumerate(refs)]), "invalid")
    a.free()
