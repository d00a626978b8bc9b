"""Captured tree calls of more than one launch group, in the layer form too."""
import ctypes as C

import numpy as np
import pytest

import trees
from kvl_mla import inputs, lib
from test_gpu_tree import KINDS, L, batch_device, hidden, models  # noqa: F401
from trees import Device, State, fn, ints, pointers, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [[4, 9], [64] * 4 + [30, 3], [1] * 70])
def test_captured_layer_replays(models, kind, sizes):  # noqa: F811
    cfg, layer, w = models("kimi")
    lens = [(37 * i) % 500 for i in range(len(sizes))]
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    n1, n2 = inputs.normal_bf16(1, "n1", (cfg.hidden_size,), 1.0, 0.1), inputs.normal_bf16(2, "n2", (cfg.hidden_size,), 1.0, 0.1)
    h = hidden(cfg, 0xD1, sum(sizes))
    dh, dn = Device(h), Device(h)
    u16 = lambda a: trees.abi.ptr(a, C.c_uint16)  # noqa: E731
    counts, parents, arr = ints(sizes), ints(sum(ps, [])), pointers(states)
    call = lambda: fn("attention_layer_%stree_device", kind)(dh.p, dn.p, counts, parents, len(sizes), C.byref(cfg), C.byref(w),  # noqa: E731
                                                            u16(n1), u16(n2), arr, lib.NO_ADVANCE)
    lib.check(call(), "eager")
    want = dh.get(), dn.get()
    lib.check(L.kvl_mla_capture_begin(), "capture")
    rc = call()
    g = C.c_void_p()
    lib.check(L.kvl_mla_capture_end(C.byref(g)), "capture end")
    lib.check(rc, "captured layer")
    for r in range(4):
        dh.put(h)
        dn.put(np.zeros_like(h))
        lib.check(L.kvl_mla_graph_launch(g), "replay")
        np.testing.assert_array_equal(dh.get(), want[0], err_msg=f"replay {r}")
        np.testing.assert_array_equal(dn.get(), want[1], err_msg=f"replay {r}")
        batch_device(kind, cfg, w, states, ps, hidden(cfg, r, sum(sizes)), lib.NO_ADVANCE)
        lib.check(L.kvl_mla_synchronize(), "sync")
    L.kvl_mla_graph_destroy(g)
    for b in (dh, dn):
        b.free()
    for s in states:
        s.free()
