"""A launch that fails in the middle of a batched call on branching histories: the states of the launches before it
are done and say so in len, the others are as they were. Runs without a GPU, the HIP runtime's device calls
replaced by host memory and launches that do nothing (fake_hip.cpp)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

CHILD = r'''
import ctypes as C, sys
sys.path[:0] = [{here!r}, {root!r}, {pkg!r}]
import numpy as np
import trees
from kvl_mla import inputs, lib
from trees import State, fn, ints, pointers

kind, what = sys.argv[1:]
fake = C.CDLL({fake!r})
cfg = inputs.config(**trees.TINY)

if what == "fork":
    src = State(kind, cfg, 40).load(1, 30)
    dsts = [State(kind, cfg, 40).load(2 + i, 9) for i in range(50)]
    row0, row1 = [i % 8 for i in range(50)], [10 + i % 20 for i in range(50)]
    call = lambda: fn("compressed_%sstate_fork_batch_device", kind)(pointers(dsts), pointers([src] * 50), ints(row0), ints(row1), 50)
    states, first, before, after = dsts, 48, [9] * 50, row1
elif what == "accept":
    states = [State(kind, cfg, 40).load(i, 30) for i in range(40)]
    call = lambda: fn("compressed_%sstate_accept_batch_device", kind)(pointers(states), ints([20] * 40), ints([2] * 40), ints([1, 3] * 40), 40)
    first, before, after = 32, [30] * 40, [22] * 40
else:
    layer = inputs.make_layer(cfg, 3)
    w = layer.struct()
    states = [State(kind, cfg, 40).load(i, 10) for i in range(70)]
    p = C.c_void_p(C.addressof((C.c_float * 65536)()))
    tree = lambda n, flags: fn("decode_compressed_%stree_batch_device", kind)(p, p, ints([2] * n), ints([-1, 0] * n), n, C.byref(cfg), C.byref(w),
                                                                            pointers(states[:n]), flags)
    call = lambda: tree(70, 0)
    first, before, after = 64, [10] * 70, [12] * 70
    lib.check(tree(64, lib.NO_ADVANCE), "warm")
    group = fake.fake_hip_launches()
    lib.check(tree(64, lib.NO_ADVANCE), "count")
    group = fake.fake_hip_launches() - group

lens = lambda: [s.s.len for s in states]
fake.fake_hip_fail_at(1)
assert call() == -1 and "launch" in lib.last_error(), lib.last_error()
assert lens() == before, lens()
fake.fake_hip_fail_at(2 if what != "tree" else group + 1)
assert call() == -1
assert lens() == after[:first] + before[first:], lens()
if what != "tree":
    for s, n in zip(states, before):
        s.s.len = n
fake.fake_hip_fail_at(0)
lib.check(call(), "call")
assert all(a > b for a, b in zip(lens(), before)) if what == "tree" else lens() == after
print("ok")
'''


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake") / "libfake_hip.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-I/opt/rocm/include", os.path.join(HERE, "fake_hip.cpp"), "-o", so], check=True)
    return so


@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("what", ["fork", "accept", "tree"])
def test_states_after_a_failed_launch(fake, kind, what):
    root = os.path.dirname(HERE)
    code = CHILD.format(here=HERE, root=root, pkg=os.path.join(root, "in-c-test_amd"), fake=fake)
    env = dict(os.environ, LD_PRELOAD=":".join([fake] + os.environ.get("LD_PRELOAD", "").split(":")).rstrip(":"))
    r = subprocess.run([sys.executable, "-c", code, kind, what], env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
