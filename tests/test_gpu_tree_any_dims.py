"""Tree decodes at dims whose nope dim is larger than the latent rank (a head's projected query is then longer
than the row it is scored against), more nodes in a launch than a slice of them takes."""
import numpy as np
import pytest

import trees
from kvl_mla import inputs
from test_gpu_tree import KINDS, batch_device, hidden
from trees import TOL, State, off, reference, tree

pytestmark = pytest.mark.gpu

SHORT = dict(trees.TINY, qk_nope_dim=12)                   # R 6, DN 12
WIDE = dict(trees.LAB, num_heads=3, qk_nope_dim=80)        # R 32, DN 80
DIMS = {
    "one": dict(trees.TINY, hidden_size=1, num_heads=1, qk_nope_dim=1, qk_rope_dim=2, v_head_dim=1, kv_lora_rank=1),
    "odd": dict(trees.TINY, hidden_size=9, num_heads=3, qk_nope_dim=3, qk_rope_dim=2, v_head_dim=5, kv_lora_rank=7),
    "largest": dict(trees.KIMI, hidden_size=256, num_heads=2, qk_nope_dim=512, qk_rope_dim=256, v_head_dim=64, kv_lora_rank=1024),
    "nope64": dict(trees.KIMI, qk_nope_dim=64),
    "nope200": dict(trees.KIMI, qk_nope_dim=200),
    "v64": dict(trees.KIMI, v_head_dim=64),
    "heads8": dict(trees.KIMI, num_heads=8),
    "rank256": dict(trees.KIMI, kv_lora_rank=256),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", [SHORT, WIDE], ids=["short", "wide"])
@pytest.mark.parametrize("lens,sizes", [([30, 70], [60, 50]), ([9, 0, 300, 64, 65], [64, 64, 64, 64, 9])])
def test_batch_at_more_nope_than_latent_columns(kind, dims, lens, sizes):
    cfg = inputs.config(**dims)
    layer = inputs.fast_layer(cfg, 0x7E)
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n + 1).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    x = hidden(cfg, 0x55, sum(sizes))
    got = batch_device(kind, cfg, layer.struct(), states, ps, x)
    at = 0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        e = off(got[at:at + n], reference(cfg, layer, x[at:at + n], ps[i], m, states[i].pull(0, m + n), kind))
        assert e <= TOL, (i, m, n, e)
        at += n
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("lens,sizes", [([40], [7]), ([0, 130], [12, 5]), ([70, 9], [64, 30])])
def test_batch_at_other_dims(kind, dims, lens, sizes):
    cfg = inputs.config(**DIMS[dims])
    layer = inputs.fast_layer(cfg, 0x7F)
    print(f"[dims] {kind} {dims} {lens} {sizes}", flush=True)
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n + 1).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    x = hidden(cfg, 0x56, sum(sizes))
    got = batch_device(kind, cfg, layer.struct(), states, ps, x)
    at = 0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        e = off(got[at:at + n], reference(cfg, layer, x[at:at + n], ps[i], m, states[i].pull(0, m + n), kind))
        assert e <= TOL, (i, m, n, e)
        at += n
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", [dict(trees.KIMI, num_heads=64), dict(trees.KIMI, hidden_size=4096)], ids=["heads64", "hidden4096"])
def test_batch_of_large_projections(kind, dims):
    """Projections of so many rows that their largest tiles are taken; the rows are a decode's of few nodes."""
    cfg = inputs.config(**dims)
    layer = inputs.fast_layer(cfg, 0x80)
    w = layer.struct()
    sizes, lens = [64, 64, 64, 63], [20, 50, 0, 33]
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    x = hidden(cfg, 0x57, sum(sizes))
    got = batch_device(kind, cfg, w, states, ps, x)
    at = 0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        rows = states[i].pull(0, m + n)
        some = [0, 1, n // 2, n - 1]
        e = off(got[at:at + n][some], reference(cfg, layer, x[at:at + n], ps[i], m, rows, kind, some))
        assert e <= TOL, (i, m, n, e)
        few = State(kind, cfg, m + 8).load(i, m)
        batch_device(kind, cfg, w, [few], [ps[i][:8]], x[at:at + 8])
        for a, b in zip(few.pull(m, m + 8), rows):
            np.testing.assert_array_equal(a, b[m:m + 8])
        few.free()
        at += n
    for s in states:
        s.free()
