"""Tree decodes at dims whose nope dim is larger than the latent rank (a head's projected query is then longer
than the row it is scored against), more nodes in a launch than a slice of them takes."""
import pytest

import trees
from kvl_mla import inputs
from test_gpu_tree import KINDS, batch_device, hidden
from trees import TOL, State, off, reference, tree

pytestmark = pytest.mark.gpu

SHORT = dict(trees.TINY, qk_nope_dim=12)                   # R 6, DN 12
WIDE = dict(trees.LAB, num_heads=3, qk_nope_dim=80)        # R 32, DN 80


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
