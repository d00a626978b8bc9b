"""How near the tree decodes come to 64 bits (trees.TOL is a bound of the worst case; these hold the kernels to
the error that their operands' bits make likely).

Errors here are norms of a node's output, relative. An fp32 operand as two bf16 parts is off by 2^-18.8 of itself,
root mean square: the hi part leaves a residual that is even over half a step, 2^-8, the lo part rounds that to 8
bits (rms over its binades 2^-18.2 for values in [1, 2), whose own rms is 1.5). Each element is off for itself, so a
product with such an operand is off by about that share in norm. On the way to the output lie the weights, the
heads' outputs and the rows where they are FP32: sqrt(3) * 2^-18.8 = 3.8e-6. On the way to the logits, whose root mean
square is 0.6 for the inputs drawn here, lie x, q_nope, the query and again FP32 rows: 2 * 0.6 * 2^-18.8 = 2.6e-6.
Together 4.6e-6 (BF16 and Q8 rows 3.9e-6); NEAR is twice that and a little."""
import numpy as np
import pytest

import trees
from kvl_mla import inputs, lib
from test_gpu_tree import batch_device, hidden, models  # noqa: F401
from trees import State, f64, fn, ints, pointers, reference, tree

pytestmark = pytest.mark.gpu

NEAR = 1e-5


def relative(got, want):
    """The largest relative error, in norm, of a node's output."""
    return float((np.linalg.norm(got.astype(np.float64) - want, axis=-1) / np.linalg.norm(want, axis=-1)).max())


def latent_queries(cfg, layer, x):
    """[count, heads, R]: the nodes' queries against latents, with the softmax scale."""
    NH, DN, DR, DV, R = cfg.num_heads, cfg.qk_nope_dim, cfg.qk_rope_dim, cfg.v_head_dim, cfg.kv_lora_rank
    q = (x.astype(np.float64) @ f64(layer.q_proj).T).reshape(-1, NH, DN + DR)
    kvb = f64(layer.kv_b_proj).reshape(NH, DN + DV, R)
    return np.stack([np.matmul(kvb[h, :DN].T, q[:, h, :DN].T).T for h in range(NH)], 1) / np.sqrt(DN + DR)


def put_rows(st, lat, key):
    """The state's rows become these, rounded to its format."""
    n, a = len(lat), st.arrays()
    lat, key = lat.astype(np.float32), key.astype(np.float32)
    if st.kind == "f32":
        a[0][:n], a[1][:n] = lat, key
    elif st.kind == "bf16":
        a[0][:n], a[1][:n] = inputs.f32_to_bf16_bits(lat), inputs.f32_to_bf16_bits(key)
    else:
        scale = (np.abs(lat).max(1) / np.float32(127)).astype(np.float32)
        a[0][:n] = np.clip(np.rint(lat / scale[:, None]), -127, 127).astype(np.int8)
        a[1][:n], a[2][:n] = scale, inputs.f32_to_bf16_bits(key)
    st.s.len = n
    lib.check(fn("compressed_%sstate_sync", st.kind)(st.ref()), "sync")
    return st


def first_row_weight(cfg, layer, x, st, ctx):
    """The softmax weight of row 0 in each head of a node that attends the history alone, keys left out."""
    lat = trees.values(st.rows(0, ctx), st.kind)[0]
    s = latent_queries(cfg, layer, x[None])[0] @ lat.T
    w = np.exp(s - s.max(1, keepdims=True))
    return w[:, 0] / w.sum(1)


@pytest.mark.parametrize("kind,ctx", [("f32", 32768), ("bf16", 32768), ("q8", 2048), ("q8", 32768), ("q8", 131072)])
def test_first_row_that_draws_much_of_the_weight(models, kind, ctx):  # noqa: F811
    """The usual history of a trained model: its first token draws more than half of the attention, and the latents
    share a mean, so that what is lost of the many small weights adds up. Eight trees of 32 nodes, so that a split
    holds a quarter of the history. NEAR, and as much again for the sums over a split: two additions per chunk of
    32 rows and eight of its rows at a time, each off by 2^-25 of the sum in the mean and not always up or down."""
    cfg, layer, w = models("kimi")
    n, batch = 32, 8
    rng = np.random.default_rng(ctx)
    base = 4 * hidden(cfg, 0xE1, 1)
    x = (base + 0.1 * rng.standard_normal((batch * n, cfg.hidden_size))).astype(np.float32)
    mean = 2 * rng.standard_normal(cfg.kv_lora_rank)
    lat = mean + 0.5 * rng.standard_normal((ctx, cfg.kv_lora_rank))
    key = 0.2 * rng.standard_normal((ctx, cfg.qk_rope_dim))
    q = latent_queries(cfg, layer, base)[0]
    rest = q @ (lat[1:] - mean).T
    target = np.log(1.5 * np.exp(rest).sum(1))
    lat[0] = mean + np.linalg.lstsq(q, target, rcond=None)[0]
    key[0] = 0
    states = [State(kind, cfg, ctx + n) for _ in range(batch)]
    put_rows(states[0], lat, key)
    del lat, rest
    lib.check(fn("compressed_%sstate_fork_batch_device", kind)(pointers(states[1:]), pointers(states[:1] * (batch - 1)), ints([0] * (batch - 1)),
                                                              ints([ctx] * (batch - 1)), batch - 1), "fork")
    share = first_row_weight(cfg, layer, x[1], states[0], ctx)
    assert share.min() > 0.3 and share.max() < 0.9, share
    p = tree("any", n, 1)
    got = batch_device(kind, cfg, w, states, [p] * batch, x).reshape(batch, n, -1)
    some = [1, n - 1] if ctx < 100000 else [1]
    for b in (0, batch - 1):
        rows = states[b].pull(0, ctx + n)
        e = relative(got[b][some], reference(cfg, layer, x[b * n:(b + 1) * n], p, ctx, rows, kind, some))
        print(f"[precision] {kind} {ctx} rows, tree {b}: {e:.2e}", flush=True)
        assert e <= 2 * NEAR, (b, e)
    for s in states:
        s.free()
