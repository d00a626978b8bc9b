"""How near the tree decodes come to 64 bits: trees.TOL is a bound of the worst case, these hold the outputs to
the error that their operands' bits make likely, and the stored rows to their definition.

Errors here are norms of a node's output, relative. An fp32 operand as two bf16 parts is off by 2^-18.8 of itself,
root mean square: the hi part leaves a residual that is even over half a step, 2^-8, the lo part rounds that to 8
bits (rms over its binades 2^-18.2 for values in [1, 2), whose own rms is 1.5). Each element is off for itself, so a
product with such an operand is off by about that share in norm. On the way to the output lie the weights, the
heads' outputs and the rows where they are FP32: sqrt(3) * 2^-18.8 = 3.8e-6. On the way to the logits, whose root mean
square is 0.6 for the inputs drawn here, lie x, q_nope, the query and again FP32 rows: 2 * 0.6 * 2^-18.8 = 2.6e-6.
Together 4.6e-6 (BF16 and Q8 rows 3.9e-6); NEAR is twice that and a little."""
import ctypes as C

import numpy as np
import pytest

import trees
from kvl_mla import inputs, lib
from test_gpu_tree import KINDS, L, batch_device, hidden, models  # noqa: F401
from trees import ONE, State, f32p, f64, fn, ints, pointers, reference, tree, tree_host

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


def rope_scores(cfg, layer, x, keys, pos):
    """[count, heads]: what the rotated query of each node, at one position, scores against its own key."""
    NH, DN, DR = cfg.num_heads, cfg.qk_nope_dim, cfg.qk_rope_dim
    q = (x.astype(np.float64) @ f64(layer.q_proj).T).reshape(-1, NH, DN + DR)
    a = pos * cfg.rope_theta ** (-2.0 * np.arange(DR // 2) / DR)
    e, o = q[..., DN::2], q[..., DN + 1::2]
    qr = np.concatenate([e * np.cos(a) - o * np.sin(a), o * np.cos(a) + e * np.sin(a)], -1)
    return (qr * keys[:, None]).sum(-1) / np.sqrt(DN + DR)


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
    32 rows and eight of its rows at a time, each off by 2^-25 of the sum in the mean and not always up or down.
    A rope_theta of its own past 65536 rows: the table of the usual one grows with the positions, and other tests
    count on positions that it does not reach."""
    cfg, layer, w = models("kimi")
    if ctx > 65536:
        cfg = inputs.config(**dict(trees.KIMI, rope_theta=30000.0))
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


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,sizes", [([400], [7]), ([0, 33, 1000], [1, 5, 12]), ([5000, 64, 700], [64, 30, 20]),
                                        ([90 + 77 * i for i in range(13)], [1] * 13)])
def test_outputs_near_64_bits(models, kind, lens, sizes):  # noqa: F811
    cfg, layer, w = models("kimi")
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    x = hidden(cfg, 0xE2, sum(sizes))
    got = batch_device(kind, cfg, w, states, ps, x)
    at, worst = 0, 0.0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        want = reference(cfg, layer, x[at:at + n], ps[i], m, states[i].pull(0, m + n), kind)
        worst = max(worst, relative(got[at:at + n], want))
        at += n
    print(f"[precision] {kind} {lens} {sizes}: {worst:.2e}", flush=True)
    assert worst <= NEAR
    for s in states:
        s.free()


def row_bounds(cfg, layer, x, parents, ctx):
    """trees.new_rows and how far its latents and keys may be off before they are stored. A projection's element is
    off by at most 2^-17 of the sum of its terms' sizes (x as two bf16 parts), and by 2^-24 of it for each of the
    fp32 additions in a row (H / 64 in a lane, then at most 24); a latent by that through its factors, and through
    its row's norm by the row's weighted mean of such errors; a key by its pair's, both to first order, with the
    few fp32 roundings on the way."""
    R, DR = cfg.kv_lora_rank, cfg.qk_rope_dim
    lat, key = trees.new_rows(cfg, layer, x, parents, ctx)
    wa, g = f64(layer.kv_a_proj), np.abs(f64(layer.kv_a_norm))
    y = x.astype(np.float64) @ wa.T
    dy = (2.0 ** -17 + (cfg.hidden_size / 64 + 24) * 2.0 ** -24) * (np.abs(x).astype(np.float64) @ np.abs(wa).T)
    yl, dl = np.abs(y[:, :R]), dy[:, :R]
    inv = 1 / np.sqrt((yl * yl).mean(1, keepdims=True) + cfg.rms_eps)
    drms = (yl * dl).mean(1, keepdims=True) * inv * inv
    blat = 1.01 * g * inv * (dl + yl * (drms + 2.0 ** -21))
    e, o = np.abs(y[:, R::2]), np.abs(y[:, R + 1::2])
    bkey = 1.01 * (dy[:, R::2] + dy[:, R + 1::2] + 2.0 ** -22 * (e + o))
    return lat, key, blat, np.concatenate([bkey, bkey], 1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["tiny", "lab", "nine", "kimi"])
@pytest.mark.parametrize("ctx,n", [(0, 3), (77, 8), (77, 40), (9999, 20)])
def test_rows_equal_their_definition(models, kind, dims, ctx, n):  # noqa: F811
    """The stored rows against RMSNorm and the rotation at position ctx + depth in 64 bits, not against another
    decode's. Rounding to the format: half a step, for Q8 of the row's scale."""
    cfg, layer, w = models(dims)
    p, x = tree("any", n, ctx + n), hidden(cfg, 0xE3 + n, n)
    st = State(kind, cfg, ctx + n).load(1, ctx)
    tree_host(st, layer, x, p, w)
    rows = st.rows(ctx, ctx + n)
    got = trees.values(rows, kind)
    lat, key, blat, bkey = row_bounds(cfg, layer, x, p, ctx)
    half = 2.0 ** -24 if kind == "f32" else 2.0 ** -8
    bkey = bkey * (1 + half) + half * np.abs(key)
    if kind == "q8":
        scale = rows[1].astype(np.float64)
        want = np.abs(lat).max(1) / 127
        assert (np.abs(scale - want) <= blat.max(1) / 127 + 2.0 ** -23 * want).all()
        blat = blat + (0.5 + 2.0 ** -14) * scale[:, None]  # 127 codes, each product off by 2^-23 twice
    else:
        blat = blat * (1 + half) + half * np.abs(lat)
    assert (np.abs(got[0] - lat) <= blat).all(), float((np.abs(got[0] - lat) / blat).max())
    assert (np.abs(got[1] - key) <= bkey).all(), float((np.abs(got[1] - key) / bkey).max())
    st.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [7, 12, 70])
def test_special_rows_equal_decoded_rows(models, kind, n):  # noqa: F811
    """Nodes whose rows meet the special cases (all zero, overflowing, NaN, infinite, subnormal products), through
    the projection of few nodes and of many: the rows of single-token decodes (NaN compares equal)."""
    cfg, layer, w = models("kimi")
    ctx, x = 5, hidden(cfg, 0xE4, n)
    x[1] = 0.0
    with np.errstate(over="ignore"):
        x[2] *= np.float32(1e38)
    x[3, 100] = np.nan
    x[4] *= np.float32(1e-30)
    x[5, 0] = np.inf
    x[6, 2047] = -3.3e38
    sizes = [n] if n <= 64 else [40, n - 40]
    ps = [[-1] * k for k in sizes]
    states = [State(kind, cfg, ctx + k).load(2, ctx) for k in sizes]
    batch_device(kind, cfg, w, states, ps, x)
    rows = [np.concatenate(a) for a in zip(*[s.pull(ctx, ctx + k) for s, k in zip(states, sizes)])]
    for i in range(n) if n < 20 else range(7):
        one = State(kind, cfg, ctx + 1).load(2, ctx)
        out = np.zeros((1, cfg.hidden_size), np.float32)
        lib.check(getattr(L, ONE[kind])(f32p(out), f32p(x[i:i + 1].copy()), ctx, C.byref(cfg), C.byref(w), one.ref()), "one")
        for a, b in zip(one.rows(ctx, ctx + 1), rows):
            a, b = (inputs.bf16_bits_to_f32(v) if v.dtype == np.uint16 else v for v in (a[0], b[i]))
            np.testing.assert_array_equal(a, b, err_msg=str(i))
        one.free()
    for s in states:
        s.free()


def test_q8_rows_of_the_smallest_scales(models):  # noqa: F811
    """Every history row of a scale near the least normal number, over long splits: the sums of the weights stay
    finite, and what is left of the output is the nodes' own rows'."""
    cfg, layer, w = models("kimi")
    ctx, n, batch = 40000, 8, 8
    states = [State("q8", cfg, ctx + n).load(3, 0) for _ in range(batch)]
    a = states[0].arrays()
    rng = np.random.default_rng(4)
    a[0][:ctx] = rng.integers(-127, 128, (ctx, cfg.kv_lora_rank))
    a[1][:ctx] = np.float32(2e-38) * rng.random(ctx, np.float32)  # some of them subnormal
    states[0].s.len = ctx
    lib.check(fn("compressed_%sstate_sync", "q8")(states[0].ref()), "sync")
    lib.check(fn("compressed_%sstate_fork_batch_device", "q8")(pointers(states[1:]), pointers(states[:1] * (batch - 1)), ints([0] * (batch - 1)),
                                                              ints([ctx] * (batch - 1)), batch - 1), "fork")
    p, x = tree("any", n, 1), hidden(cfg, 0xE5, n)
    got = batch_device("q8", cfg, w, states, [p] * batch, np.concatenate([x] * batch)).reshape(batch, n, -1)
    some = [0, n - 1]
    want = reference(cfg, layer, x, p, ctx, states[-1].pull(0, ctx + n), "q8", some)
    for b in range(batch):
        assert relative(got[b][some], want) <= 2 * NEAR
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("exponents,keys", [(range(18, 28), False), ((40, 47, 48, 49, 50, 51, 52, 55, 58), True)], ids=["past integers", "huge"])
def test_large_logits(models, kind, exponents, keys):  # noqa: F811
    """Logits of 2^21 to 2^30 (past 2^24 in steps of 2 to 128), and with keys as large as the queries up to 2^118, of
    either sign, equal over the history's rows, whose scale lies just below a power of two: the weights stay finite.
    Each head takes the history's row or the node's own; nodes whose heads do that by a margin of 2^-8 of the logit
    are compared."""
    cfg, layer, w = models("kimi")
    ctx, n = 100, 24
    rng = np.random.default_rng(6)
    lat = rng.integers(-127, 128, cfg.kv_lora_rank).astype(np.float64)
    lat[0] = 127
    key = rng.standard_normal(cfg.qk_rope_dim)
    st = State(kind, cfg, ctx + n)
    compared = 0
    for e in exponents:
        st.s.len = 0
        put_rows(st, np.tile(lat, (ctx, 1)), np.tile(key * 2.0 ** e * keys, (ctx, 1)))
        if kind == "q8":
            st.arrays()[1][:ctx] = np.float32(2 - 2.0 ** -23)
            lib.check(fn("compressed_%sstate_sync", kind)(st.ref()), "sync")
        x = (hidden(cfg, 0xE6, n) * np.float32(2.0 ** e)).astype(np.float32)
        p = [-1] * n
        got = tree_host(st, layer, x, p, w)
        assert np.isfinite(got).all(), e
        rows = st.rows(0, ctx + n)
        want = reference(cfg, layer, x, p, ctx, rows, kind)
        lats, ks = trees.values(rows, kind)
        q = latent_queries(cfg, layer, x)
        a = np.matmul(q, lats[0]) + rope_scores(cfg, layer, x, np.tile(ks[:1], (n, 1)), ctx)
        b = np.stack([q[i] @ lats[ctx + i] for i in range(n)]) + rope_scores(cfg, layer, x, ks[ctx:], ctx)
        for i in range(n):
            if (np.abs(a[i] - b[i]) > 2.0 ** -8 * np.abs(a[i]) + 64).all():
                compared += 1
                assert relative(got[i:i + 1], want[i:i + 1]) <= NEAR, (e, i)
    assert compared > 20
    st.free()
