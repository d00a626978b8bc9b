"""Tree decodes, forked states and accepted paths on the GPU.

Outputs are held to the definition in 64 bits over the rows that the state stores (trees.reference),
within trees.TOL; the stored rows to those that single-token decodes of each path append, bit for bit."""
import ctypes as C

import numpy as np
import pytest

import trees
from kvl_mla import inputs, lib
from trees import BLOCK, ONE, TOL, Device, State, f32p, fn, ints, off, path_to, pointers, reference, tree, tree_host

pytestmark = pytest.mark.gpu

L = lib.load()
KINDS = ["f32", "bf16", "q8"]
DIMS = {"tiny": trees.TINY, "lab": trees.LAB, "nine": trees.NINE, "kimi": trees.KIMI}


@pytest.fixture(scope="module")
def models():
    got = {}

    def get(name, seed=0x7E):
        if name not in got:
            cfg = inputs.config(**DIMS[name])
            layer = inputs.fast_layer(cfg, seed)
            w = layer.struct()
            lib.check(L.kvl_mla_bind_weights(C.byref(cfg), C.byref(w)), "bind")
            got[name] = cfg, layer, w
        return got[name]

    yield get
    for _, _, w in got.values():
        L.kvl_mla_release_weights(C.byref(w))


def hidden(cfg, seed, n):
    return np.ascontiguousarray(inputs.hidden(cfg, seed, n))


def batch_device(kind, cfg, w, states, parents, x, flags=0, out=None):
    dx, do = Device(x), Device(x if out is None else out)
    call = fn("decode_compressed_%stree_batch_device", kind)
    lib.check(call(do.p, dx.p, ints([len(p) for p in parents]), ints(sum(parents, [])), len(states), C.byref(cfg), C.byref(w),
                   pointers(states), flags), "tree batch")
    got = do.get()
    dx.free()
    do.free()
    return got


# ------------------------------------------------------------------ one tree ---------------

SHAPES = [("one", 1), ("chain", 7), ("star", 5), ("any", 3), ("any", 17), ("any", 64), ("chain", 64)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("ctx", [0, 1, 31, 32, 33, 64, 65, 257, 1000])
def test_tree_equals_definition(models, kind, dims, ctx):
    cfg, layer, w = models(dims)
    for k, (shape, n) in enumerate(SHAPES):
        if dims == "nine" and n > 20:
            continue
        print(f"[tree] {kind} {dims} ctx {ctx} {shape} {n}", flush=True)
        parents = tree(shape, n, 5 * ctx + k)
        st = State(kind, cfg, ctx + n + 3).load(ctx + k, ctx)
        x = hidden(cfg, 0x100 + ctx + k, n)
        got = tree_host(st, layer, x, parents, w)
        assert st.s.len == ctx + n
        want = reference(cfg, layer, x, parents, ctx, st.rows(0, ctx + n), kind)
        e = off(got, want)
        assert e <= TOL, (shape, n, e)
        # host rows and device rows are the same
        for a, b in zip(st.rows(ctx, ctx + n), st.pull(ctx, ctx + n)):
            np.testing.assert_array_equal(a, b)
        st.free()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_long_history(models, kind):
    cfg, layer, w = models("kimi")
    for ctx, n in [(4097, 9), (12345, 33), (20000, 2), (9999, 64)]:
        print(f"[tree] {kind} long {ctx} {n}", flush=True)
        parents = tree("any", n, ctx)
        st = State(kind, cfg, ctx + n).load(ctx, ctx)
        x = hidden(cfg, ctx, n)
        got = tree_host(st, layer, x, parents, w)
        e = off(got, reference(cfg, layer, x, parents, ctx, st.rows(0, ctx + n), kind))
        assert e <= TOL, (ctx, n, e)
        st.free()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_sharp_softmax(models, kind):
    """Logits of +-100 and more: a few rows carry the whole weight, the reference maximum moves often.
    A logit's own error is up to S 3 * 2^-18 of itself here, S <= 200, and enters a weight as it is."""
    cfg, layer, w = models("kimi")
    ctx, n = 3333, 6
    st = State(kind, cfg, ctx + n).load(1, ctx, spread=12.0)
    x = 4 * hidden(cfg, 0x21, n)
    parents = tree("any", n, 2)
    got = tree_host(st, layer, x, parents, w)
    want = reference(cfg, layer, x, parents, ctx, st.rows(0, ctx + n), kind)
    e = off(got, want)
    assert e <= (8 + 3 * 200) * 2.0 ** -18, e
    st.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["lab", "kimi"])
def test_rows_equal_path_decodes(models, kind, dims):
    """Every node's row is the one that a single-token decode of its path appends; a chain is a block."""
    cfg, layer, w = models(dims)
    ctx, n = 70, 9
    parents = tree("any", n, 3)
    st = State(kind, cfg, ctx + n).load(9, ctx)
    x = hidden(cfg, 0x33, n)
    got = tree_host(st, layer, x, parents, w)
    rows = st.rows(ctx, ctx + n)
    for i in range(n):
        p = path_to(parents, i)
        one = State(kind, cfg, ctx + n).load(9, ctx)
        out = np.zeros((1, cfg.hidden_size), np.float32)
        for j, node in enumerate(p):
            lib.check(getattr(L, ONE[kind])(f32p(out), f32p(x[node:node + 1].copy()), ctx + j, C.byref(cfg), C.byref(w), one.ref()), "one")
        for a, b in zip(one.rows(ctx + len(p) - 1, ctx + len(p)), rows):
            np.testing.assert_array_equal(a[0], b[i])
        # the single-token decode of Q8 rows takes its query in 15 bits (2.5e-5 of the output's norm)
        assert off(got[i:i + 1], out.astype(np.float64)) <= (5e-4 if kind == "q8" else 2 * TOL)
        one.free()
    chain, block = State(kind, cfg, ctx + n).load(9, ctx), State(kind, cfg, ctx + n).load(9, ctx)
    tree_host(chain, layer, x, tree("chain", n), w)
    out = np.zeros_like(x)
    lib.check(getattr(L, BLOCK[kind])(f32p(out), f32p(x), n, ctx, C.byref(cfg), C.byref(w), block.ref()), "block")
    for a, b in zip(chain.rows(0, ctx + n), block.rows(0, ctx + n)):
        np.testing.assert_array_equal(a, b)
    for s in (st, chain, block):
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["lab", "kimi"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
def test_other_branches_do_not_reach_a_node(models, kind, dims, bad):
    """A node whose hidden state is not finite spoils its own row and descendants, nothing else."""
    cfg, layer, w = models(dims)
    ctx, n = 50, 12
    parents = [-1, 0, 0, 1, 1, 2, 2, 3, -1, 8, 9, 4]
    x = hidden(cfg, 0x44, n)
    clean, spoilt = State(kind, cfg, ctx + n).load(4, ctx), State(kind, cfg, ctx + n).load(4, ctx)
    want = tree_host(clean, layer, x, parents, w)
    x[2, :] = bad
    got = tree_host(spoilt, layer, x, parents, w)
    for i in range(n):
        if 2 not in path_to(parents, i):
            np.testing.assert_array_equal(got[i], want[i], err_msg=str(i))
    assert not np.isfinite(got[2]).all()
    for s in (clean, spoilt):
        s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_behind_the_tree_stay(models, kind):
    cfg, layer, w = models("kimi")
    st = State(kind, cfg, 60).load(6, 60).upload()
    before = st.rows(0, 60)
    lib.check(fn("compressed_%sstate_truncate", kind)(st.ref(), 40), "truncate")
    tree_host(st, layer, hidden(cfg, 1, 5), tree("any", 5), w)
    for k, (a, b) in enumerate(zip(st.rows(0, 60), before)):
        for got in (a, device_array(st, k, 0, 60)):
            np.testing.assert_array_equal(got[:40], b[:40])
            np.testing.assert_array_equal(got[45:], b[45:])
    st.free()


# ------------------------------------------------------------------ batches ----------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims,lens,sizes", [
    ("lab", [0, 5, 90], [3, 1, 12]),
    ("lab", [30, 70], [60, 50]),
    ("nine", [40, 100, 0], [50, 30, 2]),
    ("kimi", [700, 0, 33, 1500, 64], [5, 3, 1, 8, 2]),
    ("kimi", [900, 40, 2000, 300], [64, 30, 40, 1]),
    ("kimi", [100 + 37 * i for i in range(13)], [1] * 13),
    ("kimi", [64 * i for i in range(70)], [1 + i % 2 for i in range(70)]),
])
def test_batch_equals_definition(models, kind, dims, lens, sizes):
    cfg, layer, w = models(dims)
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n + 1).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    x = hidden(cfg, 0x55, sum(sizes))
    first = batch_device(kind, cfg, w, states, ps, x, lib.NO_ADVANCE)
    assert [s.s.len for s in states] == lens
    got = batch_device(kind, cfg, w, states, ps, x)
    np.testing.assert_array_equal(first, got)
    assert [s.s.len for s in states] == [m + n for m, n in zip(lens, sizes)]
    at = 0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        rows = states[i].pull(0, m + n)
        e = off(got[at:at + n], reference(cfg, layer, x[at:at + n], ps[i], m, rows, kind))
        assert e <= TOL, (i, m, n, e)
        at += n
    # the residual form, onto another buffer and onto the input itself (the sum is one more rounding)
    for s, m in zip(states, lens):
        s.s.len = m
    base = hidden(cfg, 0x56, sum(sizes))
    res = batch_device(kind, cfg, w, states, ps, x, lib.RESIDUAL | lib.NO_ADVANCE, out=base)
    np.testing.assert_allclose(res, base + got, rtol=0, atol=float(np.abs(base).max() + np.abs(got).max()) * 2.0 ** -23)
    d = Device(x)
    lib.check(fn("decode_compressed_%stree_batch_device", kind)(d.p, d.p, ints(sizes), ints(sum(ps, [])), len(states), C.byref(cfg),
                                                               C.byref(w), pointers(states), lib.RESIDUAL | lib.NO_ADVANCE), "in place")
    np.testing.assert_allclose(d.get(), x + got, rtol=0, atol=float(np.abs(x).max() + np.abs(got).max()) * 2.0 ** -23)
    d.free()
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_batch_of_large_trees(models, kind):
    """Several launch groups, each with work for more than a round of workgroups; ragged trees and splits."""
    cfg, layer, w = models("kimi")
    sizes, lens = [64, 63, 61, 64, 62, 64, 64, 5], [3500, 3471, 3049, 4000, 3500, 3001, 3333, 31]
    ps = [tree("any", n, 20 + i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    x = hidden(cfg, 0x57, sum(sizes))
    got = batch_device(kind, cfg, w, states, ps, x)
    at = 0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        some = sorted({0, n - 1, n // 2, n // 3, n - 3, n - 2})
        want = reference(cfg, layer, x[at:at + n], ps[i], m, states[i].pull(0, m + n), kind, some)
        e = off(got[at:at + n][some], want)
        assert e <= TOL, (i, m, n, e)
        at += n
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [9, 16, 17, 32, 33, 63])
def test_rows_of_any_count_equal_few(models, kind, n):
    """A node's row does not depend on how many nodes are decoded with it, nor on where x lies."""
    cfg, layer, w = models("kimi")
    p, x, ctx = tree("any", n, n), hidden(cfg, 0x60 + n, n), 20
    rows = []
    for k in (n, 1, 4, 8):
        st = State(kind, cfg, ctx + n).load(1, ctx)
        batch_device(kind, cfg, w, [st], [p[:k]], x[:k])
        rows.append(st.pull(ctx, ctx + k))
        st.free()
    st = State(kind, cfg, ctx + n).load(1, ctx)
    tree_host(st, layer, x, p, w)
    rows.append(st.rows(ctx, ctx + n))
    st.free()
    for other in rows[1:]:
        for a, b in zip(rows[0], other):
            np.testing.assert_array_equal(a[:len(b)], b)


@pytest.mark.parametrize("kind", KINDS)
def test_many_nodes_equal_few(models, kind):
    """The rows of a batch of many nodes are those of its trees alone, bit for bit, and a node that is not
    finite stays within its tree there too."""
    cfg, layer, w = models("kimi")
    sizes, lens = [40, 50, 33], [90, 10, 200]
    ps = [tree("any", n, 30 + i) for i, n in enumerate(sizes)]
    x = hidden(cfg, 0x58, sum(sizes))
    x[44, :] = np.nan
    both = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    got = batch_device(kind, cfg, w, both, ps, x)
    at = 0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        alone = State(kind, cfg, m + n).load(i, m)
        out = batch_device(kind, cfg, w, [alone], [ps[i]], x[at:at + n])
        rows = [k for k in range(n) if at + k != 44]
        for a, b in zip(alone.pull(m, m + n), both[i].pull(m, m + n)):
            np.testing.assert_array_equal(a[rows], b[rows])
        # so are those of the tree's first nodes, which take the projection of few
        few = State(kind, cfg, m + 8).load(i, m)
        batch_device(kind, cfg, w, [few], [ps[i][:8]], x[at:at + 8])
        for a, b in zip(few.pull(m, m + 8), both[i].pull(m, m + 8)):
            np.testing.assert_array_equal(a[rows[:7]], b[rows[:7]])
        few.free()
        fine = [k for k in range(n) if at + k != 44 and not (i == 1 and 4 in path_to(ps[1], k))]
        assert off(got[at:at + n][fine], out[fine].astype(np.float64)) <= 2 * TOL
        alone.free()
        at += n
    assert not np.isfinite(got[44]).all()
    for s in both:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [[7], [30, 9], [64, 40]])
def test_unaligned_buffers(models, kind, sizes):
    """Hidden states and outputs 4 bytes off a 16-byte boundary: the aligned call's outputs; the words
    around the output stay."""
    cfg, layer, w = models("kimi")
    ps = [tree("any", n, 3 + i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, 400).load(i, 300 + i) for i in range(len(sizes))]
    x = hidden(cfg, 0x59, sum(sizes))
    want = batch_device(kind, cfg, w, states, ps, x, lib.NO_ADVANCE)
    room = np.full(x.size + 8, 7.25, np.float32)
    placed = room.copy()
    placed[1:1 + x.size] = x.ravel()
    dx, do = Device(placed), Device(room)
    lib.check(fn("decode_compressed_%stree_batch_device", kind)(do.p + 4, dx.p + 4, ints([len(p) for p in ps]), ints(sum(ps, [])),
                                                               len(states), C.byref(cfg), C.byref(w), pointers(states),
                                                               lib.NO_ADVANCE), "tree batch")
    got = do.get()
    assert off(got[1:1 + x.size].reshape(x.shape), want.astype(np.float64)) <= 2 * TOL
    np.testing.assert_array_equal(got[[0, *range(1 + x.size, room.size)]], 7.25)
    np.testing.assert_array_equal(dx.get(), placed)
    for b in (dx, do):
        b.free()
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ctx", [0, 37, 64, 300])
def test_rows_behind_the_history_do_not_enter(models, kind, ctx):
    """What a dropped draft left behind the history, not finite here, has no effect."""
    cfg, layer, w = models("kimi")
    n = 6
    x, p = hidden(cfg, 0x5A, n), tree("any", n, 5)
    st, clean = State(kind, cfg, 400).load(3, 400), State(kind, cfg, 400).load(3, 400)
    for a in st.arrays():
        if a.dtype == np.float32:
            a[ctx:] = np.nan
        elif a.dtype == np.uint16:
            a[ctx:] = 0x7FC0
    lib.check(fn("compressed_%sstate_sync", kind)(st.ref()), "sync")
    st.upload()
    for s in (st, clean):
        lib.check(fn("compressed_%sstate_truncate", kind)(s.ref(), ctx), "truncate")
    np.testing.assert_array_equal(tree_host(st, layer, x, p, w), tree_host(clean, layer, x, p, w))
    for s in (st, clean):
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [4096, 328])
def test_other_hidden_sizes(models, kind, size):
    """The attention's dims of KIMI under another hidden size: other projections, few nodes and many."""
    cfg = inputs.config(**dict(trees.KIMI, hidden_size=size))
    layer = inputs.fast_layer(cfg, 0x5D)
    w = layer.struct()
    lib.check(L.kvl_mla_bind_weights(C.byref(cfg), C.byref(w)), "bind")
    for sizes in ([5], [20, 9], [60, 50]):
        ps = [tree("any", n, i) for i, n in enumerate(sizes)]
        states = [State(kind, cfg, 300 + n).load(i, 200 + i) for i, n in enumerate(sizes)]
        x = hidden(cfg, 0x5E, sum(sizes))
        got = batch_device(kind, cfg, w, states, ps, x)
        at = 0
        for i, n in enumerate(sizes):
            rows = states[i].pull(0, 200 + i + n)
            e = off(got[at:at + n], reference(cfg, layer, x[at:at + n], ps[i], 200 + i, rows, kind))
            assert e <= TOL, (sizes, i, e)
            at += n
        for s in states:
            s.free()
    L.kvl_mla_release_weights(C.byref(w))


def test_q8_scales_of_all_sizes(models):
    """Q8 rows whose scales run from zero over the smallest numbers to the usual ones: small scales must
    not push the other rows' weights out of range."""
    cfg, layer, w = models("kimi")
    ctx, n = 700, 9
    st = State("q8", cfg, ctx + n).load(8, ctx)
    sc = st.arrays()[1]
    sc[0:100] = 0
    sc[100:200] = np.float32(1e-40)
    sc[200:300] = np.float32(1e-30)
    sc[300:400] *= np.float32(1e-6)
    sc[650:] *= np.float32(3)
    lib.check(fn("compressed_%sstate_sync", "q8")(st.ref()), "sync")
    x, p = hidden(cfg, 0x5B, n), tree("any", n, 6)
    got = tree_host(st, layer, x, p, w)
    e = off(got, reference(cfg, layer, x, p, ctx, st.rows(0, ctx + n), "q8"))
    assert e <= 3 * TOL, e  # three times the logits
    st.free()


@pytest.mark.parametrize("kind", KINDS)
def test_long_histories_of_zero_rows(models, kind):
    """Rows of zeros (Q8: of scale zero too), many to a split: every row has the weight 1."""
    cfg, layer, w = models("kimi")
    ctx, n, batch = 40000, 32, 8
    states = [State(kind, cfg, ctx + n) for _ in range(batch)]
    states[0].s.len = ctx  # as initialised: zeros
    for a in states[0].arrays():
        a[:] = 0
    lib.check(fn("compressed_%sstate_sync", kind)(states[0].ref()), "sync")
    lib.check(fn("compressed_%sstate_fork_batch_device", kind)(pointers(states[1:]), pointers(states[:1] * (batch - 1)), ints([0] * (batch - 1)),
                                                              ints([ctx] * (batch - 1)), batch - 1), "fork")
    p = tree("any", n, 1)
    x = hidden(cfg, 0x5C, n)
    got = batch_device(kind, cfg, w, states, [p] * batch, np.concatenate([x] * batch)).reshape(batch, n, -1)
    some = [0, n - 1]
    want = reference(cfg, layer, x, p, ctx, states[-1].pull(0, ctx + n), kind, some)
    for b in range(batch):
        e = off(got[b][some], want)
        assert e <= TOL, (b, e)
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [[4], [9, 1, 30], [60, 50], [1, 1, 1], [64, 64, 64, 63, 60]])
def test_layer_form(models, kind, sizes):
    cfg, layer, w = models("kimi")
    lens = [333, 20, 800, 50, 0][:len(sizes)]
    ps = [tree("any", n, 7 + i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    n1, n2 = inputs.normal_bf16(1, "n1", (cfg.hidden_size,), 1.0, 0.1), inputs.normal_bf16(2, "n2", (cfg.hidden_size,), 1.0, 0.1)
    h = hidden(cfg, 0x66, sum(sizes))
    dh, dn = Device(h), Device(h)
    u16 = lambda a: trees.abi.ptr(a, C.c_uint16)  # noqa: E731
    lib.check(fn("attention_layer_%stree_device", kind)(dh.p, dn.p, ints(sizes), ints(sum(ps, [])), len(sizes), C.byref(cfg), C.byref(w),
                                                       u16(n1), u16(n2), pointers(states), 0), "layer")
    got, post = dh.get(), dn.get()
    at = 0
    for i, (m, n) in enumerate(zip(lens, sizes)):
        x = trees.rms64(h[at:at + n].astype(np.float64), trees.f64(n1), cfg.rms_eps)
        att = reference(cfg, layer, x, ps[i], m, states[i].pull(0, m + n), kind)
        e = np.abs((got[at:at + n] - h[at:at + n].astype(np.float64)) - att).max() / np.abs(att).max()
        # the sum with h rounds to 2^-24 of a value up to |h| + |attention|
        assert e <= TOL + 2.0 ** -23 * np.abs(h).max() / np.abs(att).max(), (i, e)
        at += n
    want = trees.rms64(got.astype(np.float64), trees.f64(n2), cfg.rms_eps)
    assert off(post, want) <= 2.0 ** -20
    for b in (dh, dn):
        b.free()
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [[3], [50, 40]])
def test_layer_form_on_unaligned_buffers(models, kind, sizes):
    cfg, layer, w = models("kimi")
    ps = [tree("any", n, 4 + i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, 400).load(i, 250 + i) for i in range(len(sizes))]
    n1, n2 = inputs.normal_bf16(1, "n1", (cfg.hidden_size,), 1.0, 0.1), inputs.normal_bf16(2, "n2", (cfg.hidden_size,), 1.0, 0.1)
    h = hidden(cfg, 0x67, sum(sizes))
    u16 = lambda a: trees.abi.ptr(a, C.c_uint16)  # noqa: E731
    got = []
    for at in (0, 4):
        placed = np.full(h.size + 8, 3.5, np.float32)
        placed[at // 4:at // 4 + h.size] = h.ravel()
        dh, dn = Device(placed), Device(np.full_like(placed, 3.5))
        lib.check(fn("attention_layer_%stree_device", kind)(dh.p + at, dn.p + at, ints(sizes), ints(sum(ps, [])), len(sizes), C.byref(cfg),
                                                           C.byref(w), u16(n1), u16(n2), pointers(states), lib.NO_ADVANCE), "layer")
        for d in (dh, dn):
            a = d.get()
            got.append(a[at // 4:at // 4 + h.size].reshape(h.shape))
            rest = np.r_[a[:at // 4], a[at // 4 + h.size:]]
            np.testing.assert_array_equal(rest, 3.5)
            d.free()
    for a, b in ((got[0], got[2]), (got[1], got[3])):
        assert off(b, a.astype(np.float64)) <= 2 * TOL
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_captured_tree_replays(models, kind):
    """A graph of the tree call repeats its result on every replay, other work and waits between."""
    cfg, layer, w = models("kimi")
    sizes, lens = [6, 11], [500, 90]
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
    x = hidden(cfg, 0x77, sum(sizes))
    want = batch_device(kind, cfg, w, states, ps, x, lib.NO_ADVANCE)
    dx, do = Device(x), Device(x)
    call = lambda: fn("decode_compressed_%stree_batch_device", kind)(do.p, dx.p, ints(sizes), ints(sum(ps, [])), 2, C.byref(cfg),  # noqa: E731
                                                                   C.byref(w), pointers(states), lib.NO_ADVANCE)
    lib.check(L.kvl_mla_capture_begin(), "capture")
    rc = call()
    g = C.c_void_p()
    lib.check(L.kvl_mla_capture_end(C.byref(g)), "capture end")
    lib.check(rc, "captured tree")
    for r in range(4):
        do.put(np.zeros_like(x))
        lib.check(L.kvl_mla_graph_launch(g), "replay")
        np.testing.assert_array_equal(do.get(), want, err_msg=f"replay {r}")
        other = hidden(cfg, r, sum(sizes))  # eager work on other inputs, through the same workspace
        batch_device(kind, cfg, w, states, ps, other, lib.NO_ADVANCE)
        lib.check(L.kvl_mla_synchronize(), "sync")
    L.kvl_mla_graph_destroy(g)
    # row moves are refused inside a capture
    lib.check(L.kvl_mla_capture_begin(), "capture")
    rcs = [fn("compressed_%sstate_accept_batch_device", kind)(pointers(states), ints([10, 10]), ints([1, 1]), ints([1, 1]), 2),
           fn("compressed_%sstate_fork_batch_device", kind)(pointers(states[:1]), pointers(states[1:]), ints([0]), ints([5]), 1)]
    why = lib.last_error()
    lib.check(L.kvl_mla_capture_end(C.byref(g)), "capture end")
    L.kvl_mla_graph_destroy(g)
    assert rcs == [-1, -1] and "capture" in why
    assert [s.s.len for s in states] == lens
    for b in (dx, do):
        b.free()
    for s in states:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_two_graphs_in_turn(models, kind):
    """Two captured trees of different sizes, replayed in turn: they share the library's workspaces."""
    cfg, layer, w = models("kimi")
    plans = [([8, 3], [700, 20]), ([50, 64], [90, 1200]), ([1], [333])]
    calls, wants, graphs, keep = [], [], [], []
    for k, (sizes, lens) in enumerate(plans):
        ps = [tree("any", n, i + k) for i, n in enumerate(sizes)]
        states = [State(kind, cfg, m + n).load(i, m) for i, (m, n) in enumerate(zip(lens, sizes))]
        x = hidden(cfg, 0x7A + k, sum(sizes))
        wants.append(batch_device(kind, cfg, w, states, ps, x, lib.NO_ADVANCE))
        dx, do = Device(x), Device(x)
        keep.append((states, dx, do))
        calls.append(lambda do=do, dx=dx, sizes=sizes, ps=ps, states=states: fn("decode_compressed_%stree_batch_device", kind)(
            do.p, dx.p, ints(sizes), ints(sum(ps, [])), len(sizes), C.byref(cfg), C.byref(w), pointers(states), lib.NO_ADVANCE))
    for call in calls:
        lib.check(L.kvl_mla_capture_begin(), "capture")
        rc = call()
        g = C.c_void_p()
        lib.check(L.kvl_mla_capture_end(C.byref(g)), "capture end")
        lib.check(rc, "captured tree")
        graphs.append(g)
    for r in range(3):
        for k, (states, dx, do) in enumerate(keep):
            do.put(np.zeros(do.shape, np.float32))
        for g in graphs:
            lib.check(L.kvl_mla_graph_launch(g), "replay")
        for k, (states, dx, do) in enumerate(keep):
            np.testing.assert_array_equal(do.get(), wants[k], err_msg=f"replay {r} of {k}")
        lib.check(calls[r % 3](), "eager")
        lib.check(L.kvl_mla_synchronize(), "sync")
    for g in graphs:
        L.kvl_mla_graph_destroy(g)
    for states, dx, do in keep:
        for s in (*states, dx, do):
            s.free()


@pytest.mark.parametrize("kind", KINDS)
def test_host_calls_are_refused_in_a_capture(models, kind):
    cfg, layer, w = models("kimi")
    a, b = State(kind, cfg, 80).load(1, 40), State(kind, cfg, 80).load(2, 50)
    x = hidden(cfg, 0x7D, 3)
    want = tree_host(a, layer, x, [-1, 0, 0], w)
    lib.check(fn("compressed_%sstate_truncate", kind)(a.ref(), 40), "truncate")
    out = np.full_like(x, np.nan)
    lib.check(L.kvl_mla_capture_begin(), "capture")
    rcs = [fn("decode_compressed_%stree_bf16", kind)(f32p(out), f32p(x), ints([-1, 0, 0]), 3, 40, C.byref(cfg), C.byref(w), a.ref())]
    whys = [lib.last_error()]
    for name, args in (("fork", (a.ref(), b.ref(), 0, 50)), ("accept", (b.ref(), 40, ints([1]), 1))):
        rcs.append(fn("compressed_%sstate_" + name, kind)(*args))
        whys.append(lib.last_error())
    g = C.c_void_p()
    lib.check(L.kvl_mla_capture_end(C.byref(g)), "capture end")
    L.kvl_mla_graph_destroy(g)
    assert rcs == [-1] * 3 and all("capture" in y for y in whys), whys
    assert np.isnan(out).all() and (a.s.len, b.s.len) == (40, 50)
    np.testing.assert_array_equal(tree_host(a, layer, x, [-1, 0, 0], w), want)
    for s in (a, b):
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims,sizes,launches", [
    ("kimi", [7], [1, 1, 0, 1, 1, 1]), ("kimi", [60, 50], [1, 1, 0, 1, 1, 1]), ("kimi", [64] * 5, [2, 2, 0, 2, 2, 2]),
    ("lab", [60, 50], [1, 2, 0, 1, 2, 2]),
])
def test_stage_timing(models, kind, dims, sizes, launches):
    """A tree decode's launches are bracketed as the other decodes' are."""
    cfg, layer, w = models(dims)
    ps = [tree("any", n, i) for i, n in enumerate(sizes)]
    states = [State(kind, cfg, 200).load(i, 100) for i in range(len(sizes))]
    x = hidden(cfg, 0x7E, sum(sizes))
    want = batch_device(kind, cfg, w, states, ps, x, lib.NO_ADVANCE)
    ms, count = (C.c_double * 6)(), (C.c_int * 6)()
    lib.check(L.kvl_mla_timing_enable(1), "timing")
    try:
        lib.check(L.kvl_mla_timing_read(ms, count), "read")
        got = batch_device(kind, cfg, w, states, ps, x, lib.NO_ADVANCE)
        lib.check(L.kvl_mla_timing_read(ms, count), "read")
    finally:
        L.kvl_mla_timing_enable(0)
    np.testing.assert_array_equal(got, want)
    assert list(count) == launches
    assert all((t > 0) == (n > 0) for t, n in zip(ms, count))
    for s in states:
        s.free()


def test_two_threads(models):
    """Calls from two threads take turns; each thread reads its own errors."""
    import threading
    cfg, layer, w = models("kimi")
    want, got, fails = {}, {}, []

    def work(k):
        try:
            st = State("bf16", cfg, 400).load(k, 300 + k)
            x, p = hidden(cfg, 0x90 + k, 5 + k), tree("any", 5 + k, k)
            for _ in range(5):
                got[k] = tree_host(st, layer, x, p, w)
                assert fn("compressed_%sstate_accept", "bf16")(st.ref(), 900 + k, ints([0]), 1) == -1
                assert f"row {300 + k}" not in lib.last_error() and f"row {900 + k}" in lib.last_error().replace("from row", "row")
                lib.check(fn("compressed_%sstate_truncate", "bf16")(st.ref(), 300 + k), "truncate")
            want[k] = reference(cfg, layer, x, p, 300 + k, st.rows(0, 305 + 2 * k), "bf16")
            st.free()
        except Exception as e:  # noqa: BLE001
            fails.append(e)

    ts = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not fails, fails
    for k in range(2):
        assert off(got[k], want[k]) <= TOL


# ------------------------------------------------------------------ copies -----------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["tiny", "lab", "kimi"])
def test_fork_host(models, kind, dims):
    cfg = models(dims)[0]
    for n, r0, r1 in [(1, 0, 1), (40, 0, 40), (40, 7, 33), (130, 129, 130), (55, 5, 5), (600, 1, 600)]:
        src, dst = State(kind, cfg, n + 2).load(n, n), State(kind, cfg, n + 9).load(n + 1, r0 + 2 if r0 + 2 <= n else r0)
        kept, tail = dst.rows(0, r0), dst.rows(r1, n + 9)
        lib.check(fn("compressed_%sstate_fork", kind)(dst.ref(), src.ref(), r0, r1), "fork")
        assert dst.s.len == r1 and src.s.len == n
        for got in (dst.rows(0, r1), dst.pull(0, r1)):
            for a, b, k in zip(got, src.rows(0, r1), kept):
                np.testing.assert_array_equal(a[r0:], b[r0:])
                np.testing.assert_array_equal(a[:r0], k)
        for a, b in zip(dst.rows(r1, n + 9), tail):
            np.testing.assert_array_equal(a, b)
        for s in (src, dst):
            s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["tiny", "kimi"])
def test_fork_batch_device(models, kind, dims):
    """One source to many and many to many, in one call of more pairs than a launch takes; the rows
    around the copied ones stay, on the device too."""
    cfg = models(dims)[0]
    rng = np.random.default_rng(5)
    n = 53
    srcs = [State(kind, cfg, 400).load(i, 300 + 7 * i) for i in range(5)]
    pick = [int(rng.integers(0, 5)) if i > 20 else 0 for i in range(n)]
    dsts = [State(kind, cfg, 420).load(100 + i, 390) for i in range(n)]
    for d in dsts:
        d.upload()
    r1 = [int(rng.integers(0, 300)) for _ in range(n)]
    r0 = [int(rng.integers(0, b + 1)) for b in r1]
    lib.check(fn("compressed_%sstate_fork_batch_device", kind)(pointers(dsts), pointers([srcs[k] for k in pick]), ints(r0), ints(r1), n), "fork")
    for i, d in enumerate(dsts):
        assert d.s.len == r1[i]
        own = State(kind, cfg, 420).load(100 + i, 390)
        before = own.rows(0, 390)
        for k, (a, s, b) in enumerate(zip(d.pull(0, r1[i]), srcs[pick[i]].rows(0, r1[i]), before)):
            np.testing.assert_array_equal(a[r0[i]:], s[r0[i]:], err_msg=f"{i} {k}")
            np.testing.assert_array_equal(a[:r0[i]], b[:r0[i]], err_msg=f"{i} {k}")
            # behind the copied rows the device still holds the destination's old ones
            np.testing.assert_array_equal(device_array(d, k, r1[i], 390), b[r1[i]:], err_msg=f"{i} {k}")
        own.free()
    for s in srcs + dsts:
        s.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["tiny", "lab", "kimi"])
def test_fork_of_one_range_to_many(models, kind, dims):
    """Neighbouring pairs of one source and one range are copied together, whatever the range's
    alignment; a pair of another range or source between them is not."""
    cfg = models(dims)[0]
    srcs = [State(kind, cfg, 700).load(i, 600 + i) for i in range(2)]
    pairs = [(0, 3, 577), (0, 3, 577), (0, 3, 577), (1, 3, 577), (0, 3, 577), (0, 4, 577), (0, 3, 576), (1, 0, 601), (1, 0, 601),
             (1, 5, 6), (1, 5, 6), (0, 9, 9), (0, 9, 9), (0, 1, 600), (0, 1, 600)]
    dsts = [State(kind, cfg, 650).load(50 + i, 640).upload() for i in range(len(pairs))]
    old = [d.rows(0, 640) for d in dsts]
    lib.check(fn("compressed_%sstate_fork_batch_device", kind)(pointers(dsts), pointers([srcs[k] for k, _, _ in pairs]),
                                                              ints([lo for _, lo, _ in pairs]), ints([hi for _, _, hi in pairs]),
                                                              len(pairs)), "fork")
    for i, (k, lo, hi) in enumerate(pairs):
        assert dsts[i].s.len == hi
        for j, (src, was) in enumerate(zip(srcs[k].rows(0, 600), old[i])):
            now = device_array(dsts[i], j, 0, 640)
            np.testing.assert_array_equal(now[lo:min(hi, 600)], src[lo:hi], err_msg=f"{i} {j}")
            np.testing.assert_array_equal(now[:lo], was[:lo], err_msg=f"{i} {j}")
            np.testing.assert_array_equal(now[hi:], was[hi:], err_msg=f"{i} {j}")
    for s in srcs + dsts:
        s.free()


def device_array(st, k, lo, hi):
    """Rows [lo, hi) of array k of a state, from its device address."""
    p, a = st.addresses(), st.arrays()[k]
    out = np.empty_like(a[lo:hi])
    e = a[:1].nbytes
    if out.nbytes:
        lib.check(L.kvl_mla_copy_to_host(out.ctypes.data, p[k] + lo * e, out.nbytes), "d2h")
    return out


@pytest.mark.parametrize("kind", KINDS)
def test_forked_state_decodes_as_its_source(models, kind):
    cfg, layer, w = models("kimi")
    src, dst = State(kind, cfg, 900).load(2, 777), State(kind, cfg, 900)
    lib.check(fn("compressed_%sstate_fork_batch_device", kind)(pointers([dst]), pointers([src]), ints([0]), ints([777]), 1), "fork")
    x, p = hidden(cfg, 3, 8), tree("any", 8, 1)
    a, b = batch_device(kind, cfg, w, [src], [p], x), batch_device(kind, cfg, w, [dst], [p], x)
    np.testing.assert_array_equal(a, b)
    for s in (src, dst):
        s.free()


# ------------------------------------------------------------------ accepted paths ---------

PATHS = [[], [0], [3], [0, 1, 2], [0, 2, 3, 9], [63], [1, 62, 63], list(range(64)), list(range(1, 64)), list(range(0, 64, 2)),
         [5] + list(range(20, 64))]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["tiny", "lab", "kimi"])
def test_accept_moves_rows(models, kind, dims):
    cfg = models(dims)[0]
    for i, path in enumerate(PATHS):
        n, start = 64, 1 + 11 * i
        st = State(kind, cfg, start + n + 4).load(i, start + n)
        if i % 2:  # the rows may be on the device already, or on the host only
            st.upload()
        before = st.rows(0, start + n)
        lib.check(fn("compressed_%sstate_accept", kind)(st.ref(), start, ints(path), len(path)), "accept")
        assert st.s.len == start + len(path)
        rows = list(range(start)) + [start + j for j in path]
        for got in (st.rows(0, len(rows)), st.pull(0, len(rows))):
            for a, b in zip(got, before):
                np.testing.assert_array_equal(a, b[rows])
        for k, b in enumerate(before):  # rows behind the path: as they were
            np.testing.assert_array_equal(device_array(st, k, len(rows), start + n), b[len(rows):])
        st.free()


@pytest.mark.parametrize("kind", KINDS)
def test_accept_batch_device(models, kind):
    """More states than a launch takes, each with its own path, among them ones with nothing to move."""
    cfg = models("lab")[0]
    rng = np.random.default_rng(9)
    n = 75
    states, starts, paths, before = [], [], [], []
    for i in range(n):
        size, start = int(rng.integers(1, 65)), int(rng.integers(0, 200))
        st = State(kind, cfg, start + size).load(i, start + size)
        before.append(st.rows(0, start + size))
        keep = int(rng.integers(0, size + 1))
        paths.append(list(range(keep)) if i % 5 == 0 else sorted(rng.choice(size, keep, replace=False).tolist()))
        states.append(st)
        starts.append(start)
    lib.check(fn("compressed_%sstate_accept_batch_device", kind)(pointers(states), ints(starts), ints([len(p) for p in paths]),
                                                                ints(sum(paths, [])), n), "accept")
    for st, start, p, b in zip(states, starts, paths, before):
        assert st.s.len == start + len(p)
        rows = list(range(start)) + [start + j for j in p]
        for a, c in zip(st.pull(0, len(rows)), b):
            np.testing.assert_array_equal(a, c[rows])
        st.free()


# ------------------------------------------------------------------ a run of them ----------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", ["lab", "kimi"])
def test_speculative_run_equals_serial_decoding(models, kind, dims):
    """Prefill, then rounds of fork, tree, accept; the state that remains is the serial decode's of the
    accepted tokens bit for bit, and the accepted nodes' outputs its outputs."""
    cfg, layer, w = models(dims)
    H, prompt = cfg.hidden_size, 45
    rng = np.random.default_rng(8)
    px = hidden(cfg, 0xA0, prompt)
    main, serial, spare = (State(kind, cfg, 200) for _ in range(3))
    for s in (main, serial):
        lib.check(fn("compressed_%sstate_prefill_bf16", kind)(f32p(px), prompt, C.byref(cfg), C.byref(w), s.ref()), "prefill")
    for r in range(5):
        start, n = main.s.len, int(rng.integers(1, 14))
        parents = tree("any", n, 20 + r)
        x = hidden(cfg, 0xB0 + r, n)
        # a copy keeps the context; it takes over only what it does not have yet
        lib.check(fn("compressed_%sstate_fork", kind)(spare.ref(), main.ref(), spare.s.len, start), "fork")
        host = r % 2 == 0
        got = tree_host(main, layer, x, parents, w) if host else batch_device(kind, cfg, w, [main], [parents], x)
        path = path_to(parents, int(rng.integers(0, n)))
        if host:
            lib.check(fn("compressed_%sstate_accept", kind)(main.ref(), start, ints(path), len(path)), "accept")
        else:
            lib.check(fn("compressed_%sstate_accept_batch_device", kind)(pointers([main]), ints([start]), ints([len(path)]), ints(path), 1), "accept")
        for j, node in enumerate(path):
            out = np.zeros((1, H), np.float32)
            lib.check(getattr(L, ONE[kind])(f32p(out), f32p(x[node:node + 1].copy()), start + j, C.byref(cfg), C.byref(w), serial.ref()), "one")
            assert off(got[node:node + 1], out.astype(np.float64)) <= (5e-4 if kind == "q8" else 2 * TOL)
        assert main.s.len == serial.s.len == start + len(path)
        for a, b in zip(main.pull(0, main.s.len), serial.rows(0, serial.s.len)):
            np.testing.assert_array_equal(a, b)
        for a, b in zip(spare.pull(0, start), serial.rows(0, start)):
            np.testing.assert_array_equal(a, b)
    for s in (main, serial, spare):
        s.free()


def test_tree_past_32_bit_offsets(models):
    """An FP32 state whose latent array passes 2^31 bytes: a tree at its end against the block decode of
    the same chain. A rope_theta of its own: the table of the usual one grows with the positions, and other
    tests count on positions that it does not reach."""
    _, layer, w = models("kimi")
    cfg = inputs.config(**dict(trees.KIMI, rope_theta=30000.0))
    ctx, n = 1_100_000, 6
    st = State("f32", cfg, ctx + n)
    lib.check(L.kvl_mla_compressed_state_fill_synthetic(st.ref(), 0, ctx, 77), "fill")
    x = hidden(cfg, 0xC1, n)
    dx, do = Device(x), Device(x)
    lib.check(L.kvl_mla_decode_compressed_tree_batch_device(do.p, dx.p, ints([n]), ints(tree("chain", n)), 1, C.byref(cfg), C.byref(w),
                                                            pointers([st]), 0), "tree")
    got = do.get()
    rows = st.pull(ctx - 3, ctx + n)
    lib.check(L.kvl_mla_compressed_state_truncate(st.ref(), ctx), "truncate")
    want = np.zeros_like(x)
    lib.check(L.kvl_mla_decode_compressed_block_bf16(f32p(want), f32p(x), n, ctx, C.byref(cfg), C.byref(w), st.ref()), "block")
    for a, b in zip(rows, st.pull(ctx - 3, ctx + n)):
        np.testing.assert_array_equal(a, b)
    assert off(got, want.astype(np.float64)) <= 2 * TOL
    st.free()
    for b in (dx, do):
        b.free()


def test_rows_past_32_bit_offsets(models):
    """The last rows of FP32 states whose latent arrays pass 2^32 bytes, copied and compacted."""
    cfg = models("kimi")[0]
    n = 2_200_000
    st, copy = State("f32", cfg, n), State("f32", cfg, n)
    lib.check(L.kvl_mla_compressed_state_fill_synthetic(st.ref(), 0, n, 77), "fill")
    lib.check(L.kvl_mla_compressed_state_fill_synthetic(copy.ref(), 0, n - 9, 78), "fill")
    rows, own = st.pull(n - 9, n), copy.pull(n - 12, n - 9)
    lib.check(L.kvl_mla_compressed_state_fork_batch_device(pointers([copy]), pointers([st]), ints([n - 9]), ints([n]), 1), "fork")
    for a, b, c in zip(copy.pull(n - 12, n), rows, own):
        np.testing.assert_array_equal(a[3:], b)
        np.testing.assert_array_equal(a[:3], c)
    lib.check(L.kvl_mla_compressed_state_accept_batch_device(pointers([copy]), ints([n - 9]), ints([3]), ints([1, 4, 8]), 1), "accept")
    for a, b in zip(copy.pull(n - 9, n - 6), rows):
        np.testing.assert_array_equal(a, b[[1, 4, 8]])
    for s in (st, copy):
        s.free()
