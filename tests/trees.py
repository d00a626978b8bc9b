"""What the tests of branching histories share: states with given rows, tree shapes, and the
definition of a tree decode in 64 bits."""
import ctypes as C

import numpy as np

from kvl_mla import abi, inputs, lib

TINY = dict(hidden_size=16, num_heads=2, qk_nope_dim=4, qk_rope_dim=4, v_head_dim=4, kv_lora_rank=6, rms_eps=1e-6,
            rope_theta=10000.0)
LAB = dict(hidden_size=64, num_heads=4, qk_nope_dim=8, qk_rope_dim=8, v_head_dim=8, kv_lora_rank=32, rms_eps=1e-6,
           rope_theta=10000.0)
KIMI = dict(inputs.KIMI)
# the attention's dims of KIMI with another head count: the route for any dims
NINE = dict(KIMI, num_heads=9, hidden_size=192)

TYPES = {"f32": abi.KvlMlaCompressedState, "bf16": abi.KvlMlaCompressedBF16State, "q8": abi.KvlMlaCompressedQ8State}
TAG = {"f32": "", "bf16": "bf16_", "q8": "q8_"}
BLOCK = {"f32": "kvl_mla_decode_compressed_block_bf16", "bf16": "kvl_mla_decode_compressed_bf16_block_bf16",
         "q8": "kvl_mla_decode_compressed_q8_block_bf16"}
ONE = {"f32": "kvl_mla_decode_compressed_bf16", "bf16": "kvl_mla_decode_compressed_bf16_bf16",
       "q8": "kvl_mla_decode_compressed_q8_bf16"}

# Share of an output's largest value that a result may be off. The products take their 32-bit operands
# as two bf16 parts, each rounded to nearest: what is left out is at most 2^-18 of the value, and for a
# product of two such operands (the fp32 rows) twice that. On the way from x to the output lie eight
# such products (x, q_nope, the query, the rows twice, the weights, the mix, the heads), and an error of
# a logit, itself up to the sum of three such terms of magnitude S, enters a weight S-fold. With
# S <= 12 (the inputs' logits): (8 + 3 * 12) 2^-18 = 1.7e-4.
TOL = 1.7e-4


def f32p(a):
    return a.ctypes.data_as(abi.f32p)


def ints(v):
    return (C.c_int * max(1, len(v)))(*[int(i) for i in v])


def fn(name, kind):
    """The entry point of a format; name holds a %s for its tag."""
    return getattr(lib.load(), "kvl_mla_" + name % TAG[kind])


class State:
    """A state whose host rows the test sets and reads."""

    def __init__(self, kind, cfg, capacity):
        self.kind, self.cfg, self.cap, self.s = kind, cfg, capacity, TYPES[kind]()
        lib.check(fn("compressed_%sstate_init", kind)(C.byref(self.s), C.byref(cfg), capacity), "init")

    def ref(self):
        return C.byref(self.s)

    def arrays(self):
        s, n, R, DR = self.s, self.cap, self.cfg.kv_lora_rank, self.cfg.qk_rope_dim
        view = lambda p, *shape: np.ctypeslib.as_array(p, (int(np.prod(shape)),)).reshape(shape)  # noqa: E731
        if self.kind == "q8":
            return [view(s.latent_q8, n, R), view(s.latent_scale, n), view(s.rope_bf16, n, DR)]
        return [view(s.latent, n, R), view(s.rope, n, DR)]

    def rows(self, lo, hi):
        return [a[lo:hi].copy() for a in self.arrays()]

    def load(self, seed, n, spread=1.0):
        """n rows of normalised latents and rotated keys, drawn from seed."""
        R, DR = self.cfg.kv_lora_rank, self.cfg.qk_rope_dim
        rng = np.random.default_rng(seed)
        lat = (spread * rng.standard_normal((n, R))).astype(np.float32)
        key = rng.standard_normal((n, DR)).astype(np.float32)
        a = self.arrays()
        if self.kind == "f32":
            a[0][:n], a[1][:n] = lat, key
        elif self.kind == "bf16":
            a[0][:n], a[1][:n] = inputs.f32_to_bf16_bits(lat), inputs.f32_to_bf16_bits(key)
        else:
            scale = (np.abs(lat).max(1) / np.float32(127)).astype(np.float32) if n else np.zeros(0, np.float32)
            a[0][:n] = np.clip(np.rint(lat / scale[:, None]), -127, 127).astype(np.int8)
            a[1][:n], a[2][:n] = scale, inputs.f32_to_bf16_bits(key)
        self.s.len = n
        lib.check(fn("compressed_%sstate_sync", self.kind)(self.ref()), "sync")
        return self

    def addresses(self):
        """The device arrays, rows [0, len) of the host uploaded where they were not yet."""
        p = [C.c_void_p() for _ in self.arrays()]
        lib.check(fn("compressed_%sstate_device_rows", self.kind)(self.ref(), *[C.byref(q) for q in p]), "device rows")
        return [q.value for q in p]

    def upload(self):
        self.addresses()
        return self

    def pull(self, lo, hi):
        if hi > lo:
            lib.check(fn("compressed_%sstate_pull", self.kind)(self.ref(), lo, hi - lo), "pull")
        return self.rows(lo, hi)

    def free(self):
        fn("compressed_%sstate_free", self.kind)(self.ref())


def values(rows, kind):
    """Stored rows as 64-bit latents and keys."""
    if kind == "q8":
        return rows[0].astype(np.float64) * rows[1].astype(np.float64)[:, None], inputs.bf16_bits_to_f32(rows[2]).astype(np.float64)
    if kind == "bf16":
        return tuple(inputs.bf16_bits_to_f32(r).astype(np.float64) for r in rows)
    return tuple(r.astype(np.float64) for r in rows)


def tree(shape, n, seed=0):
    rng = np.random.default_rng(seed)
    if shape == "chain":
        return list(range(-1, n - 1))
    if shape == "star":
        return [-1] * n
    return [-1] + [int(rng.integers(-1, i)) for i in range(1, n)]


def path_to(parents, i):
    p = []
    while i >= 0:
        p.insert(0, i)
        i = parents[i]
    return p


def f64(bits):
    return inputs.bf16_bits_to_f32(bits).astype(np.float64)


def rms64(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def reference(cfg, layer, x, parents, ctx, rows, kind, nodes=None):
    """out [count, hidden] of a tree decode in 64 bits over `rows`, the state's rows [0, ctx + count)
    as it stores them (the appended ones among them); of the given nodes only, if any are given."""
    NH, DN, DR, DV, R = cfg.num_heads, cfg.qk_nope_dim, cfg.qk_rope_dim, cfg.v_head_dim, cfg.kv_lora_rank
    lat, key = values(rows, kind)
    kvb = f64(layer.kv_b_proj).reshape(NH, DN + DV, R)
    wo = f64(layer.o_proj)
    q = (x.astype(np.float64) @ f64(layer.q_proj).T).reshape(-1, NH, DN + DR)
    inv = cfg.rope_theta ** (-2.0 * np.arange(DR // 2) / DR)
    out = []
    for i in range(len(parents)) if nodes is None else nodes:
        p = path_to(parents, i)
        a = (ctx + len(p) - 1) * inv
        e, o = q[i, :, DN::2], q[i, :, DN + 1::2]
        qr = np.concatenate([e * np.cos(a) - o * np.sin(a), o * np.cos(a) + e * np.sin(a)], -1)
        ql = np.einsum("hd,hdr->hr", q[i, :, :DN], kvb[:, :DN])
        at = list(range(ctx)) + [ctx + j for j in p]
        s = (ql @ lat[at].T + qr @ key[at].T) / np.sqrt(DN + DR)
        w = np.exp(s - s.max(1, keepdims=True))
        mix = (w / w.sum(1, keepdims=True)) @ lat[at]
        out.append(wo @ np.einsum("hr,hdr->hd", mix, kvb[:, DN:]).reshape(-1))
    return np.array(out)


def new_rows(cfg, layer, x, parents, ctx):
    """The tree's rows in 64 bits, before they are stored: latents [count, R], keys [count, DR]."""
    R, DR = cfg.kv_lora_rank, cfg.qk_rope_dim
    kva = x.astype(np.float64) @ f64(layer.kv_a_proj).T
    lat = rms64(kva[:, :R], f64(layer.kv_a_norm), cfg.rms_eps)
    pos = np.array([ctx + len(path_to(parents, i)) - 1 for i in range(len(parents))])
    a = pos[:, None] * cfg.rope_theta ** (-2.0 * np.arange(DR // 2) / DR)
    e, o = kva[:, R::2], kva[:, R + 1::2]
    return lat, np.concatenate([e * np.cos(a) - o * np.sin(a), o * np.cos(a) + e * np.sin(a)], -1)


def off(got, want):
    """Largest difference as a share of the largest value."""
    return float(np.abs(got.astype(np.float64) - want).max() / max(np.abs(want).max(), 1e-30))


def tree_host(st, layer, x, parents, w=None):
    """The host-buffer call; its outputs."""
    w = w or layer.struct()
    out = np.full((len(parents), st.cfg.hidden_size), np.float32(np.nan))
    lib.check(fn("decode_compressed_%stree_bf16", st.kind)(f32p(out), f32p(x), ints(parents), len(parents), st.s.len,
                                                          C.byref(st.cfg), C.byref(w), st.ref()), "tree")
    return out


def pointers(states):
    T = TYPES[states[0].kind]
    return (C.POINTER(T) * len(states))(*[C.pointer(s.s) for s in states])


class Device:
    """A device buffer holding an array."""

    def __init__(self, a):
        L = lib.load()
        self.shape, self.nbytes = a.shape, a.nbytes
        self.p = L.kvl_mla_device_alloc(a.nbytes + 16)
        self.put(a)

    def put(self, a):
        a = np.ascontiguousarray(a)
        lib.check(lib.load().kvl_mla_copy_to_device(self.p, a.ctypes.data, a.nbytes), "h2d")

    def get(self):
        out = np.empty(self.shape, np.float32)
        lib.check(lib.load().kvl_mla_copy_to_host(out.ctypes.data, self.p, out.nbytes), "d2h")
        return out

    def free(self):
        lib.load().kvl_mla_device_free(self.p)
