"""The operators of branching histories, as measurable cases: drafts in the shape of a tree, copies of
a history, and the step back to one accepted path.

A case is one pass at the Kimi-VL MLA shapes (hidden 2048, 16 heads, kv_lora_rank 512, nope 128,
rope 64, v 128):

  tree    the drafted tokens of each sequence, nodes of a tree over its latent history (fp32, bf16 or
          row-wise Q8), through one layer's attention: every node attends the history, its ancestors
          and itself, and its row is appended. Stream-ordered over device buffers; `host`: one
          sequence through host buffers, as a token loop calls a layer; `layer`: with the norms and
          the residual sum around it. A tree of one node is the decode of a single token;
  fork    states become copies of others: the rows lo .. hi - 1 of each;
  accept  after a verified tree: the draft rows come over from the state that holds them, and the
          accepted path's rows stay, moved up to the context.

Hidden states are values of a bf16 model. Where `own` is false the same is computed by elementary
torch operations, in 32 bits; the latent rows in 64, since their rounding to codes or to bf16 has
borders.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

H, NH, DN, DR, DV, R = 2048, 16, 128, 64, 128, 512
QD = DN + DR
EPS, THETA = 1e-5, 50000.0
ROW_BYTES = {"f32": 4 * (R + DR), "bf16": 2 * (R + DR), "q8": R + 4 + 2 * DR}
WEIGHT_BYTES = 2 * (NH * QD * H + (R + DR) * H + R + NH * (DN + DV) * R + H * NH * DV)


def listed():
    return [
        # a short chat, a few drafted continuations
        {"name": "tree_f32_400_7", "kind": "tree", "state": "f32", "batch": 1, "lo": 400, "hi": 400, "nodes": 7, "host": False, "layer": False},
        # the generator's own loop: one sequence, host buffers, an odd tree over 9000 rows
        {"name": "tree_q8_9000_13_host", "kind": "tree", "state": "q8", "batch": 1, "lo": 9000, "hi": 9000, "nodes": 13, "host": True, "layer": False},
        # sequences whose drafter proposed nothing: single tokens, mixed ages
        {"name": "tree_bf16_13x1", "kind": "tree", "state": "bf16", "batch": 13, "lo": 600, "hi": 20000, "nodes": 1, "host": False, "layer": False},
        # a serving batch with trees of up to 24 nodes
        {"name": "tree_bf16_8x24", "kind": "tree", "state": "bf16", "batch": 8, "lo": 1000, "hi": 12000, "nodes": 24, "host": False, "layer": False},
        # a full-precision state through the attention half of a decoder layer
        {"name": "tree_f32_3x17_layer", "kind": "tree", "state": "f32", "batch": 3, "lo": 700, "hi": 9000, "nodes": 17, "host": False, "layer": True},
        # one long sequence, the widest tree
        {"name": "tree_q8_32k_64", "kind": "tree", "state": "q8", "batch": 1, "lo": 32768, "hi": 32768, "nodes": 64, "host": False, "layer": False},
        # 8 sequences of 32K tokens, trees of 32
        {"name": "tree_q8_8x32k_32", "kind": "tree", "state": "q8", "batch": 8, "lo": 32768, "hi": 32768, "nodes": 32, "host": False, "layer": False},
        # two branches from a short prompt
        {"name": "fork_f32_2x900", "kind": "fork", "state": "f32", "pairs": 2, "one": True, "lo": 0, "hi": 900},
        # beams changing places: each takes over what another has beyond their common rows
        {"name": "fork_bf16_6x_tail", "kind": "fork", "state": "bf16", "pairs": 6, "one": False, "lo": 2311, "hi": 7777},
        # four samples of one 32K context
        {"name": "fork_q8_4x32k", "kind": "fork", "state": "q8", "pairs": 4, "one": True, "lo": 0, "hi": 32768},
        # a verified tree of 13 nodes, five of them accepted, in the states of 27 layers
        {"name": "accept_bf16_27", "kind": "accept", "state": "bf16", "states": 27, "ctx": 2100, "nodes": 13, "keep": 5},
        # one layer's states of 20 sequences, the widest trees, a long path
        {"name": "accept_q8_20", "kind": "accept", "state": "q8", "states": 20, "ctx": 5000, "nodes": 64, "keep": 17},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "fork", "accept"])
    state = rng.choice(["f32", "bf16", "q8"])
    if kind == "tree":
        # the shortest histories go to the full-precision state, the longest to the coded one
        low, high = {"f32": (1, 9000), "bf16": (500, 20000), "q8": (5000, 32768)}[state]
        batch = rng.choice([1, 1, _log_int(rng, 2, 13)])
        lo = _log_int(rng, low, high)
        hi = _log_int(rng, lo, high)
        nodes = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 2, 64)])
        nodes = max(1, min(nodes, 5_000_000 // (batch * hi), 512 // batch))
        return {"kind": "tree", "state": state, "batch": batch, "lo": lo, "hi": hi, "nodes": nodes,
                "host": batch == 1 and rng.random() < 0.4, "layer": state == "f32" and batch > 1 and rng.random() < 0.4}
    if kind == "fork":
        hi = _log_int(rng, 1, 32768)
        return {"kind": "fork", "state": state, "pairs": rng.randint(1, 6 if state != "f32" else 3), "one": rng.random() < 0.5,
                "lo": rng.choice([0, rng.randint(0, hi - 1)]), "hi": hi}
    nodes = _log_int(rng, 1, 64)
    return {"kind": "accept", "state": state, "states": _log_int(rng, 1, 20 if state == "q8" else 27), "ctx": _log_int(rng, 1, 8000),
            "nodes": nodes, "keep": rng.randint(1, nodes)}


# ------------------------------------------------------------------ inputs ----------------

def _gen(seed, *tags):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + sum((i + 1) * 7919 * int(t) for i, t in enumerate(tags))) % (1 << 62))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _weights(seed):
    """bf16 weights on the GPU: matrices N(0, 0.02), the norms 1 + N(0, 0.02)."""
    g = _gen(seed, 1)
    w = {"q": 0.02 * _randn(g, NH * QD, H), "kva": 0.02 * _randn(g, R + DR, H), "norm": 1 + 0.02 * _randn(g, R),
         "kvb": 0.02 * _randn(g, NH * (DN + DV), R), "o": 0.02 * _randn(g, H, NH * DV),
         "n1": 1 + 0.02 * _randn(g, H), "n2": 1 + 0.02 * _randn(g, H)}
    return {k: v.to(torch.bfloat16) for k, v in w.items()}


def _rows(seed, i, n, state):
    """n rows as the library stores them: normalised latents and rotated keys of unit scale."""
    g = _gen(seed, 2, i)
    lat, key = _randn(g, n, R), 0.9 * _randn(g, n, DR)
    if state == "f32":
        return [lat, key]
    if state == "bf16":
        return [lat.to(torch.bfloat16), key.to(torch.bfloat16)]
    scale = lat.abs().amax(1) / 127
    return [torch.clamp(torch.round(lat / scale[:, None]), -127, 127).to(torch.int8), scale, key.to(torch.bfloat16)]


def _lengths(case):
    """The histories' lengths: fixed by the case, spread over lo .. hi."""
    rng = np.random.default_rng(1000003 * case["batch"] + 1009 * case["lo"] + case["hi"])
    return [int(n) for n in rng.integers(case["lo"], case["hi"] + 1, size=case["batch"])]


def _trees(case):
    """Each sequence's tree as parents (-1: a child of the history's last token), fixed by the case:
    the first sequence has `nodes` nodes, the others between a third of them and all; a node hangs
    on the context, on one of the latest nodes, or anywhere."""
    rng = random.Random(31 * case["nodes"] + case["lo"])
    trees = []
    for b in range(case["batch"]):
        n = case["nodes"] if b == 0 else rng.randint((case["nodes"] + 2) // 3, case["nodes"])
        trees.append([rng.choice([-1, rng.randint(max(0, i - 4), i - 1), rng.randint(0, i - 1)]) if i else -1 for i in range(n)])
    return trees


def _path(case):
    """The accepted nodes of each state's tree (the states of a case share it), fixed by the case."""
    return sorted(random.Random(7 * case["nodes"] + case["keep"]).sample(range(case["nodes"]), case["keep"]))


def _starts(case):
    """The contexts' lengths of an accept: one for all layers of a sequence, or each its own."""
    rng = np.random.default_rng(case["ctx"])
    return [case["ctx"] if case["state"] == "bf16" else int(n)
            for n in rng.integers((case["ctx"] + 1) // 2, case["ctx"] + 1, size=case["states"])]


def _x(case, seed):
    n = sum(len(t) for t in _trees(case))
    return _randn(_gen(seed, 3), n, H).to(torch.bfloat16).float()


def _padded(rows, cap):
    """Rows of several states in one array, [states, cap, ...]."""
    return [torch.stack([torch.nn.functional.pad(r[k], (0, 0) * (r[k].dim() - 1) + (0, cap - r[k].shape[0])) for r in rows])
            for k in range(len(rows[0]))]


def prepare(case, seed):
    st = {"case": case}
    if case["kind"] == "tree":
        lens, trees = _lengths(case), _trees(case)
        st["w"], x = _weights(seed), _x(case, seed)
        rows = [_rows(seed, i, n, case["state"]) for i, n in enumerate(lens)]
        st["x"] = x.cpu().numpy() if case["host"] else x
        if own:
            _prepare_tree(st, rows, lens, trees)
        else:
            T, B, n = max(len(t) for t in trees), case["batch"], x.shape[0]
            depth, anc, place, at = [], np.zeros((B, T, T), bool), np.full((B, T), n, np.int64), 0
            for b, t in enumerate(trees):
                dep = []
                for i, p in enumerate(t):
                    dep.append(0 if p < 0 else dep[p] + 1)
                    anc[b, i] = anc[b, p] if p >= 0 else False
                    anc[b, i, i] = True
                    place[b, i] = at + i
                anc[b, len(t):, 0] = True  # places without a node: any row
                depth += [lens[b] + d for d in dep]
                at += len(t)
            st["rows"] = _padded(rows, max(lens))
            st["past"] = torch.arange(max(lens), device="cuda")[None, :] >= torch.tensor(lens, device="cuda")[:, None]
            st["hide"] = ~torch.from_numpy(anc).cuda()
            st["place"] = torch.from_numpy(place).cuda()
            st["back"] = torch.from_numpy(np.flatnonzero(place.reshape(-1) < n)).cuda()
            st["pos"] = torch.tensor(depth, device="cuda")
            st["sizes"] = [len(t) for t in trees]
    elif case["kind"] == "fork":
        sources = 1 if case["one"] else case["pairs"]
        src = [_rows(seed, i, case["hi"], case["state"]) for i in range(sources)]
        kept = [_rows(seed, 64 + i, case["lo"], case["state"]) for i in range(case["pairs"])]
        if own:
            _prepare_fork(st, src, kept)
        else:
            st["src"] = _padded(src, case["hi"])
            st["dst"] = _padded(kept, case["hi"])
    else:
        starts, keep = _starts(case), _path(case)
        src = [_rows(seed, i, n + case["nodes"], case["state"]) for i, n in enumerate(starts)]
        if own:
            _prepare_accept(st, src, starts, keep)
        else:
            cap = max(starts) + case["nodes"]
            st["src"], st["dst"] = _padded(src, cap), _padded(src, cap)
            first = torch.tensor(starts, device="cuda")[:, None]
            st["who"] = torch.arange(case["states"], device="cuda")[:, None]
            st["all"] = first + torch.arange(case["nodes"], device="cuda")
            st["from"] = first + torch.tensor(keep, device="cuda")
            st["to"] = first + torch.arange(case["keep"], device="cuda")
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------------ plain form ------------

def _rotate(v, positions):
    """Pairs (2i, 2i + 1) of the last dimension to (i, DR / 2 + i), rotated by position."""
    inv = THETA ** (-2 * torch.arange(DR // 2, dtype=torch.float64, device=v.device) / DR)
    a = (positions.double()[:, None] * inv).reshape((-1,) + (1,) * (v.dim() - 2) + (DR // 2,))
    c, s = torch.cos(a).to(v.dtype), torch.sin(a).to(v.dtype)
    return torch.cat([v[..., 0::2] * c - v[..., 1::2] * s, v[..., 1::2] * c + v[..., 0::2] * s], -1)


def _norm(x, w):
    return x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w.to(x.dtype)


def _stored(lat, key, state):
    """New rows as the state holds them, from 64 bits."""
    if state == "f32":
        return [lat.float(), key.float()]
    if state == "bf16":
        return [lat.float().to(torch.bfloat16), key.float().to(torch.bfloat16)]
    scale = lat.abs().amax(1) / 127
    return [torch.clamp(torch.round(lat / scale[:, None]), -127, 127).to(torch.int8), scale.float(), key.float().to(torch.bfloat16)]


def _values(rows, state):
    """Stored rows as 32-bit latents and keys."""
    if state == "q8":
        return rows[0].float() * rows[1][..., None], rows[2].float()
    return rows[0].float(), rows[1].float()


def _plain_tree(st):
    case, w, state = st["case"], st["w"], st["case"]["state"]
    x = torch.from_numpy(st["x"]).cuda() if case["host"] else st["x"]
    h, x = x, _norm(x, w["n1"]) if case["layer"] else x
    B, T = st["place"].shape
    q = (x @ w["q"].float().T).reshape(-1, NH, QD)
    kva = x.double() @ w["kva"].double().T
    new = _stored(_norm(kva[:, :R], w["norm"]), _rotate(kva[:, R:], st["pos"]), state)
    kvb = w["kvb"].float().reshape(NH, DN + DV, R)
    q = torch.cat([torch.bmm(q[..., :DN].transpose(0, 1).contiguous(), kvb[:, :DN].contiguous()).transpose(0, 1),
                   _rotate(q[..., DN:], st["pos"])], -1) / math.sqrt(QD)
    q = torch.cat([q, torch.zeros_like(q[:1])])[st["place"]].reshape(B, T * NH, R + DR)
    lat, key = _values(st["rows"], state)
    nlat, nkey = _values(new, state)
    pad = lambda v: torch.cat([v, torch.zeros_like(v[:1])])[st["place"]]  # noqa: E731
    nlat, nkey = pad(nlat), pad(nkey)
    s = torch.bmm(q, torch.cat([lat, key], -1).transpose(1, 2).contiguous())
    s = s.masked_fill_(st["past"][:, None, :], -math.inf)
    sn = torch.bmm(q, torch.cat([nlat, nkey], -1).transpose(1, 2).contiguous()).reshape(B, T, NH, T)
    sn = sn.masked_fill_(st["hide"][:, :, None, :], -math.inf).reshape(B, T * NH, T)
    m = torch.maximum(s.amax(-1, keepdim=True), sn.amax(-1, keepdim=True))
    p, pn = torch.exp_(s.sub_(m)), torch.exp_(sn.sub_(m))
    mix = (torch.bmm(p, lat) + torch.bmm(pn, nlat)) / (p.sum(-1, keepdim=True) + pn.sum(-1, keepdim=True))
    mix = mix.reshape(B * T, NH, R)[st["back"]]
    heads = torch.bmm(mix.transpose(0, 1).contiguous(), kvb[:, DN:].transpose(1, 2).contiguous()).transpose(0, 1).reshape(-1, NH * DV)
    out = heads @ w["o"].float().T
    if case["host"]:
        if state == "q8":
            new = [(new[0].float() * new[1][:, None]).to(torch.bfloat16), new[2]]
        return {"out": out.cpu(), "rows": [v.cpu() for v in new]}
    if state == "q8":
        new = new[1:]
    new = [list(v.split(st["sizes"])) for v in new]
    if case["layer"]:
        return {"h": h + out, "n2": _norm(h + out, w["n2"]), "rows": new}
    return {"out": out, "rows": new}


def run(st):
    if own:
        return _run(st)
    case = st["case"]
    if case["kind"] == "tree":
        return _plain_tree(st)
    if case["kind"] == "fork":
        for d, s in zip(st["dst"], st["src"]):
            d[:, case["lo"]:] = s[:, case["lo"]:]
        return [list(d) for d in st["dst"]]
    for d, s in zip(st["dst"], st["src"]):
        d[st["who"], st["all"]] = s[st["who"], st["all"]]
        d[st["who"], st["to"]] = d[st["who"], st["from"]]
    return [[d[i, n:n + case["keep"]] for i, n in enumerate(_starts(case))] for d in st["dst"]]


def work(case):
    rb = ROW_BYTES[case["state"]]
    if case["kind"] == "fork":  # one read of each source, one write of each copy
        n = case["hi"] - case["lo"]
        return {"bytes": rb * n * (case["pairs"] + (1 if case["one"] else case["pairs"])), "flops": 0}
    if case["kind"] == "accept":  # the draft rows come over, the accepted ones move
        return {"bytes": 2 * rb * case["states"] * (case["nodes"] + case["keep"]), "flops": 0}
    lens, trees = _lengths(case), _trees(case)
    nodes = sum(len(t) for t in trees)
    pairs = 0
    for n, t in zip(lens, trees):
        depth = []
        for p in t:
            depth.append(0 if p < 0 else depth[p] + 1)
        pairs += sum(n + d + 1 for d in depth)
    return {"bytes": WEIGHT_BYTES + rb * (sum(lens) + nodes) + (3 if case["layer"] else 2) * 4 * H * nodes,
            "flops": nodes * WEIGHT_BYTES + 2 * pairs * NH * (2 * R + DR)}


# ------------------------------------------------------------------ 64-bit results --------

def exact(case, seed):
    """Node by node: the rows that a node sees are gathered, and its attention taken over them."""
    if case["kind"] != "tree":
        return None
    w = {k: v.double() for k, v in _weights(seed).items()}
    lens, trees, state = _lengths(case), _trees(case), case["state"]
    x = h = _x(case, seed).double()
    if case["layer"]:
        x = x / (x.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w["n1"]
    freq = torch.tensor([THETA ** (-2.0 * i / DR) for i in range(DR // 2)], dtype=torch.float64, device="cuda")

    def turn(v, pos):
        z = torch.complex(v[..., 0::2], v[..., 1::2]) * torch.polar(torch.ones_like(freq), pos * freq)
        return torch.cat([z.real, z.imag], -1)

    up, down = w["kvb"].reshape(NH, DN + DV, R)[:, :DN], w["kvb"].reshape(NH, DN + DV, R)[:, DN:]
    outs, lats, keys, at = [], [], [], 0
    for b, (n, tree) in enumerate(zip(lens, trees)):
        hist = _rows(seed, b, n, state)
        hl = hist[0].double() * hist[1].double()[:, None] if state == "q8" else hist[0].double()
        hk = hist[-1].double()
        nl, nk, seen = [], [], []
        for i, p in enumerate(tree):
            seen.append(([] if p < 0 else seen[p]) + [i])
            pos = n + len(seen[i]) - 1
            c = w["kva"] @ x[at + i]
            lat = c[:R] / (c[:R].pow(2).mean() + EPS).sqrt() * w["norm"]
            key = turn(c[R:], pos)
            lats.append(lat)
            keys.append(key)
            if state == "q8":
                step = lat.abs().max() / 127
                lat = (lat / step).round().clamp(-127, 127) * step
            elif state == "bf16":
                lat = lat.to(torch.bfloat16).double()
            nl.append(lat)
            nk.append(key if state == "f32" else key.to(torch.bfloat16).double())
            q = (w["q"] @ x[at + i]).reshape(NH, QD)
            qa, qr = (q[:, None, :DN] @ up)[:, 0], turn(q[:, DN:], pos)
            el, ek = torch.stack([nl[j] for j in seen[i]]), torch.stack([nk[j] for j in seen[i]])
            s = torch.cat([qa @ hl.T + qr @ hk.T, qa @ el.T + qr @ ek.T], 1) / math.sqrt(QD)
            p_ = torch.softmax(s, 1)
            mix = p_[:, :n] @ hl + p_[:, n:] @ el
            outs.append(w["o"] @ (down @ mix[..., None]).reshape(-1))
        at += len(tree)
    out = torch.stack(outs)
    if case["host"]:
        return {"out": out, "rows": [torch.stack(lats), torch.stack(keys)] if state == "f32" else [None, None]}
    rows = [None, None]
    if state == "f32":
        rows = [list(torch.stack(v).split([len(t) for t in trees])) for v in (lats, keys)]
    if case["layer"]:
        r = h + out
        return {"h": r, "n2": r / (r.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w["n2"], "rows": rows}
    return {"out": out, "rows": rows}


# ------------------------------------------------------------------ the framework ---------

CALL = {"f32": "", "bf16": "bf16_", "q8": "q8_"}


def _library():
    path = os.path.join(os.getcwd(), "in-c-test_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from kvl_mla import abi, lib
    return abi, lib


def _bits(t):
    t = t.contiguous()
    return (t.view(torch.int16) if t.dtype == torch.bfloat16 else t).cpu().numpy()


class _Weights:
    """A layer's weights bound to the library for as long as a program keeps them."""

    def __init__(self, cfg, w):
        import ctypes as C
        abi, lib = _library()
        self.w = {k: _bits(v).view(np.uint16) for k, v in w.items()}
        p = {k: abi.ptr(v, C.c_uint16) for k, v in self.w.items()}
        self.struct = abi.KvlMlaBF16(p["q"], p["kva"], p["norm"], p["kvb"], p["o"])
        self.n1, self.n2 = p["n1"], p["n2"]
        self.release = lib.load().kvl_mla_release_weights
        lib.check(lib.load().kvl_mla_bind_weights(C.byref(cfg), C.byref(self.struct)), "bind weights")

    def __del__(self):
        import ctypes as C
        self.release(C.byref(self.struct))


class _Device:
    """What torch takes a device buffer from: its address, shape and type, and the state that owns it."""

    def __init__(self, owner, address, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (address, False), "version": 2}


class _State:
    """One sequence's state, its rows on host and device."""

    def __init__(self, cfg, state, capacity, rows):
        import ctypes as C
        abi, lib = _library()
        self.kind, self.capacity, L = state, capacity, lib.load()
        self.type = {"f32": abi.KvlMlaCompressedState, "bf16": abi.KvlMlaCompressedBF16State, "q8": abi.KvlMlaCompressedQ8State}[state]
        self.s, name = self.type(), "kvl_mla_compressed_%sstate_" % CALL[state]
        self.free = getattr(L, name + "free")
        self.truncate = getattr(L, name + "truncate")
        lib.check(getattr(L, name + "init")(C.byref(self.s), C.byref(cfg), capacity), "state init")
        n = rows[0].shape[0]
        for a, t in zip(self.host(), rows):
            a[:n] = _bits(t).view(a.dtype)
        self.s.len = n
        at = [C.c_void_p() for _ in rows]
        lib.check(getattr(L, name + "device_rows")(C.byref(self.s), *[C.byref(p) for p in at]), "device rows")
        self.at = [p.value for p in at]

    def host(self):
        import ctypes as C
        s, cap = self.s, self.capacity

        def of(p, *shape):
            a = (p._type_ * math.prod(shape)).from_address(C.addressof(p.contents))
            a.owner = self  # the rows live as long as a view of them
            return np.ctypeslib.as_array(a).reshape(shape)

        if self.kind == "q8":
            return [of(s.latent_q8, cap, R), of(s.latent_scale, cap), of(s.rope_bf16, cap, DR)]
        return [of(s.latent, cap, R), of(s.rope, cap, DR)]

    def device(self, lo, hi):
        """Rows lo .. hi - 1 on the device, as tensors that look into the state."""
        half = {"f32": ["<f4", "<f4"], "bf16": ["<i2", "<i2"], "q8": ["|i1", "<f4", "<i2"]}[self.kind]
        shape = {"q8": [(self.capacity, R), (self.capacity,), (self.capacity, DR)]}.get(self.kind, [(self.capacity, R), (self.capacity, DR)])
        got = [torch.as_tensor(_Device(self, p, s, k), device="cuda") for p, s, k in zip(self.at, shape, half)]
        return [(t.view(torch.bfloat16) if t.dtype == torch.int16 else t)[lo:hi] for t in got]

    def __del__(self):
        import ctypes as C
        self.free(C.byref(self.s))


def _pointers(states):
    import ctypes as C
    return (C.POINTER(states[0].type) * len(states))(*[C.pointer(s.s) for s in states])


def _ints(v):
    import ctypes as C
    return (C.c_int * len(v))(*v)


def _begin(st):
    import ctypes as C
    abi, lib = _library()
    st["L"], st["lib"], st["cfg"] = lib.load(), lib, abi.KvlMlaConfig(H, NH, DN, DR, DV, R, EPS, THETA)
    lib.check(st["L"].kvl_mla_init(), "init")
    st["cfgp"] = C.byref(st["cfg"])


def _prepare_tree(st, rows, lens, trees):
    import ctypes as C
    case = st["case"]
    _begin(st)
    st["w"] = _Weights(st["cfg"], st["w"])
    st["wp"] = C.byref(st["w"].struct)
    st["states"] = [_State(st["cfg"], case["state"], n + len(t), r) for n, t, r in zip(lens, trees, rows)]
    st["arr"] = _pointers(st["states"])
    st["counts"], st["parents"] = _ints([len(t) for t in trees]), _ints([p for t in trees for p in t])
    name = "kvl_mla_decode_compressed_%stree_" % CALL[case["state"]]
    if case["host"]:
        s, n, t = st["states"][0], lens[0], len(trees[0])
        st["fn"], st["out"], st["start"] = getattr(st["L"], name + "bf16"), np.zeros((t, H), np.float32), n
        st["rows"] = [a[n:n + t] for a in s.host()]
    else:
        st["fn"] = getattr(st["L"], "kvl_mla_attention_layer_%stree_device" % CALL[case["state"]] if case["layer"] else name + "batch_device")
        st["out"] = torch.empty_like(st["x"])
        got = [s.device(n, n + len(t)) for s, n, t in zip(st["states"], lens, trees)]
        st["rows"] = [list(v) for v in zip(*got)][1 if case["state"] == "q8" else 0:]
        if case["layer"]:
            st["h"] = torch.empty_like(st["x"])


def _prepare_fork(st, src, kept):
    case = st["case"]
    _begin(st)
    st["src"] = [_State(st["cfg"], case["state"], case["hi"], r) for r in src]
    st["dst"] = [_State(st["cfg"], case["state"], case["hi"], r) for r in kept]
    st["from"] = _pointers([st["src"][0 if case["one"] else i] for i in range(case["pairs"])])
    st["to"] = _pointers(st["dst"])
    st["lo"], st["hi"] = _ints([case["lo"]] * case["pairs"]), _ints([case["hi"]] * case["pairs"])
    st["fn"] = getattr(st["L"], "kvl_mla_compressed_%sstate_fork_batch_device" % CALL[case["state"]])
    st["rows"] = [list(v) for v in zip(*[s.device(0, case["hi"]) for s in st["dst"]])]


def _prepare_accept(st, src, starts, keep):
    case = st["case"]
    n, k = case["states"], case["keep"]
    _begin(st)
    st["src"] = [_State(st["cfg"], case["state"], a + case["nodes"], r) for a, r in zip(starts, src)]
    st["dst"] = [_State(st["cfg"], case["state"], a + case["nodes"], r) for a, r in zip(starts, src)]
    st["from"], st["to"] = _pointers(st["src"]), _pointers(st["dst"])
    st["lo"], st["hi"] = _ints(starts), _ints([a + case["nodes"] for a in starts])
    st["counts"], st["path"] = _ints([k] * n), _ints(keep * n)
    name = "kvl_mla_compressed_%sstate_" % CALL[case["state"]]
    st["fork"], st["accept"] = getattr(st["L"], name + "fork_batch_device"), getattr(st["L"], name + "accept_batch_device")
    st["rows"] = [list(v) for v in zip(*[s.device(a, a + k) for s, a in zip(st["dst"], starts)])]


def _run(st):
    import ctypes as C
    case, L, lib = st["case"], st["L"], st["lib"]
    if case["kind"] == "fork":
        lib.check(st["fn"](st["to"], st["from"], st["lo"], st["hi"], case["pairs"]), "fork")
        return st["rows"]
    if case["kind"] == "accept":
        n = case["states"]
        lib.check(st["fork"](st["to"], st["from"], st["lo"], st["hi"], n), "fork")
        lib.check(st["accept"](st["to"], st["lo"], st["counts"], st["path"], n), "accept")
        return st["rows"]
    out, x = st["out"], st["x"]
    if case["host"]:  # every draft rejected: the state is back at the context afterwards
        p = lambda a: a.ctypes.data_as(C.POINTER(C.c_float))  # noqa: E731
        s = st["states"][0]
        lib.check(st["fn"](p(out), p(x), st["parents"], case["nodes"], st["start"], st["cfgp"], st["wp"], st["arr"][0]), "tree")
        lib.check(s.truncate(st["arr"][0], st["start"]), "truncate")
        rows = [torch.from_numpy(a) for a in st["rows"]]
        if case["state"] == "q8":
            rows = [(rows[0].float() * rows[1][:, None]).to(torch.bfloat16), rows[2]]
        return {"out": out, "rows": [r.view(torch.bfloat16) if r.dtype == torch.uint16 else r for r in rows]}
    if case["layer"]:
        h = st["h"]
        rc = L.kvl_mla_copy_kernel(h.data_ptr(), x.data_ptr(), 4 * x.numel())
        rc |= st["fn"](h.data_ptr(), out.data_ptr(), st["counts"], st["parents"], case["batch"], st["cfgp"], st["wp"], st["w"].n1,
                       st["w"].n2, st["arr"], lib.NO_ADVANCE)
        lib.check(rc, "layer")
        return {"h": h, "n2": out, "rows": st["rows"]}
    lib.check(st["fn"](out.data_ptr(), x.data_ptr(), st["counts"], st["parents"], case["batch"], st["cfgp"], st["wp"], st["arr"],
                       lib.NO_ADVANCE), "tree")
    return {"out": out, "rows": st["rows"]}
