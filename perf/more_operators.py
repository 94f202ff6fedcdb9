"""Linear attention with a decay for each head, and the end of a block, as cases that can be timed.

Four kinds of pass:

* ``scan``:  linear attention with a decay for each head over whole sequences
             (``head_decay_scan``), with packed segments, an initial state and shared key heads
             where the case says so;
* ``train``: the same forward and its gradients, that of the decays among them where the case
             learns them;
* ``step``:  one token of a served batch (``head_decay_step``);
* ``join``:  the end of a block (``block_join``): the norm after it, its gate, dropout from a
             counter-based generator, the residual scale and sum, and the next block's norm; with
             the gradients where the case trains.

``own`` chooses between the framework's kernels and the plain form: elementary torch operations
in 32 bits, rounded once at the end.  ``exact`` computes a case in 64 bits: the recurrence token
by token, the block's end and its gradients from their formulas.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
CHUNK = 64
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _scan(name, nb, T, r, p, heads, dtype="bf16", nbk=None, segments=1, state=False,
          learn=False, kind="scan"):
    return {"name": name, "kind": kind, "nb": nb, "nbk": nbk or nb, "T": T, "r": r, "p": p,
            "heads": heads, "dtype": dtype, "segments": segments, "state": state, "learn": learn}


def _train(name, nb, T, r, p, heads, **kw):
    return _scan(name, nb, T, r, p, heads, kind="train", **kw)


def _step(name, nb, r, p, heads, dtype="bf16", nbk=None):
    return {"name": name, "kind": "step", "nb": nb, "nbk": nbk or nb, "r": r, "p": p,
            "heads": heads, "dtype": dtype}


def _join(name, rows, D, dtype="bf16", stream="fp32", gate="sigmoid", post=True, vector=True,
          drop=0.0, grads=False):
    """``stream``: the residual stream's type; ``vector``: a residual scale for each column."""
    return {"name": name, "kind": "join", "rows": rows, "D": D, "dtype": dtype, "stream": stream,
            "gate": gate, "post": post, "vector": vector, "drop": drop, "grads": grads}


def listed():
    return [
        # a turn's last 7 tokens on a kept state: launches and host latency
        _scan("scan_T7", 8, 7, 64, 64, 8, state=True),
        # an ordinary batch of prompts at head size 64 (B = 4, H = 8)
        _scan("scan_T8192_hd64", 32, 8192, 64, 64, 8),
        # prompts of different odd lengths packed one behind the other, fp16, two value heads a
        # key head, head size 96, states kept
        _scan("scan_packed_hd96", 12, 10007, 96, 96, 12, dtype="fp16", nbk=6, segments=5,
              state=True),
        # one long prompt, 8 heads of 128
        _scan("scan_T131072_hd128", 8, 131072, 128, 128, 8),
        # training steps of a small model's layer (B = 8, H = 12)
        _train("train_T4096_hd64", 96, 4096, 64, 64, 12),
        # a layer with two value heads a key head over packed documents whose decays are
        # learned, head size 128
        _train("train_packed_hd128", 16, 8192, 128, 128, 8, nbk=8, segments=6, learn=True),
        # one token of one prompt, eager, fp32; one of a served batch (128 requests, 16 heads)
        _step("step_nb8_fp32", 8, 64, 64, 8, dtype="fp32"),
        _step("step_nb2048", 2048, 128, 128, 16, nbk=1024),
        # a block's end for 16 requests' tokens, fp32
        _join("join_16", 16, 512, dtype="fp32", gate=None, vector=False),
        # a long prompt's (8 heads of 128), bf16 on a residual stream in fp32
        _join("join_T131072", 131072, 1024),
        # a training step's (B = 8, T = 4096, 12 heads of 64), bf16 throughout, with dropout
        _join("join_train_32768", 32768, 768, stream="bf16", drop=0.1, grads=True),
        # packed documents in fp16, an odd width, a silu gate, heavier dropout
        _join("join_train_odd", 10007, 1531, dtype="fp16", gate="silu", vector=False, drop=0.25,
              grads=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _nameless(c):
    return {k: v for k, v in c.items() if k != "name"}


def _heads(rng, hi):
    """(sequences, key sequences, heads): heads and nbk divide nb."""
    group = rng.choice([1, 1, 1, 2, 4])
    kh = _log(rng, 1, max(1, min(16, hi // group)))
    batch = _log(rng, 1, max(1, hi // (group * kh)))
    return batch * kh * group, batch * kh, kh * group


def _size(rng):
    return rng.choice([64, 64, 128, 128, 32, 96, rng.randint(16, 128)])


def draw(rng):
    kind = rng.choice(["scan", "scan", "train", "train", "step", "join", "join"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind == "join":
        grads = rng.random() < 0.5
        D = rng.choice([_log(rng, 64, 8192), _log(rng, 8, 1024) * 8, 1024])
        top = max(1, (32768 * 768 if grads else 131072 * 1024) // (D if dtype != "fp32" else 2 * D))
        return _nameless(_join("", _log(rng, 1, top), D, dtype=dtype,
                               stream=rng.choice([dtype, "fp32"]),
                               gate=rng.choice([None, "linear", "sigmoid", "silu"]),
                               post=rng.random() < 0.8, vector=rng.random() < 0.5,
                               drop=rng.choice([0.0, 0.1, rng.uniform(0.01, 0.6)]), grads=grads))
    r = _size(rng)
    p = r if rng.random() < 0.7 else _size(rng)
    if kind == "step":
        nb, nbk, heads = _heads(rng, 2048)
        return _nameless(_step("", nb, r, p, heads, dtype, nbk=nbk))
    # a third of the largest case's work at most in 16 bits, a tenth in fp32
    budget = (8 * 131072 * 128 * 128 // 3 if kind == "scan" else 96 * 4096 * 64 * 64)
    budget //= 1 if dtype == "bf16" else 3
    nb, nbk, heads = _heads(rng, 96)
    top = max(1, min(131072 if kind == "scan" else 8192, budget // (nb * r * p)))
    T = _log(rng, 1, top)
    segments = rng.choice([1, 1, rng.randint(2, 8)]) if T >= 16 else 1
    return _nameless(_scan("", nb, T, r, p, heads, dtype=dtype, nbk=nbk, segments=segments,
                           state=rng.random() < 0.5, kind=kind,
                           learn=kind == "train" and rng.random() < 0.5))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _unit(g, dt, *shape):
    """Rows of length one, rounded to the type: what a layer's query and key norms leave."""
    x = _normal(g, *shape)
    return (x / x.norm(dim=-1, keepdim=True)).to(dt)


def _log_decays(g, heads):
    """One log decay a head, from slow (1/1024 a token) to fast (1/2)."""
    return -torch.exp(torch.rand(heads, device=DEV, generator=g) * math.log(512.0)) / 1024.0


def _offsets(c, seed):
    """Segment borders: 0, sorted distinct cuts, T."""
    cuts = random.Random(seed).sample(range(1, c["T"]), c["segments"] - 1)
    return [0] + sorted(cuts) + [c["T"]]


def _scan_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    nb, nbk, T, r, p = c["nb"], c["nbk"], c["T"], c["r"], c["p"]
    q, k = _unit(g, dt, nbk, T, r), _unit(g, dt, nbk, T, r)
    v = _normal(g, nb, T, p).to(dt)
    logA = _log_decays(g, c["heads"])
    S0 = _normal(g, c["segments"], nb, r, p) if c["state"] else None
    dO = _normal(g, nb, T, p).to(dt) if c["kind"] == "train" else None
    if S0 is not None and c["segments"] == 1:
        S0 = S0[0]
    return q, k, v, logA, S0, dO


def _step_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    nb, nbk, r, p = c["nb"], c["nbk"], c["r"], c["p"]
    q, k = _unit(g, dt, nbk, r), _unit(g, dt, nbk, r)
    return q, k, _normal(g, nb, p).to(dt), _log_decays(g, c["heads"]), _normal(g, nb, r, p)


def _join_inputs(c, seed):
    """The block's output, the residual stream, the gate, the weights of the norm after the
    block, of the residual scale and of the next norm, the generator's seed, and the gradients
    of both results.  An absent one is None; a residual scale of one number is a float."""
    g, dt, hd = _gen(seed), DTYPES[c["dtype"]], DTYPES[c["stream"]]
    rows, D = c["rows"], c["D"]
    f = (0.5 * _normal(g, rows, D)).to(dt)
    h = (2.0 * _normal(g, rows, D)).to(hd)
    z = _normal(g, rows, D).to(dt) if c["gate"] else None
    w1 = (1.0 + 0.1 * _normal(g, D)) if c["post"] else None
    w2 = 1.0 + 0.1 * _normal(g, D)
    s = 0.25 + 0.05 * _normal(g, D) if c["vector"] else 0.25 + (seed % 64) / 256.0
    key = torch.randint(0, 2 ** 62, (1,), device=DEV, generator=g) if c["drop"] else None
    dh = _normal(g, rows, D).to(hd) if c["grads"] else None
    dx = _normal(g, rows, D).to(dt) if c["grads"] else None
    return f, h, z, w1, s, w2, key, dh, dx


def _learned(ts):
    return [t for t in ts if torch.is_tensor(t) and t.is_floating_point()]


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind in ("scan", "train"):
        q, k, v, logA, S0, dO = _scan_inputs(c, seed)
        offsets = _offsets(c, seed)
        s = {"kind": kind, "x": (q, k, v, logA), "S0": S0, "dO": dO, "scale": c["r"] ** -0.5,
             "offsets": offsets, "learn": c["learn"]}
        if own:
            from smat_attention_amd import attention as A
            s["segments"] = A.Segments(offsets, DEV) if c["segments"] > 1 else None
        if kind == "train":
            s["leaves"] = [q, k, v] + [t for t in (S0,) if t is not None]
            s["leaves"] += [logA] if c["learn"] else []
            for t in s["leaves"]:
                t.requires_grad_(True)
        return s
    if kind == "step":
        x = _step_inputs(c, seed)
        return {"kind": kind, "x": x, "next": torch.empty_like(x[-1]), "scale": c["r"] ** -0.5}
    f, h, z, w1, sc, w2, key, dh, dx = _join_inputs(c, seed)
    s = {"kind": kind, "x": (f, h, z, w1, sc, w2, key), "d": (dh, dx), "gate": c["gate"],
         "drop": c["drop"], "grads": c["grads"]}
    if c["grads"]:
        s["leaves"] = _learned((f, h, z, w1, sc, w2))
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _decay_segment(q, k, v, la, scale, S):
    """One segment of every sequence in chunks; fp32 (nb, T, .) and (nb,) in, (o, S) out."""
    nb, T, r = q.shape
    C, f = CHUNK, torch.nn.functional.pad
    nc = -(-T // C)
    pad = nc * C - T
    q, k, v = (f(t, (0, 0, 0, pad)).reshape(nb, nc, C, t.shape[-1]) for t in (q, k, v))
    i = torch.arange(C, device=q.device, dtype=torch.float32)
    la = la[:, None]
    low = i[:, None] >= i
    D = torch.exp(la[:, :, None] * (i[:, None] - i).clamp(min=0)) * low
    e = torch.exp(la * (i + 1))[:, None, :, None]
    # the last chunk's padded tokens are zeros and do not decay the state either
    n = torch.full((nc,), float(C), device=q.device)
    n[-1] -= pad
    w = torch.exp(la[:, :, None] * (n[:, None] - 1 - i).clamp(min=0))[..., None]
    aC = torch.exp(la * n)[..., None, None]
    D = D[:, None]
    KV = (w * k).transpose(-1, -2).contiguous() @ v
    before = []
    for c in range(nc):
        before.append(S)
        S = aC[:, c] * S + KV[:, c]
    P = (q @ k.transpose(-1, -2).contiguous()) * D
    o = P @ v + e * (q @ torch.stack(before, 1))
    return scale * o.reshape(nb, nc * C, -1)[:, :T], S


def _decay_plain(s):
    q, k, v, logA = (t.float() for t in s["x"])
    nb, group = v.shape[0], v.shape[0] // q.shape[0]
    q, k = (t.repeat_interleave(group, 0) for t in (q, k))
    la = logA.repeat(nb // logA.shape[0])
    outs, states = [], []
    off = s["offsets"]
    for i, (a, b) in enumerate(zip(off, off[1:])):
        if s["S0"] is None:
            S = torch.zeros(nb, q.shape[-1], v.shape[-1], device=q.device)
        else:
            S = s["S0"][i] if len(off) > 2 else s["S0"]
        o, S = _decay_segment(q[:, a:b], k[:, a:b], v[:, a:b], la, s["scale"], S)
        outs.append(o)
        states.append(S)
    return torch.cat(outs, 1).to(s["x"][2].dtype), torch.stack(states) if len(off) > 2 \
        else states[0]


def _step_plain(s):
    q, k, v, logA, S = s["x"]
    nb, group = v.shape[0], v.shape[0] // q.shape[0]
    qf, kf = (t.float().repeat_interleave(group, 0)[:, :, None] for t in (q, k))
    a = torch.exp(logA).repeat(nb // logA.shape[0])
    S2 = S * a[:, None, None] + kf * v.float()[:, None, :]
    return (s["scale"] * (S2 * qf).sum(1)).to(v.dtype), S2


def _words(key, rows, D):
    """The generator's 32-bit words for rows x D places, as int64: Philox 4x32 of ten rounds
    (Salmon et al., SC 2011), key = the seed's two halves, counter = (column // 4, row, 0, 0)."""
    low = 0xFFFFFFFF
    blocks = -(-D // 4)
    key = key.reshape(())
    k0, k1 = key & low, (key >> 32) & low
    c0 = torch.arange(blocks, device=DEV).expand(rows, blocks)
    c1 = torch.arange(rows, device=DEV)[:, None].expand(rows, blocks)
    c2 = c3 = torch.zeros(rows, blocks, dtype=torch.int64, device=DEV)
    for _ in range(10):
        # the products' 64 bits wrap in int64 without loss
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((b >> 32) & low) ^ c1 ^ k0, b & low,
                          ((a >> 32) & low) ^ c3 ^ k1, a & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], -1).reshape(rows, 4 * blocks)[:, :D]


def _join_plain(s):
    f, h, z, w1, sc, w2, key = s["x"]
    y = f.float()
    if w1 is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w1
    if s["gate"]:
        g = z.float()
        if s["gate"] != "linear":
            sig = 1.0 / (1.0 + torch.exp(-g))
            g = sig if s["gate"] == "sigmoid" else g * sig
        y = g * y
    if key is not None:
        keep = _words(key, *f.shape) >= round(s["drop"] * 2 ** 32)
        y = y * (keep.float() * (1.0 / (1.0 - s["drop"])))
    h2 = h.float() + sc * y
    x = h2 * torch.rsqrt((h2 * h2).mean(-1, keepdim=True) + EPS) * w2
    return h2.to(h.dtype), x.to(f.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s, kind = state, state["kind"]
    if own:
        from smat_attention_amd import attention as A
    if kind in ("scan", "train"):
        with torch.set_grad_enabled(kind == "train"):
            if own:
                o, S = A.head_decay_scan(*s["x"], scale=s["scale"], state=s["S0"],
                                         segments=s["segments"], return_state=True)
            else:
                o, S = _decay_plain(s)
        if kind == "scan":
            return {"o": o, "S": S}
        grads = torch.autograd.grad(o, s["leaves"], s["dO"])
        names = ["dq", "dk", "dv"] + ["dS0"] * (s["S0"] is not None) + ["dlogA"] * s["learn"]
        return {"o": o.detach(), **dict(zip(names, grads))}
    if kind == "step":
        if own:
            o = A.head_decay_step(*s["x"], scale=s["scale"], out_state=s["next"])
            return {"o": o, "S": s["next"]}
        o, S = _step_plain(s)
        return {"o": o, "S": S}
    with torch.set_grad_enabled(s["grads"]):
        if own:
            f, h, z, w1, sc, w2, key = s["x"]
            h2, x = A.block_join(f, h, post_weight=w1, gate=z, gate_kind=s["gate"] or "linear",
                                 scale=sc, pre_weight=w2, eps=EPS, dropout=s["drop"], seed=key)
        else:
            h2, x = _join_plain(s)
    if not s["grads"]:
        return {"h": h2, "x": x}
    grads = torch.autograd.grad((h2, x), s["leaves"], s["d"])
    names = [n for n, t in zip(("df", "dh", "dgate", "dpost", "dscale", "dpre"), s["x"])
             if torch.is_tensor(t)]
    return {"h": h2.detach(), "x": x.detach(), **dict(zip(names, grads))}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, eb = case, DTYPES[case["dtype"]].itemsize
    if c["kind"] == "join":
        n, hb = c["rows"] * c["D"], DTYPES[c["stream"]].itemsize
        gate = eb if c["gate"] else 0
        one = n * (2 * eb + 2 * hb + gate)
        if not c["grads"]:
            return {"bytes": one + 12 * c["D"], "flops": 12.0 * n}
        # dh, dx in; df, dh and the gate's gradient out
        return {"bytes": one + n * (2 * eb + 2 * hb + gate) + 24 * c["D"], "flops": 40.0 * n}
    nb, nbk, r, p = c["nb"], c["nbk"], c["r"], c["p"]
    T = c.get("T", 1)
    keys, values = nbk * T * r * eb, nb * T * p * eb
    flops = 4.0 * nb * T * r * p
    if c["kind"] == "step":
        return {"bytes": 2 * keys + 2 * values + 2 * nb * r * p * 4, "flops": flops}
    states = c["segments"] * nb * r * p * 4 * (2 if c["state"] else 1)
    if c["kind"] == "scan":
        return {"bytes": 2 * keys + 2 * values + states, "flops": flops}
    # q, k, v, dO in, o and three gradients out
    states = 2 * c["segments"] * nb * r * p * 4 if c["state"] else 0
    return {"bytes": 4 * keys + 4 * values + states, "flops": 3 * flops}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _scan64(c, seed):
    """The recurrence token by token; with the gradients, its adjoint from the kept states."""
    q, k, v, logA, S0, dO = _scan_inputs(c, seed)
    off, scale, train = _offsets(c, seed), c["r"] ** -0.5, c["kind"] == "train"
    nb, nbk, T, heads = c["nb"], c["nbk"], c["T"], c["heads"]
    group, many = nb // nbk, c["segments"] > 1
    # token-major copies, each key head repeated for its value heads
    q, k = (t.double().repeat_interleave(group, 0).transpose(0, 1).contiguous() for t in (q, k))
    v = v.double().transpose(0, 1).contiguous()
    a = logA.double().exp().repeat(nb // heads)[:, None, None]
    o = torch.empty_like(v)
    before, finals = [], []
    begin = {t: i for i, t in enumerate(off[:-1])}
    S = None
    for t in range(T):
        if t in begin:
            if t:
                finals.append(S)
            S = torch.zeros(nb, c["r"], c["p"], dtype=torch.float64, device=DEV) if S0 is None \
                else (S0[begin[t]] if many else S0).double()
        if train:
            before.append(S)
        S = torch.baddbmm(S * a, k[t, :, :, None], v[t, :, None])
        o[t] = torch.bmm(q[t, :, None], S)[:, 0]
    finals.append(S)
    got = {"o": (scale * o).transpose(0, 1)}
    if not train:
        got["S"] = torch.stack(finals) if many else finals[0]
        return got
    do = scale * dO.double().transpose(0, 1)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dl = torch.zeros(nb, dtype=torch.float64, device=DEV)
    ends = set(off[1:])
    dS0 = torch.empty(len(off) - 1, nb, c["r"], c["p"], dtype=torch.float64, device=DEV)
    for t in range(T - 1, -1, -1):
        if t + 1 in ends:
            dS = torch.zeros(nb, c["r"], c["p"], dtype=torch.float64, device=DEV)
        S1 = before.pop() * a
        dS = torch.baddbmm(dS, q[t, :, :, None], do[t, :, None])
        S2 = torch.baddbmm(S1, k[t, :, :, None], v[t, :, None])
        dq[t] = torch.bmm(S2, do[t, :, :, None])[..., 0]
        dk[t] = torch.bmm(dS, v[t, :, :, None])[..., 0]
        dv[t] = torch.bmm(k[t, :, None], dS)[:, 0]
        if c["learn"]:
            dl += (dS * S1).sum((1, 2))
        dS = dS * a
        if t in begin:
            dS0[begin[t]] = dS
    fold = lambda x: x.transpose(0, 1).reshape(nbk, group, T, c["r"]).sum(1)
    got.update(dq=fold(dq), dk=fold(dk), dv=dv.transpose(0, 1))
    if S0 is not None:
        got["dS0"] = dS0 if many else dS0[0]
    if c["learn"]:
        got["dlogA"] = dl.reshape(nb // heads, heads).sum(0)
    return got


def _step64(c, seed):
    q, k, v, logA, S = (t.double() for t in _step_inputs(c, seed))
    group = c["nb"] // c["nbk"]
    q, k = (t.repeat_interleave(group, 0) for t in (q, k))
    a = logA.exp().repeat(c["nb"] // c["heads"])[:, None, None]
    S = S * a + k[:, :, None] * v[:, None]
    return {"o": c["r"] ** -0.5 * torch.bmm(q[:, None], S)[:, 0], "S": S}


def _kept(key, rows, D, drop):
    """Which places are kept, from the generator on the host in unsigned 64 bits."""
    key, m = int(key.item()), np.uint64(0xFFFFFFFF)
    x = [np.zeros((rows, -(-D // 4)), np.uint64) for _ in range(4)]
    x[0] += np.arange(-(-D // 4), dtype=np.uint64)
    x[1] += np.arange(rows, dtype=np.uint64)[:, None]
    k = [np.uint64(key & 0xFFFFFFFF), np.uint64(key >> 32)]
    half = np.uint64(32)
    for _ in range(10):
        u, w = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(w >> half) ^ x[1] ^ k[0], w & m, (u >> half) ^ x[3] ^ k[1], u & m]
        k = [(k[0] + np.uint64(0x9E3779B9)) & m, (k[1] + np.uint64(0xBB67AE85)) & m]
    words = np.stack(x, -1).reshape(rows, -1)[:, :D]
    return torch.from_numpy(words >= np.uint64(round(drop * 2 ** 32))).to(DEV)


def _join64(c, seed):
    f, h, z, w1, s, w2, key, dh, dx = _join_inputs(c, seed)
    f, h = f.double(), h.double()
    D = c["D"]
    norm = lambda t: (t.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    y, r1 = f, None
    if w1 is not None:
        r1 = norm(f)
        y = f * r1 * w1.double()
    gate = slope = None
    if c["gate"]:
        z = z.double()
        sig = torch.sigmoid(z)
        gate, slope = {"linear": (z, torch.ones_like(z)), "sigmoid": (sig, sig * (1 - sig)),
                       "silu": (z * sig, sig * (1 + z * (1 - sig)))}[c["gate"]]
    m = _kept(key, c["rows"], D, c["drop"]).double() / (1 - c["drop"]) if c["drop"] else 1.0
    u = m * y * (1.0 if gate is None else gate)
    sd = s.double() if c["vector"] else s
    h2 = h + sd * u
    r2 = norm(h2)
    got = {"h": h2, "x": h2 * r2 * w2.double()}
    if not c["grads"]:
        return got
    dx = dx.double()
    t = w2.double() * dx
    dh2 = dh.double() + r2 * t - h2 * r2 ** 3 * (t * h2).mean(-1, keepdim=True)
    du = dh2 * m * sd
    dy = du if gate is None else du * gate
    got["df"] = dy
    if w1 is not None:
        t1 = w1.double() * dy
        got["df"] = r1 * t1 - f * r1 ** 3 * (t1 * f).mean(-1, keepdim=True)
    got["dh"] = dh2
    if gate is not None:
        got["dgate"] = du * y * slope
    if w1 is not None:
        got["dpost"] = (dy * f * r1).sum(0)
    if c["vector"]:
        got["dscale"] = (dh2 * u).sum(0)
    got["dpre"] = (dx * h2 * r2).sum(0)
    return got


def exact(case, seed):
    with torch.no_grad():
        if case["kind"] == "step":
            return _step64(case, seed)
        if case["kind"] == "join":
            return _join64(case, seed)
        return _scan64(case, seed)
