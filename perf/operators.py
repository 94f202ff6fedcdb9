"""The gated delta rule and drafted trees over the decode cache, as cases that can be timed.

Four kinds of pass:

* ``scan``:  the gated delta rule over whole sequences (``gated_delta_scan``), with packed
             segments, an initial state and shared key heads where the case says so;
* ``train``: the same forward and its gradients;
* ``step``:  one token of a served batch (``gated_delta_step``);
* ``tree``:  a drafted tree verified against a decoder's cache, and the state that each
             request's accepted path leaves (``SmatDecoder.tree_step`` / ``tree_state``).

``own`` chooses between the framework's kernels and the plain form: elementary torch operations
in 32 bits, rounded once at the end.  ``exact`` computes a case in 64 bits token by token.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
CHUNK = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _scan(name, nb, T, r, p, dtype="bf16", nbk=None, segments=1, state=False, kind="scan"):
    return {"name": name, "kind": kind, "nb": nb, "nbk": nbk or nb, "T": T, "r": r, "p": p,
            "dtype": dtype, "segments": segments, "state": state}


def _train(name, nb, T, r, p, **kw):
    return _scan(name, nb, T, r, p, kind="train", **kw)


def _step(name, nb, r, p, dtype="bf16", nbk=None):
    return {"name": name, "kind": "step", "nb": nb, "nbk": nbk or nb, "r": r, "p": p,
            "dtype": dtype}


def _tree(name, requests, heads, nodes, depth, B, hd, dtype="bf16"):
    return {"name": name, "kind": "tree", "requests": requests, "heads": heads, "nodes": nodes,
            "depth": depth, "B": B, "hd": hd, "dtype": dtype}


def listed():
    return [
        # a turn's last 7 tokens on a kept state: launches and host latency
        _scan("scan_T7", 8, 7, 64, 64, state=True),
        # a short prompt in fp32, 4 heads of 64
        _scan("scan_fp32_T1024", 4, 1024, 64, 64, dtype="fp32"),
        # an ordinary batch of prompts at head size 64 (B = 4, H = 8)
        _scan("scan_T8192_hd64", 32, 8192, 64, 64),
        # prompts of different odd lengths packed one behind the other, fp16, two value heads a
        # key head, head size 96, states kept
        _scan("scan_packed_hd96", 12, 10007, 96, 96, dtype="fp16", nbk=6, segments=5, state=True),
        # one long prompt, 8 heads of 128
        _scan("scan_T131072_hd128", 8, 131072, 128, 128),
        # training steps of a small model's layer (B = 8, H = 12)
        _train("train_T4096_hd64", 96, 4096, 64, 64),
        # a layer with two value heads a key head over packed documents, head size 128
        _train("train_packed_hd128", 16, 8192, 128, 128, nbk=8, segments=6),
        # one token of one prompt, eager, fp32; one of a served batch (128 requests, 16 heads)
        _step("step_nb8_fp32", 8, 64, 64, dtype="fp32"),
        _step("step_nb2048", 2048, 128, 128, nbk=1024),
        # eight drafted tokens of one prompt of 8 heads; 64-node trees of 16 requests
        _tree("tree_1x8", 1, 8, 8, 5, 33, 64),
        _tree("tree_16x64", 16, 8, 64, 8, 131, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _nameless(c):
    return {k: v for k, v in c.items() if k != "name"}


def _heads(rng, hi):
    """(value heads, key heads) times sequences: nbk divides nb."""
    group = rng.choice([1, 1, 1, 2, 4])
    nbk = _log(rng, 1, max(1, hi // group))
    return nbk * group, nbk


def _size(rng):
    return rng.choice([64, 64, 128, 128, 32, 96, rng.randint(16, 128)])


def draw(rng):
    kind = rng.choice(["scan", "scan", "train", "train", "step", "tree"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind == "tree":
        c = _tree("", _log(rng, 1, 16), rng.choice([4, 8, 12]), _log(rng, 1, 64),
                  rng.randint(1, 12), _log(rng, 4, 131), _size(rng), dtype)
        if c["requests"] * c["heads"] * c["hd"] > 128 * 128:
            c["requests"] = max(1, 128 * 128 // (c["heads"] * c["hd"]))
        return _nameless(c)
    r = _size(rng)
    p = r if rng.random() < 0.7 else _size(rng)
    if kind == "step":
        nb, nbk = _heads(rng, 2048)
        return _nameless(_step("", nb, r, p, dtype, nbk=nbk))
    # a third of the largest case's work at most in 16 bits, a tenth in fp32
    budget = (8 * 131072 * 128 * 128 // 3 if kind == "scan" else 96 * 4096 * 64 * 64)
    budget //= 1 if dtype == "bf16" else 3
    nb, nbk = _heads(rng, 96)
    top = max(1, min(131072 if kind == "scan" else 8192, budget // (nb * r * p)))
    T = _log(rng, 1, top)
    segments = rng.choice([1, 1, rng.randint(2, 8)]) if T >= 16 else 1
    return _nameless(_scan("", nb, T, r, p, dtype=dtype, nbk=nbk, segments=segments,
                           state=rng.random() < 0.5, kind=kind))


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


def _gates(g, nb, *shape):
    """Log decays -rate softplus(x), one rate a head from slow (1/64) to fast (4), and write
    strengths in (0, 1)."""
    rate = torch.exp(torch.rand(nb, *[1] * len(shape), device=DEV, generator=g)
                     * math.log(256.0)) / 64.0
    logA = -rate * torch.nn.functional.softplus(_normal(g, nb, *shape) - 2.0)
    return logA, torch.sigmoid(_normal(g, nb, *shape))


def _offsets(c, seed):
    """Segment borders: 0, sorted distinct cuts, T."""
    cuts = random.Random(seed).sample(range(1, c["T"]), c["segments"] - 1)
    return [0] + sorted(cuts) + [c["T"]]


def _scan_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    nb, nbk, T, r, p = c["nb"], c["nbk"], c["T"], c["r"], c["p"]
    q, k = _unit(g, dt, nbk, T, r), _unit(g, dt, nbk, T, r)
    v = _normal(g, nb, T, p).to(dt)
    logA, beta = _gates(g, nb, T)
    S0 = _normal(g, c["segments"], nb, r, p) if c["state"] else None
    dO = _normal(g, nb, T, p).to(dt) if c["kind"] == "train" else None
    return q, k, v, logA, beta, S0, dO


def _step_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    nb, nbk, r, p = c["nb"], c["nbk"], c["r"], c["p"]
    q, k = _unit(g, dt, nbk, r), _unit(g, dt, nbk, r)
    v = _normal(g, nb, p).to(dt)
    logA, beta = (t[:, 0] for t in _gates(g, nb, 1))
    return q, k, v, logA.contiguous(), beta.contiguous(), _normal(g, nb, r, p)


def _tree_inputs(c, seed):
    """Features of the drafted tokens (elu + 1 of normals), values with their ones column, the
    cache of a decoder (sums of about 64 landmark and 64 recent tokens), the requests' positions,
    trees and accepted nodes (-1: none)."""
    g, dt, rng = _gen(seed), DTYPES[c["dtype"]], random.Random(seed)
    R, nb, M, r, p = c["requests"], c["requests"] * c["heads"], c["nodes"], c["hd"], c["hd"] + 1
    Phi = (torch.nn.functional.elu(_normal(g, nb, M, r)) + 1).to(dt)
    Psi = (torch.nn.functional.elu(_normal(g, nb, M, r) * r ** -0.5) + 1).to(dt)
    Vb = _normal(g, nb, M, p)
    Vb[..., -1] = 1.0
    Vb = Vb.to(dt)
    U = _normal(g, nb, c["B"], r, p) * 8
    S = _normal(g, nb, r, p) * 8
    for t in (U, S):
        t[..., -1] = 64.0 + 16.0 * torch.rand(t.shape[:-1], device=DEV, generator=g)
    parents = []
    for _ in range(R):
        par, depth = [], []
        for j in range(M):
            pick = rng.choice([-1] + [a for a in range(j) if depth[a] < c["depth"] - 1][-6:])
            par.append(pick)
            depth.append(0 if pick < 0 else depth[pick] + 1)
        parents.append(par)
    i = rng.randint(0, 1000)
    ahead = [rng.randint(0, 20) for _ in range(R)]
    nodes = [rng.randint(-1, M - 1) for _ in range(R)]
    return Phi, Psi, Vb, U, S, parents, i, ahead, nodes


def prepare(case, seed):
    c, kind = case, case["kind"]
    if own:
        from smat_attention_amd import attention as A
    if kind in ("scan", "train"):
        q, k, v, logA, beta, S0, dO = _scan_inputs(c, seed)
        scale, offsets = c["r"] ** -0.5, _offsets(c, seed)
        if S0 is not None and c["segments"] == 1:
            S0 = S0[0]
        s = {"kind": kind, "x": (q, k, v, logA, beta), "S0": S0, "dO": dO, "scale": scale,
             "offsets": offsets}
        if own:
            s["segments"] = A.Segments(offsets, DEV) if c["segments"] > 1 else None
        if kind == "train":
            for t in s["x"] + ((S0,) if S0 is not None else ()):
                t.requires_grad_(True)
        return s
    if kind == "step":
        x = _step_inputs(c, seed)
        return {"kind": kind, "x": x, "next": torch.empty_like(x[-1]), "scale": c["r"] ** -0.5}
    Phi, Psi, Vb, U, S, parents, i, ahead, nodes = _tree_inputs(c, seed)
    s = {"kind": kind, "x": (Phi, Psi, Vb), "nodes": torch.tensor(nodes, device=DEV,
                                                                 dtype=torch.int32)}
    ahead = torch.tensor(ahead, device=DEV, dtype=torch.int32)
    if own:
        s["tree"] = A.DraftTree(parents, DEV)
        s["dec"] = A.SmatDecoder.from_cache(U, S, i, ahead=ahead)
        return s
    M = c["nodes"]
    anc = torch.zeros(c["requests"], M, M)
    for b, par in enumerate(parents):
        for j in range(M):
            if par[j] >= 0:
                anc[b, j] = anc[b, par[j]]
            anc[b, j, j] = 1.0
    depth = anc.sum(-1).long() - 1
    s.update(U=U, S=S, anc=anc.to(DEV), depth=depth.to(DEV), i=i, ahead=ahead.long())
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _unit_lower_inverse(A):
    """(I + A)^{-1} of strictly lower A (..., C, C), C a power of two, by doubling: with the
    diagonal blocks inverted, [[X, 0], [Y, Z]]^{-1} = [[X', 0], [-Z' Y X', Z']]."""
    C = A.shape[-1]
    if C == 1:
        return torch.ones_like(A)
    h = C // 2
    X = _unit_lower_inverse(A[..., :h, :h])
    Z = _unit_lower_inverse(A[..., h:, h:])
    Y = -(Z @ A[..., h:, :h].contiguous()) @ X
    return torch.cat([torch.cat([X, torch.zeros_like(X)], -1), torch.cat([Y, Z], -1)], -2)


def _delta_segment(q, k, v, logA, beta, scale, S):
    """One segment of every sequence in chunks; fp32 (nb, T, .) in, (o, S) out."""
    nb, T, r = q.shape
    p, C = v.shape[-1], CHUNK
    pad, f = (-T) % C, torch.nn.functional.pad
    nc = (T + pad) // C
    q, k, v = (f(t, (0, 0, 0, pad)).reshape(nb, nc, C, t.shape[-1]) for t in (q, k, v))
    L = f(logA, (0, pad)).reshape(nb, nc, C).cumsum(-1)
    b = f(beta, (0, pad)).reshape(nb, nc, C, 1)
    low = torch.ones(C, C, device=q.device, dtype=torch.bool).tril()
    D = torch.exp((L[..., :, None] - L[..., None, :]).masked_fill(~low, float("-inf")))
    kT = k.transpose(-1, -2).contiguous()
    inv = _unit_lower_inverse((b * (k @ kT) * D).tril(-1))
    P = (q @ kT) * D
    eL, eC, aC = (torch.exp(t)[..., None] for t in (L, L[..., -1:] - L, L[..., -1:]))
    o = []
    for c in range(nc):
        U = inv[:, c] @ (b[:, c] * (v[:, c] - eL[:, c] * (k[:, c] @ S)))
        o.append(eL[:, c] * (q[:, c] @ S) + P[:, c] @ U)
        S = aC[:, c] * S + (eC[:, c] * k[:, c]).transpose(1, 2).contiguous() @ U
    return scale * torch.cat(o, 1)[:, :T], S


def _delta_plain(s):
    q, k, v, logA, beta = (t.float() for t in s["x"])
    nb, group = v.shape[0], v.shape[0] // q.shape[0]
    q, k = (t.repeat_interleave(group, 0) for t in (q, k))
    outs, states = [], []
    off = s["offsets"]
    for i, (a, b) in enumerate(zip(off, off[1:])):
        if s["S0"] is None:
            S = torch.zeros(nb, q.shape[-1], v.shape[-1], device=q.device)
        else:
            S = s["S0"][i] if len(off) > 2 else s["S0"]
        o, S = _delta_segment(q[:, a:b], k[:, a:b], v[:, a:b], logA[:, a:b], beta[:, a:b],
                              s["scale"], S)
        outs.append(o)
        states.append(S)
    return torch.cat(outs, 1).to(s["x"][2].dtype), torch.stack(states) if len(off) > 2 \
        else states[0]


def _step_plain(s):
    q, k, v, logA, beta, S = s["x"]
    group = v.shape[0] // q.shape[0]
    qf, kf = (t.float().repeat_interleave(group, 0)[:, :, None] for t in (q, k))
    S1 = S * torch.exp(logA)[:, None, None]
    u = beta[:, None] * (v.float() - (S1 * kf).sum(1))
    S2 = S1 + kf * u[:, None, :]
    return (s["scale"] * (S2 * qf).sum(1)).to(v.dtype), S2


def _tree_plain(s):
    Phi, Psi, Vb = (t.float() for t in s["x"])
    U, S, anc, depth = s["U"], s["S"], s["anc"], s["depth"]
    nb, M = Phi.shape[:2]
    heads = nb // anc.shape[0]
    anc, depth = anc.repeat_interleave(heads, 0), depth.repeat_interleave(heads, 0)
    at = (s["i"] + s["ahead"].repeat_interleave(heads, 0)[:, None] + depth) % U.shape[1]
    N = Phi @ S + ((Phi @ Psi.transpose(1, 2).contiguous()) * anc) @ Vb
    seq = torch.arange(nb, device=U.device)
    N = N + torch.stack([(Phi[:, j, :, None] * U[seq, at[:, j]]).sum(1) for j in range(M)], 1)
    node = s["nodes"].long().repeat_interleave(heads, 0)
    path = torch.where((node >= 0)[:, None], anc[seq, node.clamp(min=0)], 0.0)
    S2 = S + (Psi * path[..., None]).transpose(1, 2).contiguous() @ Vb
    return N[..., :-1] / N[..., -1:], S2


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
                o, S = A.gated_delta_scan(*s["x"], scale=s["scale"], state=s["S0"],
                                          segments=s["segments"], return_state=True)
            else:
                o, S = _delta_plain(s)
        if kind == "scan":
            return {"o": o, "S": S}
        leaves = s["x"] + ((s["S0"],) if s["S0"] is not None else ())
        grads = torch.autograd.grad(o, leaves, s["dO"])
        names = ("dq", "dk", "dv", "dlogA", "dbeta", "dS0")
        return {"o": o.detach(), **dict(zip(names, grads))}
    if kind == "step":
        if own:
            o = A.gated_delta_step(*s["x"], scale=s["scale"], out_state=s["next"])
            return {"o": o, "S": s["next"]}
        o, S = _step_plain(s)
        return {"o": o, "S": S}
    if own:
        Phi, Psi, Vb = s["x"]
        return {"o": s["dec"].tree_step(Phi, Psi, Vb, s["tree"]),
                "S": s["dec"].tree_state(Psi, Vb, s["tree"], s["nodes"])}
    o, S = _tree_plain(s)
    return {"o": o, "S": S}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, eb = case, DTYPES[case["dtype"]].itemsize
    if c["kind"] == "tree":
        R, nb, M, r, p = c["requests"], c["requests"] * c["heads"], c["nodes"], c["hd"], c["hd"] + 1
        levels = min(c["depth"], M, c["B"])
        rows = nb * M * ((2 * r + p) * eb + (p - 1) * 4)
        return {"bytes": nb * r * p * 4 * (2 + levels) + rows,
                "flops": nb * 2.0 * M * (2 * r * p + 0.5 * levels * (r + p)) + 2.0 * nb * r * p}
    nb, nbk, r, p = c["nb"], c["nbk"], c["r"], c["p"]
    T = c.get("T", 1)
    keys, values = nbk * T * r * eb, nb * T * p * eb
    flops = 7.0 * nb * T * r * p
    if c["kind"] == "step":
        return {"bytes": 2 * keys + 2 * values + nb * 8 + 2 * nb * r * p * 4, "flops": flops}
    states = c["segments"] * nb * r * p * 4 * (2 if c["state"] else 1)
    if c["kind"] == "scan":
        return {"bytes": 2 * keys + 2 * values + nb * T * 8 + states, "flops": flops}
    # q, k, v, dO in, o and three gradients out; the gates and theirs
    states = 2 * c["segments"] * nb * r * p * 4 if c["state"] else 0
    return {"bytes": 4 * keys + 4 * values + nb * T * 16 + states, "flops": 3 * flops}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _scan64(c, seed):
    """The recurrence token by token; with the gradients, its adjoint from the kept states."""
    q, k, v, logA, beta, S0, dO = _scan_inputs(c, seed)
    off, scale, train = _offsets(c, seed), c["r"] ** -0.5, c["kind"] == "train"
    nb, nbk, T = c["nb"], c["nbk"], c["T"]
    group = nb // nbk
    # token-major copies, each key head repeated for its value heads
    q, k = (t.double().repeat_interleave(group, 0).transpose(0, 1).contiguous() for t in (q, k))
    v, a, b = (t.double().transpose(0, 1).contiguous() for t in (v, logA.double().exp(), beta))
    o = torch.empty_like(v)
    before, finals = [], []
    begin = {t: i for i, t in enumerate(off[:-1])}
    S = None
    for t in range(T):
        if t in begin:
            if t:
                finals.append(S)
            S = torch.zeros(nb, c["r"], c["p"], dtype=torch.float64, device=DEV) if S0 is None \
                else S0[begin[t]].double()
        if train:
            before.append(S)
        S = S * a[t, :, None, None]
        w = torch.baddbmm(v[t, :, None], k[t, :, None], S, alpha=-1.0)
        S = torch.baddbmm(S, k[t, :, :, None], b[t, :, None, None] * w)
        o[t] = torch.bmm(q[t, :, None], S)[:, 0]
    finals.append(S)
    got = {"o": (scale * o).transpose(0, 1)}
    if not train:
        got["S"] = torch.stack(finals) if len(off) > 2 else finals[0]
        return got
    do = scale * dO.double().transpose(0, 1)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dl, db = torch.empty_like(a), torch.empty_like(b)
    ends = set(off[1:])
    dS0 = torch.empty(len(off) - 1, nb, c["r"], c["p"], dtype=torch.float64, device=DEV)
    for t in range(T - 1, -1, -1):
        if t + 1 in ends:
            dS = torch.zeros(nb, c["r"], c["p"], dtype=torch.float64, device=DEV)
        S1 = before.pop() * a[t, :, None, None]
        kc, kr = k[t, :, :, None], k[t, :, None]
        w = v[t, :, None] - kr @ S1
        u = b[t, :, None, None] * w
        S2 = S1 + kc * u
        dS = dS + q[t, :, :, None] * do[t, :, None]
        dq[t] = (S2 * do[t, :, None]).sum(-1)
        du = kr @ dS
        dw = b[t, :, None, None] * du
        db[t] = (du * w).sum((1, 2))
        dv[t] = dw[:, 0]
        dk[t] = (dS * u).sum(-1) - (S1 * dw).sum(-1)
        dS = dS - kc * dw
        dl[t] = (dS * S1).sum((1, 2))
        dS = dS * a[t, :, None, None]
        if t in begin:
            dS0[begin[t]] = dS
    fold = lambda x: x.transpose(0, 1).reshape(nbk, group, T, c["r"]).sum(1)
    got.update(dq=fold(dq), dk=fold(dk), dv=dv.transpose(0, 1), dlogA=dl.transpose(0, 1),
               dbeta=db.transpose(0, 1))
    if S0 is not None:
        got["dS0"] = dS0 if len(off) > 2 else dS0[0]
    return got


def _step64(c, seed):
    q, k, v, logA, beta, S = (t.double() for t in _step_inputs(c, seed))
    group = c["nb"] // c["nbk"]
    q, k = (t.repeat_interleave(group, 0) for t in (q, k))
    S = S * logA.exp()[:, None, None]
    w = v - torch.bmm(k[:, None], S)[:, 0]
    S = S + k[:, :, None] * (beta[:, None] * w)[:, None]
    return {"o": c["r"] ** -0.5 * torch.bmm(q[:, None], S)[:, 0], "S": S}


def _tree64(c, seed):
    """Node by node: each node's state is its parent's with its own token added."""
    Phi, Psi, Vb, U, S, parents, i, ahead, nodes = _tree_inputs(c, seed)
    H, M = c["heads"], c["nodes"]
    o = torch.empty(Phi.shape[0], M, c["hd"], dtype=torch.float64, device=DEV)
    after = S.double()
    for b, par in enumerate(parents):
        rows = slice(b * H, (b + 1) * H)
        root, states, depth = S[rows].double(), [], []
        for j in range(M):
            depth.append(0 if par[j] < 0 else depth[par[j]] + 1)
            mine = root if par[j] < 0 else states[par[j]]
            mine = mine + Psi[rows, j].double()[:, :, None] * Vb[rows, j].double()[:, None]
            states.append(mine)
            table = mine + U[rows, (i + ahead[b] + depth[j]) % c["B"]].double()
            N = (Phi[rows, j].double()[:, :, None] * table).sum(1)
            o[rows, j] = N[:, :-1] / N[:, -1:]
        if nodes[b] >= 0:
            after[rows] = states[nodes[b]]
    return {"o": o, "S": after}


def exact(case, seed):
    with torch.no_grad():
        if case["kind"] == "step":
            return _step64(case, seed)
        if case["kind"] == "tree":
            return _tree64(case, seed)
        return _scan64(case, seed)
