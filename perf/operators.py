"""Timing cases of the row operators of `mignn.attention`: root-mean-square
norm with the residual's addition, rotary positions over several axes, and
cross attention of one mesh's rows to an encoder's states of another length.

A case is a dict of plain values.  `prepare` makes its inputs on the GPU,
`run` is one pass of the operator (a training case: forward and gradients),
`work` the bytes and operations that the pass cannot do without, `exact` the
same outputs from the definition in 64 bits.  `own` chooses between the plain
form (elementary torch operations in 32 bits) and the framework's kernels.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
BASE = 10000.0
# positions are cell centres in the unit box; the lowest axis frequency turns
# once over the box's 2 pi / CELLS fraction, the highest resolves one cell
CELLS = 256.0
SCORE_BYTES = 1 << 31      # the plain forms keep this much of the scores at a time


def _attention():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "gnn-bfs-rans_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mignn import attention
    return attention


# --------------------------------------------------------------------------
# cases

def _norm(rows, width, dtype, residual, train, name=None):
    case = {"op": "rms_norm", "rows": rows, "width": width, "dtype": dtype,
            "residual": residual, "train": train}
    return dict(case, name=name) if name else case


def _rot(rows, heads, head_dim, axes, dtype, interleaved, train, name=None):
    case = {"op": "rotary", "rows": rows, "heads": heads, "head_dim": head_dim, "axes": axes,
            "dtype": dtype, "interleaved": interleaved, "train": train}
    return dict(case, name=name) if name else case


def _cross(batch, q_len, k_len, ragged, heads, kv_heads, head_dim, dtype, masked, train,
           name=None):
    case = {"op": "cross", "batch": batch, "q_len": q_len, "k_len": k_len, "ragged": ragged,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "masked": masked, "train": train}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one probe point's row ahead of its projections: latency
        _norm(1, 128, "f32", True, False, "norm_probe"),
        # a training step over the 49,181-node graph of the step-flow case
        _norm(49181, 256, "f32", True, True, "norm_train_f32"),
        # states of a million-cell mesh in 16 bits, served
        _norm(1000000, 128, "bf16", True, False, "norm_mesh_bf16"),
        # one probe point's query heads, rotated by its coordinates: latency
        _rot(1, 4, 32, 3, "f32", False, False, "rotary_probe"),
        # the query heads of a million-cell mesh
        _rot(1000000, 4, 32, 3, "f32", False, False, "rotary_mesh_f32"),
        # training over the 49,181-node graph, two axes, 16 bits
        _rot(49181, 8, 64, 2, "bf16", True, True, "rotary_train_bf16"),
        # one probe point against the 12,225 states of the step-flow mesh
        _cross(1, 1, 12225, 0, 4, 4, 32, "f32", False, False, "cross_probe_f32"),
        # one probe in each of 64 meshes of unlike sizes, shared key heads
        _cross(64, 1, 20000, 5, 8, 2, 64, "bf16", True, False, "cross_probes_bf16"),
        # every cell of the step-flow mesh against every state, some left out
        _cross(1, 12225, 12225, 0, 4, 4, 32, "f32", True, False, "cross_mesh_f32"),
        # three snapshots' cells against a few hundred coarse states, trained
        _cross(3, 12225, 257, 7, 4, 4, 64, "f32", True, True, "cross_coarse_train_f32"),
        # a fine mesh against a coarse one, trained in 16 bits
        _cross(1, 49181, 4096, 0, 4, 2, 64, "bf16", False, True, "cross_fine_train_bf16"),
        # the largest: long states, wide heads
        _cross(2, 16384, 16384, 0, 8, 8, 128, "f16", False, False, "cross_wide_f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rms_norm", "rotary", "cross", "cross"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.5
    if op == "rms_norm":
        # widths: every hidden size the layers take (a multiple of 8), odd ones between
        width = _log_int(rng, 32, 1024)
        rows = _log_int(rng, 1, 128000000 // width)
        return _norm(rows, width, dtype, rng.random() < 0.75, train)
    if op == "rotary":
        heads = rng.choice([1, 2, 3, 4, 8])
        head_dim = 2 * rng.randint(8, 64)
        rows = _log_int(rng, 1, 128000000 // (heads * head_dim))
        return _rot(rows, heads, head_dim, rng.randint(1, 3), dtype, rng.random() < 0.5, train)
    kv_heads = rng.choice([1, 2, 4])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    head_dim = rng.choice([16, 24, 32, 40, 64, 64, 96, 128])
    batch = _log_int(rng, 1, 64)
    k_len = _log_int(rng, 1, 20000)
    # up to 16384 queries, and no more score products than the largest listed case
    # (12 flops a product and column in training where a forward pass has 4)
    room = 2 * 16384 * 16384 * 8 * 128 // (batch * k_len * heads * head_dim * (3 if train else 1))
    q_len = 1 if rng.random() < 0.25 else _log_int(rng, 1, max(1, min(16384, room)))
    return _cross(batch, q_len, k_len, rng.randint(0, 9), heads, kv_heads, head_dim, dtype,
                  rng.random() < 0.5, train)


def _lens(case):
    """The sequences' lengths: all alike where `ragged` is 0, else spread over
    a quarter to the whole of the case's lengths."""
    b, lq, lk = case["batch"], case["q_len"], case["k_len"]
    if not case["ragged"]:
        return [lq] * b, [lk] * b
    rng = random.Random(case["ragged"])
    ql = [max(1, int(lq * rng.uniform(0.25, 1.0))) for _ in range(b)]
    kl = [max(1, int(lk * rng.uniform(0.25, 1.0))) for _ in range(b)]
    return ql, kl


def _pairs(case):
    """The rotated pairs of each axis: as even as they divide."""
    half, axes = case["head_dim"] // 2, case["axes"]
    return tuple(half // axes + (1 if a < half % axes else 0) for a in range(axes))


# --------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    train = case["train"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=DEV).mul_(scale).to(dt)

    state = {"case": case}
    if case["op"] == "rms_norm":
        n, h = case["rows"], case["width"]
        state["x"] = normal(n, h)
        state["weight"] = (1.0 + 0.1 * torch.randn(h, generator=gen, device=DEV)).to(dt)
        # the stream that the layers add up: wider than one layer's output
        state["residual"] = normal(n, h, scale=3.0) if case["residual"] else None
        if train:
            state["dy"] = normal(n, h)
            state["ds"] = normal(n, h) if case["residual"] else None
        leaves = ("x", "weight", "residual")
    elif case["op"] == "rotary":
        t, heads, d = case["rows"], case["heads"], case["head_dim"]
        state["x"] = normal(t, heads, d)
        state["pos"] = torch.rand(t, case["axes"], generator=gen, device=DEV)
        if train:
            state["dy"] = normal(t, heads, d)
        if own:
            state["axes"] = _attention().RotaryAxes(
                _pairs(case), base=BASE, scales=(CELLS,) * case["axes"],
                interleaved=case["interleaved"], device=DEV)
        else:
            state["axes"] = _turn_table(case)
        leaves = ("x",)
    else:
        ql, kl = _lens(case)
        d = case["head_dim"]
        state["q"] = normal(sum(ql), case["heads"], d)
        state["k"] = normal(sum(kl), case["kv_heads"], d)
        state["v"] = normal(sum(kl), case["kv_heads"], d)
        state["key_mask"] = (torch.rand(sum(kl), generator=gen, device=DEV) < 0.9
                             if case["masked"] else None)
        if train:
            state["dy"] = normal(sum(ql), case["heads"], d)
        if own:
            state["plan"] = _attention().CrossPlan(
                ql, kl, heads=case["heads"], kv_heads=case["kv_heads"], head_dim=d, dtype=dt,
                device=DEV, train=train)
        else:
            state["lens"] = (ql, kl)
        leaves = ("q", "k", "v")
    if own and train:
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


def _turn_table(case):
    """(frequency of each pair in 64 bits, axis of each pair)."""
    freq, axis = [], []
    for a, m in enumerate(_pairs(case)):
        freq += [CELLS * BASE ** (-i / m) for i in range(m)]
        axis += [a] * m
    return (torch.tensor(freq, dtype=torch.float64, device=DEV),
            torch.tensor(axis, dtype=torch.long, device=DEV))


# --------------------------------------------------------------------------
# one pass

def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "rms_norm":
        return _plain_norm(state, case)
    if case["op"] == "rotary":
        return _plain_rotary(state, case)
    return _plain_cross(state, case)


def _run_own(state, case):
    ops = _attention()
    if case["op"] == "rms_norm":
        x, w, r = state["x"], state["weight"], state["residual"]
        res = ops.rms_norm(x, w, residual=r, eps=EPS)
        if not case["train"]:
            return res
        if r is None:
            return (res,) + torch.autograd.grad(res, (x, w), state["dy"])
        return res + torch.autograd.grad(res, (x, w, r), (state["dy"], state["ds"]))
    if case["op"] == "rotary":
        y = ops.rotary(state["x"], state["pos"], state["axes"])
        if not case["train"]:
            return y
        return (y,) + torch.autograd.grad(y, (state["x"],), state["dy"])
    q, k, v = state["q"], state["k"], state["v"]
    o = ops.cross_attention(q, k, v, state["plan"], key_mask=state["key_mask"])
    if not case["train"]:
        return o
    return (o,) + torch.autograd.grad(o, (q, k, v), state["dy"])


def _plain_norm(state, case):
    x, w, r = state["x"], state["weight"], state["residual"]
    dt = x.dtype
    s = x.float()
    if r is not None:
        s = s + r.float()
    rstd = torch.rsqrt((s * s).mean(1, keepdim=True) + EPS)
    xh = s * rstd
    y = (xh * w.float()).to(dt)
    if not case["train"]:
        return y if r is None else (y, s.to(dt))
    dy = state["dy"].float()
    g = dy * w.float()
    ds = rstd * (g - xh * (g * xh).mean(1, keepdim=True))
    dw = (dy * xh).double().sum(0).to(dt)
    if r is None:
        return y, ds.to(dt), dw
    ds = (ds + state["ds"].float()).to(dt)
    return y, s.to(dt), ds, dw, ds


def _plain_turn(x, cos, sin, interleaved):
    xf = x.float()
    half = xf.shape[-1] // 2
    if interleaved:
        a, b = xf[..., 0::2], xf[..., 1::2]
        out = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = xf[..., :half], xf[..., half:]
        out = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return out.to(x.dtype)


def _plain_rotary(state, case):
    freq, axis = state["axes"]
    ang = state["pos"].double()[:, axis] * freq
    cos, sin = ang.cos().float().unsqueeze(1), ang.sin().float().unsqueeze(1)
    y = _plain_turn(state["x"], cos, sin, case["interleaved"])
    if not case["train"]:
        return y
    return y, _plain_turn(state["dy"], cos, -sin, case["interleaved"])


def _plain_cross(state, case):
    q, k, v, mask = state["q"], state["k"], state["v"], state["key_mask"]
    ql, kl = state["lens"]
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    g = hq // hk
    scale = 1.0 / math.sqrt(d)
    train = case["train"]
    out = torch.empty_like(q)
    if train:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    q0 = k0 = 0
    for lq, lk in zip(ql, kl):
        ks = k[k0:k0 + lk].float().permute(1, 0, 2)                   # [hk, lk, d]
        vs = v[k0:k0 + lk].float().permute(1, 0, 2)
        ms = None if mask is None else mask[k0:k0 + lk]
        if ms is not None:
            vs = vs * ms[None, :, None]
        if train:
            dks, dvs = torch.zeros_like(ks), torch.zeros_like(vs)
        step = max(1, SCORE_BYTES // (4 * hq * lk))
        for a in range(q0, q0 + lq, step):
            n = min(step, q0 + lq - a)

            def rows(t):        # [n, hq, d] -> [hk, g n, d]
                return (t[a:a + n].float().view(n, hk, g, d).permute(1, 2, 0, 3)
                        .reshape(hk, g * n, d))

            def back(t):        # [hk, g n, d] -> [n, hq, d]
                return t.view(hk, g, n, d).permute(2, 0, 1, 3).reshape(n, hq, d).to(q.dtype)

            qs = rows(q)
            s = torch.matmul(qs, ks.transpose(1, 2)) * scale
            if ms is not None:
                s = s.masked_fill(~ms, -math.inf)
            m = s.amax(-1, keepdim=True)
            m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
            p = torch.exp(s - m)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, torch.ones_like(total), total)
            o = torch.matmul(p, vs)
            out[a:a + n] = back(o)
            if train:
                do = rows(state["dy"])
                dvs += torch.matmul(p.transpose(1, 2), do)
                dp = torch.matmul(do, vs.transpose(1, 2))
                dsc = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
                dq[a:a + n] = back(torch.matmul(dsc, ks))
                dks += torch.matmul(dsc.transpose(1, 2), qs)
        if train:
            dk[k0:k0 + lk] = dks.permute(1, 0, 2).to(k.dtype)
            dv[k0:k0 + lk] = dvs.permute(1, 0, 2).to(v.dtype)
        q0, k0 = q0 + lq, k0 + lk
    return (out, dq, dk, dv) if train else out


# --------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    train = case["train"]
    if case["op"] == "rms_norm":
        n, h, r = case["rows"], case["width"], case["residual"]
        # forward: x, weight and y, with a residual r and s; gradients: dy (and
        # ds) read, dx (the residual's is the same numbers, but its own output) and dw written
        tensors = (4 if r else 2) + ((4 if r else 2) if train else 0)
        flops = n * h * (5 + (8 if train else 0))
        return {"bytes": (tensors * n * h + h * (2 if train else 1)) * es, "flops": flops}
    if case["op"] == "rotary":
        t, width = case["rows"], case["heads"] * case["head_dim"]
        passes = 2 if train else 1
        return {"bytes": passes * 2 * t * width * es + t * case["axes"] * 4,
                "flops": passes * 3 * t * width}
    ql, kl = _lens(case)
    d, hq, hk = case["head_dim"], case["heads"], case["kv_heads"]
    products = sum(a * b for a, b in zip(ql, kl)) * hq * d * 2
    qn, kn = sum(ql) * hq * d, sum(kl) * hk * d
    nbytes = (2 * qn + 2 * kn) * es + (sum(kl) if case["masked"] else 0)
    if train:      # dy read, the three gradients written; dP, dV, dQ, dK
        nbytes += (2 * qn + 2 * kn) * es
    return {"bytes": nbytes, "flops": products * (6 if train else 2)}


# --------------------------------------------------------------------------
# the definitions in 64 bits

def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    f64 = {n: t.double() for n, t in state.items()
           if torch.is_tensor(t) and t.is_floating_point()}
    with torch.enable_grad():
        if case["op"] == "rms_norm":
            return _exact_norm(case, f64)
        if case["op"] == "rotary":
            return _exact_rotary(case, f64)
        return _exact_cross(case, f64, state["key_mask"], state["lens"])


def _exact_norm(case, t):
    x = t["x"].requires_grad_(case["train"])
    w = t["weight"].requires_grad_(case["train"])
    r = t.get("residual")
    s = x
    if r is not None:
        s = x + r.requires_grad_(case["train"])
    y = s / torch.sqrt((s ** 2).sum(1, keepdim=True) / case["width"] + EPS) * w
    if not case["train"]:
        return y if r is None else (y, s)
    if r is None:
        return (y.detach(),) + torch.autograd.grad(y, (x, w), t["dy"])
    return (y.detach(), s.detach()) + torch.autograd.grad((y, s), (x, w, r), (t["dy"], t["ds"]))


def _exact_rotary(case, t):
    """Pairs as complex numbers, turned by exp(i angle)."""
    angles = []
    for a, m in enumerate(_pairs(case)):
        freq = np.power(BASE, -np.arange(m, dtype=np.float64) / m) * CELLS
        angles.append(t["pos"][:, a:a + 1] * torch.from_numpy(freq).to(DEV))
    ang = torch.cat(angles, 1)
    turn = torch.polar(torch.ones_like(ang), ang).unsqueeze(1)

    def apply(x, factor):
        n, heads, d = x.shape
        if case["interleaved"]:
            z = torch.view_as_complex(x.reshape(n, heads, d // 2, 2).contiguous())
            return torch.view_as_real(z * factor).reshape(n, heads, d)
        z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * factor
        return torch.cat([z.real, z.imag], -1)

    y = apply(t["x"], turn)
    return (y, apply(t["dy"], turn.conj())) if case["train"] else y


def _exact_cross(case, t, mask, lens):
    """Head by head and a stretch of queries at a time; gradients by automatic
    differentiation of the forward definition."""
    q, k, v = t["q"], t["k"], t["v"]
    train = case["train"]
    group = case["heads"] // case["kv_heads"]
    root = math.sqrt(case["head_dim"])
    out = torch.zeros_like(q)
    grads = tuple(torch.zeros_like(x) for x in (q, k, v))
    qa = ka = 0
    for lq, lk in zip(*lens):
        keep = torch.arange(ka, ka + lk, device=q.device)
        if mask is not None:
            keep = keep[mask[ka:ka + lk]]
        stretch = max(1, (1 << 27) // max(1, lk))
        for h in range(case["heads"] if keep.numel() else 0):
            kh, vh = k[keep, h // group], v[keep, h // group]
            for a in range(qa, qa + lq, stretch):
                b = min(a + stretch, qa + lq)
                qh = q[a:b, h]
                if train:
                    qh, kh, vh = (x.detach().requires_grad_(True) for x in (qh, kh, vh))
                o = torch.softmax(qh @ kh.t() / root, 1) @ vh
                out[a:b, h] = o.detach()
                if train:
                    gq, gk, gv = torch.autograd.grad(o, (qh, kh, vh), t["dy"][a:b, h])
                    grads[0][a:b, h] = gq
                    grads[1][keep, h // group] += gk
                    grads[2][keep, h // group] += gv
        qa, ka = qa + lq, ka + lk
    return (out,) + grads if train else out
