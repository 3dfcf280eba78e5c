"""GPU parity of the row operators (mignn.attention: rms_norm, rotary,
cross_attention) against the float64 restatements in oracle/attention_oracle.py.

Tolerances come from counting roundings.  u = 2^-24 is fp32's half step, h the
half step of the rows' type (bf16 2^-8 / 2 = finfo.eps / 2, fp16 2^-11, fp32 u).
A sum of n terms in fp32 is off by at most (n + 2) u times the sum of the terms'
absolute values ("magnitude", from the oracle), and each stored value once more
by h of itself:

  rms_norm   sums of <= 64 terms a lane and 6 butterfly steps (70 u of the sum,
             35 u of its root), 4 roundings in y: 48 u; gradients take a second
             such sum: 128 u of their magnitude; dw adds n rows: (n + 128) u
  rotary     sine and cosine from a fraction rounded to fp32 (2 pi 2^-26) and 2
             ulp of sincospi, three roundings of the product: 8 u (|u| + |v|)
  attention  a score is off by e = (d + 6) u of its magnitude S, which moves its
             weight by the factor 1 +- 2 e; sums over L keys and the statistics:
             r = 2 (d + 6) u S + (L + 16) u of the output's magnitude.  16-bit
             rows: P and dS are rounded to the rows' type ahead of the products
             over keys or rows, once more h of the magnitude each (2 h where dS
             carries P's as well).  Gradients: 2 r (P's error and that of <do, o>).
"""

import math

import pytest
import torch

from mignn import _lib
from mignn import attention as A
from oracle import attention_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    _lib.lib()


def half_step(dt):
    return torch.finfo(dt).eps / 2


def rnd(*shape, seed=0, dt=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dt).to(DEV)


def close(got, ref, bound, dt, what=""):
    """|got - ref| <= bound + the store's rounding (and fp16's subnormal step)."""
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -140
    lim = bound + half_step(dt) * (ref.abs() + bound) + tiny
    err = (got - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (err > lim)
    assert not over.any(), (f"{what}: {int(over.sum())} of {err.numel()} over, worst "
                            f"{(err / lim).max().item():.2f} of the bound at "
                            f"{int((err / lim).argmax())}")


# ---------------------------------------------------------------------------
# rms_norm

NORM_SHAPES = [(1, 128), (1, 1), (3, 5), (7, 8), (1000, 96), (513, 257), (130, 507), (65, 1023),
               (9, 1024), (5, 2048), (3, 2047), (0, 64), (40000, 64)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,h", NORM_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(n, h, dt, residual):
    x, w = rnd(n, h, seed=1, dt=dt), rnd(h, seed=2, dt=dt)
    r = rnd(n, h, seed=3, dt=dt, scale=3.0) if residual else None
    res = A.rms_norm(x, w, residual=r)
    y, s = res if residual else (res, None)
    ry, rs, rstd = orc.rms_norm(x, w, r)
    mag = x.double().cpu().abs() + (r.double().cpu().abs() if residual else 0.0)
    close(y, ry, 48 * U * (rstd * mag * w.double().cpu().abs()), dt, "y")
    if residual:
        close(s, rs, U * mag, dt, "s")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,h", NORM_SHAPES)
@pytest.mark.parametrize("residual,weight32", [(True, False), (False, True)])
def test_rms_norm_backward(n, h, dt, residual, weight32):
    wt = torch.float32 if weight32 else dt
    x, w = rnd(n, h, seed=1, dt=dt).requires_grad_(), rnd(h, seed=2, dt=wt).requires_grad_()
    r = rnd(n, h, seed=3, dt=dt, scale=3.0).requires_grad_() if residual else None
    dy, ds = rnd(n, h, seed=4, dt=dt), rnd(n, h, seed=5, dt=dt) if residual else None
    if residual:
        y, s = A.rms_norm(x, w, residual=r)
        gx, gw, gr = torch.autograd.grad((y, s), (x, w, r), (dy, ds))
        assert torch.equal(gx, gr)
    else:
        gx, gw = torch.autograd.grad(A.rms_norm(x, w), (x, w), dy)
    assert gw.dtype == wt
    rx, rw, mx, mw = orc.rms_norm_grads(x.detach(), w.detach(), r.detach() if residual else None,
                                        1e-6, dy, ds)
    # the residual's sum carries u of |x| + |r|, which s may cancel
    if residual:
        _, s64, rstd = orc.rms_norm(x.detach(), w.detach(), r.detach())
        extra = (x.detach().double().cpu().abs() + r.detach().double().cpu().abs() + s64.abs())
        t = dy.double().cpu()
        mw = mw + (t.abs() * extra * rstd).sum(0)
        g = (t * w.detach().double().cpu()).abs()
        mx = mx + rstd ** 3 * (extra * (g * s64.abs()).mean(1, keepdim=True)
                               + s64.abs() * (g * extra).mean(1, keepdim=True))
    close(gx, rx, 128 * U * mx, dt, "dx")
    close(gw, rw, (n + 128) * U * mw, wt, "dw")


def test_rms_norm_strides_partial_grads_and_zero_rows():
    base = rnd(20, 300, seed=7)
    x = base[:, 30:130]                       # row stride 300, pointer off 16 bytes
    w = rnd(100, seed=8)
    assert torch.equal(A.rms_norm(x, w), A.rms_norm(x.contiguous(), w))
    xt = rnd(100, 20, seed=9).t()             # columns not contiguous
    assert torch.equal(A.rms_norm(xt, w), A.rms_norm(xt.contiguous(), w))
    xe = base[:1, :100].expand(20, 100)       # one row for all
    assert torch.equal(A.rms_norm(xe, w), A.rms_norm(xe.contiguous(), w))
    # eps keeps an all-zero row finite; only the stream's gradient; only the weight's
    z = torch.zeros(3, 100, device=DEV, requires_grad=True)
    y, s = A.rms_norm(z, w, residual=torch.zeros(3, 100, device=DEV))
    assert (y == 0).all()
    g, = torch.autograd.grad(s.sum(), z, retain_graph=True)
    assert (g == 1).all()
    assert torch.isfinite(torch.autograd.grad(y.sum(), z)[0]).all()
    wg = w.clone().requires_grad_()
    gw, = torch.autograd.grad(A.rms_norm(x, wg).sum(), wg)
    rw = orc.rms_norm_grads(x, w, None, 1e-6, torch.ones(20, 100))
    close(gw, rw[1], 148 * U * rw[3], torch.float32)
    # an expanded gradient (stride 0), and the same tensor as x and residual
    xg = x.contiguous().requires_grad_()
    y, s = A.rms_norm(xg, w, residual=xg)
    g2, = torch.autograd.grad((y + s).sum(), xg)
    rx, _, mx, _ = orc.rms_norm_grads(x, w, x, 1e-6, torch.ones(20, 100), torch.ones(20, 100))
    close(g2, 2 * rx, 2 * 130 * U * mx, torch.float32)


def test_rms_norm_nan_stays_in_its_row():
    x = rnd(70, 96, seed=1)
    ref = A.rms_norm(x, torch.ones(96, device=DEV))
    x[13, 5], x[40, 95] = float("nan"), float("inf")
    y = A.rms_norm(x, torch.ones(96, device=DEV))
    ok = torch.ones(70, dtype=torch.bool, device=DEV)
    ok[13] = ok[40] = False
    assert torch.equal(y[ok], ref[ok]) and y[13].isnan().all() and y[40, 95].isnan()


# ---------------------------------------------------------------------------
# rotary

@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,d,pairs", [
    (1, 4, 32, (6, 5, 5)), (37, 3, 20, (4, 4)), (130, 1, 6, (1, 1, 1)), (1000, 8, 64, (16, 16)),
    (77, 2, 40, (7, 0, 6)), (5, 2, 2, (1,)), (0, 2, 8, (4,)), (19, 5, 128, (22, 21, 21)),
    (64, 1, 66, (11, 11, 10, 1)), (3, 2, 8200, (4096,)), (700, 1, 4, (1, 1)), (2, 300, 16, (8,))])
def test_rotary_and_gradient(n, heads, d, pairs, dt, interleaved):
    x = rnd(n, heads, d, seed=1, dt=dt).requires_grad_()
    pos = torch.rand(n, len(pairs), generator=torch.Generator().manual_seed(2)).to(DEV)
    scales = tuple(100.0 * (a + 1) for a in range(len(pairs)))
    axes = A.RotaryAxes(pairs, scales=scales, interleaved=interleaved)
    y = A.rotary(x, pos, axes)
    dy = rnd(n, heads, d, seed=3, dt=dt)
    gx, = torch.autograd.grad(y, x, dy)
    for got, src, inv in ((y, x.detach(), False), (gx, dy, True)):
        ref = orc.rotary(src, pos, pairs, scales=scales, interleaved=interleaved, inverse=inv)
        mag = src.double().cpu().abs()
        m = sum(pairs)
        bound = torch.zeros_like(mag)
        if interleaved:
            b = mag[..., 0:2 * m:2] + mag[..., 1:2 * m:2]
            bound[..., 0:2 * m:2] = bound[..., 1:2 * m:2] = b
        else:
            b = mag[..., :m] + mag[..., m:2 * m]
            bound[..., :m] = bound[..., m:2 * m] = b
        close(got, ref, 8 * U * bound, dt)
        assert torch.equal(got[..., 2 * m:], src[..., 2 * m:])


@pytest.mark.parametrize("pt", [torch.float32, torch.float64, torch.int32, torch.int64])
def test_rotary_far_positions_strides_and_types(pt):
    """Positions of 1e8 and above (2^40 where the type holds them): the angle's
    turns are formed in fp64, whose product is off by 2^-53 of them."""
    big = 2 ** 40 if pt in (torch.float64, torch.int64) else 10 ** 8
    pos = (torch.tensor([[0, 1], [3, big], [-big, 7], [big - 1, -5]])).to(pt).to(DEV)
    qkv = rnd(4, 3, 2, 16, seed=1)
    axes = A.RotaryAxes((4, 4))
    x = qkv[:, 1]                                  # a head block of a fused projection
    y = A.rotary(x, pos, axes)
    ref = orc.rotary(x, pos, (4, 4))
    mag = x.double().cpu().abs()
    bound = (8 * U + 8 * 2.0 ** -53 * big) * (mag + mag.roll(8, 2))
    close(y, ref, bound, torch.float32)
    wide = torch.empty(4, 4, dtype=pt, device=DEV)
    wide[:, ::2] = pos
    assert torch.equal(A.rotary(x, wide[:, ::2], axes), y)
    assert torch.equal(A.rotary(x.transpose(0, 1).contiguous().transpose(0, 1), pos, axes), y)
    assert torch.equal(A.rotary(qkv[:1, 1].expand(4, 2, 16), pos, axes),
                       A.rotary(qkv[:1, 1].expand(4, 2, 16).contiguous(), pos, axes))


def test_rotary_odd_alignment():
    flat = rnd(1 + 50 * 3 * 30, seed=4, dt=torch.bfloat16)
    x = flat[1:].view(50, 3, 30)                   # rows 2 bytes off
    pos = torch.arange(50, device=DEV)[:, None]
    axes = A.RotaryAxes((15,))
    assert torch.equal(A.rotary(x, pos, axes), A.rotary(x.clone(), pos, axes))


# ---------------------------------------------------------------------------
# cross attention

CROSS = [
    # q_lens, k_lens, heads, kv_heads, d
    ([1], [1], 1, 1, 32), ([1], [33], 4, 4, 32), ([5], [0], 2, 1, 16), ([0], [7], 2, 2, 8),
    ([33, 0, 1, 130], [65, 4, 0, 257], 4, 2, 24), ([3, 1, 2], [700, 31, 32], 8, 2, 64),
    ([129], [129], 2, 2, 40), ([64], [200], 3, 1, 96), ([70, 70], [40, 150], 4, 4, 128),
    ([1] * 9, [1, 2, 3, 15, 16, 17, 63, 64, 900], 8, 1, 72), ([300], [3], 4, 1, 56),
    ([2], [5000], 4, 4, 32), ([2100], [20], 4, 2, 64), ([260], [1111], 2, 2, 104),
    ([2, 1], [3000, 70], 8, 2, 48), ([7, 90], [100, 40], 32, 1, 32), ([31], [300], 6, 2, 128),
]


def cross_bounds(ref, dt, d, klens, qlens, group):
    h = half_step(dt) if dt != torch.float32 else 0.0
    s = ref["score_mag"].max().item() if ref["score_mag"].numel() else 0.0
    lk, lr = max(klens, default=0), max(qlens, default=0) * group
    base = 2 * (d + 6) * U * s
    r = base + (lk + 16) * U
    return {"out": (r + h) * ref["out_mag"],
            "dq": (2 * (r + (lk + d + 16) * U) + 2 * h) * ref["dq_mag"],
            "dk": (2 * (r + (lr + lk + d + 16) * U) + 2 * h) * ref["dk_mag"],
            "dv": (base + (lr + lk + 16) * U + h) * ref["dv_mag"]}


def cross_inputs(ql, kl, heads, kv, d, dt, seed=0, masked="none"):
    q, k, v = (rnd(sum(n), m, d, seed=seed + i, dt=dt)
               for i, (n, m) in enumerate(((ql, heads), (kl, kv), (kl, kv))))
    mask = None
    if masked != "none":
        mask = torch.rand(sum(kl), generator=torch.Generator().manual_seed(seed + 9)) < 0.6
        if masked == "empty" and kl:
            mask[:kl[0]] = False              # the first sequence keeps no key
        # what the mask leaves out may hold anything
        for t, val in ((k, float("nan")), (v, float("inf"))):
            t[~mask.to(DEV)] = val
        mask = mask.to(DEV)
    return q, k, v, mask


def clean(t, mask):
    return t if mask is None else torch.where(mask[:, None, None], t, torch.zeros_like(t))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("masked", ["none", "some", "empty"])
@pytest.mark.parametrize("ql,kl,heads,kv,d", CROSS)
def test_cross_attention(ql, kl, heads, kv, d, dt, masked):
    q, k, v, mask = cross_inputs(ql, kl, heads, kv, d, dt, masked=masked)
    plan = A.CrossPlan(ql, kl, heads=heads, kv_heads=kv, head_dim=d, dtype=dt)
    with torch.no_grad():
        served = A.cross_attention(q, k, v, plan, key_mask=mask)
    for t in (q, k, v):
        t.requires_grad_()
    out = A.cross_attention(q, k, v, plan, key_mask=mask)
    do = rnd(*q.shape, seed=5, dt=dt)
    grads = torch.autograd.grad(out, (q, k, v), do)
    ref = orc.cross_attention(q, clean(k, mask), clean(v, mask), ql, kl, mask, None, do)
    bound = cross_bounds(ref, dt, d, kl, ql, heads // kv)
    close(served, ref["out"], bound["out"], dt, "out (no gradients)")
    close(out, ref["out"], bound["out"], dt, "out")
    for name, g in zip(("dq", "dk", "dv"), grads):
        close(g, ref[name], bound[name], dt, name)
    if masked == "empty" and ql and kl:
        assert (out[:ql[0]] == 0).all() and (grads[0][:ql[0]] == 0).all()
    if mask is not None:
        assert (grads[1][~mask] == 0).all() and (grads[2][~mask] == 0).all()


@pytest.mark.parametrize("dt", TYPES)
def test_cross_attention_scale_and_large_scores(dt):
    """A given scale, and scores far beyond exp's range (a softmax that picks
    one key)."""
    ql, kl = [40], [90]
    q, k, v, _ = cross_inputs(ql, kl, 2, 1, 32, dt, seed=3)
    plan = A.CrossPlan(ql, kl, heads=2, kv_heads=1, head_dim=32, dtype=dt)
    for scale in (0.01, 1.0, 30.0):
        ref = orc.cross_attention(q, k, v, ql, kl, None, scale)
        out = A.cross_attention(q, k, v, plan, scale=scale)
        close(out, ref["out"], cross_bounds(ref, dt, 32, kl, ql, 2)["out"], dt, f"scale {scale}")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ql,kl", [([200], [700]), ([1], [4000])])
def test_cross_attention_strides(ql, kl, dt):
    """Heads inside a fused projection, rows at an odd alignment, broadcast
    keys, transposed heads: the same results as from contiguous copies."""
    d, n, m = 32, sum(ql), sum(kl)
    plan = A.CrossPlan(ql, kl, heads=2, kv_heads=2, head_dim=d, dtype=dt)
    kvf = rnd(m, 4, d, seed=1, dt=dt)
    flat = rnd(3 + n * 2 * d, seed=2, dt=dt)
    q = flat[3:].view(n, 2, d)
    k, v = kvf[:, 1:3], kvf[:, ::2]
    run = lambda *a: A.cross_attention(*a, plan)  # noqa: E731
    want = run(q.clone(), k.contiguous(), v.contiguous())
    assert torch.equal(run(q, k, v), want)
    assert torch.equal(run(q, k.transpose(0, 1).contiguous().transpose(0, 1), v), want)
    one = k[:, :1].expand(m, 2, d)                    # one head's keys for both
    assert torch.equal(run(q, one, v), run(q, one.contiguous(), v))
    # gradients: of a broadcast input summed, for an expanded output gradient
    kk = k[:, :1].contiguous().requires_grad_()
    qq, vv = q.clone().requires_grad_(), v.contiguous().requires_grad_()
    out = run(qq, kk.expand(m, 2, d), vv)
    got = torch.autograd.grad(out.sum(), (qq, kk, vv))
    k2 = one.contiguous().requires_grad_()
    out = run(qq, k2, vv)
    ref = torch.autograd.grad(out, (qq, k2, vv), torch.ones_like(out))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[2], ref[2])
    assert torch.equal(got[1], ref[1].sum(1, keepdim=True))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ql,kl", [([700], [900]), ([2], [6000]), ([5000], [17])])
def test_cross_attention_is_deterministic_and_stream_safe(ql, kl, dt):
    """Equal bits from run to run, from another stream, and in gradients asked
    for one at a time."""
    q, k, v, mask = cross_inputs(ql, kl, 4, 2, 64, dt, masked="some")
    plan = A.CrossPlan(ql, kl, heads=4, kv_heads=2, head_dim=64, dtype=dt)
    for t in (q, k, v):
        t.requires_grad_()
    do = rnd(*q.shape, seed=5, dt=dt)

    def step():
        out = A.cross_attention(q, k, v, plan, key_mask=mask)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), do)
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    again = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    for i, t in enumerate((q, k, v)):
        for x in (q, k, v):
            x.requires_grad_(x is t)
        out = A.cross_attention(q, k, v, plan, key_mask=mask)
        assert torch.equal(torch.autograd.grad(out, t, do)[0], first[1 + i])


@pytest.mark.parametrize("up", [2.0 ** -9, 1.0, 2.0 ** 9])
@pytest.mark.parametrize("ql,kl", [([2], [5000]), ([130], [300]), ([900], [9])])
def test_cross_attention_fp16_range(ql, kl, up):
    """fp16 rows with output gradients and values far from 1: P and dS leave
    fp16's range (dS up to 2^9 2^6 sqrt(d) and more, down to 2^-9 / 5000), the
    gradients do not."""
    dt, d = torch.float16, 64
    q, k, v, _ = cross_inputs(ql, kl, 2, 1, d, dt, seed=3)
    v = (v.float() * (8.0 if up > 1 else 1.0)).to(dt)
    do = rnd(*q.shape, seed=8, dt=dt, scale=up)
    # rows of very unlike gradients in one tile
    do[::3] = do[::3] * 2.0 ** -7
    plan = A.CrossPlan(ql, kl, heads=2, kv_heads=1, head_dim=d, dtype=dt)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(A.cross_attention(*leaves, plan, scale=0.03), leaves, do)
    ref = orc.cross_attention(q, k, v, ql, kl, None, 0.03, do)
    assert max(ref[n].abs().max().item() for n in ("dq", "dk", "dv")) < 65504
    bound = cross_bounds(ref, dt, d, kl, ql, 2)
    for name, g in zip(("dq", "dk", "dv"), grads):
        close(g, ref[name], bound[name], dt, name)


def test_cross_attention_nan_in_a_query_stays_in_its_row():
    ql, kl = [100], [300]
    q, k, v, _ = cross_inputs(ql, kl, 2, 2, 32, torch.float32)
    plan = A.CrossPlan(ql, kl, heads=2, head_dim=32)
    ref = A.cross_attention(q, k, v, plan)
    q[57, 1, 3] = float("nan")
    out = A.cross_attention(q, k, v, plan)
    assert out[57, 1].isnan().all()
    keep = torch.ones(100, 2, dtype=torch.bool, device=DEV)
    keep[57, 1] = False
    assert torch.equal(out[keep], ref[keep])


def test_cross_attention_gradient_matches_differences():
    """<gradient, way> against central differences of the kernel's own forward,
    with the truncation taken from the oracle's differences at the same step."""
    ql, kl, d, e = [20, 7], [50, 90], 32, 2.0 ** -5
    q, k, v, mask = cross_inputs(ql, kl, 4, 2, d, torch.float32, masked="some")
    k, v = clean(k, mask), clean(v, mask)
    plan = A.CrossPlan(ql, kl, heads=4, kv_heads=2, head_dim=d)
    do = rnd(*q.shape, seed=5)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(A.cross_attention(*leaves, plan, key_mask=mask), leaves, do)
    ref = orc.cross_attention(q, k, v, ql, kl, mask, None, do)
    bound = cross_bounds(ref, torch.float32, d, kl, ql, 2)
    for i, name in enumerate(("dq", "dk", "dv")):
        way = rnd(*(q, k, v)[i].shape, seed=20 + i)
        num, onum, slack = 0.0, 0.0, 0.0
        for s in (1, -1):
            args = [t + s * e * way if j == i else t for j, t in enumerate((q, k, v))]
            out = A.cross_attention(*args, plan, key_mask=mask)
            o = orc.cross_attention(*args, ql, kl, mask)
            num += s * (out.double().cpu() * do.double().cpu()).sum().item() / (2 * e)
            onum += s * (o["out"] * do.double().cpu()).sum().item() / (2 * e)
            b = cross_bounds(o, torch.float32, d, kl, ql, 2)["out"] + U * o["out"].abs()
            slack += (b * do.double().cpu().abs()).sum().item() / (2 * e)
        w = way.double().cpu()
        exact = (ref[name] * w).sum().item()
        mine = (grads[i].double().cpu() * w).sum().item()
        gslack = ((bound[name] + U * ref[name].abs()) * w.abs()).sum().item()
        assert abs(num - onum) <= slack, name
        assert abs(mine - exact) <= gslack, name
        assert abs(mine - num) <= slack + gslack + abs(onum - exact), name


def test_operators_in_captured_graphs():
    """Two graphs over one plan and one RotaryAxes, replayed in turn with new
    inputs and eager calls between: each replay equals the eager result."""
    ql, kl, d = [65, 3], [400, 90], 32
    plan = A.CrossPlan(ql, kl, heads=4, kv_heads=2, head_dim=d)
    axes = A.RotaryAxes((8, 8))
    w = rnd(4 * d, seed=9)

    def make():
        st = {n: torch.empty(s, device=DEV) for n, s in
              (("q", (68, 4 * d)), ("k", (490, 2, d)), ("v", (490, 2, d)), ("qp", (68, 2)),
               ("kp", (490, 2)), ("do", (68, 4, d)))}
        return st

    def fill(st, seed):
        for i, t in enumerate(st.values()):
            t.copy_(rnd(*t.shape, seed=seed + i))

    def step(st):
        leaves = [st[n].detach().requires_grad_() for n in ("q", "k", "v")]
        y, s = A.rms_norm(leaves[0], w, residual=leaves[0])
        q = A.rotary(y.view(68, 4, d), st["qp"], axes)
        o = A.cross_attention(q, A.rotary(leaves[1], st["kp"], axes), leaves[2], plan)
        return (o.detach(), s.detach()) + torch.autograd.grad(o, leaves, st["do"])

    states, graphs, outs = [make(), make()], [], []
    for i, st in enumerate(states):
        fill(st, 10 * i)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(st)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(st))
        graphs.append(g)
    for rep in range(3):
        for i in (0, 1):
            fill(states[i], 100 * rep + 10 * i)
            graphs[i].replay()
        for i in (0, 1):
            for a, b in zip(outs[i], step(states[i])):
                assert torch.equal(a, b)


def test_gradients_are_first_order_only():
    """create_graph gives the gradients; differentiating them again is refused."""
    x = rnd(6, 32, seed=1).requires_grad_()
    w = torch.ones(32, device=DEV, requires_grad=True)
    axes = A.RotaryAxes((8,))
    plan = A.CrossPlan([6], [6], heads=1, head_dim=32)

    def ops():
        yield A.rms_norm(x, w)
        yield A.rms_norm(x, w, residual=x)[0]
        yield A.rotary(x.view(6, 1, 32), torch.arange(6, device=DEV)[:, None], axes)
        yield A.cross_attention(*(x.view(6, 1, 32),) * 3, plan)
    for y in ops():
        plain, = torch.autograd.grad(y.square().sum(), x, retain_graph=True)
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        assert torch.equal(g.detach(), plain) and g.requires_grad
        with pytest.raises(RuntimeError, match="first order only"):
            g.sum().backward(retain_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("queries", [1, 40])
def test_cross_attention_offsets_past_32_bits(queries):
    """17 million keys of 128 bf16 columns (2^31.02 elements) of which the mask
    keeps some at both ends: outputs and gradients equal those of the kept keys."""
    n, d = 17_000_000, 128
    keep = torch.cat([torch.arange(0, 60), torch.arange(n - 90, n)])
    k = torch.zeros(n, 1, d, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    ks, vs = rnd(150, 1, d, seed=1, dt=torch.bfloat16), rnd(150, 1, d, seed=2, dt=torch.bfloat16)
    k[keep.to(DEV)], v[keep.to(DEV)] = ks, vs
    mask = torch.zeros(n, dtype=torch.bool, device=DEV)
    mask[keep.to(DEV)] = True
    q, do = (rnd(queries, 2, d, seed=s, dt=torch.bfloat16) for s in (3, 4))
    plan = A.CrossPlan([queries], [n], heads=2, kv_heads=1, head_dim=d, dtype=torch.bfloat16)
    for t in (q, k, v):
        t.requires_grad_()
    out = A.cross_attention(q, k, v, plan, key_mask=mask)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    ref = orc.cross_attention(q, ks, vs, [queries], [150], None, None, do)
    # (the sums run over 150 weights that are not 0)
    bound = cross_bounds(ref, torch.bfloat16, d, [150], [queries], 2)
    close(out, ref["out"], bound["out"], torch.bfloat16, "out")
    close(dq, ref["dq"], bound["dq"], torch.bfloat16, "dq")
    close(dk[keep.to(DEV)], ref["dk"], bound["dk"], torch.bfloat16, "dk")
    close(dv[keep.to(DEV)], ref["dv"], bound["dv"], torch.bfloat16, "dv")
    assert dk[~mask].count_nonzero() == 0 and dv[~mask].count_nonzero() == 0


def test_norm_and_rotary_offsets_past_32_bits():
    n, h = 17_000_000, 128
    x = torch.empty(n, h, dtype=torch.bfloat16, device=DEV)
    x[:] = rnd(1, h, seed=1, dt=torch.bfloat16)
    x[-300:] = rnd(300, h, seed=2, dt=torch.bfloat16)
    w = rnd(h, seed=3, dt=torch.bfloat16)
    y = A.rms_norm(x, w)
    assert torch.equal(y[-300:], A.rms_norm(x[-300:].clone(), w))
    assert torch.equal(y[:-300], y[:1].expand(n - 300, h))
    del y
    pos = torch.zeros(n, 1, dtype=torch.int64, device=DEV)
    pos[-300:, 0] = torch.arange(300, device=DEV) * 1000
    axes = A.RotaryAxes((16,))
    y = A.rotary(x.view(n, 4, 32), pos, axes)
    assert torch.equal(y[-300:], A.rotary(x[-300:].clone().view(300, 4, 32), pos[-300:], axes))
    assert torch.equal(y[:-300], x[:-300].view(-1, 4, 32))


def test_cross_attention_from_two_threads_and_streams():
    """Two threads, each on its own stream, over one plan: every result is the
    single call's."""
    import threading
    ql, kl, d = [300, 5], [900, 4000], 64
    plan = A.CrossPlan(ql, kl, heads=4, kv_heads=2, head_dim=d, dtype=torch.bfloat16)
    sets = [cross_inputs(ql, kl, 4, 2, d, torch.bfloat16, seed=30 * i)[:3] for i in (0, 1)]
    want = [A.cross_attention(*s, plan) for s in sets]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    got[i].append(A.cross_attention(*sets[i], plan))
            st.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_cross_attention_wide_strides_are_copied():
    """Rows further apart than the kernels' offsets reach (2^23 elements)."""
    base = torch.zeros(4, (1 << 23) + 64, device=DEV)
    base[:, :64] = rnd(4, 64, seed=1)
    q = base[:, :64].unflatten(1, (2, 32))
    plan = A.CrossPlan([4], [4], heads=2, head_dim=32)
    c = q.contiguous()
    assert torch.equal(A.cross_attention(q, q, q, plan), A.cross_attention(c, c, c, plan))


# ---------------------------------------------------------------------------
# the operators together: the block and the surrogate that calls it

def block_oracle(blk, x, pos, context, cpos, ql, kl, mask=None):
    """CrossAttention.forward in float64 (autograd through it gives its gradients)."""
    def norm(t, w):
        return t / torch.sqrt((t * t).mean(1, keepdim=True) + blk.eps) * w
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in blk.named_parameters()}
    x, context = (t.detach().double().cpu().requires_grad_() for t in (x, context))
    half, d = blk.head_dim // 2, blk.head_dim
    pairs = [half // blk.axes + (a < half % blk.axes) for a in range(blk.axes)]

    def turn(t, ps):
        ang = torch.stack([ps[:, a].double().cpu() * blk.position_scale * blk.base ** (-i / m)
                           for a, m in enumerate(pairs) for i in range(m)], 1)[:, None]
        u, v = t[..., :half], t[..., half:]
        return torch.cat([u * ang.cos() - v * ang.sin(), v * ang.cos() + u * ang.sin()], 2)
    lin = lambda t, n: t @ p[n + ".weight"].T + p[n + ".bias"]  # noqa: E731
    q = turn(lin(norm(x, p["norm_x"]), "lin_query").view(-1, blk.heads, d), pos)
    c = norm(context, p["norm_context"])
    k = turn(lin(c, "lin_key").view(-1, blk.kv_heads, d), cpos)
    v = lin(c, "lin_value").view(-1, blk.kv_heads, d)
    g, rows, qa, ka = blk.heads // blk.kv_heads, [], 0, 0
    for lq, lk in zip(ql, kl):
        keep = torch.arange(ka, ka + lk)
        if mask is not None:
            keep = keep[mask.cpu()[ka:ka + lk]]
        heads = [torch.softmax(q[qa:qa + lq, h] @ k[keep, h // g].T / math.sqrt(d), 1)
                 @ v[keep, h // g] if keep.numel() else 0.0 * q[qa:qa + lq, h]
                 for h in range(blk.heads)]
        rows.append(torch.cat(heads, 1))
        qa, ka = qa + lq, ka + lk
    s = x + lin(torch.cat(rows), "lin_out")
    return norm(s, p["norm_out"]), s, x, context, p


@pytest.mark.parametrize("kv", [4, 2])
@pytest.mark.parametrize("ql,kl,masked", [([150, 33], [40, 300], False), ([70, 5, 9], [64, 0, 31], True),
                                          ([1], [500], False)])
def test_block(ql, kl, kv, masked):
    """norm, projections, rotation, attention and the residual's norm in one
    run: outputs and every gradient against the float64 block.  Bound: each of
    the ~8 steps loses what its own test grants (at most (h + L + 64) u of its
    magnitude, widths 64, L <= 300), through weights of norm about 1: 2^-24 *
    8 * 512 = 2^-12 of the largest value of the tensor."""
    blk = A.CrossAttention(64, 4, kv)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for n, t in blk.named_parameters():
            t.copy_(torch.randn(t.shape, generator=g) * (0.1 if t.dim() == 1 else 0.125)
                    + (1.0 if n.startswith("norm") else 0.0))
    blk = blk.to(DEV)
    x, ctx = rnd(sum(ql), 64, seed=2).requires_grad_(), rnd(sum(kl), 64, seed=3).requires_grad_()
    pos = torch.rand(sum(ql), 3, generator=g).to(DEV)
    cpos = torch.rand(sum(kl), 3, generator=g).to(DEV)
    mask = (torch.rand(sum(kl), generator=g) < 0.7).to(DEV) if masked else None
    plan = blk.plan(ql, kl)
    y, s = blk(x, pos, ctx, cpos, plan, key_mask=mask)
    dy, ds = rnd(*y.shape, seed=4), rnd(*y.shape, seed=5)
    names, params = zip(*blk.named_parameters())
    grads = torch.autograd.grad((y, s), (x, ctx) + params, (dy, ds))
    ry, rs, rx, rc, rp = block_oracle(blk, x, pos, ctx, cpos, ql, kl, mask)
    ref = torch.autograd.grad((ry, rs), (rx, rc) + tuple(rp[n] for n in names),
                              (dy.double().cpu(), ds.double().cpu()))
    for name, a, b in [("y", y, ry), ("s", s, rs)] + list(zip(("x", "context") + names, grads, ref)):
        err = (a.detach().double().cpu() - b.detach()).abs().max().item()
        assert err <= 2.0 ** -12 * max(b.abs().max().item(), 1e-3), (name, err)
    with torch.no_grad():
        k, v = blk.keys_values(ctx, cpos)
        y2, s2 = blk.attend(x, pos, k, v, plan, mask)
    assert (y2 - y).abs().max() <= 2.0 ** -12 * y.abs().max()
    assert (s2 - s).abs().max() <= 2.0 ** -12 * s.abs().max()


def grid(nx, ny, nz, seed=0):
    from mignn.synthetic import grid_graph
    return grid_graph(nx, ny, nz, device=DEV, permute_seed=seed)


@pytest.mark.parametrize("layer_type", ["GCN", "GAT"])
def test_surrogate_with_context(layer_type):
    """FlowGNNSurrogate(cross_heads): eval forward equals its parts run by hand,
    a training step reaches every parameter, and the context's nodes matter."""
    from mignn import Data, FlowGNNSurrogate
    m = FlowGNNSurrogate(hidden_dim=64, num_layers=4, layer_type=layer_type, dropout=0.0,
                         cross_heads=4).to(DEV)
    x, ei = grid(8, 6, 5)
    cx, cei = grid(4, 3, 3, seed=1)
    ctx = Data(x=cx, edge_index=cei)
    m.eval()
    with torch.no_grad():
        y = m(x, ei, context=ctx)
        enc, states = m.encoder(x, ei), m.encoder(cx, cei)
        plan = m.cross.plan([x.shape[0]], [cx.shape[0]], train=False)
        h, _ = m.cross(enc, x, states, cx, plan)
        assert torch.equal(y, m.decoder(h, ei))
        assert torch.equal(y, m(x, ei, context=ctx, plan=plan))
        assert not torch.equal(y, m(x, ei, context=Data(x=cx[:20], edge_index=cei[:, :0])))
    m.train()
    out = m(x, ei, context=ctx)
    out.square().mean().backward()
    missing = [n for n, p in m.named_parameters() if p.grad is None or not p.grad.abs().sum() > 0]
    # (an attention output bias or a layer's bias ahead of a batch norm may have gradient 0)
    assert not [n for n in missing if "bias" not in n], missing


def test_surrogate_batch_of_graphs_reads_its_own_context():
    """Two graphs with contexts of unlike size in one batch: each graph's
    attention equals that of the graph alone."""
    from mignn import Batch, Data
    blk = A.CrossAttention(64, 4).to(DEV)
    graphs = [grid(5, 4, 3), grid(4, 4, 4, seed=2)]
    ctxs = [grid(3, 3, 3, seed=3), grid(6, 3, 3, seed=4)]
    b = Batch.from_data_list([Data(x=x.cpu(), edge_index=e.cpu()) for x, e in graphs])
    cb = Batch.from_data_list([Data(x=x.cpu(), edge_index=e.cpu()) for x, e in ctxs])
    ql = A.graph_lengths(b.batch, b.num_nodes)
    kl = A.graph_lengths(cb.batch, cb.num_nodes)
    assert ql == [60, 64] and kl == [27, 54]
    h, c = rnd(124, 64, seed=1), rnd(81, 64, seed=2)
    with torch.no_grad():
        y, _ = blk(h, b.x.to(DEV), c, cb.x.to(DEV), blk.plan(ql, kl))
        a0 = c0 = 0
        for n, k in zip(ql, kl):
            one, _ = blk(h[a0:a0 + n], b.x[a0:a0 + n].to(DEV), c[c0:c0 + k], cb.x[c0:c0 + k].to(DEV),
                         blk.plan([n], [k]))
            assert (one - y[a0:a0 + n]).abs().max() <= 2.0 ** -12 * y.abs().max()
            a0, c0 = a0 + n, c0 + k


def test_plan_and_axes_dropped_while_another_stream_reads_them():
    """A plan and axes made on one stream, read by another and dropped: their
    memory is not handed out again before the reader is done."""
    x = rnd(3000, 3000, seed=1)
    q = rnd(300, 2, 32, seed=2)
    pos = torch.arange(300, device=DEV)[:, None]
    plan = A.CrossPlan([300], [300], heads=2, head_dim=32)
    axes = A.RotaryAxes((16,))
    sizes = [plan._lists.numel(), 8 * axes.freq.numel(), 4 * axes.axis.numel()]
    held = {t.data_ptr() for t in (plan._lists, axes.freq, axes.axis)}
    want = A.cross_attention(q, q, q, plan), A.rotary(q, pos, axes)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):
            x @ x
        got = A.cross_attention(q, q, q, plan), A.rotary(q, pos, axes)
    del plan, axes
    new = {torch.empty(n, dtype=torch.uint8, device=DEV).data_ptr() for n in sizes}
    busy = not side.query()
    side.synchronize()
    assert not busy or not held & new
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_out_of_memory_is_torch_s_error():
    x, pos = torch.zeros(1, 1, 64, device=DEV), torch.zeros(1, 1, device=DEV)
    with pytest.raises(torch.OutOfMemoryError):
        A.rotary(x.expand(1 << 33, 1, 64), pos.expand(1 << 33, 1), A.RotaryAxes((32,)))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("h", [8, 128, 257, 2048])
def test_rms_norm_weight_gradient_around_one_block(dt, h):
    """Rows on both sides of where one block takes all of them."""
    vec = 4 if dt == torch.float32 else 8
    lanes = 1
    while lanes < 64 and lanes < -(-h // vec):
        lanes *= 2
    edge = 4 * 4 * (64 // lanes)
    for n in (1, 2, edge - 1, edge, edge + 1, 2 * edge + 3):
        for wt in {dt, torch.float32}:
            x, dy = rnd(n, h, seed=n, dt=dt), rnd(n, h, seed=n + 1, dt=dt)
            w = rnd(h, seed=3, dt=wt).requires_grad_()
            gw, = torch.autograd.grad(A.rms_norm(x, w), w, dy)
            _, rw, _, mw = orc.rms_norm_grads(x, w.detach(), None, 1e-6, dy)
            close(gw, rw, (n + 128) * U * mw, wt, f"dw of {n} rows")
