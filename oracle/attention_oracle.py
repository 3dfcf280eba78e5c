"""float64 CPU restatements of the row operators (mignn.attention) from their
formulas, with the sums of absolute values that the tests' rounding bounds
are made of.  Test infrastructure only."""

import math

import torch


def rms_norm(x, weight, residual=None, eps=1e-6):
    x, w = x.double().cpu(), weight.double().cpu()
    s = x if residual is None else x + residual.double().cpu()
    rstd = 1.0 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    return s * rstd * w, s, rstd


def rms_norm_grads(x, weight, residual, eps, dy, ds=None):
    """(dx, dw) and the magnitudes (|terms| of dx, |terms| of dw)."""
    _, s, rstd = rms_norm(x, weight, residual, eps)
    w, dy = weight.double().cpu(), dy.double().cpu()
    g = dy * w
    c = (g * s).mean(1, keepdim=True) * rstd ** 2
    dx = rstd * (g - s * c)
    mag = rstd * (g.abs() + s.abs() * (g * s).abs().mean(1, keepdim=True) * rstd ** 2)
    if ds is not None:
        dx = dx + ds.double().cpu()
        mag = mag + ds.double().cpu().abs()
    t = dy * s * rstd
    return dx, t.sum(0), mag, t.abs().sum(0)


def rotary(x, pos, pairs, base=10000.0, scales=None, interleaved=False, inverse=False):
    x, pos = x.double().cpu(), pos.cpu().double()
    scales = (1.0,) * len(pairs) if scales is None else scales
    cols = []
    for a, m in enumerate(pairs):
        for i in range(m):
            cols.append(pos[:, a] * scales[a] * base ** (-i / m))
    ang = torch.stack(cols, 1)[:, None, :] * (-1.0 if inverse else 1.0)
    n = sum(pairs)
    y = x.clone()
    if interleaved:
        u, v = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y[..., 0:2 * n:2] = u * ang.cos() - v * ang.sin()
        y[..., 1:2 * n:2] = v * ang.cos() + u * ang.sin()
    else:
        u, v = x[..., :n], x[..., n:2 * n]
        y[..., :n] = u * ang.cos() - v * ang.sin()
        y[..., n:2 * n] = v * ang.cos() + u * ang.sin()
    return y


def cross_attention(q, k, v, q_lens, k_lens, key_mask=None, scale=None, dout=None):
    """{"out"} and, given dout, {"dq", "dk", "dv"}; each with its magnitude
    under "<name>_mag" (the sum of its terms' absolute values), and "score_mag":
    per (query, head) the largest scale sum_d |q||k| of the row."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    do = None if dout is None else dout.double().cpu()
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    g = hq // hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = {n: torch.zeros_like(q) for n in ("out", "out_mag", "dq", "dq_mag")}
    out.update({n: torch.zeros_like(k) for n in ("dk", "dk_mag", "dv", "dv_mag")})
    out["score_mag"] = torch.zeros(q.shape[:2], dtype=torch.float64)
    qa = ka = 0
    for lq, lk in zip(q_lens, k_lens):
        keep = torch.arange(ka, ka + lk)
        if key_mask is not None:
            keep = keep[key_mask.cpu()[ka:ka + lk]]
        if keep.numel() and lq:
            for h in range(hq):
                qh, kh, vh = q[qa:qa + lq, h], k[keep, h // g], v[keep, h // g]
                p = torch.softmax(scale * (qh @ kh.T), 1)
                o = p @ vh
                out["out"][qa:qa + lq, h] = o
                out["out_mag"][qa:qa + lq, h] = p @ vh.abs()
                out["score_mag"][qa:qa + lq, h] = scale * (qh.abs() @ kh.abs().T).amax(1)
                if do is None:
                    continue
                doh = do[qa:qa + lq, h]
                dp = doh @ vh.T
                ds = p * (dp - (doh * o).sum(1, keepdim=True)) * scale
                dsm = p * (doh.abs() @ vh.abs().T
                           + (doh.abs() * (p @ vh.abs())).sum(1, keepdim=True)) * scale
                out["dq"][qa:qa + lq, h] = ds @ kh
                out["dq_mag"][qa:qa + lq, h] = dsm @ kh.abs()
                out["dk"][keep, h // g] += ds.T @ qh
                out["dk_mag"][keep, h // g] += dsm.T @ qh.abs()
                out["dv"][keep, h // g] += p.T @ doh
                out["dv_mag"][keep, h // g] += p.T @ doh.abs()
        qa, ka = qa + lq, ka + lk
    return out
