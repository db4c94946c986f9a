"""The definitions of the per-head norm and rotation, the 8-bit cache and the attention over it, in f64 on the CPU."""
import torch

MIN_SCALE = 2.0 ** -60


def angles(positions, frequencies, axis_pairs):
    """(..., pairs) angles of positions (axes, ...)."""
    parts, at = [], 0
    for a, n in enumerate(axis_pairs):
        parts.append(positions[a].double().unsqueeze(-1) * frequencies[at:at + n])
        at += n
    return torch.cat(parts, -1)


def transform(x, gain, norm, eps, angle, interleaved):
    """x (..., heads, d) in f64; angle (..., pairs) or None; returns the transformed heads."""
    if norm:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        if gain is not None:
            x = x * gain
    if angle is None or angle.shape[-1] == 0:
        return x
    n = angle.shape[-1]
    c, s = angle.cos().unsqueeze(-2), angle.sin().unsqueeze(-2)
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)


def e4m3(x):
    """To the nearest e4m3 value, ties to even, saturating."""
    mag = x.abs().clamp_min(2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(mag)) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def scale_for(top):
    """The smallest power of two >= MIN_SCALE with top <= 448 scale."""
    m, e = torch.frexp(top / 448.0)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(top > 0, torch.exp2(e.double()), torch.zeros_like(top)).clamp_min(MIN_SCALE)


def attention(q, k, v, alpha, visible):
    """q (m, heads, d), k, v (n, kv_heads, d), visible (m, n): out (m, heads, d), lse (m, heads), and the sums of |w v|."""
    group = q.shape[1] // k.shape[1]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("mhd,nhd->mhn", q, kk) * alpha
    s = s.masked_fill(~visible[:, None, :], -torch.inf)
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full(q.shape[:2], -torch.inf, dtype=torch.float64)
    w = torch.exp(s - lse.clamp_min(-1e300).unsqueeze(-1))
    w = torch.where(visible[:, None, :], w, torch.zeros_like(w))
    vis = visible.any(0)
    vv = torch.where(vis[:, None, None], vv, torch.zeros_like(vv))
    return torch.einsum("mhn,nhd->mhd", w, vv), lse, torch.einsum("mhn,nhd->mhd", w, vv.abs())
