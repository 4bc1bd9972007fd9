"""Attention of any mask plainly and in 64 bits, with bounds for what the kernels' roundings may add: those that scored_reference.py derives, for a given `keep`
in the place of a causal mask, ids and a prefix."""
import math

import torch


def windowed(M, N, window, sinks, prefix=None, device="cuda"):
    """[1 or B, 1, M, N]: what a causal mask with a window, its sinks and prefixes leaves visible."""
    i, j = torch.arange(M, device=device)[:, None] + max(0, N - M), torch.arange(N, device=device)
    keep = ((j <= i) & ((i - j < window) | (j < sinks)))[None, None]
    return keep if prefix is None else keep | (j < prefix.long()[:, None, None, None])


def attention_64(q, k, v, do, keep, sm_scale=None, cap=None, slopes=None, sub=None):
    """{"o", "dq", "dk", "dv"}: (value, bound) of each; the gradients where there is a `do`. `sub`: what an entry of P may lack absolutely, of a row whose sum is at
    least 1, where that is not the type's (below)."""
    B, H, M, D = q.shape
    Hk, N = k.shape[1:3]
    G, gap, dev, dtype = H // Hk, max(0, N - M), q.device, q.dtype
    u = torch.finfo(dtype).eps / 2
    half = dtype != torch.float32
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    Q, K, V = (x.detach().double() for x in (q, k, v))
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    s = Q @ K.mT * scale
    err = (D + 2) * 2.0 ** -23 * scale * (Q.abs() @ K.abs().mT)  # absolute error of a score
    far = torch.arange(M, device=dev)[:, None] + gap - torch.arange(N, device=dev)
    x, f = s, torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        x, f = cap * t, 1 - t * t
        err = err * f + 4e-6 * x.abs()
    if slopes is not None:
        bias = slopes.double()[:, None, None] * far.abs()
        x, err = x - bias, err + 4 * 2.0 ** -24 * (x.abs() + bias.abs())
    keep = keep.expand(B, H, M, N)
    x = x.masked_fill(~keep, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e300)
    p = (x - top).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    err = torch.where(p > 1e-30, err + 2.0 ** -23 * (x.abs() + top.abs()), 0.0)
    rel = 2 * err.amax((-2, -1), keepdim=True) + 2.0 ** -20
    acc = N * 2.0 ** -23
    up = u if half else 0.0
    # An entry below the type's least normal number is off by up to half the step there; and the 16-bit kernels' exponentials are 0 below fp32's least normal number,
    # 2^-126, which is bf16's as well: an entry of bf16 may lack that much, 2^8 half steps. (A key at a distance of 450 with a slope of 0.2 has exp(-90) = 2^-130.)
    if sub is None:
        sub = max(torch.finfo(dtype).smallest_normal * u, 2.0 ** -126) if half else 0.0
    seen = keep.double()
    tiny = torch.finfo(dtype).tiny if dtype != torch.float16 else 2.0 ** -24
    o = p @ V
    o_err = (up + rel + acc) * (p @ V.abs()) + sub * (seen @ V.abs()) + u * o.abs()
    out = {"o": (o, o_err * (1 + u) + 4 * tiny)}
    if do is None:
        return out
    DO = do.detach().double()
    accm = G * M * 2.0 ** -23
    dv = p.mT @ DO
    dv_err = (up + rel + accm) * (p.mT @ DO.abs()) + sub * (seen.mT @ DO.abs())
    dp, delta = DO @ V.mT, (DO * o).sum(-1, keepdim=True)
    dp_err = D * 2.0 ** -23 * (DO.abs() @ V.abs().mT)
    delta_err = (DO.abs() * (o_err + D * 2.0 ** -23 * o.abs())).sum(-1, keepdim=True)
    ds = p * (dp - delta) * f
    f_err = (2.0 ** -21 + 2 * err / cap) if cap else 0.0
    ds_err = sub * seen + (up + rel) * ds.abs() + p * ((f + f_err) * (dp_err + delta_err) + f_err * (dp - delta).abs())
    dq, dk = ds @ K * scale, ds.mT @ Q * scale
    dq_err = scale * ((ds_err + acc * ds.abs()) @ K.abs())
    dk_err = scale * ((ds_err + accm * ds.abs()).mT @ Q.abs())
    group = lambda g: g.reshape(B, Hk, G, N, D).sum(2)  # noqa: E731
    dk, dv, dk_err, dv_err = map(group, (dk, dv, dk_err, dv_err))
    for name, g, e in (("dq", dq, dq_err), ("dk", dk, dk_err), ("dv", dv, dv_err)):
        out[name] = g, (e + u * g.abs()) * (1 + u) + 4 * tiny
    return out


def check(got, want, what):
    value, bound = want
    assert got.isfinite().all(), what
    off = (got.double() - value).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1, f"{what}: {worst:.2f} times its bound, at most {off.max().item():.3g} off"


def paged_keep(length, n, window=None, sinks=0, parents=None, prefix=0, device="cuda"):
    """[n, length]: which places of a sequence's cache each of its last n tokens sees; `parents` of drafted ones, a list."""
    base = length - n
    keep = torch.zeros(n, length, dtype=torch.bool)
    j = torch.arange(length)
    for t in range(n):
        if base + t < 0:
            continue
        if parents is None:
            row = (j <= base + t) & ((base + t - j < window) | (j < sinks)) if window else j <= base + t
            keep[t] = row | (j < prefix)
            continue
        branch = [t]
        while parents[branch[-1]] >= 0:
            branch.append(parents[branch[-1]])
        depth = len(branch) - 1
        keep[t] = (j < base) & ((base + depth - j < window) | (j < sinks)) if window else j < base
        for up, a in enumerate(branch):
            if base + a >= 0 and (not window or up < window or base + depth - up < sinks):
                keep[t, base + a] = True
    return keep.to(device)
