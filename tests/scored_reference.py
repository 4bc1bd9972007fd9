"""Attention with capped, biased and prefix-masked scores, plainly and in 64 bits, with bounds for what the kernels' roundings may add.

Bounds. A rounding to the inputs' type is off by at most u = eps / 2, relative to the value; one to fp32 by 2^-24. The 16-bit kernels round P (and dS)
to the inputs' type before the second products and every result once; sums, scores, statistics are fp32. With n terms a fp32 sum (in any
order, also cut off instead of rounded) is off by at most n 2^-23 of the sum of its terms' sizes. `rel` is a bound for the relative error of an entry of
P that comes from its score: twice (numerator and sum) the absolute error of the exponent.
Below the type's least normal number a rounding is off by up to half the step there, `sub` (fp16: 2^-25 for all below 2^-14), whatever the
value: each entry of P or dS may add that much, in the forward over a sum of the row that is at least 1."""
import math

import torch


def attention_64(q, k, v, do, causal, sm_scale, eq, ek, cap, slopes, prefix):
    """{"o", "dq", "dk", "dv"}: (value, bound) of each, and "keep"."""
    B, H, M, D = q.shape
    Hk, N = k.shape[1:3]
    G, gap, dev, dtype = H // Hk, max(0, N - M), q.device, q.dtype
    u = torch.finfo(dtype).eps / 2
    half = dtype != torch.float32
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    Q, K, V, DO = (x.detach().double() for x in (q, k, v, do))
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    s = Q @ K.mT * scale
    err = (D + 2) * 2.0 ** -23 * scale * (Q.abs() @ K.abs().mT)  # absolute error of a score
    far = torch.arange(M, device=dev)[:, None] + gap - torch.arange(N, device=dev)
    x, f = s, torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        x, f = cap * t, 1 - t * t
        # the polynomial 3.0e-6 of the value, the other form a few 2^-23 of the cap where tanh > 0.71; arithmetic a few 2^-24 more
        err = err * f + 4e-6 * x.abs()
    if slopes is not None:
        bias = slopes.double()[:, None, None] * far.abs()
        x, err = x - bias, err + 4 * 2.0 ** -24 * (x.abs() + bias.abs())
    keep = torch.ones(B, 1, M, N, dtype=torch.bool, device=dev)
    if causal:
        keep = keep & (far >= 0)
        if prefix is not None:
            keep = keep | (torch.arange(N, device=dev) < prefix.long()[:, None, None, None])
    if eq is not None:
        keep = keep & ((eq[..., None] >= 0) | (eq[..., None] == ek[:, :, None, :]))
    x = x.masked_fill(~keep, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e300)
    p = (x - top).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    # 2^-22 for exp2 (relative), 2^-24 of the exponent for its argument's rounding; exponents far below the maximum carry no weight
    err = torch.where(p > 1e-30, err + 2.0 ** -23 * (x.abs() + top.abs()), 0.0)
    rel = 2 * err.amax((-2, -1), keepdim=True) + 2.0 ** -20
    acc = N * 2.0 ** -23
    up = u if half else 0.0  # the rounding of P and dS
    sub = torch.finfo(dtype).smallest_normal * u if half else 0.0
    seen = keep.double()
    o = p @ V
    o_err = (up + rel + acc) * (p @ V.abs()) + sub * (seen @ V.abs()) + u * o.abs()
    dv = p.mT @ DO
    accm = G * M * 2.0 ** -23
    dv_err = (up + rel + accm) * (p.mT @ DO.abs()) + sub * (seen.mT @ DO.abs())
    dp, delta = DO @ V.mT, (DO * o).sum(-1, keepdim=True)
    dp_err = D * 2.0 ** -23 * (DO.abs() @ V.abs().mT)
    # (delta takes what the rounding of o leaves out, too)
    delta_err = (DO.abs() * (o_err + D * 2.0 ** -23 * o.abs())).sum(-1, keepdim=True)
    ds = p * (dp - delta) * f
    # f = 1 - tanh^2 is off by some 2^-22 in absolute terms and by the score's error. (f + e)(d + g) - f d = f g + e d + e g: the last term is all there
    # is where f is 0 (a score far beyond the cap) and so is d = dP - delta (a row of one key).
    f_err = (2.0 ** -21 + 2 * err / cap) if cap else 0.0
    ds_err = sub * seen + (up + rel) * ds.abs() + p * ((f + f_err) * (dp_err + delta_err) + f_err * (dp - delta).abs())
    dq, dk = ds @ K * scale, ds.mT @ Q * scale
    dq_err = scale * ((ds_err + acc * ds.abs()) @ K.abs())
    dk_err = scale * ((ds_err + accm * ds.abs()).mT @ Q.abs())
    group = lambda g: g.reshape(B, Hk, G, N, D).sum(2)  # noqa: E731
    dk, dv, dk_err, dv_err = map(group, (dk, dv, dk_err, dv_err))
    tiny = torch.finfo(dtype).tiny if dtype != torch.float16 else 2.0 ** -24
    out = {"keep": keep}
    for name, g, e in (("o", o, o_err), ("dq", dq, dq_err + u * dq.abs()), ("dk", dk, dk_err + u * dk.abs()), ("dv", dv, dv_err + u * dv.abs())):
        out[name] = g, e * (1 + u) + 4 * tiny
    return out
