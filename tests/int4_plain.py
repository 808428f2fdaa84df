"""The 4-bit page format and the operators on it in plain torch, for the tests: the
format's formula in fp32 step by step (codes are whole numbers: they have to be the
same), attention in 64 bits."""
import math

import torch

BF = torch.bfloat16


def quantise(x, group):
    """fp32 rows [..., dim] -> codes uint8 [..., dim / 2], params bf16 [..., 2, dim / group]."""
    y = x.float().unflatten(-1, (-1, group))
    odd = ~torch.isfinite(y).all(-1)
    low, high = y.amin(-1), y.amax(-1)
    odd |= ~torch.isfinite(high - low)
    s = ((high - low) / torch.full_like(low, 15.0)).to(BF).float()
    c = (low + 8.0 * s).to(BF).float()
    flat = s < 2.0 ** -126
    s, c = s.masked_fill(flat, 0.0), torch.where(flat, low.to(BF).float(), c)
    s, c = s.masked_fill(odd, 0.0), c.masked_fill(odd, math.nan)
    u = torch.round((y - c.unsqueeze(-1)) / s.unsqueeze(-1)).clamp(-8, 7)
    u = torch.where((s == 0).unsqueeze(-1), torch.zeros_like(u), u).to(torch.int32).add(8).flatten(-2)
    codes = (u[..., 0::2] | u[..., 1::2] << 4).to(torch.uint8)
    return codes, torch.stack([s, c], -2).to(BF)


def values(codes, params):
    """What codes and params stand for, in 64 bits (exact but for sums of far exponents)."""
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double() - 8
    s, c = params.double().unbind(-2)
    return (c.unsqueeze(-1) + s.unsqueeze(-1) * u.unflatten(-1, (s.shape[-1], -1))).flatten(-2)


def turn(x, cos, sin, interleaved):
    """Rotary positions in fp32, each product rounded; cos and sin [N, 1, rot / 2]."""
    x, rot = x.float(), cos.shape[-1] * 2
    y = x.clone()
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * cos - b * sin, b * cos + a * sin
    return y


def attend(q, k, v, scale):
    """q [Hq, D], k and v [T, Hkv, D] in 64 bits -> [Hq, D] and the log-sum-exp [Hq]."""
    hq, d = q.shape
    t, hkv, _ = k.shape
    if t == 0:
        return torch.zeros(hq, d, dtype=torch.float64, device=q.device), \
            torch.full((hq,), -math.inf, dtype=torch.float64, device=q.device)
    s = torch.einsum("hgd,thd->hgt", q.double().view(hkv, hq // hkv, d), k) * scale
    return torch.einsum("hgt,thd->hgd", s.softmax(-1), v).reshape(hq, d), s.logsumexp(-1).reshape(hq)


def attention_error(q, k, v, kparams, scale, longest):
    """A bound on what attention in fp32 over 4-bit pages is off before the output is rounded,
    relative to max |v|. Scores in base 2: sums of dim + 8 terms, none of which, nor a partial
    sum, passes (15 s + |c|) sum |q|, each addition losing 2^-23 (tensor cores cut). Both sums of
    the softmax get it. Weights: in two bf16 parts (2^-16) and the exponential (2^-22) for the
    centres; times the scale, in fp16 for the codes, half a step or 2^-11 for bf16 queries (and
    its remainder, then 2^-22, for fp16 ones), of s |u - 8| = |v - c|, at most 2 max |v|; sums
    over the tokens in steps of 8 or more, of terms up to 3 max |v| (|c| + 8 s)."""
    if k.numel() == 0:
        return 0.0
    s, c = kparams.double().unbind(-2)
    most = float((15 * s + c.abs()).nan_to_num(0.0).max()) * float(q.double().abs().sum(-1).max())
    d = q.shape[-1]
    part = 2.0 ** -10 if q.dtype == BF else 0.0
    return 2 * (d + 8) * 2.0 ** -23 * most * abs(scale) + 3 * 2.0 ** -16 + part + (longest / 8 + 16) * 3 * 2.0 ** -23
