"""The decoding operators in 64 bits, from their definitions, for the tests; and how far from these a result may be.

Every bound is the sum of the roundings that the operator's documentation admits; `U` is the relative error of one rounding to a type."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half the smallest subnormal number


def rotary(x, positions, table, layout):
    """x [tokens, heads, dim] -> (result, its bound) in float64."""
    half = table.shape[1] // 2
    inside = (positions >= 0) & (positions < table.shape[0])
    t = table.double()[positions.long().clamp(0, max(0, table.shape[0] - 1))]
    cos, sin = t[:, None, :half], t[:, None, half:]
    y = x.double().clone()
    at_a = slice(0, half) if layout == 'half' else slice(0, 2 * half, 2)
    at_b = slice(half, 2 * half) if layout == 'half' else slice(1, 2 * half, 2)
    a, b = y[..., at_a].clone(), y[..., at_b].clone()
    y[..., at_a], y[..., at_b] = a * cos - b * sin, b * cos + a * sin
    y[..., :2 * half] = torch.where(inside[:, None, None], y[..., :2 * half], 0.0)
    # two products and a sum, each off by 2^-24 of its size
    bound = torch.zeros_like(y)
    bound[..., at_a] = 2.0 ** -23 * ((a * cos).abs() + (b * sin).abs())
    bound[..., at_b] = 2.0 ** -23 * ((b * cos).abs() + (a * sin).abs())
    return y, bound + U[x.dtype] * y.abs() + TINY[x.dtype]


def cached(x):
    """Rows as the cache keeps them, computed as documented in float32: (codes, scales)."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    zero = ~(amax >= 2.0 ** -100)
    limit = torch.full_like(amax, 127.0)
    codes = torch.where(bad | zero, torch.zeros_like(x), torch.round(x * (limit / amax)))
    scales = torch.where(bad, torch.full_like(amax, math.nan), torch.where(zero, torch.zeros_like(amax), amax / limit))
    return codes, scales[..., 0]


def attention(q, k, v, fresh, mask, scale):
    """One sequence: q [t, heads, dim], k and v [n, kv_heads, dim] (restored rows, float64).  (out, lse, bound of out, bound of lse)."""
    t, heads, dim = q.shape
    n, kv_heads = k.shape[:2]
    qd = q.double().unflatten(1, (kv_heads, heads // kv_heads))
    s = torch.einsum('thgd,nhd->hgtn', qd, k) * scale
    size = torch.einsum('thgd,nhd->hgtn', qd.abs(), k.abs()) * scale
    at = torch.arange(n, device=q.device)
    old = n - fresh
    seen = (at <= old + torch.arange(t, device=q.device)[:, None]) if mask is None else torch.cat(
        [torch.ones((t, max(old, 0)), dtype=torch.bool, device=q.device), mask[:, max(0, -old):fresh].bool()], -1)
    s = torch.where(seen, s, -math.inf)
    vd = torch.where(seen[None, None, :, :, None].any(2).any(1).any(0)[..., 0][:, None, None], v, 0.0) if n else v  # what nobody sees
    top = s.amax(-1, keepdim=True) if n else torch.full(s.shape[:-1] + (1,), -math.inf, device=q.device, dtype=torch.float64)
    p = torch.where(seen, (s - torch.where(top.isinf() & (top < 0), 0.0, top)).exp(), 0.0)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, p)
    out = torch.einsum('hgtn,nhd->thgd', p, vd).flatten(1, 2)
    lse = (top + total.log())[..., 0].permute(2, 0, 1).flatten(1)
    # scores: float sums of exact products, 2^-20 of the sum of magnitudes; exponentials: 2^-22, and 2^-23 of their argument
    ds = torch.where(seen, 2.0 ** -20 * size + 2.0 ** -22 + 2.0 ** -23 * s.abs(), 0.0).amax(-1) if n else torch.zeros(s.shape[:-1], device=q.device, dtype=torch.float64)
    ds = ds.permute(2, 0, 1)                                                               # [t, kv_heads, group]
    spread = torch.einsum('hgtn,nhd->thgd', p, vd.abs())
    # probabilities rounded to f16: 2^-11 of each, and 2^-32 of the largest value where they are small; sums in float
    few = n * 2.0 ** -32 * (vd.abs().amax() if n else 0.0)
    bound = ((2 * ds[..., None] + 2.0 ** -11 + n * 2.0 ** -26 + 2.0 ** -20) * spread + few).flatten(1, 2)
    return out, lse, bound + U[q.dtype] * out.abs() + TINY[q.dtype], (ds + 2.0 ** -21 + n * 2.0 ** -26).flatten(1) + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)


def log_probs(logits, tokens, top):
    """(log_probs, entropy, top values, indices) in float64, and the bounds of the first two."""
    x = logits.double()
    lse = torch.logsumexp(x, -1, keepdim=True)
    logp = x - lse
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][..., :top]
    largest = x.masked_fill(x.isinf(), 0.0).abs().amax(-1, keepdim=True)
    span = torch.where(p > 1e-30, (x - x.amax(-1, keepdim=True)).abs(), 0.0).amax(-1)
    # a thread's float sum of vocab / 512 terms, then 2^-23 of the size of the numbers that are subtracted
    d = 2.0 ** -24 * (x.shape[-1] / 512 + 64) + 2.0 ** -22 * largest + 2.0 ** -23 * lse.abs()
    return (logp.gather(-1, tokens.long()), entropy, logp.gather(-1, order), order), (d, (d[..., 0] * 2 + 2.0 ** -20) * (2 + span))
