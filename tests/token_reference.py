"""Plain 64-bit forms of the linears on int8 tokens and of the layers of experts, with bounds of what the kernels may be off by.

Every bound is a sum of the roundings that the operators name: half a step of a type is eps / 2 relative (float16 2^-11, bfloat16 2^-8, float32 2^-24), and
half its smallest subnormal number absolutely."""
import torch

F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least_half(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def silu_mul(g, u, dg, du):
    """silu(g) * u of exact g and u with bounds dg, du of their errors, and the result's bound.  The exponential is off by 2 + 1.16 |g| units of 2^-23 (CUDA's bound of
    __expf), the quotient by two; silu's slope is at most 1.1."""
    s = g * torch.sigmoid(g)
    ds = s.abs() * (6 + 1.2 * g.abs().clamp(max=100)) * 2 * F32 + 1.1 * dg
    z = s * u
    return z, (ds * u.abs() + s.abs() * du + ds * du + z.abs() * 2 * F32)


def quantized(x, norm, eps):
    """(codes before rounding, scales) of tokens, in 64 bits."""
    y = x.double()
    amax = (y * norm.double() if norm is not None else y).abs().amax(-1)
    if norm is not None:
        y = y * norm.double()
    codes = torch.where(amax[..., None] > 0, y * (127 / amax.clamp(min=1e-300))[..., None], 0.0)
    scales = amax / 127
    if norm is not None:
        scales = scales / torch.sqrt(x.double().square().mean(-1) + eps)
    return codes, scales


def product(a, a_scale, weight, scale, layout, bias, residual, pairs, dtype):
    """(result, bound) of the int8 product on its own inputs: the sum is exact, its conversion and two factors are a rounding each, bias and residual one."""
    w = weight.double() if layout == 'KN' else weight.double().t()
    y = (a.double() @ w) * scale.double() * a_scale.double()[..., None]
    d = y.abs() * 4 * F32
    if bias is not None:
        y = y + bias.double()
        d = d + (y.abs() + d) * F32
    if pairs:
        y, d = silu_mul(y[..., 0::2], y[..., 1::2], d[..., 0::2], d[..., 1::2])
    if residual is not None:
        y = y + residual.double()
        d = d + (y.abs() + d) * F32
    return y, d + (y.abs() + d) * half_step(dtype) + least_half(dtype)


def experts(x, chosen, weights, gate_up, s1, down, s2, residual):
    """(result, bound) of a layer of experts.  x and h are at most 2^-22 of their row's largest element off (whole numbers of up to 2^22, at least 2^21 for the largest, rounded); what stands for the sum of
    n products in float is off by no more than (n / 8 + 32) roundings of 2^-23 of their magnitudes (float sums run eight or more products at a time; whole ones are exact).
    A row of x or h whose largest element is below 2^-98 may be zeros, as the layer's documentation says: an element is then off by itself, by the largest at most."""
    rows, hidden = x.shape
    inner = down.shape[2]
    xd = x.double()
    out, bound = torch.zeros_like(xd), torch.zeros_like(xd)

    def held(least, most):  # how far elements of a row are held, whose largest lies between these
        return torch.where(least < 2.0 ** -98, most, most * 2.0 ** -22)

    largest = xd.abs().amax(-1, keepdim=True)
    dx = held(largest, largest)
    for e in range(down.shape[0]):
        share = torch.where(chosen == e, weights.double(), 0.0)
        token = (chosen == e).any(-1).nonzero()[:, 0]
        if len(token) == 0:
            continue
        share, size = share[token].sum(-1, keepdim=True), share[token].abs().sum(-1, keepdim=True)
        w1, w2 = gate_up[e].double() * s1[e].double()[:, None], down[e].double() * s2[e].double()[:, None]
        y = xd[token] @ w1.t()
        dy = xd[token].abs() @ w1.abs().t() * ((hidden / 8 + 32) * 2 * F32) + dx[token] * w1.abs().sum(1)
        h, dh = silu_mul(y[:, 0::2], y[:, 1::2], dy[:, 0::2], dy[:, 1::2])
        dh = dh + held((h.abs() - dh).amax(-1, keepdim=True), (h.abs() + dh).amax(-1, keepdim=True))
        o = h @ w2.t()
        do = dh @ w2.abs().t() + (h.abs() + dh) @ w2.abs().t() * ((inner / 8 + 32) * 2 * F32)
        out[token] += share * o
        bound[token] += size * (do + o.abs() * 4 * F32)
    bound = bound + out.abs() * 8 * F32
    if residual is not None:
        out = out + residual.double()
        bound = bound + out.abs() * F32
    return out, bound + (out.abs() + bound) * half_step(x.dtype) + least_half(x.dtype)


def check(got, want, bound):
    """All elements within their bounds; where it should be NaN, NaN."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), 'NaN in other places: {} for {}'.format(int(got.isnan().sum()), int(want.isnan().sum()))
    over = ((got - want).abs() > bound) & ~want.isnan()
    assert not over.any(), '{} of {} elements off by up to {:.3g} times their bound, first at {}'.format(
        int(over.sum()), over.numel(), ((got - want).abs() / bound)[over].max().item(), over.nonzero()[0].tolist())
