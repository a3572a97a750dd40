"""64-bit oracle of the 8-bit cache and of norm + rotation, and what a kernel
may be off by."""

import torch

BLOCK = 32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def held(x, fmt):
    """What one sequence's [S, H, hd] raw values stand for once stored:
    complete blocks coded, the rest as it is; fp64."""
    x = x.double().cpu()
    S = x.shape[0] // BLOCK * BLOCK
    out = x.clone()
    for lo in range(0, S, BLOCK):
        b = x[lo:lo + BLOCK]
        mag = torch.where(torch.isfinite(b), b.abs(), torch.zeros(()).double())
        a = mag.amax((0, 2), keepdim=True)
        b = torch.nan_to_num(b, nan=0.0, posinf=3e300, neginf=-3e300)
        b = torch.minimum(torch.maximum(b, -a), a)
        a = a.clamp(min=2.0 ** -100)
        if fmt == "int8":
            # the definition's two fp32 roundings
            mul, scale = (127 / a).float(), (a / 127).float()
            code = torch.round((b.float() * mul).double()).clamp(-127, 127)
            out[lo:lo + BLOCK] = code * scale.double()
        else:
            e = torch.ceil(torch.log2(a / 448))
            e = torch.where(a <= 448 * torch.exp2(e - 1), e - 1, e)
            e = torch.where(a > 448 * torch.exp2(e), e + 1, e)
            y = b * torch.exp2(-e)
            lead = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
            step = torch.exp2(lead - 3)
            out[lo:lo + BLOCK] = torch.round(y / step) * step * torch.exp2(e)
    return out


def attention(q, k, v, start, scale):
    """q [T, qH, hd] at positions start.. over what k, v [n, kvH, hd] hold ->
    (out [T, qH, hd], bound on a kernel's error before its last rounding)."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    T, n = q.shape[0], k.shape[0]
    group = q.shape[1] // k.shape[1]
    v = torch.nan_to_num(v)
    k = k.repeat_interleave(group, 1).permute(1, 2, 0)
    v = v.repeat_interleave(group, 1).transpose(0, 1)
    qt = q.transpose(0, 1)
    s = qt @ k * scale
    late = torch.arange(n) > start + torch.arange(T)[:, None]
    s = s.masked_fill(late, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    out = p @ v / total
    # Scores are sums of hd exact products in fp32: off by at most
    # hd * 2^-24 * sum |q k| scale, the scaling and exp2 add 2^-20; a weight
    # then by twice that (its own and the row's largest), and by 2^-11 from
    # its rounding to fp16 (the incomplete block's are finer). Weights under
    # 2^-14 are off by 2^-25 each instead, against a sum of 1 at least.
    ds = 2.0 ** -24 * q.shape[2] * (qt.abs() @ k.abs()).amax(-1, keepdim=True) \
        * abs(scale) + 2.0 ** -20
    # a sum over all weights carries the weights' relative error as well
    size = p @ v.abs() / total
    bound = size * (2.0 ** -11 + 4 * ds) + n * 2.0 ** -25 * v.abs().amax()
    return out.transpose(0, 1), bound.transpose(0, 1)


def attention_tight(q, k, v, start, scale, step, weight=2.0 ** -11):
    """As :func:`attention`, with a bound that knows that a weight under
    2^-20 of the row's largest is off by at most `step` of it: for each token
    that the row sees, times that token's own largest value (the cache's
    kernel for that: 2^-32 fp8, 2^-31 int8; a V scale may lie 2 under the
    reference of the others, so int8 tests give 2^-30)."""
    out, _ = attention(q, k, v, start, scale)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    T, n = q.shape[0], k.shape[0]
    group = q.shape[1] // k.shape[1]
    k = k.repeat_interleave(group, 1).permute(1, 2, 0)
    v = v.repeat_interleave(group, 1).transpose(0, 1).abs()
    qt = q.transpose(0, 1)
    late = torch.arange(n) > start + torch.arange(T)[:, None]
    s = (qt @ k * scale).masked_fill(late, float("-inf"))
    p = torch.softmax(s, -1)
    size = p @ v
    ds = 2.0 ** -24 * q.shape[2] * (qt.abs() @ k.abs()).masked_fill(late, 0) \
        .amax(-1, keepdim=True) * abs(scale) + 2.0 ** -20
    # numerator and denominator each carry a weight's own error and
    # twice the error of two scores; the row's largest weight over the sum is
    # the largest of p. Tokens whose weight fp32 cannot hold add nothing.
    held = (p > 2.0 ** -140).double()
    floor = step * p.amax(-1, keepdim=True) * (held @ v.amax(-1, keepdim=True))
    bound = (size + out.abs().transpose(0, 1)) * (weight + 4 * ds) + floor
    return out, bound.transpose(0, 1)


def norm_rope(x, w, cos, sin, pos, eps, interleaved):
    """x [B, T, H, hd], pos [B, T] -> (fp64 result, error bound before the
    last rounding)."""
    x, cos, sin = x.double().cpu(), cos.double().cpu(), sin.double().cpu()
    y = x
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) \
            * w.double().cpu()
    n = cos.shape[1]
    c, s = cos[pos.cpu()].unsqueeze(2), sin[pos.cpu()].unsqueeze(2)
    out = y.clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved \
        else (slice(0, n), slice(n, 2 * n))
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., a] * s + y[..., b] * c
    # fp32 inside: the sum of squares, its root and two products are off by
    # at most 24 * 2^-24 of a value; a turn adds three roundings of the two
    # products' sizes. Tables may carry a factor.
    f = float(max(cos.abs().max(), sin.abs().max(), 1.0))
    bound = 2.0 ** -24 * 30 * 2 * f * y.abs().amax(-1, keepdim=True)
    return out, bound.expand_as(out)


def check(got, want, bound, dtype):
    got = got.double().cpu()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    room = bound + half_step(dtype) * (want.abs() + bound) + tiny
    off = (got - want).abs()
    assert torch.isfinite(got).all()
    worst = (off / room).max() if off.numel() else 0.0
    assert (off <= room).all(), f"{float(worst):.3g} times the bound"


def tables(S, rot, device="cpu", factor=1.0, base=10000.0):
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = torch.arange(S, dtype=torch.float64)[:, None] * inv
    return ((ang.cos() * factor).float().to(device),
            (ang.sin() * factor).float().to(device))
