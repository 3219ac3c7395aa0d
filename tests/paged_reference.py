"""Plain 64-bit forms of the paged-cache operators and of packed attention, for the tests: loops over sequences and heads."""
import math

import torch


def rope(x, pos, d, adjacent, theta):
    """x [tokens][heads][d] rotated as a whole, in 64 bits."""
    freq = theta ** -(torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    angle = (pos.double().view(-1, 1) * freq).view(-1, 1, d // 2)
    c, s, z, out = angle.cos(), angle.sin(), x.double(), torch.empty_like(x, dtype=torch.float64)
    if adjacent:
        a, b = z[..., 0::2], z[..., 1::2]
        out[..., 0::2], out[..., 1::2] = a * c - b * s, a * s + b * c
    else:
        a, b = z[..., :d // 2], z[..., d // 2:]
        out[..., :d // 2], out[..., d // 2:] = a * c - b * s, a * s + b * c
    return out


def quantise(x):
    """Codes and scales of x [..., d] by the rule of the 8-bit pages, every step in 32 bits, halves away from zero."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    top = torch.where(top < 1e-36, torch.zeros_like(top), top)
    n = torch.full_like(top, 127.0)
    y = x * torch.where(top > 0, n / top, torch.zeros_like(top))
    code = torch.sign(y) * torch.floor(y.double().abs() + 0.5).float().clamp(max=127)
    return code.to(torch.int8), torch.where(top > 0, top / n, torch.ones_like(top)).squeeze(-1)


def attention(q, k, v, first, window, scale):
    """Rows q [tokens][Hq][d] at positions first ... against k, v [keys][Hkv][d], in 64 bits. Returns the result and, for error
    bounds, the softmax-weighted mean of |v| and the largest scaled sum of |q_i k_i| of a row."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    pos = torch.arange(first, first + n, device=q.device).view(-1, 1)
    key = torch.arange(k.shape[0], device=q.device).view(1, -1)
    seen = key <= pos
    if window:
        seen &= key > pos - window
    out, size, reach = (torch.zeros(n, hq, d, dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(hq):
        kk, vv = k[:, h // group].double(), v[:, h // group].double()
        s = (q[:, h].double() @ kk.T) * scale
        p = torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), -1)
        p = torch.where(seen, p, torch.zeros_like(p))
        for t in range(0, n):  # only what a token sees takes part: hidden values may be anything
            sel = seen[t]
            out[t, h] = p[t, sel] @ vv[sel]
            size[t, h] = p[t, sel] @ vv[sel].abs()
            reach[t, h] = (q[t, h].double().abs() @ kk[sel].abs().T).max() * scale if bool(sel.any()) else 0.0
    return out, size, reach


def bound(dtype, out, size, reach):
    """How far a result may be from the 64-bit one, element by element.

    bf16: the result and each softmax weight are rounded once, by at most 2^-8 of their value.
    f32: q (and packed k, v) and the weights are taken in three bf16 parts, which leave out at most 2^-24 of a value; of the nine
    products of two such values the three smallest are dropped, at most 2 * 2^-24 + 2^-32 of the whole: a score is off by less
    than 5 * 2^-24 * reach, a weight by twice that share (its own and the sum's) and 2^-24, a value by 3 * 2^-24.
    Over 8-bit pages: two f16 parts (of values brought next to 1), which leave out at most 2^-22: a score is off by 2^-22 * reach,
    a weight by twice that share and 2^-22; codes are exact.
    All: 2^-20 for exponentials, sums and the order they are taken in.
    """
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * (out.abs() + size) * 1.01 + 2.0 ** -20 * (1 + reach) * size
    return (10 * reach + 4) * 2.0 ** -24 * size + (2 * reach + 1) * 2.0 ** -22 * size + 2.0 ** -20 * (1 + reach) * size
