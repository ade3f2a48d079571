"""Plain forms of the serving operators in 64 bits, and how far a kernel may be from them."""
import math

import torch


def turn(x, positions, inv_freq, interleaved, scale, inverse=False):
    """x [B, T*G, H, D] in 64 bits, row t*G + g at positions[b, t]."""
    B, T = positions.shape
    rot = 2 * inv_freq.numel()
    a = positions.double()[:, :, None] * inv_freq.double()                       # [B, T, pairs]
    a = a.repeat_interleave(x.shape[1] // T, 1)[:, :, None]
    c, s = a.cos() * scale, a.sin() * scale * (-1 if inverse else 1)
    y = x.clone()
    if interleaved:
        p, q = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = p * c - q * s, q * c + p * s
    else:
        p, q = x[..., : rot // 2], x[..., rot // 2 : rot]
        y[..., : rot // 2], y[..., rot // 2 : rot] = p * c - q * s, q * c + p * s
    return y


def turn_bound(x, y, rot, interleaved, scale, dtype):
    """Rounding of the result (half a step), and of the sums before it.  The angle is rounded to 2^-24 of at most half a
    turn (pi 2^-24 = 1.9e-7), cosine and sine to 2^-24 of at most 1 each and the products and the sum to 2^-24: less than 1e-6
    of |x1| + |x2| together, times the factor."""
    m = torch.zeros_like(x)
    if interleaved:
        both = x[..., 0:rot:2].abs() + x[..., 1:rot:2].abs()
        m[..., 0:rot:2] = m[..., 1:rot:2] = both
    else:
        both = x[..., : rot // 2].abs() + x[..., rot // 2 : rot].abs()
        m[..., : rot // 2] = m[..., rot // 2 : rot] = both
    before = 1e-6 * scale * m
    return torch.finfo(dtype).eps / 2 * (y.abs() + before) + before + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rows_of(cache, table, n):
    """The first n rows of a sequence: [n, H, D]."""
    j = torch.arange(n, device=cache.device)
    return cache[table[j // cache.shape[1]].long(), j % cache.shape[1]]


def attend(q, keys, values, scale):
    """q [G, H, D], keys and values [n, H, D], in 64 bits -> o, lse, what bounds the error: largest scale * sum |q k| of a row, sum p |v|."""
    if keys.shape[0] == 0:
        return torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=q.dtype, device=q.device), torch.zeros_like(q[..., 0]), torch.zeros_like(q)
    s = torch.einsum("ghd,nhd->ghn", q, keys) * scale
    p = torch.softmax(s, -1)
    size = torch.einsum("ghd,nhd->ghn", q.abs(), keys.abs()).amax(-1) * abs(scale)
    return (torch.einsum("ghn,nhd->ghd", p, values), torch.logsumexp(s, -1) / math.log(2), size, torch.einsum("ghn,nhd->ghd", p, values.abs()))


def attend_bounds(o, lse, size, mass, D, dtype, turned):
    """Of o and lse.  A score is a sum of D products in 32 bits, where each addition may drop 2^-23 of what the terms' sizes add up
    to; a turned query is held in two 16-bit halves (2^-16) and turned with 1e-6.  So a probability is off by a factor of up to
    e^d, and numerator and denominator both are; a probability is also held in two halves (2^-16; 2^-24 absolute in
    fp16), and exp2 and the factors of the joins are good to 2^-20.  The result is rounded by half a step."""
    d = size * ((D + 4) * 2.0 ** -23 + (2.0 ** -16 + 2e-6 if turned else 0.0))
    rel = 2 * torch.expm1(d) + 2.0 ** -15
    tol_o = rel[..., None] * mass
    tol_o = torch.finfo(dtype).eps / 2 * (o.abs() + tol_o) + tol_o + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    tol_lse = (d + 2.0 ** -19) / math.log(2) + torch.where(lse.isfinite(), lse.abs(), 0.0) * 2.0 ** -22
    return tol_o, tol_lse


def close(got, want, tol, what):
    got, want = got.double(), want.double()
    same = (got == want) | ((got - want).abs() <= tol) | (got.isnan() & want.isnan())
    assert same.all(), f"{what}: {(~same).sum().item()} of {same.numel()} off, worst {((got - want).abs() / tol.clamp_min(1e-30))[~same].max().item():.3g} of the bound"
