"""Plain 64-bit restatements of the temporal operators, with bounds on what 32-bit arithmetic may be off by.

Each returns (results, bounds): `bounds` is how far a result computed in fp32 from the same inputs may lie, from the number
and size of its roundings (U = 2^-24 is half a step of fp32), before it is rounded to the tensors' type.  `rounded` adds that
rounding.  Step by step and stream by stream; no relation to how the kernels split the work.
"""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(ref, bound, dtype):
    """Bound after one rounding to `dtype`: half a step of the value, or of the smallest normal number below it."""
    return bound + half_step(dtype) * ((ref.abs() + bound).clamp(min=torch.finfo(dtype).tiny))


def _d(t):
    return t.double() if t is not None else None


def causal_conv(x, weight, bias=None, state=None, silu=True):
    x, weight, bias, state = _d(x), _d(weight), _d(bias), _d(state)
    B, T, D = x.shape
    W = weight.shape[0]
    xx = torch.cat([state if state is not None else x.new_zeros(B, W - 1, D), x], 1)
    s, size = x.new_zeros(B, T, D), x.new_zeros(B, T, D)
    for w in range(W):
        s = s + weight[w] * xx[:, w:w + T]
        size = size + (weight[w] * xx[:, w:w + T]).abs()
    if bias is not None:
        s, size = s + bias, size + bias.abs()
    bound = (W + 1) * U * size                              # W fused steps, each rounding a partial sum of at most `size`
    y = s
    if silu:
        y = s * torch.sigmoid(s)
        # |silu'| < 1.1; exp of an argument off by |s| U (two roundings: the constant, the product), its own two units,
        # 1 + e, the reciprocal (two units) and the product
        bound = 1.1 * bound + y.abs() * U * (2 * s.abs() + 8)
    return (y, xx[:, T:]), bound


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, softplus=True):
    x, dt, A, B, C, D, z, dt_bias, state = (_d(t) for t in (x, dt, A, B, C, D, z, dt_bias, state))
    b, T, d = x.shape
    N = A.shape[0]
    raw = dt + dt_bias if dt_bias is not None else dt
    delta = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    # step size: the sum is off by U |raw|, which moves softplus by at most that much of itself (its slope is below its
    # value); max + log1p: about ten roundings, the log's argument amplified by at most one
    rel = U * ((raw.abs() + 16) if softplus else 1.0) * torch.ones_like(raw)
    h = state if state is not None else x.new_zeros(b, N, d)
    err = torch.zeros_like(h)
    ys, bounds = [], []
    for t in range(T):
        e = delta[:, t, None] * A
        a = e.exp()
        u = (delta[:, t] * x[:, t])[:, None] * B[:, t, :, None]
        # exponent: rel of delta, the constant log2 e, two products; the exponential itself two units; then one fused step.
        # doubled for a time axis in pieces, which multiplies two such factors where this multiplies one
        ea = 2 * (e.abs() * (rel[:, t, None] + 3 * U) + 4 * U)
        eu = rel[:, t, None] + 4 * U
        err = a * err * (1 + ea) + a * h.abs() * ea + u.abs() * eu
        h = a * h + u
        err = err + 2 * U * h.abs()
        c = C[:, t, :, None]
        y = (h * c).sum(1)
        size = (h * c).abs().sum(1)
        bound = (err * c.abs()).sum(1) + U * (N + 2) * size
        if D is not None:
            y = y + D * x[:, t]
            bound = bound + U * (N + 2) * (D * x[:, t]).abs()
        if z is not None:
            g = z[:, t] * torch.sigmoid(z[:, t])
            y = y * g
            bound = bound * g.abs() * 1.01 + y.abs() * U * (2 * z[:, t].abs() + 10)
        ys.append(y)
        bounds.append(bound)
    y = torch.stack(ys, 1) if T else x.new_zeros(b, 0, d)
    return (y, h), (torch.stack(bounds, 1) if T else y, err)


def rows_of(M, lengths, offsets):
    """(stream or None, position) of every row, from host lists."""
    out = [(None, -1)] * M
    if offsets is None:
        return [(m, lengths[m]) for m in range(M)]
    for s in range(len(lengths)):
        for i in range(max(0, offsets[s + 1] - offsets[s])):
            out[offsets[s] + i] = (s, lengths[s] + i)
    return out


def rotate(x, pos, freqs, interleaved=False):
    """x [H,D] at one position; angles in 64 bits."""
    x = x.double()
    n = freqs.numel()
    c, s = torch.cos(pos * freqs.double()), torch.sin(pos * freqs.double())
    r = x.clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[:, first], x[:, second]
    r[:, first], r[:, second] = a * c - b * s, a * s + b * c
    bound = torch.zeros_like(x)
    # sine and cosine to four units, of an angle reduced in 64 bits and rounded once (pi U of it); a product and a fused step
    bound[:, first] = bound[:, second] = U * 12 * (a.abs() + b.abs())
    return r, bound


def attend(q, kp, vp, table, lengths, offsets=None, scale=None, parts=1):
    """Row by row from host copies of table, lengths and offsets.  Bad pages give NaN.  `parts`: how many numbers of the
    tensors' type a weight is multiplied as, for the bound."""
    M, Hq, Dh = q.shape
    P, Hkv, page, _ = kp.shape
    scale = Dh ** -0.5 if scale is None else scale
    out = torch.zeros((M, Hq, Dh), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    half = half_step(q.dtype)
    for m, (s, pos) in enumerate(rows_of(M, lengths, offsets)):
        if s is None or pos < 0:
            continue
        pages = [table[s][c] if c < len(table[s]) else -1 for c in range(pos // page + 1)]
        if any(not 0 <= pg < P for pg in pages):
            out[m] = math.nan
            continue
        k = kp[pages].double().transpose(0, 1).reshape(Hkv, -1, Dh)[:, :pos + 1].repeat_interleave(Hq // Hkv, 0)
        v = vp[pages].double().transpose(0, 1).reshape(Hkv, -1, Dh)[:, :pos + 1].repeat_interleave(Hq // Hkv, 0)
        qq = q[m].double()[:, None]
        score = (qq * k).sum(-1) * scale
        size = (qq * k).abs().sum(-1) * scale
        top = score.amax(-1, keepdim=True)
        p = torch.exp(score - top)
        l = p.sum(-1, keepdim=True)
        p = p / l
        out[m] = (p[..., None] * v).sum(1)
        away = (p[..., None] * v.abs()).sum(1)
        # exponents: Dh fused steps of sums below `size`, and the products with the scale (size and top enter in base 2);
        # an exponent off by e moves its weight by e, and the sum of the weights moves by no more than the largest
        e = U * ((Dh + 6) * size.amax(-1, keepdim=True) + 6 * top.abs() + 8)
        n = pos + 1
        bound[m] = away * (2 * e + U * (2 * n + 16))
        if q.dtype != torch.float32:
            # weights are rounded to the tensors' type for the product with v, the largest of those seen so far being 1 or
            # more: half a step each, and below the smallest normal number half a step of that
            # (in two parts: half a step of what the first half step left out, at least 2^7 times as fine at the low end, and twice as many products)
            bound[m] += away * half ** parts + v.abs().sum(1) * torch.finfo(q.dtype).tiny * half / l / (1 if parts == 1 else 2 ** 7)
            bound[m] += away * U * n * (parts - 1)
    return out, bound
