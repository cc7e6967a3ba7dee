"""Plain 64-bit forms of the stream operators, with bounds of the fp32 error.

Each function returns values in float64 and a bound of what an fp32 evaluation
(any order of its sums) rounded once to the output's type may differ by. U is
one fp32 rounding, relative. The bounds count roundings: a sum of n terms in
any order errs by at most n U times the sum of magnitudes.
"""
import torch

U = 2.0 ** -24
WIDE = torch.float64


def half_step(y, dtype):
    """Half a step of ``dtype`` around y, and half its smallest subnormal."""
    return y.abs() * (torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -6) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


# silu(v) = v / (1 + e^-v). The hardware exponential errs by 2 + 1.173 |v| units
# in the last place (of 2 U), the division by two; |silu'| <= 1.1.
def silu(v, error):
    y = v * torch.sigmoid(v)
    return y, 1.1 * error + y.abs() * (2 * (2 + 1.173 * v.abs()) + 6) * U + 1e-35


def bounds_of(offsets, n, length):
    if offsets is None:
        return [(i * length, (i + 1) * length) for i in range(n)]
    return list(zip(offsets[:-1], offsets[1:]))


def states_before(pool, codes):
    """Per sequence the state its code names, in float64 (zeros of a fresh one)."""
    pool = pool.to(WIDE)
    return [torch.zeros_like(pool[0, 0]) if c & 2 else pool[c >> 2, c & 1] for c in codes]


def causal_conv(x, weight, bias, act, spans, old):
    """Rows of ``spans`` (others NaN), their bounds, and the new histories."""
    dtype, taps = x.dtype, weight.shape[1]
    x, w = x.to(WIDE), weight.to(WIDE)
    b = torch.zeros(x.shape[1], dtype=WIDE) if bias is None else bias.to(WIDE)
    y, tol = torch.full_like(x, float("nan")), torch.zeros_like(x)
    new = []
    for (begin, end), h in zip(spans, old):
        line = torch.cat([h, x[begin:end]])
        parts = [w[:, j] * line[j:j + end - begin] for j in range(taps)]
        v = b + sum(parts)
        error = (taps + 1) * U * (b.abs() + sum(p.abs() for p in parts))
        if act == "silu":
            v, error = silu(v, error)
        y[begin:end], tol[begin:end] = v, error + half_step(v, dtype)
        new.append(line[end - begin:])
    return y, tol, new


def selective_scan(x, dt, a, b, c, d, z, dt_bias, softplus, spans, old):
    """Rows of ``spans`` (others NaN), their bounds, the new states and their bounds.

    The state's error E follows E' = decay E + what the row adds: the decay errs
    relatively by 4 U of the hardware's 2^x, one rounding, and the exponent's
    error (three roundings of delta * a * log2 e and delta's own); the row's
    input by delta's error and three roundings; the new state by two. Joining pieces of
    a sequence multiplies in further decays and a sum of deltas, each with the
    same relative errors; the factor 2 covers them.
    """
    dtype, channels = x.dtype, x.shape[1]
    x, dt, a, b, c = (t.to(WIDE) for t in (x, dt, a, b, c))
    per = channels // b.shape[1]
    v = dt if dt_bias is None else dt + dt_bias.to(WIDE)
    delta = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v
    # softplus'(v) |v| <= softplus(v) (|v| + 1); exp, log1p and the sum: 8 units.
    off = (v.abs() + 10) * U if softplus else U * torch.ones_like(v)
    y, tol = torch.full_like(x, float("nan")), torch.zeros_like(x)
    new, new_tol = [], []
    for (begin, end), h in zip(spans, old):
        h = h.clone()
        size, error = h.abs(), torch.zeros_like(h)
        for t in range(begin, end):
            bt = b[t].t().repeat_interleave(per, 1)
            ct = c[t].t().repeat_interleave(per, 1)
            power = delta[t] * a
            decay = torch.exp(power)
            add = delta[t] * x[t] * bt
            error = decay * error + 2 * (decay * size * (5 * U + power.abs() * (4 * U + off[t]))
                                         + add.abs() * (off[t] + 4 * U))
            h, size = decay * h + add, decay * size + add.abs()
            error = error + 4 * U * size
            out = (h * ct).sum(0)
            far = (ct.abs() * error).sum(0) + (a.shape[0] + 2) * U * (ct.abs() * size).sum(0)
            if d is not None:
                out = out + d.to(WIDE) * x[t]
                far = far + 2 * U * (out.abs() + (d.to(WIDE) * x[t]).abs())
            if z is not None:
                gate, gate_tol = silu(z[t].to(WIDE), torch.zeros_like(out))
                far = far * gate.abs() * (1 + 1e-5) + out.abs() * gate_tol + 2 * U * (out * gate).abs()
                out = out * gate
            y[t], tol[t] = out, far + half_step(out, dtype)
        new.append(h)
        new_tol.append(error + 1e-36)
    return y, tol, new, new_tol


def group_norm(x, groups, weight, bias, eps, act, alpha, reciprocal, spans):
    dtype, channels = x.dtype, x.shape[1]
    x = x.to(WIDE)
    one = torch.ones(channels, dtype=WIDE)
    w = one if weight is None else weight.to(WIDE)
    b = 0 * one if bias is None else bias.to(WIDE)
    y, tol = torch.full_like(x, float("nan")), torch.zeros_like(x)
    for begin, end in spans:
        if begin == end:
            continue
        part = x[begin:end].reshape(end - begin, groups, -1)
        count = part.shape[0] * part.shape[2]
        mean = part.mean((0, 2), keepdim=True)
        centred = part - mean
        spread = (centred ** 2).mean((0, 2), keepdim=True)
        # At least 32 threads share a sum of over 2048 terms, or a thread adds 64
        # at most; sums of squares count the squares' own roundings.
        chain = (max(count / 32, 64) + 24) * U
        mean_off = chain * (centred.abs().mean((0, 2), keepdim=True) + mean.abs())
        spread_off = 3 * chain * spread + 2 * mean_off ** 2 + 8 * U * mean_off * centred.abs().mean((0, 2), keepdim=True)
        rstd = 1 / torch.sqrt(spread + eps)
        norm = centred * rstd
        far = rstd * (mean_off + U * (part.abs() + mean.abs())) + norm.abs() * (spread_off * rstd ** 2 / 2 + 4 * U)
        norm, far = (t.expand_as(part).reshape(end - begin, channels) for t in (norm, far))
        v = norm * w + b
        far = far * w.abs() + 3 * U * ((norm * w).abs() + b.abs())
        if act == "silu":
            v, far = silu(v, far)
        elif act == "snake":
            al, re = alpha.to(WIDE), reciprocal.to(WIDE)
            wave = torch.sin(al * v)
            # |d/dv| <= 1 + |re al|; the product al v and the sine err by U |al v| + 4 U.
            far = far * (1 + (al * re).abs()) + re.abs() * (2 * U * (al * v).abs() + 8 * U) + 2 * U * v.abs()
            v = v + re * wave ** 2
        y[begin:end], tol[begin:end] = v, far + half_step(v, dtype)
    return y, tol


def int4_weights(weight, scales, group):
    """The float64 matrix that packed codes and scales stand for."""
    out, depth = weight.shape[0], 2 * weight.shape[1]
    q = torch.empty(out, depth, dtype=WIDE)
    q[:, 0::2], q[:, 1::2] = (weight % 16).to(WIDE) - 8, (weight // 16).to(WIDE) - 8
    return q * scales.to(WIDE).repeat_interleave(group, 1)[:, :depth]


def project_int4(x, weight, scales, bias, group):
    w, dtype = int4_weights(weight, scales, group), x.dtype
    x = x.to(WIDE)
    b = torch.zeros(w.shape[0], dtype=WIDE) if bias is None else bias.to(WIDE)
    y = x @ w.t() + b
    # Every term passes through at most depth / 32 + 64 sums; a tensor core's
    # sums may truncate (two U each).
    far = (x.shape[1] / 32 + 64) * 2 * U * (x.abs() @ w.abs().t() + b.abs())
    return y, far + half_step(y, dtype)
