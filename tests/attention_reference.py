"""Document attention and its gradients in 64 bits, with elementwise error bounds for results computed from 16- or
32-bit operands. Test infrastructure.

Bounds, for a type with rounding error u (half a step, torch.finfo(t).eps / 2) and e = 2^-24:
  scores        |ds| <= (head_dim + 4) e scale |q|.|k|, and the exponential and the log-sum add 2^-20 relative:
                a probability is off by r = 2 max|ds| + keys e + 2^-20 relative
  output        dy_bound = (w + r) P|v| + u (|y| + (w + r) P|v|), w = u where P is rounded to the operands' type before
                the product with v, 0 where it stays in 32 bits
  delta         sum |dy| (dy_bound + head_dim e |y|)          (it is formed from the rounded y)
  dS            (w + r)|dS| + P (head_dim e |dy|.|v| + delta's bound)
                in fp16 values below 2^-14 have an absolute step: 2^-25 for dS, 2^-35 and 2^-32 for the probabilities of dv
                and of the output, which are kept 2^10 and 2^7 above their size
                the 16-bit path's exponentials flush results below 2^-126 to zero, or (those on the FMA units) hold them at
                2^-125: an absolute step of 2^-125 per probability, times what it multiplies
                for dS that is the computed dP - delta: with d' = d + x, |P'd' - Pd| <= |P' - P| |d| + P'|x|, and
                P' <= (1 + w + r) P + 2^-125, so the error x of the difference counts with P + 2^-125, not with P alone
                (seen where a key's probabilities all vanish and d is smaller than x)
  dv, dq, dk    the same sums over absolute values, times 1 + (terms) e, plus u of the result
"""

import torch


def reference(q, k, v, spans, scale, dy=None, rounded=True):
    """(values, bounds): dicts of y and, with dy, dq, dk, dv. Tokens of no document: zero, and a bound of zero."""
    u = torch.finfo(q.dtype).eps / 2
    w = u if rounded else 0.0
    t = 2.0 ** -25 if rounded and q.dtype == torch.float16 else 0.0
    e, f = 2.0 ** -24, 2.0 ** -125
    dim, group = q.shape[-1], q.shape[2] // k.shape[2]
    names = ("y",) if dy is None else ("y", "dq", "dk", "dv")
    like = {"y": q, "dq": q, "dk": k, "dv": v}
    values = {n: torch.zeros(like[n].shape, device=q.device, dtype=torch.float64) for n in names}
    errors = {n: torch.zeros_like(values[n]) for n in names}
    for row, start, end in spans:
        n = end - start
        if n == 0:
            continue
        allowed = torch.ones(n, n, device=q.device, dtype=torch.bool).tril()
        for h in range(q.shape[2]):
            s = h // group
            qd, kd, vd = q[row, start:end, h].double(), k[row, start:end, s].double(), v[row, start:end, s].double()
            raw = qd @ kd.T * scale
            p = torch.softmax(raw.masked_fill(~allowed, float("-inf")), -1)
            ds = (dim + 4) * e * abs(scale) * (qd.abs() @ kd.abs().T)
            r = 2 * float(ds.max()) + n * e + 2.0 ** -20
            y = p @ vd
            spread = (w + r) * (p @ vd.abs()) + (t * 2 ** -7 + f) * (allowed.double() @ vd.abs())
            y_error = spread + u * (y.abs() + spread)
            values["y"][row, start:end, h], errors["y"][row, start:end, h] = y, y_error
            if dy is None:
                continue
            g = dy[row, start:end, h].double()
            terms = 1 + (n * group + dim) * e
            dp, delta = g @ vd.T, (g * y).sum(-1, keepdim=True)
            delta_error = (g.abs() * (y_error + dim * e * y.abs())).sum(-1, keepdim=True)
            slope = p * (dp - delta)
            seen = allowed.double()
            slope_error = (w + r) * slope.abs() + (t + f * (dp - delta).abs()) * seen + (p + f * seen) * (dim * e * (g.abs() @ vd.abs().T) + delta_error)
            values["dv"][row, start:end, s] += p.T @ g
            errors["dv"][row, start:end, s] += (((w + r) * p + (t * 2 ** -10 + f) * seen).T @ g.abs()) * terms + (n * group) * e * (p.T @ g.abs())
            values["dq"][row, start:end, h] = slope @ kd * scale
            errors["dq"][row, start:end, h] = abs(scale) * ((slope_error * terms + n * e * slope.abs()) @ kd.abs())
            values["dk"][row, start:end, s] += slope.T @ qd * scale
            errors["dk"][row, start:end, s] += abs(scale) * ((slope_error * terms + n * group * e * slope.abs()).T @ qd.abs())
    for n in names:
        if n != "y":
            errors[n] = errors[n] + u * (values[n].abs() + errors[n])
    return values, errors


def compare(actual, values, errors):
    for name, value in values.items():
        got = actual[name].double()
        assert torch.isfinite(got).all(), f"{name} is not finite"
        excess = (got - value).abs() - errors[name]
        # a subnormal result of a 16-bit type has an absolute step instead of a relative one
        assert float(excess.max()) <= torch.finfo(actual[name].dtype).smallest_normal, (
            f"{name}: {float(excess.max()):.3e} above its bound, largest error {float((got - value).abs().max()):.3e}")
