"""64-bit forms of the dense-attention operators and bounds on their rounding.

Every function returns (value, bound) pairs: the value in float64 and how far a
result may be from it, element by element, when products and sums are held in
fp32 and rounded to the tensors' type where the operators say so.
"""

import math

import torch

# unit roundoff of each type; fp32 sums of n terms are off by at most n EPS times the sum of magnitudes
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
EPS = 2.0 ** -24
# smallest normal of fp16: below it rounding is absolute
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}


def one_head(q, k, v, hidden, scale, dtype, dout=None):
    """q [n, D], k [m, D], v [m, Dv], hidden [n, m] of one sequence and head (float64)."""
    u, dim = UNIT[dtype], q.shape[1]
    weight = 0.0 if dtype == torch.float32 else u   # P and dS are rounded to 16-bit operands
    s = (scale * (q @ k.T)).masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[1] else s.new_full((s.shape[0], 1), -math.inf)
    e = (s - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = e.sum(-1, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    lse = torch.where(total > 0, top + total.log(), torch.full_like(total, -math.inf))[:, 0]
    reach = scale * (q.abs() @ k.abs().T).masked_fill(hidden, 0.0)
    reach = reach.amax(-1, keepdim=True) if reach.shape[1] else torch.zeros_like(total)
    # error of a weight relative to itself: its logit's, the row maximum's, the
    # exponential's (a few units) and the sum's
    rel = EPS * (2 * (dim + 8) * reach + 16 + s.shape[1])
    mass = p @ v.abs()
    out = p @ v
    tiny = TINY[dtype]
    out_bound = u * out.abs() + (weight + 2 * rel) * mass * 1.05 + 4 * tiny * (1 + v.abs().sum(0, keepdim=True))
    lse_bound = 2 * rel[:, 0] + EPS * 4 * lse.abs().masked_fill(lse == -math.inf, 0.0)
    found = {"out": (out, out_bound), "lse": (lse, lse_bound)}
    if dout is None:
        return found
    dp = dout @ v.T
    delta = (dout * out).sum(-1, keepdim=True)
    ds = scale * p * (dp - delta)
    delta_err = (dout.abs() * out_bound).sum(-1, keepdim=True) + EPS * (v.shape[1] + 4) * (dout * out).abs().sum(-1, keepdim=True)
    dp_err = EPS * (v.shape[1] + 4) * (dout.abs() @ v.abs().T)
    rel = rel + EPS * 4 * (lse[:, None].abs().masked_fill(lse[:, None] == -math.inf, 0.0))
    ds_err = scale * p * (2 * rel * (dp - delta).abs() + dp_err + delta_err) + (weight + 4 * EPS) * ds.abs()
    ds_err = (ds_err + 2 * tiny).masked_fill(hidden, 0.0)
    p_err = ((weight + 2 * rel) * p + 2 * tiny).masked_fill(hidden, 0.0)
    found["dq"] = (ds @ k, ds_err @ k.abs() + EPS * (k.shape[0] + 4) * (ds.abs() @ k.abs()))
    found["dk"] = (ds.T @ q, ds_err.T @ q.abs() + EPS * (q.shape[0] + 4) * (ds.abs().T @ q.abs()))
    found["dv"] = (p.T @ dout, p_err.T @ dout.abs() + EPS * (q.shape[0] + 4) * (p.T @ dout.abs()))
    return found


def attention(q, k, v, scale=None, causal=True, queries=None, keys=None, offset=None, dout=None):
    """q [B,T,Hq,D], k, v [B,N,H,.]; ``queries`` / ``keys``: lengths of packed sequences (batch 1)."""
    dtype, scale = q.dtype, k.shape[-1] ** -0.5 if scale is None else scale
    q, k, v = (x.detach().double() for x in (q, k, v))
    dout = None if dout is None else dout.double()
    group = q.shape[2] // k.shape[2]
    out = q.new_zeros(*q.shape[:3], v.shape[-1])
    lse = q.new_full(q.shape[:3], -math.inf)
    names = {"out": out, "lse": lse}
    if dout is not None:
        names |= {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    value = names
    bound = {n: torch.zeros_like(x) for n, x in names.items()}
    spans = []
    if queries is None:
        shift = k.shape[1] - q.shape[1] if offset is None else offset
        spans = [(b, 0, q.shape[1], 0, k.shape[1], shift) for b in range(q.shape[0])]
    else:
        bq = bk = 0
        for n, m in zip(queries, keys if keys is not None else queries):
            spans.append((0, bq, bq + n, bk, bk + m, m - n))
            bq, bk = bq + n, bk + m
    for b, q0, q1, k0, k1, shift in spans:
        rows = torch.arange(q1 - q0, device=q.device)[:, None] + shift
        cols = torch.arange(k1 - k0, device=q.device)[None]
        hidden = (cols > rows) if causal else torch.zeros(q1 - q0, k1 - k0, dtype=torch.bool, device=q.device)
        if q1 == q0:
            continue
        for h in range(q.shape[2]):
            g = h // group
            found = one_head(q[b, q0:q1, h], k[b, k0:k1, g], v[b, k0:k1, g], hidden, scale, dtype,
                             None if dout is None else dout[b, q0:q1, h])
            for n, (x, e) in found.items():
                at = (b, slice(k0, k1), g) if n in ("dk", "dv") else (b, slice(q0, q1), h)
                if n in ("dk", "dv"):
                    value[n][at] += x
                    bound[n][at] += e
                else:
                    value[n][at] = x
                    bound[n][at] = e
    for n in ("dq", "dk", "dv"):
        if n in value:   # the final rounding
            bound[n] = bound[n] + UNIT[dtype] * value[n].abs() + TINY[dtype]
    return value, bound


def check(name, got, value, bound):
    """Finite parts within the bound (and never further than it by NaN), infinities equal."""
    got = got.detach().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    wild = ~torch.isfinite(value)
    assert torch.equal(got[wild], value[wild]), f"{name}: infinite entries differ"
    off = (got - value).abs()[~wild]
    most = bound[~wild] + 1e-30
    bad = ~(off <= most)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} entries out of bound, worst {float((off / most).max()):.3g} times it, "
        f"largest difference {float(off.max()):.3g}")


def norm_rotary(x, weight, angle, eps, dout=None):
    """x [B,T,H,D], angle [B|1,T,D/2] fp32 -> y, and with dout (y, dx, dw), as (value, bound)."""
    dtype, u, dim = x.dtype, UNIT[x.dtype], x.shape[-1]
    wu = UNIT[weight.dtype]
    x, w = x.detach().double(), weight.detach().double()
    cos, sin = angle.double()[:, :, None].cos(), angle.double()[:, :, None].sin()

    def turn(z, sign):
        a, b = z.chunk(2, -1)
        return torch.cat((a * cos - sign * b * sin, sign * a * sin + b * cos), -1)

    def turn_abs(z):
        a, b = z.abs().chunk(2, -1)
        return torch.cat((a * cos.abs() + b * sin.abs(), a * sin.abs() + b * cos.abs()), -1)

    inv = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit = x * inv
    rel = EPS * (dim + 16)     # the sum of squares, rsqrt, sine and cosine, a few products
    y = turn(unit * w, 1)
    tiny = TINY[dtype]
    found = {"y": (y, u * y.abs() + rel * turn_abs(unit * w) + tiny)}
    if dout is None:
        return found
    g = dout.double()
    back = turn(g, -1)
    back_abs = turn_abs(g)
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    dw = (back * unit).sum((0, 1, 2))
    found["dw"] = (dw, wu * dw.abs() + EPS * (rows + dim + 24) * (back_abs * unit.abs()).sum((0, 1, 2))
                   + TINY[weight.dtype])
    h = back * w
    mean = (h * unit).mean(-1, keepdim=True)
    dx = (h - unit * mean) * inv
    size = (back_abs * w.abs() + unit.abs() * (back_abs * w.abs() * unit.abs()).mean(-1, keepdim=True)) * inv
    found["dx"] = (dx, u * dx.abs() + 3 * EPS * (dim + 24) * size + tiny)
    return found
