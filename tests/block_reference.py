"""64-bit forms of the decoder block's operators and bounds on their rounding.

As in dense_reference: functions return (value, bound) pairs, the bound counting
fp32 steps inside and one rounding to the tensors' type at the end.
"""

import torch

import dense_reference
from dense_reference import EPS, check  # noqa: F401

# float64 tensors are exact inputs
UNIT, TINY = ({**table, torch.float64: 0.0} for table in (dense_reference.UNIT, dense_reference.TINY))

# Row sums: a thread adds at most 32 terms, then five shuffles and at most 16
# warps follow; rsqrt is off by two units, a few products by one each.
ROW = EPS * (32 + 5 + 16 + 16)


def quantized(x, group=None):
    """(values int8, scale) of fp32 rows, or of groups of them, every step in 32 bits."""
    if group is None:
        top = x.abs().amax(-1, keepdim=True)
        fine = torch.isfinite(top)
        m = torch.where(top < 2.0 ** -100, torch.full_like(top, 2.0 ** -100), top)
        most = torch.full_like(m, 127.0)
        values = torch.where(fine, (x * torch.div(most, m)).round(), torch.zeros_like(x)).to(torch.int8)
        return values, torch.where(fine, torch.div(m, most), torch.full_like(m, float("nan")))[..., 0]
    parts = [quantized(p) for p in x.split(group, -1)]
    return torch.cat([p[0] for p in parts], -1), torch.stack([p[1] for p in parts], -1)


def restored(values, scale, group):
    wide = scale.double().repeat_interleave(group, -1)[..., :values.shape[-1]]
    return values.double() * wide


def residual_norm(x, branch, weight, post=None, gate=None, a=1.0, b=1.0, eps=1e-6, dh=None, dn=None):
    """x [B,T,D] -> h, n and, with dh and dn, the gradients, as (value, bound); gate broadcast against x."""
    dtype, u, tiny = x.dtype, UNIT[x.dtype], TINY[x.dtype]
    shapes = {"post": post, "gate": gate, "weight": weight}
    wu = {k: (0.0 if t is None else UNIT[t.dtype]) for k, t in shapes.items()}
    wt = {k: (0.0 if t is None else TINY[t.dtype]) for k, t in shapes.items()}
    gate_shape = None if gate is None else gate.shape
    x, branch, weight, post, gate = (None if t is None else t.detach().double() for t in (x, branch, weight, post, gate))
    if branch is None:
        h, eh = x, torch.zeros_like(x)
    else:
        inv_y = (branch.square().mean(-1, keepdim=True) + eps).rsqrt()
        z = branch * inv_y
        y = branch if post is None else z * post
        gy = y if gate is None else gate * y
        h = a * x + b * gy
        eh = 4 * EPS * ((a * x).abs() + (b * gy).abs()) + ROW * (b * gy).abs()
    square = h.square().mean(-1, keepdim=True) + eps
    inv = square.rsqrt()
    einv = (h.abs() * eh).mean(-1, keepdim=True) / square + ROW    # relative
    v = h * inv
    n = v * weight
    found = {"h": (h, u * h.abs() + eh + tiny),
             "n": (n, u * n.abs() + (inv * eh + v.abs() * einv) * weight.abs() * 1.01 + tiny)}
    if dn is None:
        return found
    dn = dn.double()
    dh = torch.zeros_like(x) if dh is None else dh.double()
    rows = x[..., 0].numel()
    lead = tuple(range(x.dim() - 1))
    ev = inv * eh + v.abs() * einv
    found["dweight"] = ((dn * v).sum(lead), ((dn.abs() * ev).sum(lead) + EPS * (rows + 64) * (dn * v).abs().sum(lead)) * 1.01)
    s = dn * weight
    m = (s * v).mean(-1, keepdim=True)
    em = (s.abs() * ev + (ROW + 4 * EPS) * (s * v).abs()).mean(-1, keepdim=True)
    first = m
    t = dh + (s - v * m) * inv
    et = inv * (ev * m.abs() + v.abs() * em + (einv + 8 * EPS) * (s.abs() + (v * m).abs())) + 2 * EPS * dh.abs()
    found["dx"] = (a * t, u * (a * t).abs() + abs(a) * et * 1.01 + EPS * (a * t).abs() + tiny)
    if branch is not None:
        s, es = b * t, abs(b) * et + EPS * (b * t).abs()
        if gate is not None:
            dg, eg = s * y, es * y.abs() + (ROW + 4 * EPS) * (s * y).abs()
            if gate.shape != x.shape:
                keep = gate.shape if gate.dim() == x.dim() else (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
                axes = [i for i in range(x.dim() - 1) if keep[i] == 1]
                eg = eg.sum(axes, keepdim=True) + EPS * (rows + 64) * dg.abs().sum(axes, keepdim=True)
                dg = dg.sum(axes, keepdim=True)
            dg, eg = dg.reshape(gate_shape), eg.reshape(gate_shape)
            found["dgate"] = (dg, wu["gate"] * dg.abs() + eg * 1.01 + wt["gate"])
            es, s = es * gate.abs() + EPS * (s * gate).abs(), s * gate
        if post is not None:
            found["dpost_weight"] = ((s * z).sum(lead), ((es * z.abs()).sum(lead)
                                                         + (EPS * (rows + 64) + ROW) * (s * z).abs().sum(lead)) * 1.01)
            es, s = es * post.abs() + EPS * (s * post).abs(), s * post
            m = (s * z).mean(-1, keepdim=True)
            # this row sum may be taken in the parts that make up s: their magnitudes, not the sum's, carry its rounding
            parts = (abs(b) * (post * z).abs() * (1.0 if gate is None else gate.abs())
                     * (dh.abs() + inv * ((dn * weight).abs() + (v * first).abs())))
            em = (es * z.abs() + 2 * ROW * (s * z).abs() + ROW * parts).mean(-1, keepdim=True)
            es = inv_y * (es + z.abs() * em + (2 * ROW + 8 * EPS) * (s.abs() + (z * m).abs()))
            s = (s - z * m) * inv_y
        found["dbranch"] = (s, u * s.abs() + es * 1.01 + tiny)
    for name, key in (("dweight", "weight"), ("dpost_weight", "post")):
        if name in found:
            value, bound = found[name]
            found[name] = (value, bound + wu[key] * value.abs() + wt[key])
    return found


def sigmoid_error(x):
    """Relative: an exponential off by 2 + 1.2 |x| units, a sum, a quotient off by two."""
    return EPS * (16 + 4 * x.abs())


def swiglu(gate, up, dout=None, kept=None):
    """out and, with dout, dgate and dup from ``kept`` (float64 pairs) or the inputs, as (value, bound)."""
    dtype = gate.dtype
    u, tiny = UNIT[dtype], TINY[dtype] + 2.0 ** -120
    g, y = gate.detach().double(), up.detach().double()
    out = g * torch.sigmoid(g) * y
    found = {"out": (out, (u + sigmoid_error(g)) * out.abs() + tiny * (1 + y.abs() * (1 + g.abs())))}
    if dout is None:
        return found
    d = dout.double()
    g, y = (g, y) if kept is None else kept
    s = torch.sigmoid(g)
    rel = sigmoid_error(g)
    small = tiny * (1 + d.abs() * (1 + y.abs()) * (1 + g.abs()))
    dup = d * g * s
    dgate = d * y * s * (1 + g * (1 - s))
    found["dup"] = (dup, (u + rel) * dup.abs() + small)
    found["dgate"] = (dgate, u * dgate.abs() + 2 * rel * (d * y * s).abs() * (1 + g.abs()) + small)
    return found


def int8_linear(x, x_scale, weight, weight_scale, bias, dtype):
    """Integer sums in float64 are exact."""
    sums = x.double() @ weight.double().T
    value = sums * weight_scale.double() * x_scale.double()[..., None]
    extra = torch.zeros_like(value) if bias is None else bias.double().expand_as(value)
    total = value + extra
    return total, UNIT[dtype] * total.abs() + 4 * EPS * (value.abs() + extra.abs()) + TINY[dtype]
