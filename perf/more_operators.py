"""Cases and plain forms of the decoder block's operators around its token mixer.

Three operators run a decoder block's work beside attention: the norms after
one branch and before the next, fused with the branch's gate and the residual
scale (``residual_norm``), the gated product of the feed-forward layer, which
keeps its inputs for the backward in 8 bits (``swiglu``), and the projections
in 8-bit integers with a scale for each token and output channel
(``int8_linear``).

A case is a dict of plain values.  ``run`` computes it with elementary torch
operations in 32 bits (integer sums in 64), or, with ``own`` set, through the
package's entry points; ``exact`` computes the same outputs in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
GROUP = 128             # elements that share a scale of a kept activation
TINY = 2.0 ** -100      # smallest magnitude that a scale follows
MEMORY_BYTES, LINEAR_FLOPS = 2.2e9, 1.6e12


def norm_case(name, batch, tokens, width, gate, dtype, post=True, train=False, scales="1,1"):
    """``gate``: none, width (one for the layer), sequence (one per sequence) or token (a tensor like x);
    ``scales``: of the residual and of the branch."""
    return {"name": name, "op": "norm", "batch": batch, "tokens": tokens, "width": width, "gate": gate, "dtype": dtype,
            "post": post, "train": train, "scales": scales}


def swiglu_case(name, tokens, width, dtype):
    """Forward and backward, the inputs kept in 8 bits between them."""
    return {"name": name, "op": "swiglu", "tokens": tokens, "width": width, "dtype": dtype}


def linear_case(name, tokens, inner, outer, dtype, bias=False, given="float", out=None):
    """``given``: what the tokens arrive as, float (rounded to 8 bits in the call), int8, or norm (a
    residual norm before the product gives them in 8 bits)."""
    return {"name": name, "op": "linear", "tokens": tokens, "inner": inner, "outer": outer, "dtype": dtype, "bias": bias,
            "given": given, "out": out or dtype}


def listed():
    return [
        # one step of 64 users between two blocks: the latency of a call
        norm_case("norm_step", 64, 1, 4096, "width", "bf16"),
        # a 32K prompt between two blocks, norms on both sides
        norm_case("norm_prompt", 1, 32768, 4096, "width", "bf16"),
        # the training block of four sequences, forward and backward
        norm_case("norm_train", 4, 4096, 1024, "width", "bf16", train=True),
        # training with a gate computed from the tokens, an odd width, scaled residuals
        norm_case("norm_gated", 3, 2731, 1001, "token", "f16", post=False, train=True, scales="0.7,1.4"),
        # the training block's feed-forward layer
        swiglu_case("swiglu_train", 16384, 2816, "bf16"),
        # a wide layer over packed documents whose tokens fill no tile
        swiglu_case("swiglu_wide", 8191, 11264, "f16"),
        # the smallest training step, as checks of a model run it: latency
        swiglu_case("swiglu_short", 37, 1001, "f32"),
        # one user's next token through the feed-forward layer's first product: the latency of a call
        linear_case("linear_token", 1, 1024, 5632, "bf16"),
        # a step of 64 users
        linear_case("linear_step", 64, 4096, 16384, "bf16", given="int8"),
        # logits over the vocabulary for 37 sequences
        linear_case("linear_vocab", 37, 1024, 50257, "bf16", given="int8", out="f32"),
        # a step of 200 users: norm between two blocks, then the query, key and value heads' product
        linear_case("norm_linear", 200, 4096, 6144, "bf16", given="norm"),
        # prompts through a feed-forward product
        linear_case("linear_prompt", 16384, 4096, 11264, "bf16", bias=True),
    ]


def spread(rng, low, high):
    """A whole number, even over the logarithm of the range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def width_of(rng, low, high):
    """Widths of layers: most of them whole tiles, some odd."""
    n = spread(rng, low, high)
    step = rng.choice([1, 2, 8, 16, 64, 64, 128, 128])
    return min(high, max(low, n // step * step))


def draw(rng):
    op = rng.choice(["norm", "norm_train", "swiglu", "linear", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        if op in ("norm", "norm_train"):
            case = norm_case("", spread(rng, 1, 64), spread(rng, 1, 32768), width_of(rng, 64, 16384),
                             rng.choice(["none", "width", "sequence", "token"]), dtype, rng.random() < 0.6,
                             op == "norm_train", rng.choice(["1,1", "1,1", "0.5,1", "1.5,0.25"]))
        elif op == "swiglu":
            case = swiglu_case("", spread(rng, 1, 32768), width_of(rng, 64, 16384), dtype)
        else:
            given, out = rng.choice(["float", "int8", "int8", "norm"]), rng.choice([None, None, "f32"])
            # next to the border of an 8-bit step a computed norm falls to either side with its last bit: an answer in
            # 16 bits holds that
            dtype, out = (("f16" if dtype == "f16" else "bf16"), None) if given == "norm" else (dtype, out)
            case = linear_case("", spread(rng, 1, 32768), width_of(rng, 64, 16384), width_of(rng, 64, 60000), dtype,
                               rng.random() < 0.4, given, out)
        del case["name"]
        cost = work(case)
        if cost["bytes"] <= MEMORY_BYTES and (op != "linear" or cost["flops"] <= LINEAR_FLOPS):
            return case


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        values = case["batch"] * case["tokens"] * case["width"]
        wide = 1 if case["gate"] == "token" else 0
        # x, branch and a whole gate in, h and n out; with gradients dh, dn in, dx, dbranch and a whole gate's out too
        return {"bytes": size * values * (4 + wide + (4 + wide if case["train"] else 0)),
                "flops": values * (35 if case["train"] else 12)}
    if case["op"] == "swiglu":
        values = case["tokens"] * case["width"]
        # gate, up in, product out, 8-bit copies out; then these and dproduct in, dgate and dup out
        return {"bytes": values * (6 * size + 4), "flops": values * 40}
    tokens, inner, outer = case["tokens"], case["inner"], case["outer"]
    given = {"int8": 1, "float": size, "norm": 3 * size}[case["given"]]   # norm: x, branch in, h out
    return {"bytes": tokens * inner * given + inner * outer + tokens * outer * (4 if case["out"] == "f32" else 2),
            "flops": 2 * tokens * inner * outer}


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, to=None):
        return torch.randn(shape, generator=gen, device=device).mul_(scale).add_(mean).to(to or dtype)

    state = {"case": case}
    if case["op"] == "norm":
        batch, tokens, width = case["batch"], case["tokens"], case["width"]
        # the residual stream outgrows its branches; a norm's weights lie around 1
        state["x"], state["branch"] = normal(batch, tokens, width, scale=3.0), normal(batch, tokens, width, scale=0.5)
        state["weight"] = normal(width, scale=0.1, mean=1.0, to=torch.float32)
        state["post_weight"] = normal(width, scale=0.1, mean=1.0, to=torch.float32) if case["post"] else None
        shape = {"none": None, "width": (width,), "sequence": (batch, 1, width), "token": (batch, tokens, width)}[case["gate"]]
        state["gate"] = None if shape is None else normal(*shape)
        if case["train"]:
            state["dh"], state["dn"] = normal(batch, tokens, width), normal(batch, tokens, width)
            for name in ("x", "branch", "weight", "post_weight", "gate"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
    elif case["op"] == "swiglu":
        for name in ("gate", "up"):
            state[name] = normal(case["tokens"], case["width"], scale=1.5).requires_grad_(True)
        state["dout"] = normal(case["tokens"], case["width"])
    else:
        tokens, inner, outer = case["tokens"], case["inner"], case["outer"]
        # weights rounded once, in rows that start on 16 bytes, as a program keeps them
        weight = normal(outer, inner, scale=inner ** -0.5, to=torch.float32)
        kept = torch.zeros(outer, -(-inner // 16) * 16, dtype=torch.int8, device=device)
        values, state["weight_scale"] = rounded(weight)
        kept[:, :inner] = values
        state["weight_q"] = kept[:, :inner]
        state["bias"] = normal(outer, scale=0.1, to=torch.float32) if case["bias"] else None
        x = normal(tokens, inner)
        if case["given"] == "int8":
            kept = torch.zeros(tokens, -(-inner // 16) * 16, dtype=torch.int8, device=device)
            values, state["x_scale"] = rounded(x.float())
            kept[:, :inner] = values
            state["x"] = kept[:, :inner]
        else:
            state["x"] = x
        if case["given"] == "norm":
            state["branch"] = normal(tokens, inner, scale=0.5)
            state["weight"] = normal(inner, scale=0.1, mean=1.0, to=torch.float32)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def rounded(x):
    """fp32 rows as 8-bit integers and the scale of each row, every step in 32 bits by definition."""
    top = x.abs().amax(-1, keepdim=True).clamp(min=TINY)
    most = torch.full_like(top, 127.0)   # a tensor: by a number, torch multiplies with its reciprocal
    return (x * (most / top)).round().to(torch.int8), (top / most)[..., 0]


def in_groups(x):
    """The values that rows kept in 8 bits, in groups of GROUP elements, stand for."""
    width = x.shape[-1]
    padded = torch.nn.functional.pad(x.float(), (0, -width % GROUP)).unflatten(-1, (-1, GROUP))
    values, scale = rounded(padded)
    return (values.float() * scale[..., None]).flatten(-2)[..., :width]


def gate_like(case, gate):
    return gate if gate is None or case["gate"] != "width" else gate[None, None]


def plain_norm(state):
    case = state["case"]
    a, b = (float(s) for s in case["scales"].split(","))
    x, y = state["x"].detach(), state["branch"].detach().float()
    dtype = x.dtype
    weight, post, gate = (None if state[n] is None else state[n].detach().float() for n in ("weight", "post_weight", "gate"))
    gate = gate_like(case, gate)
    if post is not None:
        inner_y = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
        unit_y = y * inner_y
        y = unit_y * post
    h = a * x.float() + b * (y if gate is None else gate * y)
    inner = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    unit = h * inner
    result = {"h": h.to(dtype), "n": (unit * weight).to(dtype)}
    if not case["train"]:
        return result
    dn = state["dn"].float()
    result["dweight"] = (dn * unit).sum((0, 1))
    dn = dn * weight
    dh = state["dh"].float() + (dn - unit * (dn * unit).mean(-1, keepdim=True)) * inner
    result["dx"] = (a * dh).to(dtype)
    dh = b * dh
    if gate is not None:
        dgate = dh * y
        axes = {"width": (0, 1), "sequence": (1,), "token": ()}[case["gate"]]
        if axes:
            dgate = dgate.sum(axes)
        result["dgate"] = dgate.reshape(state["gate"].shape).to(dtype)
        dh = dh * gate
    if post is not None:
        result["dpost_weight"] = (dh * unit_y).sum((0, 1))
        dh = dh * post
        dh = (dh - unit_y * (dh * unit_y).mean(-1, keepdim=True)) * inner_y
    result["dbranch"] = dh.to(dtype)
    return result


def plain_swiglu(state):
    gate, up, dout = state["gate"].detach(), state["up"].detach(), state["dout"].float()
    dtype = gate.dtype
    x = gate.float()
    out = (x / (1 + (-x).exp()) * up.float()).to(dtype)
    x, y = in_groups(gate), in_groups(up)
    s = 1 / (1 + (-x).exp())
    return {"out": out, "dgate": (dout * y * s * (1 + x * (1 - s))).to(dtype), "dup": (dout * x * s).to(dtype)}


def plain_linear(state):
    case = state["case"]
    result, x = {}, state["x"]
    if case["given"] == "norm":
        # in 64 bits up to the 8-bit steps: next to a border the last bit decides
        h = x.double() + state["branch"].double()
        result["h"] = h.to(x.dtype)
        x = h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * state["weight"].double()
    if case["given"] == "int8":
        scale = state["x_scale"]
    else:
        x, scale = rounded(x.float())
    # sums of 8-bit products pass 24 bits
    sums = x.double() @ state["weight_q"].double().T
    out = sums.float() * state["weight_scale"] * scale[:, None]
    if state["bias"] is not None:
        out = out + state["bias"]
    result["out"] = out.to(DTYPES[case["out"]])
    return result


# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return {"norm": plain_norm, "swiglu": plain_swiglu, "linear": plain_linear}[case["op"]](state)
    import nlogn_pisa_b200 as pisa

    if case["op"] == "norm":
        a, b = (float(s) for s in case["scales"].split(","))
        names = [n for n in ("x", "branch", "weight", "post_weight", "gate") if state[n] is not None]
        h, n = pisa.residual_norm(state["x"], state["branch"], state["weight"], post_weight=state["post_weight"],
                                  gate=state["gate"], residual_scale=a, branch_scale=b, eps=EPS)
        result = {"h": h, "n": n}
        if case["train"]:
            grads = torch.autograd.grad((h, n), [state[n] for n in names], (state["dh"], state["dn"]))
            grads = dict(zip(names, grads))
            order = ("weight", "x", "gate", "post_weight", "branch")
            result.update({"d" + name: grads[name] for name in order if name in grads})
        return result
    if case["op"] == "swiglu":
        out = pisa.swiglu(state["gate"], state["up"], checkpoint_bits=8)
        dgate, dup = torch.autograd.grad(out, (state["gate"], state["up"]), state["dout"])
        return {"out": out, "dgate": dgate, "dup": dup}
    result, x, scale = {}, state["x"], state.get("x_scale")
    if case["given"] == "norm":
        result["h"], x, scale = pisa.residual_norm(x, state["branch"], state["weight"], eps=EPS, quantize=True)
    result["out"] = pisa.int8_linear(x, state["weight_q"], state["weight_scale"], bias=state["bias"], x_scale=scale,
                                     out_dtype=DTYPES[case["out"]])
    return result


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def rms_unit(v):
    return v / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + EPS)


def exact_norm(state):
    """Through autograd on the definition in 64 bits."""
    case = state["case"]
    a, b = (float(s) for s in case["scales"].split(","))
    leaves = {n: state[n].detach().double().requires_grad_(case["train"])
              for n in ("x", "branch", "weight", "post_weight", "gate") if state[n] is not None}
    value = leaves["branch"]
    if "post_weight" in leaves:
        value = rms_unit(value) * leaves["post_weight"]
    if "gate" in leaves:
        value = value * leaves["gate"]
    h = leaves["x"] * a + value * b
    n = rms_unit(h) * leaves["weight"]
    result = {"h": h.detach(), "n": n.detach()}
    if case["train"]:
        (h * state["dh"].double() + n * state["dn"].double()).sum().backward()
        for name in ("weight", "x", "gate", "post_weight", "branch"):
            if name in leaves:
                result["d" + name] = leaves[name].grad
    return result


def stands_for(x, group):
    """What 8 bits hold of fp32 rows: a group's values are whole multiples of its scale.  The scale, its
    inverse and their product with a value are 32-bit results by definition."""
    pieces = []
    for part in x.split(group, -1):
        top = part.abs().max(-1, keepdim=True).values
        top = torch.where(top < TINY, torch.full_like(top, TINY), top)
        most = torch.full_like(top, 127.0)
        steps = torch.round(part * torch.div(most, top))
        pieces.append(steps.double() * torch.div(top, most).double())
    return torch.cat(pieces, -1)


def exact_swiglu(state):
    gate, up, dout = (state[n].detach() for n in ("gate", "up", "dout"))
    out = torch.sigmoid(gate.double()) * gate.double() * up.double()
    x, y = (stands_for(t.float(), GROUP).requires_grad_(True) for t in (gate, up))
    (torch.sigmoid(x) * x * y * dout.double()).sum().backward()
    return {"out": out, "dgate": x.grad, "dup": y.grad}


def exact_linear(state):
    case = state["case"]
    result, x = {}, state["x"]
    if case["given"] == "norm":
        h = x.double() + state["branch"].double()
        result["h"] = h
        x = (rms_unit(h) * state["weight"].double()).float()
    if case["given"] == "int8":
        x = x.double() * state["x_scale"].double()[:, None]
    else:
        x = stands_for(x.float(), x.shape[-1])
    out = x @ (state["weight_q"].double() * state["weight_scale"].double()[:, None]).T
    result["out"] = out if state["bias"] is None else out + state["bias"].double()
    return result


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": exact_norm, "swiglu": exact_swiglu, "linear": exact_linear}[case["op"]](state)
