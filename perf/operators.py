"""Cases and plain forms of the dense-attention operators.

Three operators make a full-attention layer beside the sparse one: the norm of
each query and key head with its position rotation (``qk_norm_rotary``),
causal attention over whole prompts, packed or batched, with its gradient
(``full_attention``), and attention of the newest tokens over each sequence's
own cache together with a prefix that all sequences share
(``prefix_attention``).

A case is a dict of plain values.  ``run`` computes it with elementary torch
operations in 32 bits, or, with ``own`` set, through the package's entry
points; ``exact`` computes the same outputs in 64 bits.
"""

import itertools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
# score matrices of the plain form are held whole: bounds on their elements
FORWARD_ELEMENTS, TRAIN_ELEMENTS = 32 * 16384 ** 2, 5 * 32 * 4096 ** 2
ATTENTION_FLOPS, DECODE_BYTES = 2.1e12, 400e6


def numbers(text):
    return [int(x) for x in text.split(",")]


def attention_case(name, queries, keys, heads, kv_heads, dim, dtype, train=False, packed=True):
    """``queries`` / ``keys``: lengths of each sequence; a sequence's queries are its last positions."""
    return {"name": name, "op": "attention", "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "train": train, "packed": packed}


def decode_case(name, batch, new, prefix, low, high, heads, kv_heads, dim, dtype):
    """``batch`` sequences with own caches of ``low`` to ``high`` tokens, the last ``new`` of them this step's."""
    return {"name": name, "op": "decode", "batch": batch, "new": new, "prefix": prefix, "low": low, "high": high,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def norm_case(name, batch, tokens, offset, heads, kv_heads, dim, dtype, train=False):
    return {"name": name, "op": "norm_rotary", "batch": batch, "tokens": tokens, "offset": offset, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "train": train}


def listed():
    return [
        # one short chat prompt: the latency of a call
        attention_case("prompt_short", "37", "37", 32, 8, 128, "bf16"),
        # a serving step: packed prompts of very different lengths, among them a single
        # token and a chunk that continue earlier prompts
        attention_case("prompts_packed", "1,4099,517,2048,33,1290,700,2307", "4100,4099,517,2048,2081,1290,700,2307",
                       32, 8, 128, "bf16"),
        # one long prompt
        attention_case("prompt_long", "16384", "16384", 32, 8, 128, "bf16"),
        # the training block: four sequences, one head of 64 per KV head
        attention_case("train_block", "4096,4096,4096,4096", "4096,4096,4096,4096", 16, 16, 64, "bf16", True, False),
        # training on packed documents with grouped heads
        attention_case("train_packed", "2049,511,4096,1,1535", "2049,511,4096,1,1535", 32, 8, 128, "bf16", True),
        # training in 32 bits, as checks of a model run it
        attention_case("train_f32", "1500,2596", "1500,2596", 4, 4, 64, "f32", True),
        # one user's next token over a short cache: the latency of a call
        decode_case("decode_single", 1, 1, 0, 700, 700, 32, 8, 128, "bf16"),
        # 64 users of one system prompt, with conversations of their own
        decode_case("decode_shared", 64, 1, 8192, 1, 2048, 32, 8, 128, "bf16"),
        # 16 answers about one long document
        decode_case("decode_long", 16, 1, 65536, 5, 4096, 32, 8, 128, "f16"),
        # the step of 64 users: one token each
        norm_case("norm_step", 64, 1, 4321, 32, 8, 128, "f16"),
        # a 32K prompt
        norm_case("norm_prompt", 1, 32768, 0, 32, 8, 128, "bf16"),
        # the training block
        norm_case("norm_train", 4, 4096, 0, 16, 16, 64, "bf16", True),
    ]


def spread(rng, low, high):
    """A whole number, even over the logarithm of the range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


HEADS = [(32, 8, 128), (16, 16, 64), (32, 2, 64), (4, 4, 64), (8, 2, 128), (16, 4, 80), (12, 4, 96), (20, 4, 128)]


def draw(rng):
    op = rng.choice(["attention", "attention", "train", "train", "decode", "decode", "norm", "norm_train"])
    heads, kv_heads, dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("attention", "train"):
        train = op == "train"
        longest = (2048 if train else 4096) if dtype == "f32" else (4096 if train else 16384)
        while True:
            count = spread(rng, 1, 12)
            packed = rng.random() < 0.75
            if packed:
                queries = [spread(rng, 1, longest) for _ in range(count)]
                keys = [n if train or rng.random() < 0.6 else n + spread(rng, 1, longest) for n in queries]
            else:
                queries = [spread(rng, 1, longest)] * count
                past = 0 if train or rng.random() < 0.6 else spread(rng, 1, longest)
                keys = [n + past for n in queries]
            case = attention_case("", ",".join(map(str, queries)), ",".join(map(str, keys)), heads, kv_heads, dim,
                                  dtype, train, packed)
            del case["name"]
            elements = heads * count * max(queries) * max(keys)
            if (elements <= (TRAIN_ELEMENTS if train else FORWARD_ELEMENTS)
                    and work(case)["flops"] <= ATTENTION_FLOPS * (0.02 if dtype == "f32" else 1)):
                return case
    if op == "decode":
        while True:
            prefix = 0 if rng.random() < 0.25 else spread(rng, 1, 65536)
            high = spread(rng, 1, 8192)
            new = rng.choice([1, 1, 1, 2, 4, 5])
            case = decode_case("", spread(rng, 1, 128), new, prefix, max(new, high // 50), max(new, high), heads,
                               kv_heads, dim, dtype)
            del case["name"]
            if work(case)["bytes"] <= DECODE_BYTES:
                return case
    while True:
        case = norm_case("", spread(rng, 1, 64), spread(rng, 1, 32768), spread(rng, 1, 100000), heads, kv_heads, dim,
                         dtype, op == "norm_train")
        del case["name"]
        if work(case)["bytes"] <= 600e6:
            return case


def own_lengths(case):
    """Lengths of the sequences' own caches, scattered over the case's range."""
    low, high = case["low"], case["high"]
    return [low + (b * 7919 + 5 * b * b) % (high - low + 1) for b in range(case["batch"])]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attention":
        queries, keys = numbers(case["queries"]), numbers(case["keys"])
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(queries, keys))
        rows, cols = sum(queries) * heads * dim, sum(keys) * kv_heads * dim
        if case["train"]:
            # two products forward, five backward; reads q, k, v, dout and writes out and the three gradients
            return {"bytes": size * (4 * rows + 4 * cols), "flops": 14 * pairs * heads * dim}
        return {"bytes": size * (2 * rows + 2 * cols), "flops": 4 * pairs * heads * dim}
    if case["op"] == "decode":
        own_keys = sum(own_lengths(case))
        read = 2 * (case["prefix"] + own_keys) * kv_heads * dim
        rows = 2 * case["batch"] * case["new"] * heads * dim
        pairs = case["new"] * (case["batch"] * case["prefix"] + own_keys)
        return {"bytes": size * (read + rows), "flops": 4 * pairs * heads * dim}
    values = case["batch"] * case["tokens"] * (heads + kv_heads) * dim
    # forward: x in, y out; with gradients also dy in, dx out
    return {"bytes": size * values * (4 if case["train"] else 2), "flops": values * (25 if case["train"] else 10)}


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device).to(dtype)

    state = {"case": case}
    if case["op"] == "attention":
        queries, keys = numbers(case["queries"]), numbers(case["keys"])
        if case["packed"]:
            batch, rows, cols = 1, sum(queries), sum(keys)
            state["cu_queries"], state["cu_keys"] = (
                torch.tensor(list(itertools.accumulate(n, initial=0)), dtype=torch.int32, device=device)
                for n in (queries, keys))
        else:
            batch, rows, cols = len(queries), queries[0], keys[0]
        state["q"], state["k"], state["v"] = (normal(batch, rows, heads, dim), normal(batch, cols, kv_heads, dim),
                                              normal(batch, cols, kv_heads, dim))
        if case["train"]:
            state["dout"] = normal(batch, rows, heads, dim)
            for name in ("q", "k", "v"):
                state[name].requires_grad_(True)
    elif case["op"] == "decode":
        lengths = own_lengths(case)
        capacity = -(-case["high"] // 256) * 256
        state["q"] = normal(case["batch"], case["new"], heads, dim)
        state["k"], state["v"] = (normal(case["batch"], capacity, kv_heads, dim) for _ in range(2))
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
        state["prefix_k"] = state["prefix_v"] = None
        if case["prefix"]:
            state["prefix_k"], state["prefix_v"] = (normal(case["prefix"], kv_heads, dim) for _ in range(2))
    else:
        state["q"] = normal(case["batch"], case["tokens"], heads, dim)
        state["k"] = normal(case["batch"], case["tokens"], kv_heads, dim)
        state["q_weight"], state["k_weight"] = ((1 + 0.1 * torch.randn(dim, generator=gen, device=device)).to(dtype)
                                                for _ in range(2))
        pairs = torch.arange(dim // 2, dtype=torch.float64, device=device)
        state["frequency"] = (10000.0 ** (-2 * pairs / dim)).float()
        state["positions"] = torch.arange(case["tokens"], device=device)[None] + case["offset"]
        if case["train"]:
            state["dq"], state["dk"] = normal(*state["q"].shape), normal(*state["k"].shape)
            for name in ("q", "k", "q_weight", "k_weight"):
                state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def padded_rows(cu, length, total):
    """[sequences, length] row numbers of a packed tensor (clamped) and which of them are real."""
    at = cu[:-1, None].long() + torch.arange(length, device=cu.device)[None]
    return at.clamp(max=total - 1), at < cu[1:, None]


def plain_attention(state):
    case = state["case"]
    heads, kv_heads, dim, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    group, scale = heads // kv_heads, dim ** -0.5
    lq, lk = max(numbers(case["queries"])), max(numbers(case["keys"]))
    q, k, v, dout = (None if state.get(n) is None else state[n].detach().float() for n in ("q", "k", "v", "dout"))
    if case["packed"]:
        q_at, q_real = padded_rows(state["cu_queries"], lq, q.shape[1])
        k_at, k_real = padded_rows(state["cu_keys"], lk, k.shape[1])
        q, k, v = q[0][q_at], k[0][k_at], v[0][k_at]
        dout = None if dout is None else dout[0][q_at] * q_real[..., None, None]
        count_q, count_k = state["cu_queries"].diff(), state["cu_keys"].diff()
    else:
        count_q = torch.full((q.shape[0],), lq, device=q.device)
        count_k = torch.full((q.shape[0],), lk, device=q.device)
        q_real = (torch.arange(lq, device=q.device) < lq).expand(q.shape[0], lq)
    batch = q.shape[0]

    def by_kv_head(x):  # [B, L, heads, D] -> [B, kv_heads, group * L, D]
        return x.reshape(batch, lq, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * lq, dim)

    def by_token(x):
        return x.reshape(batch, kv_heads, group, lq, dim).permute(0, 3, 1, 2, 4).reshape(batch, lq, heads, dim)

    q, k, v = by_kv_head(q), k.transpose(1, 2), v.transpose(1, 2)
    last = (count_k - count_q)[:, None] + torch.arange(lq, device=q.device)[None]  # last visible key of each query
    hidden = torch.arange(lk, device=q.device)[None, None] > last[..., None]
    hidden = (hidden | ~q_real[..., None])[:, None, None]
    p = (q @ k.transpose(-1, -2)).mul_(scale).view(batch, kv_heads, group, lq, lk)
    p.masked_fill_(hidden, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill(top == float("-inf"), 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total.masked_fill(total == 0, 1.0))
    p = p.view(batch, kv_heads, group * lq, lk)
    out = p @ v

    def rows_of(x):
        x = by_token(x)
        return (x[q_real][None] if case["packed"] else x).to(dtype)

    def keys_of(x):
        x = x.transpose(1, 2)
        return (x[k_real][None] if case["packed"] else x).to(dtype)

    if dout is None:
        return rows_of(out)
    dout = by_kv_head(dout)
    dv = p.transpose(-1, -2) @ dout
    ds = (dout @ v.transpose(-1, -2)).sub_((dout * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return {"out": rows_of(out), "dq": rows_of(ds @ k), "dk": keys_of(ds.transpose(-1, -2) @ q), "dv": keys_of(dv)}


def plain_decode(state):
    case = state["case"]
    heads, kv_heads, dim, new, batch = (case[n] for n in ("heads", "kv_heads", "dim", "new", "batch"))
    group, scale = heads // kv_heads, dim ** -0.5
    rows = state["q"].float().reshape(batch, new, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    own_q = rows.reshape(batch, kv_heads, group * new, dim)
    k, v = state["k"].float().permute(0, 2, 1, 3), state["v"].float().permute(0, 2, 1, 3)
    capacity = k.shape[2]
    scores = (own_q @ k.transpose(-1, -2) * scale).view(batch, kv_heads, group, new, capacity)
    last = state["lengths"][:, None] - new + torch.arange(new, device=k.device)[None]
    hidden = torch.arange(capacity, device=k.device) > last[..., None]
    scores = scores.masked_fill(hidden[:, None, None], float("-inf")).view(batch, kv_heads, group * new, capacity)
    if state["prefix_k"] is not None:
        all_q = rows.permute(1, 0, 2, 3, 4).reshape(kv_heads, batch * group * new, dim)
        pk, pv = state["prefix_k"].float().transpose(0, 1), state["prefix_v"].float().transpose(0, 1)
        shared = (all_q @ pk.transpose(-1, -2) * scale).view(kv_heads, batch, group * new, -1).transpose(0, 1)
        scores = torch.cat((shared, scores), -1)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == float("-inf"), 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    out = p[..., -capacity:] @ v
    if state["prefix_k"] is not None:
        shared = p[..., :-capacity].transpose(0, 1).reshape(kv_heads, batch * group * new, -1) @ pv
        out = out + shared.view(kv_heads, batch, group * new, dim).transpose(0, 1)
    out = out.reshape(batch, kv_heads, group, new, dim).permute(0, 3, 1, 2, 4)
    return out.reshape(batch, new, heads, dim).to(DTYPES[case["dtype"]])


def rotate(x, cos, sin):
    first, second = x.chunk(2, -1)
    return torch.cat((first * cos - second * sin, first * sin + second * cos), -1)


def plain_norm_rotary(state):
    angle = state["positions"].float()[..., None, None] * state["frequency"]
    cos, sin = angle.cos(), angle.sin()
    result = {}
    for name in ("q", "k"):
        x, weight = state[name].detach(), state[name + "_weight"].detach()
        y = x.float()
        inverse = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
        unit = y * inverse
        result[name] = rotate(unit * weight.float(), cos, sin).to(x.dtype)
        if state["case"]["train"]:
            back = rotate(state["d" + name].float(), cos, -sin)
            result["d" + name + "_weight"] = (back * unit).sum((0, 1, 2)).to(weight.dtype)
            back = back * weight.float()
            result["d" + name] = ((back - unit * (back * unit).mean(-1, keepdim=True)) * inverse).to(x.dtype)
    return result


# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return {"attention": plain_attention, "decode": plain_decode, "norm_rotary": plain_norm_rotary}[case["op"]](state)
    import nlogn_pisa_b200 as pisa

    if case["op"] == "attention":
        q, k, v = state["q"], state["k"], state["v"]
        out = pisa.full_attention(q, k, v, cu_seqlens=state.get("cu_queries"), cu_seqlens_k=state.get("cu_keys"))
        if not case["train"]:
            return out
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "decode":
        return pisa.prefix_attention(state["q"], state["k"], state["v"], state["lengths"],
                                     prefix_k=state["prefix_k"], prefix_v=state["prefix_v"])
    inputs = [state[n] for n in ("q", "k", "q_weight", "k_weight")]
    q, k = pisa.qk_norm_rotary(*inputs, state["frequency"], positions=state["positions"], eps=EPS)
    if not case["train"]:
        return {"q": q, "k": k}
    dq, dk, dqw, dkw = torch.autograd.grad((q, k), inputs, (state["dq"], state["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dq_weight": dqw, "dk_weight": dkw}


# ---------------------------------------------------------------------------
# 64 bits, one sequence and head at a time
# ---------------------------------------------------------------------------
def exact_attention(state):
    case = state["case"]
    group, scale = case["heads"] // case["kv_heads"], case["dim"] ** -0.5
    q, k, v, dout = (None if state.get(n) is None else state[n].detach().double() for n in ("q", "k", "v", "dout"))
    out = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    begin_q = begin_k = 0
    for index, (lq, lk) in enumerate(zip(numbers(case["queries"]), numbers(case["keys"]))):
        b = 0 if case["packed"] else index
        rows = slice(begin_q, begin_q + lq) if case["packed"] else slice(0, lq)
        cols = slice(begin_k, begin_k + lk) if case["packed"] else slice(0, lk)
        begin_q, begin_k = begin_q + lq, begin_k + lk
        future = torch.ones(lq, lk, dtype=torch.bool, device=q.device).triu(lk - lq + 1)
        for h in range(case["heads"]):
            kh, vh = k[b, cols, h // group], v[b, cols, h // group]
            weight = torch.softmax((scale * (q[b, rows, h] @ kh.T)).masked_fill(future, -math.inf), -1)
            o = weight @ vh
            out[b, rows, h] = o
            if dout is None:
                continue
            do = dout[b, rows, h]
            dv[b, cols, h // group] += weight.T @ do
            weight = scale * weight * (do @ vh.T - (do * o).sum(-1, keepdim=True))
            dq[b, rows, h] = weight @ kh
            dk[b, cols, h // group] += weight.T @ q[b, rows, h]
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["train"] else out


def exact_decode(state):
    case = state["case"]
    group, scale, new = case["heads"] // case["kv_heads"], case["dim"] ** -0.5, case["new"]
    q = state["q"].double()
    out = torch.zeros_like(q)
    for b, length in enumerate(own_lengths(case)):
        keys, values = state["k"][b, :length].double(), state["v"][b, :length].double()
        if state["prefix_k"] is not None:
            keys = torch.cat((state["prefix_k"].double(), keys))
            values = torch.cat((state["prefix_v"].double(), values))
        keys, values = keys.transpose(0, 1), values.transpose(0, 1)
        qb = q[b].transpose(0, 1).reshape(case["kv_heads"], group * new, case["dim"])
        logits = (scale * (qb @ keys.mT)).view(case["kv_heads"], group, new, -1)
        future = torch.ones(new, logits.shape[-1], dtype=torch.bool, device=q.device).triu(logits.shape[-1] - new + 1)
        weight = torch.softmax(logits.masked_fill(future, -math.inf), -1).view(case["kv_heads"], group * new, -1)
        out[b] = (weight @ values).view(case["heads"], new, case["dim"]).transpose(0, 1)
    return out


def exact_norm_rotary(state):
    half = state["case"]["dim"] // 2
    # the angle is the 32-bit product of position and frequency, by definition
    angle = (state["positions"].float()[..., None] * state["frequency"]).double()[:, :, None]
    turn = torch.polar(torch.ones_like(angle), angle)
    result = {}
    for name in ("q", "k"):
        x, weight = state[name].detach().double(), state[name + "_weight"].detach().double()
        rms = (x.pow(2).sum(-1, keepdim=True) / (2 * half) + EPS).sqrt()
        y = x / rms * weight
        z = torch.complex(y[..., :half], y[..., half:]) * turn
        result[name] = torch.cat((z.real, z.imag), -1)
        if state["case"]["train"]:
            g = state["d" + name].double()
            z = torch.complex(g[..., :half], g[..., half:]) * turn.conj()
            g = torch.cat((z.real, z.imag), -1)
            result["d" + name + "_weight"] = (g * x / rms).sum((0, 1, 2))
            g = g * weight
            result["d" + name] = g / rms - x * (g * x).sum(-1, keepdim=True) / (2 * half) / rms ** 3
    return result


def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": exact_attention, "decode": exact_decode, "norm_rotary": exact_norm_rotary}[case["op"]](state)
