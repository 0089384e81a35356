"""Operators of a serving batch's step over its cache, as cases to time and to check.

A layer of a model that answers many requests at once norms and turns each token's queries and keys,
appends its keys and values to a cache held in 8 bits, and attends over that cache, or over a long
prefix that the whole batch shares and each request's own few tokens behind it:

- norms of queries and keys for each head with the position rotation in the same pass (and the
  training step of the same, with the gradients of the norms' weights);
- tokens quantised into the cache as they are written, and a cache read back;
- attention of one token per sequence over the quantised cache;
- attention of one token per sequence over a shared prefix and the sequence's own cache.

`run` computes each in plain torch operations, or through the package where `own` is true.
"""

import math
import os
import random
import sys

import torch

own = False

ROTARY_BASE = 10000.0
EPS = 1e-6


def listed():
    return [
        # One user's next token, far into its answer: nothing but latency.
        dict(name="norm_token", op="norm", dtype="bfloat16", batch=1, tokens=1, heads=32, kv_heads=8,
             dim=128, rotary=128, interleaved=False, first=100000, packed=True, grad=False),
        # The training step of a layer with grouped KV heads.
        dict(name="norm_train", op="norm", dtype="bfloat16", batch=2, tokens=8192, heads=32, kv_heads=8,
             dim=128, rotary=128, interleaved=False, first=0, packed=False, grad=True),
        # A small model's training step: part of a head of 96 turned, in neighbouring pairs.
        dict(name="norm_partial", op="norm", dtype="float16", batch=3, tokens=1000, heads=16, kv_heads=4,
             dim=96, rotary=48, interleaved=True, first=0, packed=True, grad=True),
        # A serving batch's next token joins its caches.
        dict(name="append_token", op="append", dtype="bfloat16", cache="float8_e4m3fn", batch=32, tokens=1,
             kv_heads=8, dim=128, length=2048, ragged=False, split=0),
        # Prompts of any length join their caches.
        dict(name="append_prompt", op="append", dtype="bfloat16", cache="int8", batch=8, tokens=4096,
             kv_heads=8, dim=128, length=4200, ragged=True, split=1),
        # Caches are read back for an attention that takes 16 bits.
        dict(name="read_back", op="read", dtype="bfloat16", cache="float8_e4m3fn", batch=8,
             kv_heads=8, dim=128, length=8192, ragged=True, split=2),
        # One user's next token over a short context: launches and latencies.
        dict(name="quantized_one", op="quantized", dtype="bfloat16", cache="float8_e4m3fn", batch=1, heads=32,
             kv_heads=8, dim=128, length=2000, ragged=False, split=3),
        # A serving batch in the middle of its answers.
        dict(name="quantized_batch", op="quantized", dtype="bfloat16", cache="float8_e4m3fn", batch=32, heads=32,
             kv_heads=8, dim=128, length=16384, ragged=True, split=4),
        # Two users far into very long documents, eight heads to a KV head.
        dict(name="quantized_long", op="quantized", dtype="float16", cache="int8", batch=2, heads=64,
             kv_heads=8, dim=128, length=131072, ragged=False, split=5),
        # A few answers to one question that is not long.
        dict(name="prefix_few", op="prefix", dtype="bfloat16", batch=4, heads=32, kv_heads=8, dim=128,
             prefix=2048, length=256, ragged=True, split=6),
        # A serving batch behind a system prompt, heads of 64.
        dict(name="prefix_batch", op="prefix", dtype="float16", batch=32, heads=32, kv_heads=8, dim=64,
             prefix=16385, length=1024, ragged=True, split=7),
        # Many questions about one long document.
        dict(name="prefix_large", op="prefix", dtype="bfloat16", batch=128, heads=32, kv_heads=8, dim=128,
             prefix=32768, length=2048, ragged=True, split=8),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


# No drawn case costs more than the largest listed ones.
_MOST_NORMED = 2 * 8192 * 40 * 128
_MOST_APPENDED = 8 * 4096 * 8 * 128
_MOST_READ = 8 * 8192 * 8 * 128
_MOST_CACHED = 2 * 131072 * 8 * 128
_MOST_SHARED_SCORES = 128 * 32 * 32768
_MOST_PREFIX = 32768 * 8 * 128
_MOST_OWN = 128 * 2048 * 8 * 128


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "read", "quantized", "quantized", "prefix", "prefix"])
    half = rng.choice(["float16", "bfloat16"])
    any_dtype = rng.choice(["float16", "bfloat16", "float32"])
    cache = rng.choice(["float8_e4m3fn", "int8"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 6, 8, 16])
    batch = _log(rng, 1, 128)
    ragged, split = rng.random() < 0.6, rng.randrange(1000)
    if op == "norm":
        dim = rng.choice([64, 80, 96, 128, 256])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        batch, tokens = _log(rng, 1, 8), _log(rng, 1, 8192)
        tokens = max(1, min(tokens, _MOST_NORMED // (batch * (heads + kv) * dim)))
        return dict(op=op, dtype=any_dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv, dim=dim,
                    rotary=rotary, interleaved=rng.random() < 0.5, first=rng.choice([0, _log(rng, 1, 10 ** 6)]),
                    packed=rng.random() < 0.5, grad=rng.random() < 0.7)
    if op == "append":
        dim = rng.choice([64, 80, 96, 128, 256])
        tokens = min(_log(rng, 1, 4096), _MOST_APPENDED // (batch * kv * dim))
        return dict(op=op, dtype=any_dtype, cache=cache, batch=batch, tokens=tokens, kv_heads=kv, dim=dim,
                    length=tokens + _log(rng, 1, 200), ragged=ragged, split=split)
    dim = rng.choice([64, 128])
    if op == "read":
        length = min(_log(rng, 1, 32768), _MOST_READ // (batch * kv * dim))
        return dict(op=op, dtype=any_dtype, cache=cache, batch=batch, kv_heads=kv, dim=dim, length=length,
                    ragged=ragged, split=split)
    if op == "quantized":
        length = max(1, min(_log(rng, 1, 131072), _MOST_CACHED // (batch * kv * dim)))
        return dict(op=op, dtype=half, cache=cache, batch=batch, heads=heads, kv_heads=kv, dim=dim,
                    length=length, ragged=ragged, split=split)
    prefix = max(1, min(_log(rng, 1, 131072), _MOST_PREFIX // (kv * dim), _MOST_SHARED_SCORES // (batch * heads)))
    length = max(1, min(_log(rng, 1, 2048), _MOST_OWN // (batch * kv * dim)))
    return dict(op=op, dtype=half, batch=batch, heads=heads, kv_heads=kv, dim=dim, prefix=prefix, length=length,
                ragged=ragged, split=split)


# ------------------------------------------------------------------ inputs


def _lengths(case, longest, shift=0):
    """A number of tokens for each sequence: all the most, or anything from none up to it."""
    if not case["ragged"]:
        return [longest] * case["batch"]
    rng = random.Random(case["split"] + shift)
    return [rng.randint(0, longest) for _ in range(case["batch"])]


def _frequencies(case):
    """Radians per position of each pair."""
    half = case["rotary"] // 2
    return ROTARY_BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)


def _stored(x, kind):
    """Rows as a cache holds them: codes and a scale for each row."""
    top = 448.0 if kind == "float8_e4m3fn" else 127.0
    scale = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100) / top
    codes = (x / scale).clamp(-top, top)
    codes = codes.to(torch.float8_e4m3fn) if kind == "float8_e4m3fn" else codes.round().to(torch.int8)
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    def tokens_of(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    op, batch, kv, dim, state = case["op"], case["batch"], case["kv_heads"], case["dim"], {"case": case}
    if op == "norm":
        tokens = case["tokens"]
        for name, heads in (("q", case["heads"]), ("k", kv)):
            # A projection's output, as rows of tokens (packed) or seen head-major.
            x, dx = normal(batch, tokens, heads, dim), normal(batch, tokens, heads, dim)
            if case["packed"]:
                x, dx = x.flatten(0, 1), dx.flatten(0, 1)
            else:
                x, dx = x.transpose(1, 2), dx.transpose(1, 2)
            weight = (1 + 0.2 * torch.randn(dim, generator=gen, device="cuda")).to(dtype)
            state[name], state["d" + name] = x.requires_grad_(case["grad"]), dx
            state[name + "_weight"] = weight.requires_grad_(case["grad"])
        start = torch.randint(case["first"], case["first"] + 64, (batch, 1), generator=gen, device="cuda")
        positions = start + torch.arange(tokens, device="cuda")
        state["positions"] = positions.flatten() if case["packed"] else positions
        state["frequencies"] = _frequencies(case)
        return state
    if op == "prefix":
        state["q"] = normal(batch, case["heads"], dim)
        state["k_prefix"], state["v_prefix"] = (normal(kv, case["prefix"], dim) for _ in "kv")
        state["k_cache"], state["v_cache"] = (normal(batch, kv, case["length"], dim) for _ in "kv")
        state["lengths"] = tokens_of(_lengths(case, case["length"]))
        return state
    length = case["length"]
    # Keys and values of rows that differ in size by some powers of two.
    size = torch.exp2(torch.randint(-3, 3, (2, batch, kv, length, 1), generator=gen, device="cuda").float())
    k, k_scale = _stored(torch.randn(batch, kv, length, dim, generator=gen, device="cuda") * size[0].clamp(max=1), case["cache"])
    v, v_scale = _stored(torch.randn(batch, kv, length, dim, generator=gen, device="cuda") * size[1], case["cache"])
    state["k_cache"], state["v_cache"], state["scales"] = k, v, torch.cat((k_scale, v_scale), -1)
    if op == "append":
        tokens = case["tokens"]
        state["k"], state["v"] = (normal(batch, tokens, kv, dim).transpose(1, 2) for _ in "kv")
        state["counts"] = tokens_of(_lengths(case, tokens)) if case["ragged"] else None
        state["lengths"] = tokens_of(_lengths(case, length - tokens, 1))
        return state
    state["lengths"] = tokens_of(_lengths(case, length))
    if op == "quantized":
        state["q"] = normal(batch, case["heads"], dim)
    return state


# ------------------------------------------------------------------ the plain forms


def _turn(x, cos, sin, case):
    """float32 x (..., dim) with its first `rotary` features turned."""
    rotary = case["rotary"]
    turned = x[..., :rotary]
    if case["interleaved"]:
        first, second = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack((first * cos - second * sin, second * cos + first * sin), -1).flatten(-2)
    else:
        first, second = turned[..., : rotary // 2], turned[..., rotary // 2:]
        out = torch.cat((first * cos - second * sin, second * cos + first * sin), -1)
    return torch.cat((out, x[..., rotary:]), -1)


def _plain_norm(state):
    case = state["case"]
    # Angles of far positions lose whole radians in 32 bits.
    angle = (state["positions"].double()[..., None] * state["frequencies"]).unsqueeze(1)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    outs, gradients, weights = [], [], []
    for name in ("q", "k"):
        x, w = state[name].detach().float(), state[name + "_weight"].detach().float()
        inverse = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        unit = x * inverse
        outs.append(_turn(unit * w, cos, sin, case).to(state[name].dtype))
        if case["grad"]:
            dz = _turn(state["d" + name].float(), cos, -sin, case)
            by_weight = (dz * unit).flatten(0, -2).sum(0)
            g = dz * w
            gradients.append((inverse * (g - unit * (g * unit).mean(-1, keepdim=True))).to(x.dtype).to(state[name].dtype))
            weights.append(by_weight.to(state[name].dtype))
    return (*outs, *gradients, *weights)


def _plain_append(state):
    case, lengths = state["case"], state["lengths"]
    kind, batch, tokens, kv, dim = (case[x] for x in ("cache", "batch", "tokens", "kv_heads", "dim"))
    top = 448.0 if kind == "float8_e4m3fn" else 127.0
    counts = state["counts"] if state["counts"] is not None else torch.full_like(lengths, tokens)
    step = torch.arange(tokens, device=lengths.device)
    place = (lengths[:, None] + step).long()[:, None, :, None]
    kept = (step < counts[:, None])[:, None, :, None]
    row = place.expand(batch, kv, tokens, dim)
    for i, name in enumerate("kv"):
        x = state[name].float()
        most = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
        codes = x * (top / most)
        codes = codes.to(torch.float8_e4m3fn) if kind == "float8_e4m3fn" else codes.round().to(torch.int8)
        held = state[name + "_cache"].view(torch.uint8)
        held.scatter_(2, row, torch.where(kept, codes.view(torch.uint8), held.gather(2, row)))
        one, scales = place.expand(batch, kv, tokens, 1), state["scales"][..., i: i + 1]
        scales.scatter_(2, one, torch.where(kept, most / top, scales.gather(2, one)))
    return state["k_cache"], state["v_cache"], state["scales"], lengths + counts


def _plain_read(state):
    case = state["case"]
    there = (torch.arange(case["length"], device="cuda") < state["lengths"][:, None])[:, None, :, None]
    return tuple((state[name + "_cache"].float() * state["scales"][..., i: i + 1]).masked_fill(~there, 0)
                 .to(getattr(torch, case["dtype"])) for i, name in enumerate("kv"))


def _attend(scores, values_of):
    """Softmax over the scores' last axis (float32, -inf where there is no key), its product with the
    values and its logarithm's sum in base 2."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = values_of(weights) / torch.where(total > 0, total, torch.ones_like(total))
    return out, (torch.log2(total) + top * math.log2(math.e))[..., 0]


def _plain_quantized(state):
    case, q = state["case"], state["q"]
    batch, kv, dim = case["batch"], case["kv_heads"], case["dim"]
    q32 = q.float().reshape(batch, kv, -1, dim)
    keys = state["k_cache"].float() * state["scales"][..., 0:1]
    values = state["v_cache"].float() * state["scales"][..., 1:2]
    there = (torch.arange(case["length"], device="cuda") < state["lengths"][:, None])[:, None, None]
    scores = torch.matmul(q32, keys.transpose(2, 3).contiguous()) * dim ** -0.5
    scores = scores.masked_fill(~there, -math.inf)
    out, lse = _attend(scores, lambda weights: torch.matmul(weights, values))
    return out.reshape(q.shape).to(q.dtype), lse.reshape(q.shape[:2])


def _plain_prefix(state):
    case, q = state["case"], state["q"]
    batch, kv, dim, prefix = case["batch"], case["kv_heads"], case["dim"], case["prefix"]
    q32 = q.float().reshape(batch, kv, -1, dim)
    group = q32.shape[2]
    shared = q32.transpose(0, 1).reshape(kv, batch * group, dim)
    first = torch.matmul(shared, state["k_prefix"].float().transpose(1, 2).contiguous())
    first = first.reshape(kv, batch, group, prefix).transpose(0, 1)
    second = torch.matmul(q32, state["k_cache"].float().transpose(2, 3).contiguous())
    there = (torch.arange(case["length"], device="cuda") < state["lengths"][:, None])[:, None, None]
    scores = torch.cat((first, second.masked_fill(~there, -math.inf)), -1) * dim ** -0.5

    def values_of(weights):
        rows = weights[..., :prefix].transpose(0, 1).reshape(kv, batch * group, prefix)
        part = torch.matmul(rows, state["v_prefix"].float()).reshape(kv, batch, group, dim).transpose(0, 1)
        return part + torch.matmul(weights[..., prefix:], state["v_cache"].float())

    out, lse = _attend(scores, values_of)
    return out.reshape(q.shape).to(q.dtype), lse.reshape(q.shape[:2])


# ------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        plain = {"norm": _plain_norm, "append": _plain_append, "read": _plain_read,
                 "quantized": _plain_quantized, "prefix": _plain_prefix}
        return plain[op](state)
    if os.path.join(os.getcwd(), "triton-kernel-lab_amd") not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), "triton-kernel-lab_amd"))
    if op == "norm":
        from tklab.kernels.qk_norm_rotary import qk_norm_rotary

        leaves = [state[name] for name in ("q", "k", "q_weight", "k_weight")]
        out = qk_norm_rotary(*leaves, state["positions"], state["frequencies"], eps=EPS,
                             interleaved=case["interleaved"])
        if not case["grad"]:
            return out
        return (*out, *torch.autograd.grad(out, leaves, (state["dq"], state["dk"])))
    caches = state["k_cache"], state["v_cache"]
    if op == "append":
        from tklab.kernels.quantized_cache import append_quantized

        lengths = append_quantized(*caches, state["scales"], state["lengths"], state["k"], state["v"],
                                   state["counts"])
        return *caches, state["scales"], lengths
    if op == "read":
        from tklab.kernels.quantized_cache import read_quantized

        return read_quantized(*caches, state["scales"], state["lengths"], dtype=getattr(torch, case["dtype"]))
    if op == "quantized":
        from tklab.kernels.quantized_decode import quantized_decode

        return quantized_decode(state["q"], *caches, state["scales"], state["lengths"], return_lse=True)
    from tklab.kernels.prefix_decode import prefix_decode

    return prefix_decode(state["q"], state["k_prefix"], state["v_prefix"], *caches, state["lengths"],
                         return_lse=True)


# ------------------------------------------------------------------ from the definitions, in 64 bits


def _exact_norm(state):
    """Each pair as a complex number turned by e^(i angle), the gradients by differentiation."""
    case = state["case"]
    half = case["rotary"] // 2
    angle = state["positions"].double()[..., None] * state["frequencies"]
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)  # every head alike
    outs, gradients, weights = [], [], []
    for name in ("q", "k"):
        x = state[name].detach().double().requires_grad_(case["grad"])
        w = state[name + "_weight"].detach().double().requires_grad_(case["grad"])
        normed = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        part = normed[..., : case["rotary"]]
        pairs = part.unflatten(-1, (half, 2)) if case["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        y = torch.cat((z, normed[..., case["rotary"]:]), -1)
        outs.append(y.detach())
        if case["grad"]:
            dx, dw = torch.autograd.grad(y, (x, w), state["d" + name].double())
            gradients.append(dx)
            weights.append(dw)
    return (*outs, *gradients, *weights)


def _exact_append(state):
    """Sequence by sequence. Codes of whole numbers have no value between them: None."""
    case, kind = state["case"], state["case"]["cache"]
    top = 448.0 if kind == "float8_e4m3fn" else 127.0
    starts = state["lengths"].tolist()
    counts = state["counts"].tolist() if state["counts"] is not None else [case["tokens"]] * case["batch"]
    scales, held = state["scales"].double(), []
    for i, name in enumerate("kv"):
        values = state[name + "_cache"].double()
        for b, (n, start) in enumerate(zip(counts, starts)):
            x = state[name][b, :, :n].double()
            scale = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100) / top
            # Three bits behind the leading one, and no step finer than 2^-9.
            step = torch.exp2(torch.frexp(x / scale)[1].clamp(min=-5).double() - 4)
            values[b, :, start: start + n] = torch.round(x / scale / step) * step
            scales[b, :, start: start + n, i] = scale[..., 0]
        held.append(values if kind == "float8_e4m3fn" else None)
    ends = torch.tensor([a + b for a, b in zip(starts, counts)], dtype=torch.int32, device="cuda")
    return (*held, scales, ends)


def _exact_read(state):
    out = []
    for i, name in enumerate("kv"):
        x = torch.zeros(state[name + "_cache"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(state["lengths"].tolist()):
            x[b, :, :n] = state[name + "_cache"][b, :, :n].double() * state["scales"][b, :, :n, i, None].double()
        out.append(x)
    return tuple(out)


def _exact_attention(state, keys_and_values):
    """KV head by KV head, over the keys and values that `keys_and_values` names for each sequence."""
    case, q = state["case"], state["q"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for g in range(case["kv_heads"]):
        heads = slice(g * group, (g + 1) * group)
        for b in range(case["batch"]):
            keys, values = keys_and_values(b, g)
            if len(keys) == 0:
                continue
            scores = q[b, heads].double() @ keys.t() / math.sqrt(case["dim"])
            log = torch.logsumexp(scores, 1)
            out[b, heads] = torch.exp(scores - log[:, None]) @ values
            lse[b, heads] = log / math.log(2)
    return out, lse


def _exact_quantized(state):
    lengths = state["lengths"].tolist()

    def there(b, g):
        n = lengths[b]
        scales = state["scales"][b, g, :n].double()
        return (state["k_cache"][b, g, :n].double() * scales[:, 0:1], state["v_cache"][b, g, :n].double() * scales[:, 1:2])

    return _exact_attention(state, there)


def _exact_prefix(state):
    lengths = state["lengths"].tolist()

    def there(b, g):
        return tuple(torch.cat((state[name + "_prefix"][g], state[name + "_cache"][b, g, : lengths[b]])).double()
                     for name in "kv")

    return _exact_attention(state, there)


def exact(case, seed):
    state = prepare(case, seed)
    how = {"norm": _exact_norm, "append": _exact_append, "read": _exact_read, "quantized": _exact_quantized,
           "prefix": _exact_prefix}
    return how[case["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op, batch, kv, dim = case["op"], case["batch"], case["kv_heads"], case["dim"]
    if op == "norm":
        tokens = batch * case["tokens"]
        elements = tokens * (case["heads"] + kv) * dim
        passes, flops = (5, 18) if case["grad"] else (2, 7)
        return {"bytes": passes * elements * size + tokens * 8 * (2 if case["grad"] else 1), "flops": flops * elements}
    if op == "append":
        rows = 2 * kv * sum(_lengths(case, case["tokens"]) if case["ragged"] else [case["tokens"]] * batch)
        return {"bytes": rows * (dim * (size + 1) + 4) + batch * 12, "flops": 3 * rows * dim}
    if op == "read":
        rows, there = 2 * kv * batch * case["length"], 2 * kv * sum(_lengths(case, case["length"]))
        return {"bytes": there * (dim + 4) + rows * dim * size + batch * 4, "flops": there * dim}
    heads = case["heads"]
    keys = sum(_lengths(case, case["length"]))
    ends = batch * heads * (2 * dim * size + 4) + batch * 4
    if op == "quantized":
        return {"bytes": keys * kv * 2 * (dim + 4) + ends, "flops": 4 * keys * heads * dim}
    return {"bytes": (keys + case["prefix"]) * kv * 2 * dim * size + ends,
            "flops": 4 * (keys + batch * case["prefix"]) * heads * dim}
