"""What the operators around adapted and rotary transformer blocks are measured on, over the range of calls their users make.

Operators:
  rotary   fastbb_b200.rotary.rotary: queries and keys turned by the positions of their tokens on one to three axes (a patch
           grid, a video's frames and rows and columns), and the transposed turn that its gradient is
  diff     fastbb_b200.diff_attention.diff_attention: the difference of two softmax maps over the same values, with the learned
           weight of the second, key lengths per batch entry and the norm of every head's output
  adapter  fastbb_b200.adapters.adapter_linear: one shared projection and, beside it, the low-rank adapter of each request's rows

`listed()` holds the named cases, `draw(rng)` gives more of the same ranges. `run` computes the plain form (elementary torch
operations in 32 bits, rounded once) unless `own` is set, when it makes the calls that a user makes. `exact` gives the same
from the definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # A small model on one 224 x 224 image: 16 x 16 patches and a cls token that has no position. Launch and host time.
        {"name": "rotary_257_h6", "op": "rotary", "batch": 1, "frames": 1, "high": 16, "wide": 16, "prefix": 1, "heads": 6, "kv_heads": 6, "dim": 64,
         "axes": 2, "pairing": "half", "positions": "unit", "dtype": "fp16", "inverse": False, "packed": True},
        # One 896 x 1344 frame (64 x 96 patches and a cls token), queries and keys read out of the packed projection.
        {"name": "rotary_6145_h16", "op": "rotary", "batch": 1, "frames": 1, "high": 64, "wide": 96, "prefix": 1, "heads": 16, "kv_heads": 16, "dim": 64,
         "axes": 2, "pairing": "half", "positions": "unit", "dtype": "fp16", "inverse": False, "packed": True},
        # Video clips: integer positions in time, height and width far along the first axis, wide heads, few key heads, neighbours as pairs.
        {"name": "rotary_video_bf16", "op": "rotary", "batch": 2, "frames": 12, "high": 22, "wide": 31, "prefix": 0, "heads": 16, "kv_heads": 4, "dim": 128,
         "axes": 3, "pairing": "pairs", "positions": "int", "dtype": "bf16", "inverse": False, "packed": False},
        # The gradient's direction in fp32, four 518 x 518 images with four register tokens.
        {"name": "rotary_1374_inverse_fp32", "op": "rotary", "batch": 4, "frames": 1, "high": 37, "wide": 37, "prefix": 5, "heads": 24, "kv_heads": 24, "dim": 64,
         "axes": 2, "pairing": "half", "positions": "unit", "dtype": "fp32", "inverse": True, "packed": False},
        # One small image through one layer of a small model: latency of a launch with few tiles.
        {"name": "diff_257_h6", "op": "diff", "batch": 1, "queries": 257, "keys": 257, "heads": 6, "kv_heads": 6, "norm": True, "lam": "head",
         "ragged": False},
        # A single query over a long sequence of tokens (pooling a large image, or the cls row of a last layer).
        {"name": "diff_1_of_16385", "op": "diff", "batch": 1, "queries": 1, "keys": 16385, "heads": 8, "kv_heads": 8, "norm": True, "lam": "head",
         "ragged": False},
        # A padded batch of images of different sizes, one slot of it empty, the weight of the second map per token.
        {"name": "diff_1370_ragged", "op": "diff", "batch": 8, "queries": 1370, "keys": 1370, "heads": 6, "kv_heads": 6, "norm": True, "lam": "token",
         "ragged": True},
        # One 896 x 1344 frame with the width of a large model.
        {"name": "diff_6145_h8", "op": "diff", "batch": 1, "queries": 6145, "keys": 6145, "heads": 8, "kv_heads": 8, "norm": True, "lam": "head",
         "ragged": False},
        # One row a request, an adapter of its own for nearly each: a projection of pooled features.
        {"name": "adapter_64_single_rows", "op": "adapter", "requests": 64, "rows": 1, "ragged": False, "k": 1024, "n": 1024, "rank": 16,
         "adapters": 48, "act": "none", "residual": False},
        # Eight 224 x 224 images, each of another task: the packed query / key / value projection.
        {"name": "adapter_8x257_qkv", "op": "adapter", "requests": 8, "rows": 257, "ragged": False, "k": 768, "n": 2304, "rank": 16,
         "adapters": 6, "act": "none", "residual": False},
        # Images of different sizes packed one behind another, rows left at the end; the MLP's input layer with its activation.
        {"name": "adapter_ragged_fc1_gelu", "op": "adapter", "requests": 7, "rows": 878, "ragged": True, "k": 1024, "n": 4096, "rank": 32,
         "adapters": 12, "act": "gelu", "residual": False},
        # A large batch of 518 x 518 images: the MLP's output layer with LayerScale and residual.
        {"name": "adapter_16x1370_fc2", "op": "adapter", "requests": 16, "rows": 1370, "ragged": False, "k": 4096, "n": 1024, "rank": 64,
         "adapters": 10, "act": "none", "residual": True},
    ]


# ---------------------------------------------------------------------------------------------------------- more cases
def _spread(rng, lo, hi):
    """A whole number of lo .. hi, even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _draw_rotary(rng):
    axes = rng.choice([1, 2, 2, 3])
    heads = rng.choice([6, 12, 16, 24])
    return {"op": "rotary", "batch": _spread(rng, 1, 16), "frames": _spread(rng, 1, 16) if axes == 3 else 1, "high": _spread(rng, 1, 64),
            "wide": _spread(rng, 1, 96), "prefix": rng.choice([0, 1, 5]), "heads": heads,
            "kv_heads": rng.choice([heads, heads, heads // 3 if heads % 3 == 0 else heads // 4]), "dim": rng.choice([64, 64, 80, 128]), "axes": axes,
            "pairing": rng.choice(["half", "pairs"]), "positions": rng.choice(["unit", "int"]), "dtype": rng.choice(["fp16", "bf16", "fp32"]),
            "inverse": rng.random() < 0.3, "packed": False}


def _draw_diff(rng):
    queries, heads = _spread(rng, 1, 6145), rng.choice([3, 6, 8, 12])
    keys = queries if rng.random() < 0.7 else _spread(rng, 1, 16385)
    return {"op": "diff", "batch": _spread(rng, 1, 16), "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": rng.choice([heads, heads, heads // 3 if heads % 3 == 0 else heads // 4]), "norm": rng.random() < 0.7,
            "lam": rng.choice(["one", "head", "token"]), "ragged": rng.random() < 0.4}


def _draw_adapter(rng):
    c = rng.choice([384, 768, 1024])
    k, n = rng.choice([(c, c), (c, 4 * c) if c != 768 else (c, 1536), (4 * c, c) if c != 768 else (1536, c), (1024, 1000)])
    return {"op": "adapter", "requests": _spread(rng, 1, 64), "rows": _spread(rng, 1, 6145), "ragged": rng.random() < 0.5, "k": k, "n": n,
            "rank": rng.choice([8, 16, 32, 64]), "adapters": _spread(rng, 1, 48), "act": rng.choice(["none", "none", "gelu"]),
            "residual": rng.random() < 0.4}


def draw(rng):
    most = {}
    for case in listed():
        cost = work(case)
        for key in ("bytes", "flops"):
            most[case["op"], key] = max(most.get((case["op"], key), 0), cost[key])
    make = rng.choice([_draw_rotary, _draw_diff, _draw_adapter])
    while True:
        case = make(rng)
        cost = work(case)
        if all(cost[key] <= most[case["op"], key] for key in cost):
            return case


# ------------------------------------------------------------------------------------------------------ sizes and work
def _lengths(case):
    """Keys of each batch entry of a `diff` case: whole, or (ragged) spread from none to all of them."""
    batch, keys = case["batch"], case["keys"]
    if not case["ragged"]:
        return [keys] * batch
    return [keys * (batch - 1 - i) // max(1, batch - 1) if batch > 1 else keys // 2 for i in range(batch)]


def _counts(case):
    """Rows of each request of an `adapter` case: alike, or (ragged) growing from few to many, with the same sum at most."""
    requests, rows = case["requests"], case["rows"]
    if not case["ragged"]:
        return [rows] * requests
    total = requests * rows
    weights = [i * i for i in range(requests)]  # the first request has no rows at all
    return [total * w // max(1, sum(weights)) for w in weights]


def _grid(case):
    return case["frames"], case["high"], case["wide"]


def work(case):
    if case["op"] == "rotary":
        tokens = case["batch"] * (case["prefix"] + math.prod(_grid(case)))
        values = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * values * _BYTES[case["dtype"]] + 4 * math.prod(_grid(case)) * case["axes"], "flops": 3 * values}
    if case["op"] == "diff":
        pairs = case["queries"] * sum(_lengths(case)) * case["heads"]
        seen = sum(_lengths(case)) * case["kv_heads"] * 256
        return {"bytes": 2 * (case["batch"] * case["queries"] * case["heads"] * 256 + seen), "flops": pairs * 2 * 2 * (64 + 128)}
    rows, k, n, r = case["requests"] * case["rows"], case["k"], case["n"], case["rank"]
    used = min(case["adapters"], case["requests"])
    return {"bytes": 2 * (rows * (k + n * (2 if case["residual"] else 1)) + n * k + used * r * (k + n)), "flops": 2 * rows * (n * k + r * (k + n))}


# ------------------------------------------------------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0, mean=0.0, dtype=torch.float16):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).mul_(std).add_(mean).to(dtype)


def _ladder(case):
    """(frequency, axis) of every turned pair: each axis has a ladder of its own for its share of the pairs."""
    pairs, axes = case["dim"] // 2, case["axes"]
    theta = 10000.0 if case["positions"] == "int" else 100.0
    shares = [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]
    unit = 1.0 if case["positions"] == "int" else 2.0 * math.pi  # positions of patches on a frame go from -1 to 1
    freqs = [unit * theta ** (-j / n) for n in shares for j in range(n)]
    return freqs, [a for a, n in enumerate(shares) for _ in range(n)]


def _positions(case, g):
    t, h, w = _grid(case)
    where = torch.stack(torch.meshgrid(torch.arange(t), torch.arange(h), torch.arange(w), indexing="ij"), -1).reshape(-1, 3)[:, 3 - case["axes"]:]
    if case["positions"] == "int":
        start = torch.randint(0, 50000, (case["batch"], 1, case["axes"]), generator=g, device="cuda").cpu()  # clips begin anywhere in a film
        return (where[None] + start).to(torch.int32).cuda().contiguous()
    size = torch.tensor([t, h, w])[3 - case["axes"]:]
    return ((where + 0.5) / size * 2.0 - 1.0).float().cuda().contiguous()


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "rotary":
        b, n, h, hk, d = case["batch"], case["prefix"] + math.prod(_grid(case)), case["heads"], case["kv_heads"], case["dim"]
        dtype = _DTYPE[case["dtype"]]
        if case["packed"]:
            state["q"], state["k"], _ = _normal(g, b, n, 3, h, d, dtype=dtype).unbind(2)
        else:
            state["q"], state["k"] = _normal(g, b, n, h, d, dtype=dtype), _normal(g, b, n, hk, d, dtype=dtype)
        state["positions"] = _positions(case, g)
        freqs, axes = _ladder(case)
        state["freqs"], state["axes"] = torch.tensor(freqs, dtype=torch.float32, device="cuda"), torch.tensor(axes, device="cuda")
    elif case["op"] == "diff":
        b, nq, nk, h, hk = case["batch"], case["queries"], case["keys"], case["heads"], case["kv_heads"]
        state["q"], state["k"], state["v"] = _normal(g, b, nq, 2 * h, 64), _normal(g, b, nk, 2 * hk, 64), _normal(g, b, nk, hk, 128)
        shape = {"one": (1,), "head": (h,), "token": (b, nq, h)}[case["lam"]]
        state["lam"] = torch.rand(*shape, device="cuda", generator=g).mul_(0.6).add_(0.2)
        state["weight"] = _normal(g, 128, std=0.1, mean=1.0) if case["norm"] else None
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    else:
        counts, k, n, r, slots = _counts(case), case["k"], case["n"], case["rank"], case["adapters"]
        rows = case["requests"] * case["rows"]
        state["x"] = _normal(g, rows, k) if case["ragged"] else _normal(g, case["requests"], case["rows"], k)
        state["w"], state["b"] = _normal(g, n, k, std=0.02), _normal(g, n, std=0.1)
        state["down"], state["up"] = _normal(g, slots, r, k, std=k ** -0.5), _normal(g, slots, n, r, std=0.05)
        state["scale"] = torch.rand(slots, device="cuda", generator=g).add_(0.5)
        # every fifth request has no adapter
        ids = torch.randint(0, slots, (case["requests"],), device="cuda", generator=g)
        ids[torch.arange(case["requests"], device="cuda") % 5 == 4] = -1
        state["ids"], state["slots"] = ids.to(torch.int32), ids.tolist()
        state["offsets"] = None
        if case["ragged"]:
            state["offsets"] = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
        shape = (*state["x"].shape[:-1], n)
        state["res"], state["gamma"] = (_normal(g, *shape), _normal(g, n, std=0.1, mean=0.2)) if case["residual"] else (None, None)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["op"] == "rotary":
        from fastbb_b200.rotary import rotary_plan
        state["plan"] = rotary_plan(*_ladder(case), pairing=case["pairing"], device="cuda")
    elif own and case["op"] == "adapter":
        from fastbb_b200.adapters import Adapters
        state["adapters"] = Adapters(state["down"], state["up"], state["scale"])
    return state


# -------------------------------------------------------------------------------------------------------- a user's call
def _own(state):
    case = state["case"]
    if case["op"] == "rotary":
        from fastbb_b200.rotary import rotary
        return rotary(state["q"], state["k"], state["positions"], state["plan"], n_prefix=case["prefix"], inverse=case["inverse"])
    if case["op"] == "diff":
        from fastbb_b200.diff_attention import diff_attention
        return diff_attention(state["q"], state["k"], state["v"], state["lam"], weight=state["weight"], eps=1e-5, out_scale=0.2 if case["norm"] else 1.0,
                              key_lengths=state["lengths"])
    from fastbb_b200.adapters import adapter_linear
    return adapter_linear(state["x"], state["w"], state["adapters"], state["ids"], offsets=state["offsets"], b=state["b"],
                          act=None if case["act"] == "none" else case["act"], res=state["res"], gamma=state["gamma"])


# ----------------------------------------------------------------------------------------------------------- plain forms
def _plain_rotary(state):
    case, prefix = state["case"], state["case"]["prefix"]
    angle = state["positions"].double()[..., state["axes"]] * state["freqs"].double()  # far positions: the angle needs 64 bits
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    if case["inverse"]:
        sin = -sin
    outs = []
    for x in (state["q"], state["k"]):
        body = x[:, prefix:].float()
        if case["pairing"] == "half":
            first, second = body.chunk(2, -1)
            turned = torch.cat((first * cos - second * sin, second * cos + first * sin), -1)
        else:
            first, second = body[..., 0::2], body[..., 1::2]
            turned = torch.stack((first * cos - second * sin, second * cos + first * sin), -1).flatten(-2)
        outs.append(torch.cat((x[:, :prefix], turned.to(x.dtype)), 1))
    return tuple(outs)


def _plain_diff(state):
    case = state["case"]
    b, nq, nk, h, hk = case["batch"], case["queries"], case["keys"], case["heads"], case["kv_heads"]
    q = state["q"].float().view(b, nq, hk, h // hk, 2, 64).permute(0, 2, 3, 4, 1, 5)
    k = state["k"].float().view(b, nk, hk, 2, 64).permute(0, 2, 3, 4, 1)
    v = state["v"].float().permute(0, 2, 1, 3)
    scores = (q @ k.unsqueeze(2)) * 0.125
    if state["lengths"] is not None:
        hidden = torch.arange(nk, device="cuda") >= state["lengths"].view(b, 1, 1, 1, 1, 1)
        scores = scores.masked_fill(hidden, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    maps = (p @ v.unsqueeze(2).unsqueeze(3)) / torch.where(total == 0, 1.0, total)
    lam = state["lam"].expand(b, nq, h).permute(0, 2, 1).reshape(b, hk, h // hk, nq, 1)
    out = maps[:, :, :, 0] - lam * maps[:, :, :, 1]
    if state["weight"] is not None:
        out = out * torch.rsqrt((out * out).mean(-1, keepdim=True) + 1e-5) * state["weight"].float() * 0.2
    return out.permute(0, 3, 1, 2, 4).reshape(b, nq, h, 128).to(state["q"].dtype)


def _erf_gelu(y):
    return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))


def _plain_adapter(state):
    case = state["case"]
    x = state["x"].float().view(-1, case["k"])
    y = x @ state["w"].float().t() + state["b"].float()
    begin = 0
    for slot, count in zip(state["slots"], _counts(case)):  # the program that made the batch knows its requests
        if slot >= 0 and count > 0:
            rows = slice(begin, begin + count)
            y[rows] += (x[rows] @ state["down"][slot].float().t()) @ state["up"][slot].float().t() * state["scale"][slot]
        begin += count
    if case["act"] == "gelu":
        y = _erf_gelu(y)
    if state["res"] is not None:
        y = state["res"].float().view(y.shape) + state["gamma"].float() * y
    return y.to(torch.float16).view(*state["x"].shape[:-1], case["n"])


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "diff": _plain_diff, "adapter": _plain_adapter}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------- definitions in 64 bits
def _exact_rotary(state):
    """Each pair is a complex number, multiplied by exp(i angle)."""
    case = state["case"]
    pairs, prefix = case["dim"] // 2, case["prefix"]
    where = state["positions"].double()
    if where.dim() == 2:
        where = where[None]
    angle = torch.stack([where[:, :, int(a)] * float(f) for f, a in zip(state["freqs"].tolist(), state["axes"].tolist())], -1)
    turn = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle)[:, :, None]
    results = []
    for x in (state["q"], state["k"]):
        out = x.double().contiguous().clone()
        if case["pairing"] == "half":
            re, im = out[:, prefix:, :, :pairs], out[:, prefix:, :, pairs:]
        else:
            re, im = out[:, prefix:, :, 0::2], out[:, prefix:, :, 1::2]
        z = torch.complex(re.contiguous(), im.contiguous()) * turn
        re.copy_(z.real)
        im.copy_(z.imag)
        results.append(out)
    return tuple(results)


def _exact_diff(state):
    case = state["case"]
    b, nq, h, group = case["batch"], case["queries"], case["heads"], case["heads"] // case["kv_heads"]
    lengths = _lengths(case)
    lam = state["lam"].double().expand(b, nq, h)
    out = torch.zeros(b, nq, h, 128, dtype=torch.float64, device="cuda")
    for i in range(b):
        if lengths[i] == 0:
            continue
        for j in range(h):
            v = state["v"][i, :lengths[i], j // group].double()
            for which, sign in ((0, 1.0), (1, -1.0)):
                k = state["k"][i, :lengths[i], 2 * (j // group) + which].double()
                for lo in range(0, nq, 2048):
                    s = state["q"][i, lo:lo + 2048, 2 * j + which].double() @ k.t() / 8.0
                    o = torch.softmax(s, -1) @ v
                    out[i, lo:lo + 2048, j] += o if which == 0 else sign * lam[i, lo:lo + 2048, j, None] * o
    if case["norm"]:
        out = out / torch.sqrt(out.square().mean(-1, keepdim=True) + 1e-5) * state["weight"].double() * 0.2
    return out


def _exact_adapter(state):
    """Every adapter is added to a copy of the shared weight, and a request's rows are multiplied by that."""
    case = state["case"]
    x = state["x"].double().reshape(-1, case["k"])
    counts = _counts(case)
    out = torch.empty(x.shape[0], case["n"], dtype=torch.float64, device="cuda")
    at = 0
    w = state["w"].double()
    for slot, count in list(zip(state["slots"], counts)) + [(-1, x.shape[0] - sum(counts))]:
        full = w if slot < 0 else w + state["scale"][slot].double() * (state["up"][slot].double() @ state["down"][slot].double())
        out[at:at + count] = x[at:at + count] @ full.t()
        at += count
    out += state["b"].double()
    if case["act"] == "gelu":
        out = _erf_gelu(out)
    if case["residual"]:
        out = state["res"].double().reshape(out.shape) + state["gamma"].double() * out
    return out.view(*state["x"].shape[:-1], case["n"])


def exact(case, seed):
    state = _inputs(case, seed)
    return {"rotary": _exact_rotary, "diff": _exact_diff, "adapter": _exact_adapter}[case["op"]](state)
