"""Performance cases of weights held in microscaled 4-bit floating point.

A block of 32 consecutive elements of a row shares a scale, a power of two (8 exponent bits); every
element has a sign, two exponent bits and one mantissa bit.  Three kinds of call:

    store     quantise a matrix and read it back           MX4Manager.write / MX4Manager.read
    linear    product of quantised inputs and weights      MX4Manager.linear
    experts   the same, every row by its expert's matrix   MX4Manager.grouped_linear

With `own` false `run` computes them in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

BLOCK = 32
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # converting a model: one projection of a 7B block, written and read back
        {"name": "store_matrix", "kind": "store", "rows": 4096, "cols": 11008, "dtype": "bf16"},
        # a small table of a shape that fits nothing
        {"name": "store_odd", "kind": "store", "rows": 1001, "cols": 4099, "dtype": "fp16"},
        # one token through an attention projection of a 7B model: latency
        {"name": "linear_token", "kind": "linear", "rows": 1, "out": 4096, "in": 4096, "dtype": "bf16",
         "bias": False},
        # a batch of generation through an up projection
        {"name": "linear_batch", "kind": "linear", "rows": 16, "out": 11008, "in": 4096, "dtype": "bf16",
         "bias": False},
        # ragged in every dimension, with a bias
        {"name": "linear_odd", "kind": "linear", "rows": 333, "out": 4099, "in": 1000, "dtype": "fp16",
         "bias": True},
        # a prompt through an up projection of a 7B model
        {"name": "linear_prompt", "kind": "linear", "rows": 2048, "out": 11008, "in": 4096, "dtype": "bf16",
         "bias": False},
        # the largest matrix of a 70B model on a long prompt
        {"name": "linear_large", "kind": "linear", "rows": 8192, "out": 28672, "in": 8192, "dtype": "bf16",
         "bias": False},
        # one token that goes to two of eight experts
        {"name": "experts_token", "kind": "experts", "tokens": 1, "top_k": 2, "experts": 8, "out": 11008,
         "in": 4096, "dtype": "bf16", "bias": False, "shared": True, "dropped": 0.0},
        # a batch of generation over many small experts: first product ...
        {"name": "experts_batch", "kind": "experts", "tokens": 32, "top_k": 8, "experts": 64, "out": 1408,
         "in": 2048, "dtype": "bf16", "bias": False, "shared": True, "dropped": 0.0},
        # ... and the one that leads back, whose rows differ from expert to expert
        {"name": "experts_back", "kind": "experts", "tokens": 32, "top_k": 8, "experts": 64, "out": 2048,
         "in": 1408, "dtype": "bf16", "bias": False, "shared": False, "dropped": 0.0},
        # a prompt over eight large experts
        {"name": "experts_prompt", "kind": "experts", "tokens": 4096, "top_k": 2, "experts": 8, "out": 11008,
         "in": 4096, "dtype": "bf16", "bias": False, "shared": True, "dropped": 0.0},
        # ragged in every dimension, a padded batch: some rows have no expert
        {"name": "experts_odd", "kind": "experts", "tokens": 777, "top_k": 3, "experts": 13, "out": 1001,
         "in": 1000, "dtype": "fp16", "bias": True, "shared": True, "dropped": 0.1},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A feature count: often a multiple of 64, else anything."""
    n = _log_between(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.6 else n


def draw(rng):
    kind = rng.choice(("store", "linear", "linear", "experts", "experts"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "store":
        cols = _log_between(rng, 1, 16384)
        rows = min(_log_between(rng, 1, 32768), 128_000_000 // cols)
        return {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype}
    out, inner = _size(rng, 64, 16384), _size(rng, 64, 16384)
    if kind == "linear":
        rows = min(_log_between(rng, 1, 8192), max(1, int(1.5e12 / (out * inner))))
        return {"kind": kind, "rows": rows, "out": out, "in": inner, "dtype": dtype,
                "bias": rng.random() < 0.3}
    experts = _log_between(rng, 2, 128)
    while experts * out * inner > 400_000_000:
        out, inner = max(64, out // 2), max(64, inner // 2)
    tokens = min(_log_between(rng, 1, 4096), max(1, int(1.0e11 / (out * inner))))
    return {"kind": kind, "tokens": tokens, "top_k": rng.randint(1, min(8, experts)), "experts": experts,
            "out": out, "in": inner, "dtype": dtype, "bias": rng.random() < 0.3,
            "shared": rng.random() < 0.5, "dropped": rng.choice((0.0, 0.0, 0.05, 0.3))}


# ------------------------------------------------------------------ inputs
def _weight(g, shape, dtype):
    """Normal weights whose standard deviation of about 0.02 differs a little from row to row."""
    scale = 0.02 * torch.exp(0.2 * torch.randn(*shape[:-1], 1, generator=g, device="cuda"))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _activations(g, shape, dtype):
    """Normal activations in which about one channel of a hundred is ten times larger."""
    channel = torch.rand(shape[-1], generator=g, device="cuda")
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * torch.where(channel < 0.01, 10.0, 1.0)).to(dtype)


def _routes(g, case):
    """The top_k experts of every token; some experts are more popular; -1 where a row has none."""
    tokens, experts = case["tokens"], case["experts"]
    liking = 0.5 * torch.randn(experts, generator=g, device="cuda")
    logits = torch.randn(tokens, experts, generator=g, device="cuda") + liking
    ids = logits.topk(case["top_k"], dim=-1).indices
    lost = torch.rand(tokens, 1, generator=g, device="cuda") < case["dropped"]
    return torch.where(lost, -1, ids)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["kind"] == "store":
        return {"weight": _weight(g, (case["rows"], case["cols"]), dtype)}
    if case["kind"] == "linear":
        weight = (case["out"], case["in"])
        x = (case["rows"], case["in"])
        d = {}
    else:
        weight = (case["experts"], case["out"], case["in"])
        x = (case["tokens"],) + (() if case["shared"] else (case["top_k"],)) + (case["in"],)
        d = {"ids": _routes(g, case)}
    bias = weight[:-1]
    d["weight"] = _weight(g, weight, dtype)
    d["x"] = _activations(g, x, dtype)
    d["bias"] = torch.randn(*bias, generator=g, device="cuda").to(dtype) if case["bias"] else None
    return d


def prepare(case, seed):
    """What a program has in hand: the weights as they are held, the inputs, the experts' numbers."""
    state = _inputs(case, seed)
    state["kind"] = case["kind"]
    if own:
        import neuzip_b200 as nz
        state["manager"] = nz.MX4Manager()
    if case["kind"] == "store":
        return state
    weight = state.pop("weight")
    if own:
        state["handle"] = state["manager"].write(weight)
    else:
        state["codes"], state["scales"] = _quantise(weight)
        state["inner"] = weight.shape[-1]
    return state


# ------------------------------------------------------------------ the plain form
def _power_of_two(e):
    """2^e in 32 bits for whole numbers -127 <= e <= 127 (ldexp would round the smallest to zero)."""
    return torch.exp2(torch.clamp(e, min=-126.0)) * torch.where(e < -126.0, 0.5, 1.0)


def _quantise(w):
    """Codes (uint8, one per element, padded to whole blocks) and scale exponents (uint8) of the rows of w."""
    v = w.float()
    pad = -v.shape[-1] % BLOCK
    if pad:
        v = torch.nn.functional.pad(v, (0, pad))
    v = v.unflatten(-1, (-1, BLOCK))
    largest = v.abs().amax(-1)
    # floor(log2 a) is the exponent of a minus one: frexp gives a = m * 2^e with 0.5 <= m < 1
    exponent = torch.frexp(largest).exponent.float() - 1.0
    exponent = torch.where(largest > 0, exponent - 2.0, -127.0).clamp(min=-127.0)
    finite = torch.isfinite(largest)
    exponent = torch.where(finite, exponent, 0.0)
    # dividing by 2^e in two steps: 2^127 / 2^-127 has no reciprocal in range
    half = torch.floor(-exponent / 2)
    u = v * _power_of_two(half).unsqueeze(-1) * _power_of_two(-exponent - half).unsqueeze(-1)
    m = u.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5)
            + (m > 5.0))
    code = code + 8 * torch.signbit(u).to(torch.uint8)
    code = torch.where(finite.unsqueeze(-1), code, 0).to(torch.uint8).flatten(-2)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    return packed, torch.where(finite, exponent + 127.0, 255.0).to(torch.uint8)


def _values(codes, scales, inner):
    """The numbers that codes and scales stand for, in 32 bits."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    v = table[both.int()].unflatten(-1, (-1, BLOCK))
    s = torch.where(scales == 255, math.nan, _power_of_two(scales.float() - 127.0))
    return (v * s.unsqueeze(-1)).flatten(-2)[..., :inner]


def _plain_linear(state):
    x = state["x"]
    v = _values(*_quantise(x), x.shape[-1])
    y = v @ _values(state["codes"], state["scales"], state["inner"]).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(x.dtype)


def _plain_experts(state):
    """The rows of each expert that is named, side by side and padded to the longest, in one batched product."""
    x, ids, inner = state["x"], state["ids"], state["inner"]
    rows = ids.numel()
    v = _values(*_quantise(x), inner)
    if v.dim() == ids.dim():
        v = v.unsqueeze(-2).expand(*ids.shape, inner)
    v = v.reshape(rows, inner)
    named, which, count = torch.unique(ids.reshape(-1), return_inverse=True, return_counts=True)
    order = torch.argsort(which, stable=True)
    first = torch.cumsum(count, 0) - count
    place = torch.empty_like(which)
    place[order] = torch.arange(rows, device=x.device) - first[which[order]]
    longest = int(count.max())
    padded = torch.zeros(named.numel(), longest, inner, device=x.device)
    padded[which, place] = v
    e = named.clamp(min=0)
    w = _values(state["codes"][e], state["scales"][e], inner)
    y = torch.bmm(padded, w.transpose(1, 2))[which, place]
    expert = ids.reshape(-1, 1)
    if state["bias"] is not None:
        y = y + state["bias"].float()[expert[:, 0].clamp(min=0)]
    y = torch.where(expert >= 0, y, 0.0)
    return y.reshape(*ids.shape, -1).to(x.dtype)


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        manager = state["manager"]
        if state["kind"] == "store":
            return manager.read(manager.write(state["weight"], "weight"))
        if state["kind"] == "linear":
            return manager.linear(state["handle"], state["x"], state["bias"])
        return manager.grouped_linear(state["handle"], state["x"], state["ids"], state["bias"])
    if state["kind"] == "store":
        w = state["weight"]
        return _values(*_quantise(w), w.shape[-1]).to(w.dtype)
    return _plain_linear(state) if state["kind"] == "linear" else _plain_experts(state)


def _held(rows, cols):
    """Bytes of a quantised matrix: half a byte per element of whole blocks and one per block."""
    blocks = -(-cols // BLOCK)
    return rows * blocks * (BLOCK // 2 + 1)


def work(case):
    if case["kind"] == "store":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * 2 * n + 2 * _held(case["rows"], case["cols"]), "flops": 0}
    out, inner = case["out"], case["in"]
    if case["kind"] == "linear":
        m = case["rows"]
        moved = 2 * m * (inner + out) + _held(out, inner) + (2 * out if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * m * out * inner}
    experts, rows = case["experts"], case["tokens"] * case["top_k"]
    real = rows * (1 - case["dropped"])
    # experts that at least one token names, as if all were equally popular
    hit = experts * (1 - (1 - case["top_k"] / experts) ** (case["tokens"] * (1 - case["dropped"])))
    read = case["tokens"] if case["shared"] else rows
    moved = 2 * read * inner + 8 * rows + 2 * rows * out + hit * _held(out, inner)
    if case["bias"]:
        moved += 2 * hit * out
    return {"bytes": moved, "flops": 2 * real * out * inner}


# ------------------------------------------------------------------ 64 bits, from the definition
def _exact_values(w):
    """The nearest number of the format to every element, in 64 bits."""
    v = w.double()
    cols = v.shape[-1]
    blocks = -(-cols // BLOCK)
    full = torch.zeros(*v.shape[:-1], blocks * BLOCK, dtype=torch.float64, device=v.device)
    full[..., :cols] = v
    full = full.reshape(*v.shape[:-1], blocks, BLOCK)
    largest = full.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(largest))
    e = torch.where(torch.exp2(e) > largest, e - 1, e)          # where the logarithm was rounded up
    e = torch.where(torch.exp2(e + 1) <= largest, e + 1, e)     # or down
    scale = torch.exp2(torch.where(largest > 0, e - 2, -127.0).clamp(min=-127.0))
    scale = torch.where(torch.isfinite(largest), scale, math.nan)
    m = (full.abs() / scale).clamp(max=6.0)
    # the grid is 0.5 wide below 2, 1 wide up to 4 and 2 wide up to 6; round() takes ties to even
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    nearest = torch.round(m / step) * step
    return (torch.copysign(nearest, full) * scale).flatten(-2)[..., :cols]


def exact(case, seed):
    d = _inputs(case, seed)
    w = _exact_values(d["weight"])
    if case["kind"] == "store":
        return w
    x = _exact_values(d["x"])
    if case["kind"] == "linear":
        y = x @ w.t()
        return y if d["bias"] is None else y + d["bias"].double()
    ids = d["ids"]
    y = torch.zeros(*ids.shape, case["out"], dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        at = (ids == e).nonzero(as_tuple=True)
        rows = x[at[0]] if case["shared"] else x[at]
        part = rows @ w[e].t()
        y[at] = part if d["bias"] is None else part + d["bias"][e].double()
    return y
