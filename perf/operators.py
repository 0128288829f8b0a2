"""The 8-bit layer operators and the rotation of fused q/k/v rows, as cases that can be timed and compared.

  linear     y = (q W^T) * (scale of the token) * (scale of the channel) + bias: rows of bf16 are rounded to 8-bit integers
             with one scale each, alone or as the RMS norm of x + c * delta, and multiplied with 8-bit weights
  gated_ffn  the same for a whole feed-forward block: W_down of silu(gate) * up, whose rows become 8-bit integers again
  rotary     queries and keys of fused q/k/v rows are rotated, keys and values go to their cache rows

Weights are what an 8-bit checkpoint holds: int8 values and one fp32 scale for each output channel.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F64, BF16, I8 = torch.float32, torch.float64, torch.bfloat16, torch.int8
EPS = 1e-5


# ------------------------------------------------------------------------------------------------ cases
def _linear(rows, width, out, norm=False, bias=False, pad=0, gain=1.0):
    """pad: columns of x's buffer behind its rows (a view of a wider tensor); gain: factor of delta in the residual sum."""
    return {"op": "linear", "rows": rows, "width": width, "out": out, "norm": norm, "bias": bias, "pad": pad, "gain": gain}


def _ffn(rows, width, inter, norm=False, gain=1.0):
    return {"op": "gated_ffn", "rows": rows, "width": width, "inter": inter, "norm": norm, "gain": gain}


def _rotary(rows, heads, kv_heads, dim, rot, interleaved, first, theta, stretch=1.0, factor=1.0):
    """first: position of the first row; theta, stretch: frequencies theta^(-2 i / rot) / stretch; factor: of sines and cosines."""
    return {"op": "rotary", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "interleaved": interleaved,
            "first": first, "theta": theta, "stretch": stretch, "factor": factor}


def listed():
    return [
        # attention output of one decoded token of the 8B model: the smallest product, latency counts
        dict(_linear(1, 4096, 4096), name="linear_token_o"),
        # q, k and v of one token, behind its residual sum and norm
        dict(_linear(1, 4096, 4608, norm=True), name="linear_token_qkv"),
        # q, k and v of a 60-node draft tree of the 8B model
        dict(_linear(60, 4096, 4608, norm=True, gain=0.25), name="linear_tree_qkv"),
        # the longest sums of a tree's verify pass: the down projection
        dict(_linear(60, 16384, 4096), name="linear_tree_down"),
        # widths that no tile divides, a bias, and rows of a wider tensor
        dict(_linear(333, 713, 1001, bias=True, pad=5), name="linear_ragged"),
        # a prompt of 4096 tokens through the down projection
        dict(_linear(4096, 16384, 4096), name="linear_prompt_down"),
        # feed-forward block of one token: 200 MB of weights
        dict(_ffn(1, 4096, 16384, norm=True), name="ffn_token"),
        # of a draft tree
        dict(_ffn(60, 4096, 16384), name="ffn_tree"),
        # of a prompt
        dict(_ffn(4096, 4096, 16384, norm=True, gain=0.25), name="ffn_prompt"),
        # rotation of a draft tree's rows behind 4096 tokens
        dict(_rotary(60, 32, 2, 128, 128, False, 4096, 10000.0), name="rotary_tree"),
        # a long document's chunk, positions far beyond those of training: stretched frequencies and their factor
        dict(_rotary(8192, 32, 8, 128, 128, False, 900000, 500000.0, 8.0, 1.2079), name="rotary_far"),
        # interleaved pairs on the first quarter of heads that are no power of two
        dict(_rotary(2000, 15, 5, 80, 20, True, 17, 10000.0), name="rotary_part"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated_ffn", "gated_ffn", "rotary"])
    if op == "rotary":
        dim = rng.choice([32, 64, 72, 80, 96, 112, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4]) // 2 * 2
        kv_heads = rng.randint(1, 8)
        heads = kv_heads * rng.randint(1, 8)
        rows = _spread(rng, 1, max(1, 8192 * 6144 // ((heads + 2 * kv_heads) * dim)))
        return _rotary(min(rows, 8192), heads, kv_heads, dim, rot, rng.random() < 0.5, _spread(rng, 1, 1000000) - 1,
                       rng.choice([10000.0, 500000.0, 1000000.0]), rng.choice([1.0, 1.0, 4.0, 8.0, 32.0]), rng.choice([1.0, rng.uniform(0.8, 1.4)]))
    rows, width, out = _spread(rng, 1, 4096), _spread(rng, 64, 16384), _spread(rng, 64, 16384)
    if rng.random() < 0.5:   # half of the widths are ones that models have
        width, out = max(64, width // 64 * 64), max(64, out // 64 * 64)
    norm, gain = rng.random() < 0.5, rng.choice([1.0, rng.uniform(0.1, 1.5)])
    if op == "linear":
        return _linear(rows, width, out, norm, rng.random() < 0.3, 0 if norm else rng.choice([0, 0, rng.randint(1, 64)]), gain)
    most = 4096 * 4096 * 16384
    return _ffn(max(1, min(rows, most // (width * out))), width, out, norm, gain)


# ------------------------------------------------------------------------------------------------ inputs
def _rows(g, rows, width):
    """Hidden states: a normal spread with a few channels that are ten times as large, as trained models have."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    loud = torch.rand(width, generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 10.0, 1.0)).to(BF16)


def _weight(g, out, width):
    """A channel's largest value is 127 in most checkpoints; scales are those of weights with a spread of width^-1/2."""
    q = (torch.randn(out, width, generator=g, device="cuda") * 36).round().clamp(-127, 127).to(I8)
    scale = torch.exp(torch.randn(out, generator=g, device="cuda") * 0.2) / (36 * math.sqrt(width))
    return q, scale


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "rotary":
        n = case["heads"] + 2 * case["kv_heads"]
        s["qkv"] = torch.randn(case["rows"], n * case["dim"], generator=g, device="cuda").to(BF16)
        i = torch.arange(0, case["rot"], 2, dtype=F64, device="cuda")
        s["inv_freq"] = (case["theta"] ** (-i / case["rot"]) / case["stretch"]).to(F32)
        s["pos"] = torch.arange(case["rows"], dtype=torch.int32, device="cuda") + case["first"]
        first = int(torch.randint(0, 64, (1,), generator=g, device="cuda"))
        s["slots"] = torch.arange(case["rows"], dtype=torch.int32, device="cuda") + first
        kv = case["kv_heads"] * case["dim"]
        s["k_cache"] = torch.randn(case["rows"] + 64, kv, generator=g, device="cuda").to(BF16)
        s["v_cache"] = torch.randn(case["rows"] + 64, kv, generator=g, device="cuda").to(BF16)
        return s
    rows, width = case["rows"], case["width"]
    s["x"] = _rows(g, rows, width + case.get("pad", 0))[:, :width]
    s["norm_weight"] = s["delta"] = s["bias_values"] = None
    if case["norm"]:
        s["delta"] = _rows(g, rows, width)
        s["norm_weight"] = (1 + 0.3 * torch.randn(width, generator=g, device="cuda")).to(BF16)
    if case.get("bias"):
        s["bias_values"] = torch.randn(case["out"], generator=g, device="cuda").to(BF16)
    if case["op"] == "linear":
        s["weights"] = [_weight(g, case["out"], width)]
    else:
        s["weights"] = [_weight(g, case["inter"], width), _weight(g, case["inter"], width), _weight(g, width, case["inter"])]
    if own:
        w8a8 = _package("w8a8")
        w = s["weights"]
        s["packed"] = [w8a8.PackedLinear(*w[0])] if case["op"] == "linear" else [w8a8.PackedGateUp(*w[0], *w[1]), w8a8.PackedLinear(*w[2])]
    return s


def _package(name):
    import importlib
    at = os.path.join(ROOT, "cpm.cu_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    return importlib.import_module("cpmcu." + name)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "rotary":
        return _plain_rotary(s)
    v, factor, total = _plain_norm(s["x"], s["delta"], s["norm_weight"], s["gain"])
    if s["op"] == "linear":
        y = _plain_product(*_plain_round(v, factor), *s["weights"][0])
        y = (y if s["bias_values"] is None else y + s["bias_values"].float()).to(BF16)
    else:
        q, scale = _plain_round(v, factor)
        gate, up = (_plain_product(q, scale, *w) for w in s["weights"][:2])
        y = _plain_product(*_plain_round(gate / (1 + torch.exp(-gate)) * up, 1.0), *s["weights"][2]).to(BF16)
    return y if total is None else (y, total)


def _run_own(s):
    if s["op"] == "rotary":
        q = _package("rotary").append(s["qkv"], s["heads"], s["kv_heads"], s["dim"], s["inv_freq"], s["pos"], s["k_cache"], s["v_cache"],
                                      s["slots"], rot_dims=s["rot"], interleaved=s["interleaved"], factor=s["factor"])
        return q, s["k_cache"], s["v_cache"]
    w8a8 = _package("w8a8")
    norm = {} if s["delta"] is None else {"norm_weight": s["norm_weight"], "eps": EPS, "delta": s["delta"], "delta_scale": s["gain"]}
    if s["op"] == "linear":
        return w8a8.linear(s["x"], s["packed"][0], bias=s["bias_values"], **norm)
    return w8a8.gated_ffn(s["x"], *s["packed"], **norm)


def _plain_norm(x, delta, weight, gain):
    """(v, f, total): the row that is to be rounded is v * f.  A norm's factor is the same for a whole row, so that it does not
    change which 8-bit integers the row becomes: v is total * weight, exactly, and f multiplies the scale."""
    if weight is None:
        return x.float(), 1.0, None
    total = (x.double() + delta.double() * gain).float().to(BF16)
    t = total.float()
    return t * weight.float(), torch.rsqrt(t.square().mean(-1) + EPS), total


def _plain_round(v, factor):
    """Integers in [-127, 127], to nearest and to even at a tie (64 bits: values next to a border), and the row's scale."""
    top = v.abs().amax(-1)
    q = torch.round(v.double() * 127 / torch.where(top > 0, top, 1.0).double()[:, None]).float()
    return q, top / 127 * factor


def _plain_product(q, scale, wq, wscale):
    return (q @ wq.float().t()) * scale[:, None] * wscale


def _plain_rotary(s):
    rows, dim, rot, heads, kv = s["rows"], s["dim"], s["rot"], s["heads"], s["kv_heads"]
    x = s["qkv"].float().view(rows, heads + 2 * kv, dim)
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()   # 64 bits: angles of far positions
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    part = x[:, : heads + kv, :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if s["interleaved"] else (part[..., : rot // 2], part[..., rot // 2:])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((lo, hi), -1).flatten(-2) if s["interleaved"] else torch.cat((lo, hi), -1)
    turned = torch.cat((turned, x[:, : heads + kv, rot:]), -1).to(BF16)
    at = s["slots"].long()
    s["k_cache"][at] = turned[:, heads:].reshape(rows, -1)
    s["v_cache"][at] = s["qkv"].view(rows, heads + 2 * kv, dim)[:, heads + kv:].reshape(rows, -1)
    return turned[:, :heads].reshape(rows, -1), s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "rotary":
        n, dim = case["heads"] + 2 * case["kv_heads"], case["dim"]
        # every row in and out, positions, slots; six operations for a pair of values
        return {"bytes": case["rows"] * (4 * n * dim + 8) + 2 * case["rot"],
                "flops": 3 * case["rows"] * (case["heads"] + case["kv_heads"]) * case["rot"]}
    rows, width = case["rows"], case["width"]
    out = case["out"] if case["op"] == "linear" else width
    moved = 2 * rows * (width + out) + (4 * rows * width + 2 * width if case["norm"] else 0)   # x, y; delta, total, norm weights
    if case["op"] == "linear":
        weights, n = width * out, out
    else:
        weights, n = 3 * width * case["inter"], 2 * case["inter"] + width
    return {"bytes": moved + weights + 4 * n + (2 * out if case.get("bias") else 0), "flops": 2 * rows * weights}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    if case["op"] == "rotary":
        return _exact_rotary(prepare(case, seed))
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    x = s["x"].to(F64)
    total = None
    if s["delta"] is not None:
        # the residual stream is held in bf16: the sum is rounded to it before anything else is made of it
        total = (x + s["delta"].to(F64) * s["gain"]).to(BF16)
        x = total.to(F64)
        norm = torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS)
        x, divisor = x * s["norm_weight"].to(F64), norm
    else:
        divisor = torch.ones_like(x[:, :1])
    if case["op"] == "linear":
        y = _exact_linear(x, divisor, *s["weights"][0])
        if s["bias_values"] is not None:
            y += s["bias_values"].to(F64)
    else:
        gate, up = (_exact_linear(x, divisor, *w) for w in s["weights"][:2])
        h = gate * torch.sigmoid(gate) * up
        y = _exact_linear(h, torch.ones_like(divisor), *s["weights"][2])
    return y if total is None else (y, total.to(F64))


def _exact_linear(x, divisor, wq, wscale):
    """sum over k of (integer of x / divisor) * step * wq * wscale, where step is 1/127 of the row's largest magnitude."""
    largest = torch.linalg.vector_norm(x, ord=math.inf, dim=1, keepdim=True)
    ratio = x * (127 / 1) / largest.clamp(min=torch.finfo(F64).tiny)
    low = torch.floor(ratio)
    rest = ratio - low
    integer = low + ((rest > 0.5) | ((rest == 0.5) & (low.remainder(2) == 1)))
    y = torch.einsum("mk,nk->mn", integer, wq.to(F64))
    return y * (largest / divisor / 127) * wscale.to(F64)[None, :]


def _exact_rotary(s):
    rows, dim, rot = s["rows"], s["dim"], s["rot"]
    turn = torch.polar(torch.full((), s["factor"], dtype=F64, device="cuda"),
                       s["pos"].to(F64)[:, None] * s["inv_freq"].to(F64)[None, :])[:, None, :]     # complex numbers
    x = s["qkv"].to(F64).unflatten(1, (-1, dim))
    pairs = torch.arange(rot, device="cuda").view(-1, 2) if s["interleaved"] else torch.arange(rot, device="cuda").view(2, -1).t()
    qk = x[:, : s["heads"] + s["kv_heads"]].clone()
    z = torch.complex(qk[..., pairs[:, 0]], qk[..., pairs[:, 1]]) * turn
    qk[..., pairs[:, 0]], qk[..., pairs[:, 1]] = z.real, z.imag
    k_cache, v_cache = s["k_cache"].to(F64), s["v_cache"].to(F64)
    first = int(s["slots"][0])
    k_cache[first: first + rows] = qk[:, s["heads"]:].flatten(1)
    v_cache[first: first + rows] = x[:, s["heads"] + s["kv_heads"]:].flatten(1)
    return qk[:, : s["heads"]].flatten(1), k_cache, v_cache
