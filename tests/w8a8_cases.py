"""Plain 64-bit forms of the 8-bit linear layers, with what each output may be off by, for the GPU and the CPU tests."""
import torch

F64 = torch.float64


def ints(v):
    """Rows of v (64 bits) to integers: round(127 v / max|v|), half to even; their largest magnitude; where 127 v / max lies within 2^-14 of a border."""
    top = v.abs().amax(1, keepdim=True)
    r = torch.where(top > 0, 127 * v / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(v))
    near = ((r - r.floor()) - 0.5).abs() < 2.0 ** -14
    return r.round(), top, near


def residual(x, delta, delta_scale):
    return (x.double() + delta.double() * float(torch.tensor(delta_scale, dtype=torch.float32))).float().to(torch.bfloat16)


def source(x, norm_weight=None, eps=1e-5, delta=None, delta_scale=1.0):
    """(v, f, total)"""
    if norm_weight is None:
        return x.double(), torch.ones(x.shape[0], 1, dtype=F64, device=x.device), None
    t = x if delta is None else residual(x, delta, delta_scale)
    td = t.double()
    f = 1 / torch.sqrt((td * td).mean(1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32)))
    return td * norm_weight.double(), f, (t if delta is not None else None)


def product(v, f, q, scale, bias=None):
    """(y, what rounding to bf16 and the fp32 steps before it may change).  fp32 steps: the integer sum, the token's scale (a quotient, a norm over at
    most 131072 squares in runs of 128 and a tree, a root and two products), the channel's and the bias: fewer than 256 roundings of
    2^-24 relative to the summands."""
    r, top, _ = ints(v)
    p = (r @ q.double().t()) * (top / 127 * f) * scale.double()
    y = p if bias is None else p + bias.double()
    slack = p.abs() * 2.0 ** -16 + (0 if bias is None else bias.double().abs() * 2.0 ** -16)
    return y, y.abs() * 2.0 ** -8 + slack * (1 + 2.0 ** -8) + 1e-38


def linear(x, q, scale, bias=None, **norm):
    v, f, total = source(x, **norm)
    return (*product(v, f, q, scale, bias), total)


def ffn(x, gate, gate_scale, up, up_scale, down, down_scale, **norm):
    """The activations are fp32 sums of products with 2^-16 relative error each; an element within 2^-14 of a border of its 8-bit integer may round the
    other way, and changes the output by its step times its weight."""
    v, f, total = source(x, **norm)
    g, _ = product(v, f, gate, gate_scale)
    u, _ = product(v, f, up, up_scale)
    h = g * torch.sigmoid(g) * u
    # silu's relative error from that of g: at most (1 + |g|) times it; such activations are not near a border by more than they move
    r, top, _ = ints(h)
    ratio = torch.where(top > 0, 127 * h / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(h))
    moved = ratio.abs() * (3 + g.abs()) * 2.0 ** -16 + 2.0 ** -18
    near = ((ratio - ratio.floor()) - 0.5).abs() < moved
    y, tol = product(h, torch.ones_like(f), down, down_scale)
    flips = (near.double() @ down.double().abs().t()) * (top / 127) * down_scale.double()
    spread = (g.abs().amax(1, keepdim=True) + 4) * 2.0 ** -16      # of the scale
    return y, tol + flips + y.abs() * spread, total


def make(rows, width, out, seed=0, device="cpu", loud=True):
    g = torch.Generator(device).manual_seed(seed)
    x = torch.randn(rows, width, generator=g, device=device)
    if loud:
        x = x * torch.where(torch.rand(width, generator=g, device=device) < 0.02, 10.0, 1.0)
    q = torch.randint(-128, 128, (out, width), generator=g, device=device).to(torch.int8)
    scale = torch.rand(out, generator=g, device=device) * 2e-2 + 1e-4
    return x.to(torch.bfloat16), q, scale
