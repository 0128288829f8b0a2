"""Linear layers in 8-bit integers against their definition in 64 bits (w8a8_cases.py says what each output may be off by), at the sizes where the
division of the work changes, with odd widths and strides, and for rows with zeros, infinities and NaN."""
import pytest
import torch

import w8a8_cases as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def w8():
    import cpmcu.w8a8 as w8a8
    return w8a8


def near(got, want, tol):
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float(((got.double() - want).abs() / tol).max()))


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 8), (2, 64), (3, 100), (5, 713), (7, 4096), (4, 4104), (2, 16384), (2, 16392), (3, 40001), (33, 2048)])
def test_integers_of_rows(w8, rows, width):
    x, _, _ = ref.make(rows, width, 1, seed=width, device="cuda")
    q, scale = w8.quantize(x)
    r, top, _ = ref.ints(x.double())
    assert torch.equal(q.double(), r)                       # exactly, ties among them
    assert torch.equal(scale, (top[:, 0] / 127).float()) or float(((scale.double() - top[:, 0] / 127).abs() / top[:, 0].clamp(min=1e-30)).max()) < 2.0 ** -30


def test_integers_at_ties_and_edges(w8):
    big, tiny = float(torch.finfo(BF16).max), 2.0 ** -133
    rows = [[254.0, 1.0, 3.0, -5.0, 253.0, -1.0, 0.0, 127.0],        # ties to even
            [0.0] * 8,                                                # zeros
            [big, -big, big / 2, 1.0, 0.0, 2.0 ** 120, -1.0, big / 4],
            [tiny, -tiny, 0.0, tiny, 0.0, 0.0, 0.0, 0.0],
            [127 * tiny, 3 * tiny, -64 * tiny, 0.0, tiny, 0.0, 0.0, 0.0],
            [1.0, 2.0 ** -133, -(2.0 ** -8), 0.0, 0.5, 0.25, -0.125, 1.0]]
    x = torch.tensor(rows, dtype=BF16, device="cuda")
    q, scale = w8.quantize(x)
    r, top, _ = ref.ints(x.double())
    assert torch.equal(q.double(), r)
    assert float((scale.double() - top[:, 0] / 127).abs().max() / big) < 1e-9
    assert scale[1] == 0
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = x.clone()
        y[0, 3] = bad
        q2, s2 = w8.quantize(y)
        assert bool(torch.isnan(s2[0])) and not bool(q2[0].any())
        assert torch.equal(q2[1:], q[1:]) and torch.equal(s2[1:], scale[1:])


SIZES = [(1, 64, 64), (1, 1, 1), (1, 4096, 512), (1, 1000, 333), (1, 16384, 130), (1, 50000, 20), (1, 128, 8192),
         (2, 64, 64), (2, 1, 1), (3, 129, 127), (16, 1024, 4096), (17, 2048, 640), (60, 4096, 384), (64, 512, 20000), (64, 704, 1000),
         (65, 512, 256), (100, 4096, 1024), (128, 256, 4736), (129, 1024, 512), (256, 2048, 300), (257, 512, 512), (300, 1024, 384),
         (333, 713, 1001), (512, 4096, 2048), (700, 256, 5000), (1025, 640, 768), (40, 16384, 256), (2, 131072, 40)]


@pytest.mark.parametrize("rows,width,out", SIZES)
def test_linear(w8, rows, width, out):
    x, q, s = ref.make(rows, width, out, seed=rows + width + out, device="cuda")
    y = w8.linear(x, w8.PackedLinear(q, s))
    want, tol, _ = ref.linear(x, q, s)
    near(y, want, tol)


@pytest.mark.parametrize("rows,width,out", [(1, 4096, 640), (1, 999, 77), (2, 1024, 256), (60, 4096, 512), (60, 771, 130), (300, 2048, 512), (5, 20000, 64), (1, 60000, 16)])
@pytest.mark.parametrize("delta", [None, 1.0, 0.25])
def test_linear_behind_a_norm(w8, rows, width, out, delta):
    x, q, s = ref.make(rows, width, out, seed=rows + width, device="cuda")
    g = torch.Generator("cuda").manual_seed(5)
    w = (1 + 0.3 * torch.randn(width, generator=g, device="cuda")).to(BF16)
    bias = torch.randn(out, generator=g, device="cuda").to(BF16)
    norm = {"norm_weight": w, "eps": 1e-5}
    if delta is not None:
        norm |= {"delta": torch.randn(rows, width, generator=g, device="cuda").to(BF16), "delta_scale": delta}
    got = w8.linear(x, w8.PackedLinear(q, s), bias=bias, **norm)
    if delta is not None:
        got, total = got
        # the sum is rounded to fp32 and to bf16: one bf16 step where the first rounding meets a border of the second
        t = ref.residual(x, norm["delta"], delta)
        assert float(((total.double() - t.double()).abs() / t.double().abs().clamp(min=1e-30)).max()) <= 2.0 ** -7
        assert float((total != t).float().mean()) < 1e-3
        norm = {"norm_weight": w, "eps": 1e-5}
        want, tol, _ = ref.linear(total, q, s, bias, **norm)
    else:
        want, tol, _ = ref.linear(x, q, s, bias, **norm)
    near(got, want, tol)


def make_ffn(rows, width, inter, seed):
    x, gate, gs = ref.make(rows, width, inter, seed, "cuda")
    _, up, us = ref.make(1, width, inter, seed + 1, "cuda")
    _, down, ds = ref.make(1, inter, width, seed + 2, "cuda")
    g = 1 / width ** 0.5
    return x, (gate, gs * g), (up, us * g), (down, ds)


@pytest.mark.parametrize("rows,width,inter", [(1, 64, 64), (1, 1, 1), (1, 4096, 1024), (1, 1000, 333), (2, 128, 64), (3, 100, 65), (16, 512, 704), (60, 4096, 1024),
                                              (60, 512, 9472), (64, 256, 640), (65, 512, 512), (200, 1024, 1000), (257, 512, 512), (300, 1024, 320), (600, 2048, 2048)])
@pytest.mark.parametrize("norm", [False, True])
def test_gated_ffn(w8, rows, width, inter, norm):
    x, gate, up, down = make_ffn(rows, width, inter, rows + inter)
    more = {}
    if norm:
        more = {"norm_weight": torch.linspace(0.5, 1.5, width, device="cuda").to(BF16), "delta": x.flip(0).contiguous(), "delta_scale": 0.5}
    got = w8.gated_ffn(x, w8.PackedGateUp(*gate, *up), w8.PackedLinear(*down), **more)
    if norm:
        got, total = got
        more = {"norm_weight": more["norm_weight"]}
        x = total
    want, tol, _ = ref.ffn(x, *gate, *up, *down, **more)
    near(got, want, tol)
