"""Linear layers in 8-bit integers against their definition in 64 bits (w8a8_cases.py says what each output may be off by), at the sizes where the
division of the work changes, with odd widths and strides, and for rows with zeros, infinities and NaN."""
import pytest
import torch

import cpmcu.C as C
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


@pytest.mark.parametrize("rows", [1, 40])
def test_integers_behind_a_norm(w8, rows):
    """The identity as weights shows the integers: exactly those of t * weight, half-way values among them (the half of a row's largest magnitude, and
    rows whose largest has the mantissa 254, which have many)."""
    width = 512
    eye = w8.PackedLinear(torch.eye(width, dtype=torch.int8, device="cuda"), torch.ones(width, device="cuda"))
    g = torch.Generator("cuda").manual_seed(rows)
    for top, weight in ((254.0, 1.0), (3.0, 1.0), (1.28125, 1.953125), (1.7, 0.6), (254.0, 1.5), (127.0, 2.540625)):
        x = torch.randint(-127, 128, (rows, width), generator=g, device="cuda") * torch.tensor(top / 127 / 8, device="cuda")
        x[:, 0], x[:, 1], x[:, 2], x[:, 3] = top, top / 2, -top / 2, -top / 4
        x = x.to(BF16)
        w = torch.full((width,), weight, dtype=BF16, device="cuda")
        w[200:] = (0.5 + torch.rand(width - 200, generator=g, device="cuda")).to(BF16) * weight / 2
        r, t, _ = ref.ints(x.double() * w.double())
        y = w8.linear(x, eye, norm_weight=w)
        f = 1 / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + float(torch.tensor(1e-5)))
        assert torch.equal((y.double() / (t / 127 * f)).round(), r), (top, weight)
        assert bool((w8.linear(x, eye).double() / (x.double().abs().amax(1, keepdim=True) / 127)).round().eq(ref.ints(x.double())[0]).all())


SIZES = [(1, 64, 64), (1, 1, 1), (1, 4096, 512), (1, 1000, 333), (1, 16384, 130), (1, 50000, 20), (1, 128, 8192),
         (2, 64, 64), (2, 1, 1), (3, 129, 127), (16, 1024, 4096), (17, 2048, 640), (60, 4096, 384), (64, 512, 20000), (64, 704, 1000),
         (65, 512, 256), (100, 4096, 1024), (128, 256, 4736), (129, 1024, 512), (256, 2048, 300), (257, 512, 512), (300, 1024, 384),
         (333, 713, 1001), (512, 4096, 2048), (700, 256, 5000), (1025, 640, 768), (40, 16384, 256), (2, 131072, 40), (60, 256, 19200), (17, 384, 38016), (3, 256, 19100), (64, 512, 40000)]


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
                                              (60, 512, 9472), (60, 256, 9536), (5, 128, 9530), (30, 256, 19200), (64, 256, 640), (65, 512, 512), (200, 1024, 1000), (257, 512, 512), (300, 1024, 320), (600, 2048, 2048)])
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


# ------------------------------------------------------------------------------------------------ rows with nothing, infinities and NaN; strides; types of calls
@pytest.mark.parametrize("rows", [1, 5, 40, 100, 300])
def test_rows_of_zeros_infinities_and_nan(w8, rows):
    x, q, s = ref.make(rows, 512, 300, seed=rows, device="cuda")
    bias = torch.randn(300, device="cuda").to(BF16)
    packed = w8.PackedLinear(q, s)
    gate_up, down = w8.PackedGateUp(q, s, q.flip(0).contiguous(), s), w8.PackedLinear(*ref.make(1, 300, 512, 1, "cuda")[1:])
    clean, clean_ffn = w8.linear(x, packed, bias=bias), w8.gated_ffn(x, gate_up, down)
    for value in (0.0, float("inf"), float("-inf"), float("nan")):
        bad = x.clone()
        at = rows // 2
        if value == 0.0:
            bad[at] = 0
        else:
            bad[at, 100] = value
        rest = torch.arange(rows, device="cuda") != at
        y, f = w8.linear(bad, packed, bias=bias), w8.gated_ffn(bad, gate_up, down)
        assert torch.equal(y[rest], clean[rest]) and torch.equal(f[rest], clean_ffn[rest])     # no other row is touched
        if value == 0.0:
            assert torch.equal(y[at], bias) and not bool(f[at].any())
        else:
            assert bool(torch.isnan(y[at]).all()) and bool(torch.isnan(f[at]).all())
        g = torch.ones(512, dtype=BF16, device="cuda")
        for eps in (1e-5, 0.0):
            n = w8.linear(bad, packed, bias=bias, norm_weight=g, eps=eps)[at]
            assert torch.equal(n, bias) if value == 0.0 else bool(torch.isnan(n).all())


@pytest.mark.parametrize("rows,width,out", [(1, 257, 65), (1, 256, 64), (7, 257, 129), (33, 264, 200), (300, 130, 131)])
def test_views_of_wider_matrices(w8, rows, width, out):
    wide, q, s = ref.make(rows, width + 13, out, seed=2, device="cuda")
    q = q[:, :width].contiguous()
    for left in (0, 5, 8):
        x = wide[:, left:left + width]
        held = torch.full((rows + 2, out + 11), 7.0, dtype=BF16, device="cuda")
        y = w8.linear(x, w8.PackedLinear(q, s), out=held[1:1 + rows, 3:3 + out])
        want, tol, _ = ref.linear(x, q, s)
        near(y, want, tol)
        edge = torch.ones_like(held, dtype=torch.bool)
        edge[1:1 + rows, 3:3 + out] = False
        assert bool((held[edge] == 7).all())                    # what lies around the outputs
    # input and output columns of one matrix
    both = torch.cat((wide[:, :width], torch.zeros(rows, out, dtype=BF16, device="cuda")), 1)
    y = w8.linear(both[:, :width], w8.PackedLinear(q, s), out=both[:, width:])
    assert torch.equal(y, w8.linear(wide[:, :width], w8.PackedLinear(q, s)))


def test_empty_batches(w8):
    _, q, s = ref.make(1, 64, 32, device="cuda")
    x = torch.empty(0, 64, dtype=BF16, device="cuda")
    assert w8.linear(x, w8.PackedLinear(q, s)).shape == (0, 32)
    y, t = w8.linear(x, w8.PackedLinear(q, s), norm_weight=torch.ones(64, dtype=BF16, device="cuda"), delta=x)
    assert y.shape == (0, 32) and t.shape == (0, 64)
    _, d, ds = ref.make(1, 32, 64, device="cuda")
    assert w8.gated_ffn(x, w8.PackedGateUp(q, s, q, s), w8.PackedLinear(d, ds)).shape == (0, 64)
    assert w8.quantize(x)[0].shape == (0, 64)


def test_weights_from_bf16(w8):
    w = torch.randn(200, 333, device="cuda").to(BF16)
    q, s = w8.quantize(w)
    x, _, _ = ref.make(9, 333, 1, device="cuda")
    assert torch.equal(w8.linear(x, w8.PackedLinear.from_bf16(w)), w8.linear(x, w8.PackedLinear(q, s)))
    assert float(((q * s[:, None]).double() - w.double()).abs().max()) <= float(s.max()) * 0.5001


@pytest.mark.parametrize("rows", [1, 2, 60, 129, 600])
def test_calls_repeat_to_the_bit_and_replay_in_graphs(w8, rows):
    width, out = 2048, 1152
    x, q, s = ref.make(rows, width, out, seed=rows, device="cuda")
    packed = w8.PackedLinear(q, s)
    norm = {"norm_weight": torch.linspace(0.5, 2, width, device="cuda").to(BF16), "delta": x.flip(0).contiguous()}
    _, gate, up, down = make_ffn(1, width, 704, 4)
    gate_up, down = w8.PackedGateUp(*gate, *up), w8.PackedLinear(*down)

    def calls():
        y, t = w8.linear(x, packed, **norm)
        return y, t, w8.gated_ffn(x, gate_up, down)
    first = calls()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(calls(), first))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            kept = calls()
    x.copy_(x.roll(1, 1))                  # new values in the captured input
    norm["delta"].copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, calls()))


def test_calls_on_several_streams_at_once(w8):
    """Products that fill the device, cut tiles among them, beside one another: each waits for none of the others' CTAs."""
    work = []
    for i, (rows, width, out) in enumerate([(4096, 2048, 1280), (128, 16384, 1024), (60, 4096, 4608), (1, 8192, 8192), (700, 4096, 2304)]):
        x, q, s = ref.make(rows, width, out, seed=i, device="cuda")
        work.append((x, w8.PackedLinear(q, s)))
    want = [w8.linear(x, p) for x, p in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[] for _ in work]
    for _ in range(20):
        for i, (s, (x, p)) in enumerate(zip(streams, work)):
            with torch.cuda.stream(s):
                got[i].append(w8.linear(x, p))
    torch.cuda.synchronize()
    import cpmcu.C as C
    for s in streams:
        C.stream_check(s.cuda_stream)
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)


def test_calls_from_several_threads(w8):
    import threading
    x, q, s = ref.make(64, 1024, 512, seed=1, device="cuda")
    packed = w8.PackedLinear(q, s)
    want = w8.linear(x, packed)
    torch.cuda.synchronize()
    failed = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y = w8.linear(x, packed)
            torch.cuda.current_stream().synchronize()
            if not torch.equal(y, want):
                failed.append(1)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_offsets_beyond_32_bits(w8):
    """Inputs, integers, activations and outputs of more than 2^31 elements: the last rows are right."""
    rows, width = 70000, 33000
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    last, q, s = ref.make(300, width, 96, seed=1, device="cuda")
    x[-300:] = last
    y = w8.linear(x, w8.PackedLinear(q, s))
    want, tol, _ = ref.linear(last, q, s)
    near(y[-300:], want, tol)
    assert not bool(y[:-300].any())
    del x, y
    rows, width, out = 70000, 64, 33000
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    last, q, s = ref.make(300, width, out, seed=1, device="cuda")
    x[-300:] = last
    y = w8.linear(x, w8.PackedLinear(q, s))
    want, tol, _ = ref.linear(last, q, s)
    near(y[-300:], want, tol)
    assert not bool(y[:-300].any())
    del y
    _, up, us = ref.make(1, width, out, seed=2, device="cuda")
    _, d, ds = ref.make(1, out, width, seed=3, device="cuda")
    f = w8.gated_ffn(x, w8.PackedGateUp(q, s, up, us), w8.PackedLinear(d, ds))
    want, tol, _ = ref.ffn(last, q, s, up, us, d, ds)
    near(f[-300:], want, tol)
    assert not bool(f[:-300].any())


def test_refusals_on_the_gpu(w8):
    x, q, s = ref.make(4, 64, 32, device="cuda")
    p = w8.PackedLinear(q, s)
    with pytest.raises(ValueError, match="x must be"):
        w8.linear(x.float(), p)
    with pytest.raises(ValueError, match="x must be"):
        w8.linear(x[:, :63], p)
    with pytest.raises(ValueError, match="x must be"):
        w8.linear(x.cpu(), p)
    with pytest.raises(ValueError, match="matrix"):
        w8.linear(x[0], p)
    with pytest.raises(ValueError, match="consecutive"):
        w8.linear(torch.zeros(64, 4, dtype=BF16, device="cuda").t(), p)
    with pytest.raises(ValueError, match="consecutive"):
        w8.linear(x[:1].expand(4, 64), p)
    with pytest.raises(ValueError, match="bias"):
        w8.linear(x, p, bias=torch.zeros(31, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError, match="norm_weight"):
        w8.linear(x, p, delta=x)
    with pytest.raises(ValueError, match="delta"):
        w8.linear(x, p, norm_weight=torch.ones(64, dtype=BF16, device="cuda"), delta=x[:3])
    with pytest.raises(ValueError, match="out"):
        w8.linear(x, p, out=torch.zeros(4, 33, dtype=BF16, device="cuda"))
    square = w8.PackedLinear(*ref.make(1, 64, 64, device="cuda")[1:])
    with pytest.raises(RuntimeError, match="must not overlap"):
        w8.linear(x, square, out=x)
    with pytest.raises(ValueError, match="down must be"):
        w8.gated_ffn(x, w8.PackedGateUp(q, s, q, s), p)
    with pytest.raises(ValueError, match="scale"):
        w8.PackedLinear(q, s[:-1])
    with pytest.raises(ValueError, match="131072"):
        w8.PackedLinear(torch.zeros(1, 131073, dtype=torch.int8, device="cuda"), s[:1])


@pytest.mark.parametrize("other", ["x", "y", "bias", "norm", "delta", "total", "packed"])
@pytest.mark.parametrize("ffn", [False, True])
def test_workspace_apart(other, ffn):
    """A workspace that shares memory with what the call reads or writes is refused, before any launch; next to it is fine."""
    rows, k, n = 4, 64, 64
    lib = C.load()
    size = lib.cpmcu_w8a8_workspace_bytes(rows, n, k, 128 if ffn else 0)
    assert size > 0
    packed = [lib.cpmcu_w8a8_packed_bytes(*s) for s in (((128, 64, 1), (64, 128, 0)) if ffn else ((n, k, 0),))]
    pool = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    at = (pool.data_ptr() + 255) // 256 * 256
    place, ends = {}, {}
    for name, bytes_ in [("ws", size), ("x", 2 * rows * k), ("y", 2 * rows * n), ("bias", 2 * n), ("norm", 2 * k), ("delta", 2 * rows * k), ("total", 2 * rows * k),
                         ("packed", packed[-1]), ("up", packed[0])]:
        place[name], ends[name] = at, at + bytes_
        at = (at + bytes_ + 255) // 256 * 256
    assert at <= pool.data_ptr() + pool.numel()

    def call(p, s):
        if ffn:
            C.call("cpmcu_w8a8_ffn", p["x"], k, p["up"], p["packed"], p["norm"], 1e-5, p["delta"], 1.0, p["total"], p["y"], n, rows, k, 128, p["ws"], s, None)
        else:
            C.call("cpmcu_w8a8_linear", p["x"], k, p["packed"], p["bias"], p["norm"], 1e-5, p["delta"], 1.0, p["total"], p["y"], n, rows, n, k, p["ws"], s, None)

    call(place, size)
    if not (ffn and other == "bias"):
        for ws in (place[other], (ends[other] - 1) // 256 * 256):   # the first and the last of its bytes
            with pytest.raises(RuntimeError, match="the workspace must not overlap"):
                call({**place, "ws": ws}, 1 << 19)
    with pytest.raises(RuntimeError, match=f"needs {size} bytes"):
        call(place, size - 1)
    torch.cuda.synchronize()


# Sizes at which clusters of 2, 3, 4 and 8 CTAs have token tiles of 16, 32, 64 and 128, several of them, the last one partly filled or with a single token, and
# columns that the CTAs do not share evenly.
TILED = [(95, 2624, 256), (97, 1100, 130), (26, 7168, 256), (17, 2500, 200), (60, 16384, 512), (60, 4096, 2048), (60, 4096, 4096), (31, 2000, 700), (200, 1024, 1024),
         (225, 1000, 500), (300, 4096, 1024), (257, 4096, 1024), (290, 5760, 200), (128, 8192, 4096), (127, 6400, 4000), (65, 4096, 4096), (129, 9000, 128), (513, 300, 260),
         (66, 1000, 1500), (128, 16384, 1500), (200, 16384, 1100), (1000, 2048, 128)]


@pytest.mark.parametrize("rows,width,out", TILED)
def test_linear_of_several_token_tiles(w8, rows, width, out):
    x, q, s = ref.make(rows, width, out, seed=rows + width + out, device="cuda")
    bias = torch.randn(out, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(BF16)
    wide = torch.full((rows + 1, out + 3), 7.0, dtype=BF16, device="cuda")
    y = wide[:rows, :out]
    w8.linear(x, w8.PackedLinear(q, s), bias=bias, out=y)
    want, tol, _ = ref.linear(x, q, s, bias)
    near(y, want, tol)
    assert bool((wide[rows:] == 7).all()) and bool((wide[:, out:] == 7).all())   # nothing behind the rows and columns


@pytest.mark.parametrize("rows,width,inter", [(95, 2624, 256), (26, 7168, 250), (33, 5000, 129), (60, 4096, 1024), (200, 1024, 333), (300, 4096, 511), (290, 5760, 100), (128, 8192, 2048),
                                              (257, 2048, 512), (66, 1000, 1500), (200, 8192, 550)])
def test_gated_ffn_of_several_token_tiles(w8, rows, width, inter):
    x, gate, up, down = make_ffn(rows, width, inter, rows + inter)
    got = w8.gated_ffn(x, w8.PackedGateUp(*gate, *up), w8.PackedLinear(*down))
    want, tol, _ = ref.ffn(x, *gate, *up, *down)
    near(got, want, tol)


@pytest.mark.parametrize("rows", [1, 7, 100, 400])
@pytest.mark.parametrize("inter", [3, 333, 1001])
def test_gated_ffn_of_odd_widths(w8, rows, inter):
    """Activations are padded to whole vectors: neither the padding nor rows that are NaN or zero may reach the other rows."""
    width = 200
    x, gate, up, down = make_ffn(rows, width, inter, rows + inter)
    packed = w8.PackedGateUp(*gate, *up), w8.PackedLinear(*down)
    torch.full((1 << 22,), float("nan"), device="cuda")          # what the workspace's memory may hold
    want = w8.gated_ffn(x, *packed)
    full, tol, _ = ref.ffn(x, *gate, *up, *down)
    near(want, full, tol)
    bad = x.clone()
    bad[0, 5] = float("nan")
    if rows > 2:
        bad[rows // 2] = 0
        bad[rows - 1, 0] = float("inf")
    got = w8.gated_ffn(bad, *packed)
    assert bool(torch.isnan(got[0]).all())
    if rows > 2:
        assert bool(torch.isnan(got[rows - 1]).all()) and not bool(got[rows // 2].any())
        kept = [i for i in range(rows) if i not in (0, rows // 2, rows - 1)]
        assert torch.equal(got[kept], want[kept])


@pytest.mark.parametrize("rows,width", [(1, 5121), (3, 5121), (7, 8192), (400, 1025), (400, 2049), (400, 4099), (310, 8191), (300, 16383), (5, 16390), (2, 20001), (600, 256)])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_rows_at_odd_places(w8, rows, width, shift):
    """Rows that start anywhere and have any width give the integers and sums of the same rows side by side."""
    x, q, s = ref.make(rows, width, 40, seed=width + shift, device="cuda")
    buffer = torch.full((rows * (width + 5) + shift,), float("nan"), dtype=BF16, device="cuda")
    odd = buffer[shift:].view(rows, width + 5)[:, :width]
    odd.copy_(x)
    got, scale = w8.quantize(odd)
    r, top, _ = ref.ints(x.double())
    assert torch.equal(got.double(), r)
    assert float(((scale.double() - top[:, 0] / 127).abs() / top[:, 0].clamp(min=1e-30)).max()) < 2.0 ** -24
    packed = w8.PackedLinear(q, s)
    weight = (0.5 + torch.rand(width, generator=torch.Generator("cuda").manual_seed(1), device="cuda")).to(BF16)
    assert torch.equal(w8.linear(odd, packed), w8.linear(x.contiguous(), packed))
    y, total = w8.linear(odd, packed, norm_weight=weight, delta=x.flip(0).contiguous(), delta_scale=0.5)
    assert float((total != ref.residual(x, x.flip(0), 0.5)).float().mean()) < 1e-3
    want, tol, _ = ref.linear(total, q, s, norm_weight=weight)
    near(y, want, tol)


# Up to 16 rows and one beyond: clusters of 2, 3, 4 and 8 CTAs, columns that they share unevenly, rows longer than registers hold.
@pytest.mark.parametrize("rows", [2, 3, 4, 5, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("width,out", [(512, 128), (520, 200), (1000, 9000), (1032, 5000), (4096, 4608), (4096, 500), (16384, 4096), (16392, 130), (32768, 256), (40000, 100), (2056, 6144)])
def test_few_rows(w8, rows, width, out):
    x, q, s = ref.make(rows, width, out, seed=rows + width + out, device="cuda")
    g = torch.Generator("cuda").manual_seed(rows)
    bias = torch.randn(out, generator=g, device="cuda").to(BF16)
    weight = (0.5 + torch.rand(width, generator=g, device="cuda")).to(BF16)
    packed = w8.PackedLinear(q, s)
    want, tol, _ = ref.linear(x, q, s, bias)
    near(w8.linear(x, packed, bias=bias), want, tol)
    want, tol, _ = ref.linear(x, q, s, norm_weight=weight)
    near(w8.linear(x, packed, norm_weight=weight), want, tol)
    y, total = w8.linear(x, packed, norm_weight=weight, delta=x.flip(0).contiguous(), delta_scale=0.5)
    assert float((total != ref.residual(x, x.flip(0), 0.5)).float().mean()) < 1e-3
    want, tol, _ = ref.linear(total, q, s, norm_weight=weight)
    near(y, want, tol)


@pytest.mark.parametrize("rows", [2, 5, 16])
@pytest.mark.parametrize("width,inter", [(512, 320), (2048, 1024), (4096, 4700), (1000, 333)])
def test_gated_ffn_of_few_rows(w8, rows, width, inter):
    x, gate, up, down = make_ffn(rows, width, inter, rows + inter)
    packed = w8.PackedGateUp(*gate, *up), w8.PackedLinear(*down)
    got = w8.gated_ffn(x, *packed)
    want, tol, _ = ref.ffn(x, *gate, *up, *down)
    near(got, want, tol)
    bad = x.clone()
    bad[0, 1], bad[1] = float("inf"), 0
    again = w8.gated_ffn(bad, *packed)
    assert bool(torch.isnan(again[0]).all()) and not bool(again[1].any()) and torch.equal(again[2:], got[2:])


def test_few_rows_round_exactly(w8):
    """Behind an identity: half-way values, tiny and huge rows."""
    width = 512
    eye = w8.PackedLinear(torch.eye(width, dtype=torch.int8, device="cuda"), torch.ones(width, device="cuda"))
    g = torch.Generator("cuda").manual_seed(3)
    for rows in (2, 7, 16):
        for top in (254.0, 3.0, 127.0, 2.0 ** -126, float(torch.finfo(BF16).max)):
            x = (torch.randint(-127, 128, (rows, width), generator=g, device="cuda").double() / 127 * top).to(BF16)
            x[:, 0], x[:, 1], x[:, 2] = top, top / 2, -top / 2
            r, t, _ = ref.ints(x.double())
            y = w8.linear(x, eye)
            if top > 1e38 or top < 1e-30:   # the identity's outputs leave bf16's accuracy there: the rows' kernel says which integers
                q, scale = w8.quantize(x)
                assert torch.equal(q.double(), r) and torch.equal(y, (q.float() * scale[:, None]).to(BF16))
            else:
                assert torch.equal((y.double() / (t / 127)).round(), r), (rows, top)


CAPTURE = """
import torch, cpmcu.w8a8 as w8, cpmcu.rotary as rotary
BF16 = torch.bfloat16
w8.quantize(torch.ones(1, 8, dtype=BF16, device="cuda"))          # the one call outside of a capture
packed, x = {}, {}
shapes = [(1, 640, 300), (3, 1500, 400), (77, 2000, 500), (300, 1024, 1024), (90, 300, 20000), (1100, 512, 2048), (128, 5120, 4096)]
for s in shapes:
    g = torch.Generator("cuda").manual_seed(sum(s))
    x[s] = torch.randn(s[0], s[1], generator=g, device="cuda").to(BF16)
    packed[s] = w8.PackedLinear(torch.randint(-127, 128, (s[2], s[1]), generator=g, device="cuda").to(torch.int8), torch.rand(s[2], generator=g, device="cuda"))
qkv = torch.randn(5000, 6 * 72, device="cuda").to(BF16)
inv, pos, cache = torch.rand(36, device="cuda"), torch.arange(5000, device="cuda", dtype=torch.int32), torch.zeros(2, 5000, 72, dtype=BF16, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = {s: w8.linear(x[s], packed[s]) for s in shapes}
    q = rotary.append(qkv, 4, 1, 72, inv, pos, cache[0], cache[1], pos)
for _ in range(3): graph.replay()
torch.cuda.synchronize()
for s in shapes: assert torch.equal(y[s], w8.linear(x[s], packed[s])), s
assert torch.equal(q, rotary.append(qkv, 4, 1, 72, inv, pos, cache[0], cache[1], pos))
print("same")
"""


def test_first_calls_of_their_sizes_in_a_capture():
    """Kernels and divisions of work that the process has not used before are set up inside a capture."""
    import os
    import subprocess
    import sys
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cpm.cu_b200")
    out = subprocess.run([sys.executable, "-c", CAPTURE], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


@pytest.mark.parametrize("rows,width", [(1300, 800), (1300, 1600), (1300, 2400), (1300, 4808), (1300, 8800), (1200, 16000), (1200, 17000), (1300, 4801), (1300, 9001), (310, 1600), (310, 4104), (310, 6000)])
def test_many_rows(w8, rows, width):
    """Each way of sharing a row among threads, for plain rows, rows behind a norm, and behind a residual sum and a norm."""
    x, q, s = ref.make(rows, width, 24, seed=rows + width, device="cuda")
    got, scale = w8.quantize(x)
    r, top, _ = ref.ints(x.double())
    assert torch.equal(got.double(), r)
    packed = w8.PackedLinear(q, s)
    weight = (0.5 + torch.rand(width, generator=torch.Generator("cuda").manual_seed(1), device="cuda")).to(BF16)
    for more in ({}, {"norm_weight": weight}):
        want, tol, _ = ref.linear(x, q, s, **more)
        near(w8.linear(x, packed, **more), want, tol)
    y, total = w8.linear(x, packed, norm_weight=weight, delta=x.flip(0).contiguous(), delta_scale=0.5)
    assert float((total != ref.residual(x, x.flip(0), 0.5)).float().mean()) < 1e-3
    want, tol, _ = ref.linear(total, q, s, norm_weight=weight)
    near(y, want, tol)


@pytest.mark.parametrize("rows,inter", [(1300, 1600), (1300, 4096), (1200, 9000), (310, 2400)])
def test_gated_ffn_of_many_rows(w8, rows, inter):
    x, gate, up, down = make_ffn(rows, 256, inter, rows + inter)
    got = w8.gated_ffn(x, w8.PackedGateUp(*gate, *up), w8.PackedLinear(*down))
    want, tol, _ = ref.ffn(x, *gate, *up, *down)
    near(got, want, tol)


@pytest.mark.parametrize("rows", [1, 3, 60, 300, 1000])
def test_activations_keep_32_bits(rows):
    """silu(gate) * up as the down projection's rounding finds it, at the start of the workspace.  Integers of the rows and powers of two as scales make gate
    and up exact; what is left are an exponential (off by one unit in the last place at most, 2^-23), a sum, a quotient and a product of 2^-24 each:
    less than 6 * 2^-24 relative."""
    width, inter = 512, 320
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randint(-127, 128, (rows, width), generator=g, device="cuda")
    x[:, 7] = 127                                                       # the scale of every row is 1
    weights = [torch.zeros(inter, width, dtype=torch.int8, device="cuda") for _ in range(2)]
    at = torch.randint(0, width, (inter,), generator=g, device="cuda")   # each feature is one column of x
    for w in weights:
        w[torch.arange(inter, device="cuda"), at] = torch.randint(1, 128, (inter,), generator=g, device="cuda").to(torch.int8)
    scales = [torch.full((inter,), 2.0 ** -9, device="cuda"), torch.full((inter,), 2.0 ** -12, device="cuda")]
    down = torch.ones(width, inter, dtype=torch.int8, device="cuda")
    import cpmcu.w8a8 as w8
    gate_up, down = w8.PackedGateUp(weights[0], scales[0], weights[1], scales[1]), w8.PackedLinear(down, torch.ones(width, device="cuda"))
    size = C.load().cpmcu_w8a8_workspace_bytes(rows, width, width, inter)
    workspace = torch.zeros(size, dtype=torch.uint8, device="cuda")
    xb, y = x.to(BF16), torch.empty(rows, width, dtype=BF16, device="cuda")
    C.call("cpmcu_w8a8_ffn", xb.data_ptr(), width, gate_up.data.data_ptr(), down.data.data_ptr(), None, 1e-5, None, 1.0, None, y.data_ptr(), width, rows, width, inter,
           workspace.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    got = workspace[:rows * inter * 4].view(torch.float32).view(rows, inter).double()
    a, b = (x.double() @ w.double().t() * s.double() for w, s in zip(weights, scales))
    want = a / (1 + torch.exp(-a)) * b
    off = ((got - want).abs() / want.abs().clamp(min=1e-30)).max()
    assert float(off) < 6 * 2.0 ** -24, float(off) * 2 ** 24


def test_more_rows_than_threads_are_counted_in_32_bits(w8):
    """Narrow rows: 2^26 of them and more have over 2^31 threads."""
    rows, width, out = (1 << 26) + 300, 8, 8
    last, q, s = ref.make(300, width, out, seed=1, device="cuda")
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    x[-300:] = last
    got, scale = w8.quantize(x)
    few, few_scale = w8.quantize(last)
    assert torch.equal(got[-300:], few) and torch.equal(scale[-300:], few_scale)
    assert int(got[:-300].count_nonzero()) == 0 and int(scale[:-300].count_nonzero()) == 0
    del got, scale
    packed = w8.PackedLinear(q, s)
    guard = torch.full((1 << 28,), 7, dtype=torch.uint8, device="cuda")   # memory beside the workspace
    y = w8.linear(x, packed)
    want, tol, _ = ref.linear(last, q, s)
    near(y[-300:], want, tol)
    assert int(y[:-300].count_nonzero()) == 0 and bool((guard == 7).all())


@pytest.mark.parametrize("rows", [1, 40])
def test_copies_of_packed_weights_are_their_own(w8, rows):
    """copy.deepcopy and pickle, used at once; the copy outlives the original, and changes of one leave the other alone."""
    import copy
    import pickle
    x, q, s = ref.make(rows, 512, 300, seed=rows, device="cuda")
    gate_up, down = w8.PackedGateUp(q, s, q.flip(0).contiguous(), s), w8.PackedLinear(*ref.make(1, 300, 512, 1, "cuda")[1:])
    linear = w8.PackedLinear(q, s)
    want, block = w8.linear(x, linear), w8.gated_ffn(x, gate_up, down)
    for again in (copy.deepcopy, copy.copy, lambda w: pickle.loads(pickle.dumps(w))):
        a, g, d = again(linear), again(gate_up), again(down)
        assert a.device == linear.device and (a.data.data_ptr() == linear.data.data_ptr()) == (again is copy.copy)
        assert torch.equal(w8.linear(x, a), want) and torch.equal(w8.gated_ffn(x, g, d), block)
    a = copy.deepcopy(linear)
    a.data.zero_()
    torch.cuda.synchronize()
    assert torch.equal(w8.linear(x, linear), want) and not bool(w8.linear(x, a).any())
    a = copy.deepcopy(linear)
    linear.data.zero_()
    torch.cuda.synchronize()
    assert torch.equal(w8.linear(x, a), want)


def test_outputs_and_workspaces_that_do_not_fit(w8):
    """torch's own exception, as from any other call; the next call runs."""
    rows, out = 1 << 22, 100000
    x = torch.ones(rows, 1, dtype=BF16, device="cuda")
    wide = w8.PackedLinear(torch.ones(out, 1, dtype=torch.int8, device="cuda"), torch.ones(out, device="cuda"))
    with pytest.raises(torch.OutOfMemoryError):                     # 839 GB of outputs
        w8.linear(x, wide)
    gate_up = w8.PackedGateUp(*[t for _ in range(2) for t in (torch.ones(out, 1, dtype=torch.int8, device="cuda"), torch.ones(out, device="cuda"))])
    down = w8.PackedLinear(torch.ones(1, out, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    with pytest.raises(torch.OutOfMemoryError):                     # 1.7 TB of activations
        w8.gated_ffn(x, gate_up, down)
    assert bool((w8.linear(x[:5], wide) == 1).all())


def division(rows, width, out, gated=False):
    """(token tile, CTAs of a cluster, pairs of CTAs, cut tiles), and whether there are more tiles than run at once"""
    import ctypes
    d = (ctypes.c_int32 * 6)()
    C.call("cpmcu_debug_w8a8_division", rows, out, width, int(gated), ctypes.cast(d, ctypes.c_void_p))
    tiles = -(-out // (64 if gated else 128))
    return (d[0], d[2], d[3], d[4]), d[1] * (tiles // 2 if d[3] else tiles) > d[5]


# Every way in which a product is divided, with what find_division() makes of the sizes (148 SMs) and whether whole waves of tiles are ahead: token tiles and
# features that are partly filled, columns that end inside a block.  How many clusters of 3 CTAs and more run at once depends on how a GPU's SMs are grouped, so that
# another B200 may have others where clusters are named here.
DIVISIONS = [(2, 300, 40, (16, 0, 0, 0), False), (2, 131072, 40, (16, 0, 0, 1), False), (2, 1024, 8192, (16, 2, 0, 0), False), (2, 1024, 4608, (16, 3, 0, 0), False),
             (2, 1020, 40, (16, 4, 0, 0), False), (2, 2048, 40, (16, 8, 0, 0), False), (3000, 300, 40, (32, 0, 0, 0), False), (17, 131072, 40, (32, 0, 0, 1), False),
             (2047, 1024, 40, (32, 2, 0, 0), False), (1300, 1024, 40, (32, 3, 0, 0), False), (700, 1024, 40, (32, 4, 0, 0), False), (257, 2048, 40, (32, 8, 0, 0), False),
             (3000, 300, 130, (64, 0, 0, 0), False), (40, 131072, 40, (64, 0, 0, 1), False), (140, 12000, 6624, (64, 0, 0, 1), True), (3000, 2048, 40, (64, 2, 0, 0), False),
             (1300, 2048, 130, (64, 3, 0, 0), False), (2047, 4096, 40, (64, 4, 0, 0), False), (700, 8192, 40, (64, 8, 0, 0), False), (200, 300, 5000, (128, 0, 0, 0), False),
             (700, 131072, 40, (128, 0, 0, 1), False), (3870, 12000, 566, (128, 0, 0, 1), True), (3000, 8192, 130, (128, 2, 0, 0), False), (70, 4096, 5000, (128, 3, 0, 0), False),
             (3000, 8192, 40, (128, 4, 0, 0), False), (1300, 16384, 40, (128, 8, 0, 0), False), (4096, 300, 513, (256, 0, 0, 0), False), (2047, 131072, 40, (256, 0, 0, 1), False),
             (140, 33000, 4760, (256, 0, 0, 1), False), (1320, 6000, 3362, (256, 0, 0, 1), True), (513, 4096, 8100, (256, 0, 1, 0), True), (4096, 4096, 4608, (256, 0, 1, 0), True),
             (260, 33000, 3828, (256, 0, 1, 1), False), (1300, 131072, 130, (256, 0, 1, 1), False), (810, 12000, 4993, (256, 0, 1, 1), True), (2500, 16384, 5000, (256, 0, 1, 1), True)]


@pytest.mark.parametrize("rows,width,out,kind,waves", DIVISIONS)
def test_every_division_of_a_product(w8, rows, width, out, kind, waves):
    if kind[1] == 0:
        assert division(rows, width, out) == (kind, waves)
    x, q, s = ref.make(rows, width, out, seed=rows + width + out, device="cuda")
    bias = torch.randn(out, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(BF16)
    packed = w8.PackedLinear(q, s)
    want, tol, _ = ref.linear(x, q, s, bias)
    for pad in (3, 8 + (-out) % 8):             # rows element by element, and in vectors
        wide = torch.full((rows + 1, out + pad), 7.0, dtype=BF16, device="cuda")
        y = w8.linear(x, packed, bias=bias, out=wide[:rows, :out])
        near(y, want, tol)
        assert bool((wide[rows:] == 7).all()) and bool((wide[:, out:] == 7).all())   # nothing behind the rows and columns
        assert torch.equal(w8.linear(x, packed, bias=bias), y)                       # the same again


@pytest.mark.parametrize("rows,width,inter,kind", [(2, 1024, 4096, (16, 2, 0, 0)), (17, 300, 5000, (32, 0, 0, 0)), (40, 300, 5000, (64, 0, 0, 0)), (70, 300, 5000, (128, 0, 0, 0)),
                                                   (200, 300, 5000, (256, 0, 0, 0)), (257, 8192, 1000, (128, 2, 0, 0)), (200, 4096, 1280, (128, 3, 0, 0)),
                                                   (1300, 16384, 40, (128, 8, 0, 0)), (513, 4096, 4090, (256, 0, 1, 0)), (2047, 4096, 8190, (256, 0, 1, 0))])
def test_divisions_of_gate_and_up(w8, rows, width, inter, kind):
    if kind[1] == 0:
        assert division(rows, width, inter, gated=True)[0] == kind
    x, gate, up, down = make_ffn(rows, width, inter, rows + inter)
    got = w8.gated_ffn(x, w8.PackedGateUp(*gate, *up), w8.PackedLinear(*down))
    want, tol, _ = ref.ffn(x, *gate, *up, *down)
    near(got, want, tol)


def test_clusters_are_among_the_divisions(w8):
    got = [division(rows, width, out)[0] for rows, width, out, kind, _ in DIVISIONS if kind[1] > 0]
    assert {k[0] for k in got if k[1] > 0} == {16, 32, 64, 128} and {k[1] for k in got} >= {2, 8}


def test_cut_tiles_on_several_streams_and_in_graphs(w8):
    """Pieces of tiles, on single CTAs and on pairs, beside one another and beside other products, and replayed with other inputs."""
    sizes = [(810, 12000, 4993), (140, 12000, 6624), (1320, 6000, 3362), (260, 33000, 3828), (60, 16384, 4096), (1, 8192, 8192)]
    assert [division(*s)[0][2:] for s in sizes[:4]] == [(1, 1), (0, 1), (0, 1), (1, 1)]
    work = []
    for i, (rows, width, out) in enumerate(sizes):
        x, q, s = ref.make(rows, width, out, seed=i, device="cuda")
        work.append((x, w8.PackedLinear(q, s)))
    want = [w8.linear(x, p) for x, p in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[] for _ in work]
    for _ in range(10):
        for i, (stream, (x, p)) in enumerate(zip(streams, work)):
            with torch.cuda.stream(stream):
                got[i].append(w8.linear(x, p))
    torch.cuda.synchronize()
    for stream in streams:
        C.stream_check(stream.cuda_stream)
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = [w8.linear(x, p) for x, p in work]
    for shift in (1, 2):
        for x, _ in work:
            x.copy_(x.roll(shift, 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w8.linear(x, p)) for a, (x, p) in zip(kept, work))
        assert not any(torch.equal(a, w) for a, w in zip(kept, want))
    C.stream_check()


@pytest.mark.parametrize("rows", [1, 5, 300])
def test_rows_whose_squares_do_not_fit(w8, rows):
    """Behind a norm: NaN, not zeros; the largest rows that fit are right."""
    x, q, s = ref.make(rows, 512, 300, seed=rows, device="cuda")
    packed, weight = w8.PackedLinear(q, s), torch.linspace(0.5, 2, 512, device="cuda").to(BF16)
    clean = w8.linear(x, packed, norm_weight=weight)
    at = rows // 2
    rest = torch.arange(rows, device="cuda") != at
    big = x.clone()
    big[at] = x[at] * 2.0 ** 55                       # squares up to some 2^121 each
    want, tol, _ = ref.linear(big, q, s, norm_weight=weight)
    near(w8.linear(big, packed, norm_weight=weight), want, tol)
    big[at] = x[at] * 2.0 ** 70
    y = w8.linear(big, packed, norm_weight=weight)
    assert bool(torch.isnan(y[at]).all()) and torch.equal(y[rest], clean[rest])
    z = torch.zeros_like(big)
    y, total = w8.linear(z, packed, norm_weight=weight, delta=big)
    assert torch.equal(total[at], big[at]) and bool(torch.isnan(y[at]).all()) and torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("rows", [1, 60, 1000])
def test_activations_of_large_gates(rows):
    """The same for gates from -126 to 126: small activations keep their digits as far as fp32 has them.  Below, the product with up magnifies two roundings to
    a multiple of 2^-149, of the exponential and of the quotient."""
    width, inter = 512, 320
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randint(-127, 128, (rows, width), generator=g, device="cuda")
    x[:, 7] = 127
    weights = [torch.zeros(inter, width, dtype=torch.int8, device="cuda") for _ in range(2)]
    at = torch.randint(0, width, (inter,), generator=g, device="cuda")
    for w in weights:
        w[torch.arange(inter, device="cuda"), at] = torch.randint(1, 128, (inter,), generator=g, device="cuda").to(torch.int8)
    scales = [torch.full((inter,), 2.0 ** -7, device="cuda"), torch.full((inter,), 1.0, device="cuda")]
    import cpmcu.w8a8 as w8
    gate_up = w8.PackedGateUp(weights[0], scales[0], weights[1], scales[1])
    down = w8.PackedLinear(torch.ones(width, inter, dtype=torch.int8, device="cuda"), torch.ones(width, device="cuda"))
    size = C.load().cpmcu_w8a8_workspace_bytes(rows, width, width, inter)
    workspace = torch.zeros(size, dtype=torch.uint8, device="cuda")
    xb, y = x.to(BF16), torch.empty(rows, width, dtype=BF16, device="cuda")
    C.call("cpmcu_w8a8_ffn", xb.data_ptr(), width, gate_up.data.data_ptr(), down.data.data_ptr(), None, 1e-5, None, 1.0, None, y.data_ptr(), width, rows, width, inter,
           workspace.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    got = workspace[:rows * inter * 4].view(torch.float32).view(rows, inter).double()
    a, b = (x.double() @ w.double().t() * s.double() for w, s in zip(weights, scales))
    want = a / (1 + torch.exp(-a)) * b
    tol = want.abs() * 6 * 2.0 ** -24 + (a.abs() + 2) * b.abs() * 2.0 ** -149
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())
