"""Rotation of fused q/k/v rows against its definition in 64 bits: both layouts, parts of a head, odd widths and strides, far and negative positions,
cache slots that are skipped or out of range."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, I32, F64 = torch.bfloat16, torch.int32, torch.float64


@pytest.fixture(scope="module")
def rotary():
    import cpmcu.rotary as r
    return r


def definition(qkv, heads, kv, dim, inv_freq, pos, rot, interleaved, factor):
    """(rotated queries and keys, values, allowed error of the rotated)"""
    x = qkv.double().unflatten(1, (heads + 2 * kv, dim))
    angle = pos.double()[:, None] * inv_freq.double()
    f = float(torch.tensor(factor, dtype=torch.float32))
    cs, sn = torch.cos(angle)[:, None] * f, torch.sin(angle)[:, None] * f
    out, part = x[:, :heads + kv].clone(), x[:, :heads + kv, :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rot // 2], part[..., rot // 2:])
    new = (a * cs - b * sn, b * cs + a * sn)
    size = (a.abs() + b.abs()) * abs(f)
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = new
        size = size.repeat_interleave(2, -1)
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = new
        size = torch.cat((size, size), -1)
    # rounding to bf16; sines and cosines to 2^-20 (a turn's fraction in fp32, its functions, the factor and two more roundings)
    tol = out.abs() * 2.0 ** -8
    tol[..., :rot] += size * 2.0 ** -20 + 1e-38
    tol[..., rot:] = 0
    return out, x[:, heads + kv:], tol


SHAPES = [(32, 2, 128, 128, False), (32, 8, 128, 64, False), (15, 5, 80, 20, True), (4, 4, 80, 20, False), (3, 1, 64, 64, True), (2, 2, 96, 48, False), (1, 1, 2, 2, True),
          (5, 1, 6, 2, False), (7, 3, 10, 6, True), (8, 8, 256, 256, False), (2, 1, 256, 64, True), (1, 1, 36, 36, False), (2, 2, 1024, 1024, False), (3, 1, 64, 0, False), (40, 1, 72, 72, True)]


@pytest.mark.parametrize("heads,kv,dim,rot,interleaved", SHAPES)
@pytest.mark.parametrize("rows,pad", [(1, 0), (5, 0), (60, 8), (33, 3), (700, 2)])
def test_rotation(rotary, heads, kv, dim, rot, interleaved, rows, pad):
    g = torch.Generator("cuda").manual_seed(rows + dim)
    cols = (heads + 2 * kv) * dim
    wide = torch.randn(rows, cols + 2 * pad, generator=g, device="cuda").to(BF16)
    qkv = wide[:, pad:pad + cols]
    before = wide.clone()
    inv, _ = rotary.frequencies(max(rot, 2), 10000.0)
    inv = inv[:rot // 2].cuda()
    pos = torch.randint(-50, 2_000_000, (rows,), generator=g, device="cuda", dtype=I32)
    n = rows + 9
    slots = torch.randperm(n, generator=g, device="cuda")[:rows].to(I32)
    slots[rows // 2] = -3
    k, v = torch.randn(2, n, kv * dim, generator=g, device="cuda").to(BF16)
    k0, v0 = k.clone(), v.clone()
    q = rotary.append(qkv, heads, kv, dim, inv, pos, k, v, slots, rot_dims=rot, interleaved=interleaved, factor=1.19)
    want, values, tol = definition(qkv, heads, kv, dim, inv, pos, rot, interleaved, 1.19)
    got = q.double().unflatten(1, (heads, dim))
    assert bool(((got - want[:, :heads]).abs() <= tol[:, :heads]).all())
    kept = slots >= 0
    at = slots[kept].long()
    assert bool(((k[at].double().unflatten(1, (kv, dim)) - want[kept][:, heads:]).abs() <= tol[kept][:, heads:]).all())
    assert torch.equal(v[at].double().unflatten(1, (kv, dim)), values[kept])
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(k[rest], k0[rest]) and torch.equal(v[rest], v0[rest])          # rows that no slot names
    assert torch.equal(wide.view(torch.int16), before.view(torch.int16))
    # in place: the queries of qkv themselves
    again = rotary.append(qkv, heads, kv, dim, inv, pos, k, v, slots, rot_dims=rot, interleaved=interleaved, factor=1.19, out=qkv[:, :heads * dim])
    assert torch.equal(again, q)
    assert torch.equal(wide[:, :pad], before[:, :pad]) and torch.equal(wide[:, pad + heads * dim:], before[:, pad + heads * dim:])


def test_unrotated_elements_and_infinities_stay_apart(rotary):
    """An infinity or a NaN reaches its own pair only."""
    for interleaved in (False, True):
        qkv = torch.randn(4, 3 * 64, device="cuda").to(BF16)
        inv = rotary.frequencies(32, 10000.0)[0].cuda()
        pos = torch.arange(4, dtype=I32, device="cuda")
        k, v = torch.zeros(2, 4, 64, dtype=BF16, device="cuda")
        clean = rotary.append(qkv, 1, 1, 64, inv, pos, k, v, pos, rot_dims=32, interleaved=interleaved)
        bad = qkv.clone()
        bad[1, 40], bad[2, 5], bad[3, 6] = float("nan"), float("inf"), float("nan")
        got = rotary.append(bad, 1, 1, 64, inv, pos, k, v, pos, rot_dims=32, interleaved=interleaved)
        differ = {(int(r), int(c)) for r, c in (got != clean).nonzero()}
        pairs = {(2, 4), (2, 5), (3, 6), (3, 7)} if interleaved else {(2, 5), (2, 21), (3, 6), (3, 22)}
        assert differ == pairs | {(1, 40)}


def test_slots_beyond_the_cache_are_reported_and_not_written(rotary):
    import cpmcu.C as C
    qkv = torch.randn(3, 3 * 64, device="cuda").to(BF16)
    inv = rotary.frequencies(64, 10000.0)[0].cuda()
    pos = torch.arange(3, dtype=I32, device="cuda")
    store = torch.zeros(2, 8, 64, dtype=BF16, device="cuda")
    k, v = store[0, :4], store[1, :4]
    rotary.append(qkv, 1, 1, 64, inv, pos, k, v, torch.tensor([4, 1, 2 ** 31 - 1], dtype=I32, device="cuda"))
    with pytest.raises(RuntimeError, match="error flags 8"):
        C.call("cpmcu_stream_check", torch.cuda.current_stream().cuda_stream)
    C.call("cpmcu_stream_check", torch.cuda.current_stream().cuda_stream)      # reported once
    assert not bool(store[:, 0].any()) and not bool(store[:, 2:].any()) and bool(store[:, 1].any())


def test_queries_or_keys_alone(rotary):
    qkv = torch.randn(6, 4 * 32, device="cuda").to(BF16)
    inv = rotary.frequencies(32, 10000.0)[0].cuda()
    pos = torch.arange(6, dtype=I32, device="cuda") * 1000
    q = rotary.append(qkv, 4, 0, 32, inv, pos)
    k, v = torch.zeros(2, 6, 64, dtype=BF16, device="cuda")
    none = rotary.append(qkv, 0, 2, 32, inv, pos, k, v, torch.arange(6, dtype=I32, device="cuda"))
    assert none.shape == (6, 0)
    assert torch.equal(k, q[:, :64]) and torch.equal(v, qkv[:, 64:])
    assert rotary.append(qkv[:0], 4, 0, 32, inv, pos[:0]).shape == (0, 128)


def test_many_rows_and_graphs(rotary):
    """Row counts on both sides of the change to rings of rows, short rows in groups among them; again from a graph, in place."""
    for heads, kv, dim, rot, interleaved, rows in [(8, 2, 128, 128, False, 1183), (8, 2, 128, 128, False, 1185), (4, 1, 64, 64, True, 3551), (4, 1, 64, 32, False, 3557),
                                                   (2, 0, 64, 64, False, 20001), (0, 1, 32, 32, True, 9001), (3, 1, 64, 0, False, 9001), (24, 4, 256, 256, False, 1301)]:
        g = torch.Generator("cuda").manual_seed(rows)
        qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g, device="cuda").to(BF16)
        inv = rotary.frequencies(max(rot, 2), 500000.0)[0][:rot // 2].cuda()
        pos = torch.arange(rows, dtype=I32, device="cuda") + 100000
        slots = torch.randperm(rows, generator=g, device="cuda").to(I32)
        slots[::7] = -1
        k, v = torch.zeros(2, rows, kv * dim, dtype=BF16, device="cuda")
        q = rotary.append(qkv, heads, kv, dim, inv, pos, k, v, slots, rot_dims=rot, interleaved=interleaved)
        want, values, tol = definition(qkv, heads, kv, dim, inv, pos, rot, interleaved, 1.0)
        assert bool(((q.double().unflatten(1, (heads, dim)) if heads else want[:, :0]) - want[:, :heads]).abs().le(tol[:, :heads]).all())
        if kv:
            at = slots[slots >= 0].long()
            assert bool(((k[at].double().unflatten(1, (kv, dim)) - want[slots >= 0][:, heads:]).abs() <= tol[slots >= 0][:, heads:]).all())
            assert torch.equal(v[at].double().unflatten(1, (kv, dim)), values[slots >= 0])
            rest = torch.ones(rows, dtype=torch.bool, device="cuda")
            rest[at] = False
            assert not bool(k[rest].any()) and not bool(v[rest].any())
        again = qkv.clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                rotary.append(again, heads, kv, dim, inv, pos, k, v, slots, rot_dims=rot, interleaved=interleaved, out=again[:, :heads * dim])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again[:, :heads * dim], q) and torch.equal(again[:, heads * dim:], qkv[:, heads * dim:])


def test_offsets_beyond_32_bits(rotary):
    """Cache slots and rows whose elements lie beyond 2^31."""
    heads, kv, dim, slots_n = 2, 2, 64, 17_000_000
    k = torch.empty(slots_n, kv * dim, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    rows, ld = 40000, 60000
    wide = torch.empty(rows, ld, dtype=BF16, device="cuda")
    qkv = wide[:, 1000:1000 + (heads + 2 * kv) * dim]
    qkv.copy_(torch.randn(rows, (heads + 2 * kv) * dim, device="cuda"))
    inv = rotary.frequencies(dim, 10000.0)[0].cuda()
    pos = torch.arange(rows, dtype=I32, device="cuda")
    at = torch.arange(slots_n - rows, slots_n, device="cuda")
    for n in (rows, 200):                    # rings of rows, one CTA per row
        k[at], v[at] = 0, 0
        part = qkv[-n:]
        q = rotary.append(part, heads, kv, dim, inv, pos[-n:], k, v, at[-n:].to(I32))
        want, values, tol = definition(part, heads, kv, dim, inv, pos[-n:], dim, False, 1.0)
        assert bool(((q.double().unflatten(1, (heads, dim)) - want[:, :heads]).abs() <= tol[:, :heads]).all())
        assert bool(((k[at[-n:]].double().unflatten(1, (kv, dim)) - want[:, heads:]).abs() <= tol[:, heads:]).all())
        assert torch.equal(v[at[-n:]].double().unflatten(1, (kv, dim)), values)
        if n < rows:
            assert not bool(k[at[:-n]].any())


def test_refusals_on_the_gpu(rotary):
    qkv = torch.zeros(4, 3 * 64, dtype=BF16, device="cuda")
    inv, pos = torch.ones(32, device="cuda"), torch.zeros(4, dtype=I32, device="cuda")
    k, v = torch.zeros(2, 4, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="qkv"):
        rotary.append(qkv[:, 1:], 1, 1, 64, inv, pos, k, v, pos)
    with pytest.raises(ValueError, match="inv_freq"):
        rotary.append(qkv, 1, 1, 64, inv[1:], pos, k, v, pos)
    with pytest.raises(ValueError, match="positions"):
        rotary.append(qkv, 1, 1, 64, inv, pos.long(), k, v, pos)
    with pytest.raises(ValueError, match="v_cache"):
        rotary.append(qkv, 1, 1, 64, inv, pos, k, v[:3], pos)
    with pytest.raises(ValueError, match="slots"):
        rotary.append(qkv, 1, 1, 64, inv, pos, k, v)
    with pytest.raises(RuntimeError, match="caches must not overlap"):
        rotary.append(qkv, 1, 1, 64, inv, pos, k, k, pos)
    with pytest.raises(RuntimeError, match="query part"):
        rotary.append(qkv, 1, 1, 64, inv, pos, k, v, pos, out=qkv[:, 64:128])


@pytest.mark.parametrize("heads,kv,dim,rot,interleaved", [(3, 3, 72, 72, False), (3, 3, 72, 72, True), (12, 4, 72, 36, False), (4, 4, 80, 20, False), (4, 4, 80, 40, False), (12, 4, 96, 24, False),
                                                          (6, 2, 112, 28, False), (2, 1, 8, 4, False), (1, 1, 40, 40, True), (1, 1, 8, 8, True), (2, 1, 72, 18, False), (2, 2, 256, 4, False)])
@pytest.mark.parametrize("rows,pad", [(4100, 0), (6001, 8), (6001, 4), (4100, 1)])
def test_many_rows_of_narrow_pieces(rotary, heads, kv, dim, rot, interleaved, rows, pad):
    """Rings of rows whose heads' halves are not vectors of eight; rows at places that no bulk copy reaches."""
    test_rotation(rotary, heads, kv, dim, rot, interleaved, rows, pad)


def beyond(rotary, stream=None):
    """A call whose slots lie behind its cache, on `stream`."""
    qkv = torch.zeros(2, 3 * 64, device="cuda").to(BF16)
    inv = torch.ones(32, device="cuda")
    pos = torch.arange(2, dtype=I32, device="cuda")
    k, v = torch.zeros(2, 1, 64, dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream or torch.cuda.current_stream()):
        rotary.append(qkv, 1, 1, 64, inv, pos, k, v, pos)
    return qkv, inv, pos, k, v


def test_a_check_tells_its_own_stream_s_errors(rotary):
    import cpmcu.C as C
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    C.stream_check(a.cuda_stream)
    for _ in range(3):
        beyond(rotary, b)
        b.synchronize()
        C.stream_check(a.cuda_stream)                                 # the other stream's is neither told here
        C.stream_check()
        with pytest.raises(RuntimeError, match="error flags 8"):      # nor taken away
            C.stream_check(b.cuda_stream)
        C.stream_check(b.cuda_stream)
    # reports that arrive while other streams are being checked
    for _ in range(20):
        with torch.cuda.stream(b):
            torch.cuda._sleep(200000)
        held = beyond_behind(rotary, b)
        for _ in range(20):
            C.stream_check(a.cuda_stream)
        with pytest.raises(RuntimeError, match="error flags 8"):
            C.stream_check(b.cuda_stream)
        del held


def beyond_behind(rotary, stream):
    """The same without a synchronisation ahead of it."""
    with torch.cuda.stream(stream):
        qkv, inv, pos = torch.zeros(2, 3 * 64, dtype=BF16, device="cuda"), torch.ones(32, device="cuda"), torch.arange(2, dtype=I32, device="cuda")
        k, v = torch.zeros(2, 1, 64, dtype=BF16, device="cuda")
        rotary.append(qkv, 1, 1, 64, inv, pos, k, v, pos)
    return qkv, inv, pos, k, v


def test_checks_from_several_threads_lose_nothing(rotary):
    import threading
    import cpmcu.C as C
    told, failed = [0] * 4, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            for n in range(40):
                held = beyond_behind(rotary, stream) if n % 2 else None
                try:
                    C.stream_check(stream.cuda_stream)
                except RuntimeError as e:
                    assert "error flags 8" in str(e)
                    told[i] += 1
                del held
        except BaseException as e:   # noqa: B036 (shown by the assertion below)
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and told == [20] * 4


GRAPH = """
import torch, cpmcu.C as C, cpmcu.rotary as rotary
BF16, I32 = torch.bfloat16, torch.int32
qkv, inv, pos = torch.zeros(2, 192, dtype=BF16, device="cuda"), torch.ones(32, device="cuda"), torch.arange(2, dtype=I32, device="cuda")
k, v = torch.zeros(2, 1, 64, dtype=BF16, device="cuda")
slots = torch.zeros(2, dtype=I32, device="cuda")
slots[1] = -1
def check(stream):
    try: C.stream_check(stream.cuda_stream)
    except RuntimeError as e: return str(e)
    return ""
rotary.append(qkv, 1, 1, 64, inv, pos, k, v, slots)
a, b, late = (torch.cuda.Stream() for _ in range(3))
assert check(a) == check(b) == ""
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    assert "being captured" in check(torch.cuda.current_stream())    # and the capture goes on
    q = rotary.append(qkv, 1, 1, 64, inv, pos, k, v, slots)
for _ in range(2):
    slots.fill_(1)
    torch.cuda.synchronize()
    with torch.cuda.stream(a): graph.replay()
    a.synchronize()
    assert "flags 8" in check(a) and check(a) == ""
    assert "flags 8" in check(b) and check(b) == ""    # it could have run there
    slots.fill_(-1)
    torch.cuda.synchronize()
    with torch.cuda.stream(a): graph.replay()
    assert check(a) == check(b) == ""
assert "captured graphs" in check(late) and check(late) == ""
print("told")
"""


def test_errors_of_captured_graphs():
    import os
    import subprocess
    import sys
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cpm.cu_b200")
    out = subprocess.run([sys.executable, "-c", GRAPH], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "told" in out.stdout, out.stderr[-2000:]


DURING = """
import threading, torch, cpmcu.C as C, cpmcu.w8a8 as w8
x = torch.ones(3, 64, dtype=torch.bfloat16, device="cuda")
w = w8.PackedLinear.from_bf16(torch.ones(32, 64, dtype=torch.bfloat16, device="cuda"))
want, other = w8.linear(x, w), torch.cuda.Stream()
torch.cuda.synchronize()
def elsewhere(check):
    thread = threading.Thread(target=check)
    thread.start()
    thread.join()
done = []
for stream in (other.cuda_stream, 0):
    def check():
        C.stream_check(stream)
        done.append(stream)
    for how in (lambda: check(), lambda: elsewhere(check)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(other): held = w8.linear(x, w)
        with torch.cuda.graph(graph):
            y = w8.linear(x, w)
            how()
            z = y + 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want + 1)
assert len(done) == 4
print("captured")
"""


def test_checks_of_other_streams_during_a_capture():
    """From the thread that captures and from another one: the check ends, and the capture goes on."""
    import os
    import subprocess
    import sys
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cpm.cu_b200")
    out = subprocess.run([sys.executable, "-c", DURING], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]
