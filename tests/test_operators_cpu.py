"""What the operators on the caller's streams refuse, from C and from Python; no GPU: every refusal comes before the device is touched."""
import ctypes

import pytest
import torch

import cpmcu.C as C

PACKED, X, Y, WS = 0x10000000, 0x20000000, 0x30000000, 0x40000000   # addresses that nothing reads


def refused(name, *args):
    with pytest.raises(RuntimeError) as e:
        C.call(name, *args)
    return str(e.value)


def linear(x=X, ldx=64, packed=PACKED, bias=None, norm=None, eps=1e-5, delta=None, scale=1.0, total=None, y=Y, ldy=32, rows=4, n=32, k=64, ws=WS,
           size=1 << 30):
    return refused("cpmcu_w8a8_linear", x, ldx, packed, bias, norm, eps, delta, scale, total, y, ldy, rows, n, k, ws, size, None)


def test_linear_refusals():
    assert "sizes must be positive" in linear(rows=-1)
    assert "sizes must be positive" in linear(n=0)
    assert "sizes must be positive" in linear(k=0)
    assert "131072" in linear(k=131073, ldx=131073)
    assert "256-byte aligned" in linear(packed=None)
    assert "256-byte aligned" in linear(packed=PACKED + 16)
    assert "must not be null" in linear(x=None)
    assert "must not be null" in linear(y=None)
    assert "leading dimension" in linear(ldx=63)
    assert "leading dimension" in linear(ldy=31)
    assert "delta needs" in linear(delta=0x50000000, total=0x60000000)
    assert "come together" in linear(norm=0x70000000, delta=0x50000000)
    assert "come together" in linear(norm=0x70000000, total=0x50000000)
    assert "y must not overlap x" in linear(y=X)
    assert "y must not overlap x" in linear(y=X + 2 * 64 * 4 - 2)            # x's last element
    assert "total must not overlap" in linear(norm=0x70000000, delta=0x50000000, total=X)
    assert "total must not overlap" in linear(norm=0x70000000, delta=0x50000000, total=0x50000000)
    assert "total must not overlap" in linear(norm=0x70000000, delta=0x50000000, total=Y)
    assert "y must not overlap delta" in linear(norm=0x70000000, delta=Y, total=0x50000000)
    # rows of one wider matrix interleave and share no element: not refused for that
    assert "overlap" not in linear(ldx=96, y=X + 128, ldy=96, ws=None)          # refused later, without a workspace
    assert "y must not overlap x" in linear(ldx=96, y=X + 126, ldy=96)


def test_what_is_written_shares_nothing():
    n, d, t = 0x70000000, 0x50000000, 0x60000000
    assert "weights or the bias" in linear(bias=Y + 64)
    assert "weights or the bias" in linear(y=PACKED + 128 * 128)                  # the packed scales
    assert "weights or the bias" in linear(norm=n, delta=d, total=PACKED + 256)
    assert "weights or the bias" in linear(norm=n, delta=d, total=t, bias=t)

    def ffn(y):
        return refused("cpmcu_w8a8_ffn", X, 64, PACKED, 0x18000000, None, 1e-5, None, 1.0, None, y, 64, 4, 64, 128, WS, 1 << 30, None)

    assert "weights or the bias" in ffn(PACKED)
    assert "weights or the bias" in ffn(0x18000000)
    assert "packed must not overlap" in refused("cpmcu_w8a8_pack", PACKED + 16, Y, 4, 4, 0, PACKED, None)
    assert "packed must not overlap" in refused("cpmcu_w8a8_pack", X, PACKED + 128 * 128, 4, 4, 1, PACKED, None)
    for name in ("pos", "slots", "inv"):
        assert "positions, slots or frequencies" in rotary(**{name: Y + 8}), name
        assert "positions, slots or frequencies" in rotary(**{name: 0x60000000 + 64}), name


def test_ffn_refusals():
    def ffn(x=X, ldx=64, up=PACKED, down=PACKED, y=Y, ldy=64, rows=4, k=64, inter=128):
        return refused("cpmcu_w8a8_ffn", x, ldx, up, down, None, 1e-5, None, 1.0, None, y, ldy, rows, k, inter, WS, 1 << 30, None)
    assert "sizes must be positive" in ffn(inter=0)
    assert "131072" in ffn(inter=131073)
    assert "256-byte aligned" in ffn(up=PACKED + 128)
    assert "256-byte aligned" in ffn(down=None)
    assert "y must not overlap x" in ffn(y=X)


def test_packing_and_rounding_refusals():
    assert "part is" in refused("cpmcu_w8a8_pack", X, Y, 4, 4, 3, PACKED, None)
    assert "must not be null" in refused("cpmcu_w8a8_pack", None, Y, 4, 4, 0, PACKED, None)
    assert "256-byte aligned" in refused("cpmcu_w8a8_pack", X, Y, 4, 4, 0, PACKED + 8, None)
    assert "leading dimension" in refused("cpmcu_w8a8_quantize", X, 3, 4, 4, Y, WS, None)
    assert "must not overlap" in refused("cpmcu_w8a8_quantize", X, 4, 4, 4, X + 8, WS, None)
    for sizes in ((0, 4, 0), (4, 0, 0), (4, 131073, 0), (1 << 30, 131072, 0)):
        assert C.load().cpmcu_w8a8_packed_bytes(*sizes) == -1 and C.load().cpmcu_last_error()
    # one block of 128 x 128 and its scales; a gate/up tile has 64 features
    assert C.load().cpmcu_w8a8_packed_bytes(1, 1, 0) == C.load().cpmcu_w8a8_packed_bytes(64, 128, 1) == 128 * 128 + 512
    assert C.load().cpmcu_w8a8_packed_bytes(129, 129, 0) == 4 * 128 * 128 + 1024


def rotary(qkv=X, ld=384, rows=4, heads=4, kv=1, dim=64, rot=64, inter=0, inv=0x50000000, pos=0x51000000, q=Y, ldq=256, k=0x60000000, v=0x70000000,
           cache=16, slots=0x52000000):
    return refused("cpmcu_rotary_append", qkv, ld, rows, heads, kv, dim, rot, inter, inv, 1.0, pos, q, ldq, k, v, cache, slots, None)


def test_rotary_refusals():
    assert "sizes must be positive" in rotary(rows=-1)
    assert "sizes must be positive" in rotary(heads=0, kv=0)
    assert "even" in rotary(dim=63, rot=0)
    assert "rot_dims" in rotary(rot=66)
    assert "rot_dims" in rotary(rot=33)
    assert "512 pairs" in rotary(dim=2048, rot=1026, ld=1 << 20, ldq=1 << 20)
    assert "too wide" in rotary(dim=4098, rot=64, ld=1 << 20, ldq=1 << 20)
    assert "must not be null" in rotary(qkv=None)
    assert "must not be null" in rotary(pos=None)
    assert "must not be null" in rotary(inv=None)
    assert "must not be null" in rotary(q=None)
    assert "must not be null" in rotary(k=None)
    assert "must not be null" in rotary(slots=None)
    assert "leading dimension" in rotary(ld=383)
    assert "leading dimension" in rotary(ldq=255)
    assert "query part" in rotary(q=X, ldq=256)               # rows other than qkv's own
    assert "query part" in rotary(q=X + 2, ldq=384)
    assert "caches must not overlap" in rotary(k=X)
    assert "caches must not overlap" in rotary(v=0x60000000 + 64 * 2 * 16 - 2)
    assert "caches must not overlap" in rotary(v=Y)


def test_python_refusals():
    from cpmcu import rotary as R, w8a8 as W
    bf, i8 = torch.bfloat16, torch.int8
    with pytest.raises(ValueError):
        W.quantize(torch.zeros(4, 4))                          # fp32
    with pytest.raises(ValueError):
        W.quantize(torch.zeros(4, 4, dtype=bf))                # not on the GPU
    with pytest.raises(ValueError):
        W.quantize(torch.zeros(4, dtype=bf))
    with pytest.raises(ValueError):
        W.PackedLinear(torch.zeros(4, 4, dtype=i8), torch.zeros(4))
    with pytest.raises(ValueError):
        W.PackedGateUp(torch.zeros(4, 4, dtype=i8), torch.zeros(4), torch.zeros(4, 4, dtype=i8), torch.zeros(4))
    with pytest.raises(ValueError):
        W.linear(torch.zeros(1, 4, dtype=bf), torch.zeros(4, 4))
    with pytest.raises(ValueError):
        W.gated_ffn(torch.zeros(1, 4, dtype=bf), None, None)
    with pytest.raises(ValueError):
        R.append(torch.zeros(4, 6, dtype=bf), 1, 1, 2, torch.zeros(1), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        R.append(torch.zeros(6, dtype=bf), 1, 1, 2, torch.zeros(1), torch.zeros(4, dtype=torch.int32))


def test_plain_forms_agree_with_torch():
    """The 64-bit forms that the GPU tests hold the kernels to, against other ways of writing them."""
    import w8a8_cases as ref
    x, q, s = ref.make(5, 40, 7, seed=3)
    bias = torch.randn(7).to(torch.bfloat16)
    r, top, _ = ref.ints(x.double())
    assert int(r.abs().max()) == 127 and torch.equal(r, (127 * x.double() / top).round())
    y, _, _ = ref.linear(x, q, s, bias)
    assert torch.allclose(y, (r * top / 127) @ (q.double() * s.double()[:, None]).t() + bias.double(), rtol=1e-12)
    w = torch.rand(40).to(torch.bfloat16)
    y, _, _ = ref.linear(x, q, s, norm_weight=w)
    v = torch.nn.functional.rms_norm(x.double(), (40,), w.double(), float(torch.tensor(1e-5)))
    step = v.abs().amax(1, keepdim=True) / 127
    # the factor of the norm cancels in the integers but for its rounding at exact ties
    assert torch.allclose(y, (v / step).round() * step @ (q.double() * s.double()[:, None]).t(), rtol=1e-6, atol=float(step.max()) * 1e-3)


def test_more_rows_than_are_counted_in_32_bits():
    top = 2 ** 31 - 1
    assert "too many rows" in linear(rows=top)
    assert "too many rows" in refused("cpmcu_w8a8_ffn", X, 64, PACKED, PACKED, None, 1e-5, None, 1.0, None, Y, 64, top, 64, 64, WS, 1 << 30, None)
    assert C.load().cpmcu_w8a8_workspace_bytes(top, 32, 64, 0) == -1 and b"too many rows" in C.load().cpmcu_last_error()
    assert "too many rows" not in linear(rows=top - 256, ws=None)


def test_packed_weights_off_the_gpu_are_refused():
    """What torch.load with a map_location gives: weights whose bytes are somewhere else."""
    from cpmcu import w8a8 as W
    w = W.PackedLinear.__new__(W.PackedLinear)
    w.__setstate__({"out": 4, "width": 4, "data": torch.zeros(128 * 128 + 512, dtype=torch.uint8)})
    with pytest.raises(ValueError, match="weight must be on the GPU"):
        W.linear(torch.zeros(1, 4, dtype=torch.bfloat16), w)
    w.data = w.data[1:]
    with pytest.raises(ValueError, match="weight must be torch.uint8"):
        W.linear(torch.zeros(1, 4, dtype=torch.bfloat16), w)
    g = W.PackedGateUp.__new__(W.PackedGateUp)
    g.__setstate__({"out": 4, "width": 4, "data": torch.zeros(128 * 128 + 512, dtype=torch.uint8)})
    w.data = g.data
    with pytest.raises(ValueError, match="gate_up must be on the GPU"):
        W.gated_ffn(torch.zeros(1, 4, dtype=torch.bfloat16), g, w)
