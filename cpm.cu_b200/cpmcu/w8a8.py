"""Linear layers in 8-bit integers: weights int8 with a scale for each output channel, rows of bf16 rounded to 8-bit integers with a
scale each, exact 32-bit sums (formulas at cpmcu_w8a8_linear in include/cpmcu_b200.h).

    w = PackedLinear(q, scale)                     # once: int8 [out, in] and fp32 [out] of a checkpoint, or PackedLinear.from_bf16(weight)
    y = linear(x, w)                               # x [rows, in] bf16 -> [rows, out] bf16
    y, t = linear(x, w, norm_weight=g, delta=d)    # t = x + d, y of rms_norm(t) * g
    y = gated_ffn(x, PackedGateUp(...), w_down)    # down(silu(gate(x)) * up(x))

Calls run on torch's current stream and return without waiting; they can be captured into CUDA graphs (after a first call outside of one).  What a
kernel reports (a wait that ran out) is raised by cpmcu.C.stream_check.  Packed weights are not to be written to; copy.deepcopy and pickle keep them whole.
"""
import torch

from . import C
from . import _ops   # raises where it has not been built (`python cpm.cu_b200/build.py`)

_BF16, _I8, _F32 = torch.bfloat16, torch.int8, torch.float32


def _check(t, what, dtype, shape, device=None, rows=False):
    """rows: any distance between the rows; otherwise contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {dtype} of shape {tuple(shape)}" +
                         (f", got {t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else ""))
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{what} must be on {device or 'the GPU'}, got {t.device}")
    if t.is_contiguous():
        return
    if not rows or t.dim() != 2:
        raise ValueError(f"{what} must be contiguous")
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what} must have consecutive elements in rows that do not overlap")


def _call(name, device, *args):
    """The entry point on torch's current stream of `device`."""
    with torch.cuda.device(device):
        C.call(name, *args, torch.cuda.current_stream(device).cuda_stream)


def quantize(x):
    """(q, scale) of the rows of x [rows, in] bf16: q = round(127 x / max|x|), int8, scale = max|x| / 127, fp32."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a matrix")
    _check(x, "x", _BF16, x.shape, rows=True)
    q, scale = torch.empty(x.shape, dtype=_I8, device=x.device), torch.empty(x.shape[0], dtype=_F32, device=x.device)
    ld = x.stride(0) if x.shape[0] > 1 else max(1, x.shape[1])
    _call("cpmcu_w8a8_quantize", x.device, x.data_ptr(), ld, x.shape[0], x.shape[1], q.data_ptr(), scale.data_ptr())
    return q, scale


class _Packed:
    def __init__(self, out, width, gated, parts):
        if out < 1 or width < 1:
            raise ValueError("weights must not be empty")
        self.out, self.width, device = out, width, parts[0][0].device
        n = C.load().cpmcu_w8a8_packed_bytes(out, width, int(gated))
        if n < 0:
            raise ValueError(C.load().cpmcu_last_error().decode())
        self.data = torch.empty(n, dtype=torch.uint8, device=device)
        for part, (q, scale) in enumerate(parts, start=int(gated)):
            _call("cpmcu_w8a8_pack", device, q.data_ptr(), scale.data_ptr(), out, width, part, self.data.data_ptr())

    @property
    def device(self):
        return self.data.device

    def __setstate__(self, state):
        """Of copies and of unpickled weights.  Their bytes were not written by the packing kernel, and a call fetches weights before it waits for the work
        ahead of it in the stream: they have to be there."""
        self.__dict__.update(state)
        if self.data.is_cuda:
            torch.cuda.current_stream(self.data.device).synchronize()


class PackedLinear(_Packed):
    """A weight matrix in the kernels' layout: q [out, in] int8, scale [out] fp32."""

    def __init__(self, q, scale):
        if not isinstance(q, torch.Tensor) or q.dim() != 2:
            raise ValueError("q must be a matrix")
        _check(q, "q", _I8, q.shape)
        _check(scale, "scale", _F32, q.shape[:1], q.device)
        super().__init__(q.shape[0], q.shape[1], False, [(q, scale)])

    @classmethod
    def from_bf16(cls, weight):
        """Rounds a bf16 matrix [out, in], a scale for each row."""
        return cls(*quantize(weight))


class PackedGateUp(_Packed):
    """The gate and the up projection of a feed-forward block: q [inter, in] int8 and scale [inter] fp32 each."""

    def __init__(self, gate, gate_scale, up, up_scale):
        if not isinstance(gate, torch.Tensor) or gate.dim() != 2:
            raise ValueError("gate must be a matrix")
        _check(gate, "gate", _I8, gate.shape)
        _check(up, "up", _I8, gate.shape, gate.device)
        _check(gate_scale, "gate_scale", _F32, gate.shape[:1], gate.device)
        _check(up_scale, "up_scale", _F32, gate.shape[:1], gate.device)
        super().__init__(gate.shape[0], gate.shape[1], True, [(gate, gate_scale), (up, up_scale)])

    @classmethod
    def from_bf16(cls, gate, up):
        return cls(*quantize(gate), *quantize(up))


def linear(x, weight, bias=None, norm_weight=None, eps=1e-5, delta=None, delta_scale=1.0, out=None):
    """y [rows, out] of x [rows, in].  With norm_weight the rows are RMS norms; with delta, of t = x + delta_scale * delta, and (y, t) is
    returned.  bias [out] bf16.  x (and out) may be rows of a wider matrix."""
    if type(weight) is not PackedLinear:
        raise ValueError("weight must be a PackedLinear")
    return _ops.linear(x, weight.data, weight.out, weight.width, bias, norm_weight, eps, delta, delta_scale, out)


def gated_ffn(x, gate_up, down, norm_weight=None, eps=1e-5, delta=None, delta_scale=1.0, out=None):
    """down(silu(gate(x)) * up(x)) of x [rows, in]; norm_weight, delta and out as for linear."""
    if type(gate_up) is not PackedGateUp or type(down) is not PackedLinear:
        raise ValueError("gate_up must be a PackedGateUp and down a PackedLinear")
    width, inter = gate_up.width, gate_up.out
    if down.width != inter or down.out != width:
        raise ValueError(f"down must be [{width}, {inter}]")
    return _ops.ffn(x, gate_up.data, down.data, width, inter, norm_weight, eps, delta, delta_scale, out)
