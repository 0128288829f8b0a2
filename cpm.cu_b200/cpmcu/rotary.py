"""Rotary positions: frequencies of the scaled kinds, and the rotation of fused q/k/v rows with their append to a cache.

    inv_freq, factor = frequencies(128, 500000.0, {"rope_type": "llama3", ...}, length=max_length)
    q = append(qkv, heads, kv_heads, 128, inv_freq.cuda(), positions, k_cache, v_cache, slots, factor=factor)
"""
import math

import torch

from . import _ops   # raises where it has not been built (`python cpm.cu_b200/build.py`)

_F32, _F64 = torch.float32, torch.float64


def frequencies(rot_dims, base, scaling=None, length=None, max_position=None):
    """(inv_freq, factor): the rot_dims / 2 frequencies (fp32, CPU, computed in 64 bits) and the factor of sines and cosines.

    scaling: a checkpoint's rope_scaling dictionary ("rope_type" or "type", and the entries of that type); None or "default" is
    base^(-2 i / rot_dims).  linear: positions divided by "factor".  dynamic: a base that grows with `length` beyond max_position.  llama3: long waves
    divided by "factor", short ones kept, a ramp between.  yarn: a ramp over the pairs between the numbers of turns "beta_fast" and "beta_slow".
    longrope: "long_factor" if `length` is beyond the trained length, else "short_factor", for each pair.
    length: of the sequence that is served; max_position: of the checkpoint (max_position_embeddings), the trained length where the
    dictionary names no "original_max_position_embeddings"."""
    if rot_dims < 2 or rot_dims % 2:
        raise ValueError("rot_dims must be a positive even number")
    if not base > 1:
        raise ValueError("base must be above 1")
    s = dict(scaling or {})
    kind = s.get("rope_type", s.get("type")) or "default"
    i = torch.arange(0, rot_dims, 2, dtype=_F64) / rot_dims
    inv, factor = base ** -i, 1.0

    def entry(name, default=None):
        value = s.get(name)
        value = default if value is None else value
        if value is None:
            raise ValueError(f"rope_scaling of type {kind} needs {name!r}")
        return value

    def trained():
        return entry("original_max_position_embeddings", max_position)

    if kind == "default":
        pass
    elif kind == "linear":
        inv = inv / entry("factor")
    elif kind == "dynamic":
        f, top = entry("factor"), trained() if max_position is None else max_position
        n = max(length or top, top)
        if rot_dims > 2:
            inv = (base * ((f * n / top) - (f - 1)) ** (rot_dims / (rot_dims - 2))) ** -i
    elif kind == "llama3":
        f, low, high = entry("factor"), entry("low_freq_factor"), entry("high_freq_factor")
        turns = trained() * inv / (2 * math.pi)                       # of the trained length
        ramp = ((turns - low) / (high - low)).clamp(0, 1)             # 0: a long wave
        inv = inv / f * (1 - ramp) + inv * ramp
    elif kind == "yarn":
        f, top = entry("factor"), trained()

        def attention(scale, m):
            return 1.0 if scale <= 1 else 0.1 * m * math.log(scale) + 1.0

        if s.get("attention_factor") is not None:
            factor = float(s["attention_factor"])
        elif s.get("mscale") and s.get("mscale_all_dim"):
            factor = attention(f, s["mscale"]) / attention(f, s["mscale_all_dim"])
        else:
            factor = attention(f, 1.0)

        def pair_of(n):   # the (fractional) pair that turns n times in the trained length
            return rot_dims * math.log(top / (n * 2 * math.pi)) / (2 * math.log(base))

        first, last = pair_of(entry("beta_fast", 32)), pair_of(entry("beta_slow", 1))
        if s.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rot_dims - 1)
        if first == last:
            last += 0.001
        ramp = ((torch.arange(rot_dims // 2, dtype=_F64) - first) / (last - first)).clamp(0, 1)
        inv = inv / f * ramp + inv * (1 - ramp)
    elif kind == "longrope":
        top = trained()
        by = entry("long_factor" if length and length > top else "short_factor")
        if len(by) != rot_dims // 2:
            raise ValueError(f"longrope needs {rot_dims // 2} factors, got {len(by)}")
        inv = inv / torch.tensor(by, dtype=_F64)
        if s.get("attention_factor") is not None:
            factor = float(s["attention_factor"])
        else:
            f = entry("factor", max_position and max_position / top)
            factor = 1.0 if f <= 1 else math.sqrt(1 + math.log(f) / math.log(top))
    else:
        raise ValueError(f"rope type {kind!r} is not one of default, linear, dynamic, llama3, yarn, longrope")
    return inv.to(_F32), factor


def append(qkv, heads, kv_heads, dim, inv_freq, positions, k_cache=None, v_cache=None, slots=None, rot_dims=None, interleaved=False, factor=1.0,
           out=None):
    """Rotated queries [rows, heads * dim] of qkv [rows, (heads + 2 kv_heads) * dim] bf16; rotated keys, and values, go to rows `slots` of the
    caches [cache_rows, kv_heads * dim] (a negative slot: to none).  inv_freq [rot_dims / 2] fp32, positions and slots [rows] int32.
    rot_dims: rotated elements of each head (default: all, None).  out: where the queries go; a view of qkv's own query part is allowed."""
    return _ops.rotary_append(qkv, heads, kv_heads, dim, dim if rot_dims is None else rot_dims, interleaved, inv_freq, factor, positions, k_cache, v_cache,
                              slots, out)
