"""Frequencies of the scaled rotary kinds against the initialisers of the transformers package, and what is refused; no GPU."""
import types

import pytest
import torch

KINDS = [
    (None, {}),
    ({"rope_type": "linear", "factor": 4.0}, {}),
    ({"rope_type": "dynamic", "factor": 2.0}, {}),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}, {}),
    ({"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}, {}),
    ({"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "mscale": 1.0, "mscale_all_dim": 0.8, "beta_fast": 16, "beta_slow": 2}, {}),
    ({"rope_type": "longrope", "short_factor": [1.0 + 0.01 * i for i in range(32)], "long_factor": [1.0 + i for i in range(32)],
      "original_max_position_embeddings": 4096}, {}),
]


def transformers_frequencies(dim, base, scaling, length, max_position):
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    kind = (scaling or {}).get("rope_type", "default")
    if kind == "default":
        return 1.0 / (base ** (torch.arange(0, dim, 2, dtype=torch.int64).float() / dim)), 1.0
    params = dict(scaling, rope_theta=base)
    cfg = types.SimpleNamespace(rope_theta=base, head_dim=dim, hidden_size=dim * 4, num_attention_heads=4, max_position_embeddings=max_position,
                                rope_scaling=params, rope_parameters=params, standardize_rope_params=lambda: None,
                                original_max_position_embeddings=scaling.get("original_max_position_embeddings", max_position))
    return ROPE_INIT_FUNCTIONS[kind](cfg, "cpu", seq_len=length)


@pytest.mark.parametrize("scaling", [k for k, _ in KINDS], ids=[(k or {}).get("rope_type", "default") for k, _ in KINDS])
@pytest.mark.parametrize("length", [1000, 50000])
def test_frequencies(scaling, length):
    from cpmcu.rotary import frequencies
    inv, factor = frequencies(64, 10000.0, scaling, length=length, max_position=16384)
    want, want_factor = transformers_frequencies(64, 10000.0, scaling, length, 16384)
    assert inv.dtype == torch.float32
    # theirs are computed in fp32: a power of the base is off by up to 12 roundings of its logarithm's magnitude
    assert float(((inv.double() - want.double()) / want.double()).abs().max()) < 1e-5
    assert abs(factor - want_factor) < 1e-6


def test_refusals():
    from cpmcu.rotary import frequencies
    for args in ((63, 10000.0), (0, 10000.0), (64, 1.0), (64, 10000.0, {"rope_type": "other"}), (64, 10000.0, {"rope_type": "linear"}),
                 (64, 10000.0, {"rope_type": "llama3", "factor": 2.0}), (64, 10000.0, {"rope_type": "yarn", "factor": 2.0}),
                 (64, 10000.0, {"rope_type": "longrope", "short_factor": [1.0], "long_factor": [1.0], "original_max_position_embeddings": 10})):
        with pytest.raises(ValueError):
            frequencies(*args)


def test_dynamic_grows_beyond_the_checkpoint_s_positions():
    """As the initialiser that the engine's own models use has it: also where the dictionary names a trained length."""
    from cpmcu.rotary import frequencies
    for trained, top, length in ((4096, 16384, 10000), (4096, 16384, 50000), (8192, 4096, 6000)):
        scaling = {"rope_type": "dynamic", "factor": 4.0, "original_max_position_embeddings": trained}
        inv, _ = frequencies(64, 10000.0, scaling, length=length, max_position=top)
        want, _ = transformers_frequencies(64, 10000.0, scaling, length, top)
        assert float(((inv.double() - want.double()) / want.double()).abs().max()) < 1e-5
    alone, _ = frequencies(64, 10000.0, scaling, length=10000)                       # nothing else is known
    assert torch.equal(alone, frequencies(64, 10000.0, {"rope_type": "dynamic", "factor": 4.0}, length=10000, max_position=8192)[0])


def test_longrope_without_its_factor():
    """It is that of the dictionary, or of the checkpoint's positions to the trained ones; with neither there is no right answer."""
    from cpmcu.rotary import frequencies
    scaling = {"rope_type": "longrope", "short_factor": [1.0] * 4, "long_factor": [2.0] * 4, "original_max_position_embeddings": 4096}
    with pytest.raises(ValueError, match="'factor'"):
        frequencies(8, 10000.0, scaling)
    assert frequencies(8, 10000.0, scaling, max_position=32768)[1] == frequencies(8, 10000.0, {**scaling, "factor": 8.0})[1] > 1
    assert frequencies(8, 10000.0, {**scaling, "attention_factor": 1.25})[1] == 1.25
