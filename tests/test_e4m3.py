"""The plain functions of the cache in 8 bits against torch's own 8-bit type, and what the operators refuse on the host."""

import numpy as np
import pytest
import torch

import plain_e4m3 as plain


def test_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(plain.VALUES, codes)
    rng = np.random.default_rng(1)
    x = np.concatenate((rng.normal(0, 1, 4000) * 2.0 ** rng.uniform(-12, 8, 4000), plain.VALUES[np.isfinite(plain.VALUES)],
                        (plain.VALUES[:126] + plain.VALUES[1:127]) / 2))
    x = np.clip(x, -448.0, 448.0).astype(np.float32)
    want = torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(plain.nearest_code(x), want)


def test_sizes():
    from mini_llm_b200.kernels import ops
    assert ops.e4m3_sizes_take(64, 64, 64) and ops.e4m3_sizes_take(16, 256, 16) and ops.e4m3_sizes_take(96, 48, 112)
    for sizes in ((0, 64, 64), (64, 24, 64), (64, 64, 8), (64, 64, 24), (272, 64, 64), (64, 512, 64), (64, 64, 0), (8, 64, 64)):
        assert not ops.e4m3_sizes_take(*sizes)


def test_there_is_no_path_on_the_host():
    from mini_llm_b200.kernels import ops
    from mini_llm_b200.kernels.lib import KernelError
    pages, scales = torch.zeros((2, 1, 16, 64), dtype=torch.float8_e4m3fn), torch.zeros((2, 1, 1))
    ints = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros((1, 64), dtype=torch.bfloat16)
    with pytest.raises(KernelError, match="CUDA tensor"):
        ops.e4m3_attention(q, q, pages, pages, scales, scales, ints[None], ints, ints, ints, 1, 1, 1.0, plain=True)
    with pytest.raises(KernelError, match="CUDA tensor"):
        ops.e4m3_store(None, torch.zeros((1, 192)), 64, 128, 1, 1, 64, 64, 0, None, 1.0, ints, ints, ints[None], pages, pages, scales, scales)


def test_which_mixers_take_a_cache_in_8_bits():
    import deluvik_helpers
    import fuvolix_helpers
    import lipulorn_helpers
    import sumozen_helpers
    from mini_llm_b200.config import config_from_dict, describe_model
    from mini_llm_b200.engine.model import Model
    from mini_llm_b200.parts.base import Mixer
    from tiny_configs import TINY_A

    def refused(raw):
        return {type(p).__name__ for p in Model(describe_model(config_from_dict(raw))).parts() if isinstance(p, Mixer) and not p.takes_e4m3_cache()}

    assert refused(TINY_A) == set() and refused(sumozen_helpers.full_stack()) == set()
    assert refused(fuvolix_helpers.config([fuvolix_helpers.mlstm()])) == set()              # (keeps no pages)
    assert refused(fuvolix_helpers.full_stack()) == {"LatentAttention"}
    assert "GatedAttention" in refused(lipulorn_helpers.full_stack()) and "NormedAttention" in refused(deluvik_helpers.full_stack())
