"""MXFP4 operators without a GPU: the reference itself, refusals that need no device."""
import numpy as np
import pytest
import torch

import mx4_reference as ref
from oracle import oracle
from oxidized_gpt_oss_b200 import abi, ffn, mxfp4


def test_reference_quantiser_against_the_nearest_value_and_the_oracle():
    """The reference's codes are the nearest MXFP4 values (no other code is closer), and read back through the
    dequantisation oracle they are the values that they stand for."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((5, 96)) * np.exp(2 * rng.standard_normal((5, 96)))).astype(np.float32)
    for rule in ("floor", "noclip"):
        codes, scales = ref.quantize(x, rule)
        step = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, 1)
        got = np.concatenate([ref.E2M1, -ref.E2M1])[codes] * step
        every = ref.E2M1[None, None, :] * step[..., None]
        assert np.array_equal(np.abs(np.abs(x) - np.abs(got)), np.abs(np.abs(x)[..., None] - every).min(-1))
        back = oracle.dequantize_mxfp4_e8m0(ref.pack(codes).ravel(), scales.ravel(), 5, 96)
        assert np.array_equal((back.astype(np.uint32) << 16).view(np.float32).reshape(5, 96), got.astype(np.float32))
        if rule == "noclip":
            assert np.abs(x / step).max() <= 6


def test_null_context_is_refused():
    lib = abi.load()
    for st in (lib.oxg_quantize_mxfp4(None, None, 0, 1, 32, 32, None, 0, 0, None, None),
               lib.oxg_swiglu_quantize_mxfp4(None, None, 0, 1, 32, 64, 1.702, 7.0, 0, 0, None, None),
               lib.oxg_mxfp4_tile_scales(None, None, 1, 1, 32, None),
               lib.oxg_mxfp4_matmul(None, None, None, 1, None, None, 1, 32, None, None, 0, 1),
               lib.oxg_mxfp4_grouped_matmul(None, None, None, 1, None, 1, None, None, 1, 32, None, None, 0, 1)):
        assert st == abi.OXG_ERR_INVALID_ARG
        assert lib.oxg_last_error(None) == b"ctx is NULL"


def test_host_tensors_are_refused():
    x = torch.zeros(2, 64)
    b, s = torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(1, 2, 4, dtype=torch.uint8)
    for call in (lambda: mxfp4.quantize_mxfp4(x), lambda: ffn.swiglu_quantize_mxfp4(x), lambda: mxfp4.tile_scales(s),
                 lambda: mxfp4.mxfp4_matmul(b, s, b, s),
                 lambda: mxfp4.mxfp4_grouped_matmul(b, s, torch.zeros(1, dtype=torch.int32), b[None], s[None])):
        with pytest.raises(ValueError, match="CUDA"):
            call()
