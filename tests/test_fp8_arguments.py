"""FP8 dense path: arguments that the entry points refuse or take, beyond the first list of refusals (no GPU)."""

import ctypes

import pytest
import torch

from test_fp8_refusals import GOOD, p


@pytest.mark.parametrize("name,at", [("qk_fp8_rms_norm", 9), ("qk_fp8_quantize", 7), ("qk_fp8_quantize_blocks", 7), ("qk_fp8_gated", 14)])
@pytest.mark.parametrize("address", [17, 18, 19])
def test_scales_off_four_bytes_are_refused(name, at, address):
    """Every entry point that writes scales stores them as FP32: an address off 4 bytes would fault."""
    from qk_b200 import _lib

    args = list(GOOD[name])
    args[at] = p(address)
    assert getattr(_lib.load(), name)(*args) == _lib.QK_ERR_INVALID_ARGUMENT, _lib.last_error()
