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


@pytest.mark.parametrize("device,want", [(0, torch.device("cuda", 0)), (2, torch.device("cuda", 2)), ("cuda:0", torch.device("cuda", 0)),
                                         (None, torch.device("cuda", 1))])
def test_weights_are_laid_out_on_the_device_that_is_named(monkeypatch, device, want):
    """By its number too: 0 is a device, not "wherever the codes are"."""
    from qk_b200 import fp8

    class Codes:  # on the second GPU
        is_cuda, device, dtype = True, torch.device("cuda", 1), torch.float8_e4m3fn

        def to(self, device):
            self.moved = device
            return self

    monkeypatch.setattr(fp8, "_quantised", lambda codes, scales, by_rows, name: (codes, 0, scales))
    assert fp8.fp8_weights(Codes(), None, device).codes.moved == want
