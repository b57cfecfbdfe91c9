"""What the token operators' Python entry points refuse before they reach a GPU."""
import ctypes
import types

import pytest
import torch

from tensorium_b200 import _lib
from tensorium_b200 import tokens as K

CTX = types.SimpleNamespace(device=0, handle=ctypes.c_void_p(), raw_stream=0)  # a closed context


def test_tensors_that_are_not_on_the_gpu():
    x, w = torch.zeros(2, 16), torch.zeros(3, 16, dtype=torch.int8)
    s = torch.zeros(3)
    with pytest.raises(ValueError, match="not on the context's GPU"):
        K.int8_connected(CTX, x, w, s)
    with pytest.raises(ValueError, match="not on the context's GPU"):
        K.quantize_rows(CTX, x)
    with pytest.raises(ValueError, match="not on the context's GPU"):
        K.token_logprobs(CTX, x, torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("bad", [torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.float64), torch.zeros(3), torch.zeros(1, 2, 3)])
def test_types_and_dimensions(bad):
    for call in (lambda: K.quantize_rows(CTX, bad), lambda: K.token_logprobs(CTX, bad)):
        with pytest.raises(ValueError):
            call()


def test_activation_names():
    assert K._activation("leaky") == _lib.ACT["leaky"] and K._activation(4) == 4
    with pytest.raises(ValueError):
        K._activation("swish")


def test_null_context():
    lib = _lib.lib
    assert lib.tb_quantize_rows(None, 1, 1, None, 0, 1, None, 1, None) == _lib.TB_ERR_INVALID
    assert lib.tb_int8_gemm(None, 1, 1, 1, None, 16, None, None, 16, None, None, 4, None, 0, 1) == _lib.TB_ERR_INVALID
    assert lib.tb_int8_connected_fwd(None, 1, 1, 1, None, 0, 1, None, 16, None, None, 4, None, 0, 1) == _lib.TB_ERR_INVALID
    assert lib.tb_token_logprobs_fwd(None, 1, 1, None, 0, 1, None, 1.0, 0, None, None, None, None, None, None, None) == _lib.TB_ERR_INVALID
    assert lib.tb_token_logprobs_bwd(None, 1, 1, None, 0, 1, None, 1.0, None, None, None, None, None, None, 1) == _lib.TB_ERR_INVALID
