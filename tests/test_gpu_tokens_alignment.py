"""The token operators' C entry points turn an address that is not a multiple of its element's size into an error: each
argument in turn, the others as they should be."""
import pytest
import torch

from tensorium_b200._lib import TB_ERR_INVALID, TB_OK, lib

pytestmark = pytest.mark.gpu
ROWS, COLS, N = 3, 32, 48


@pytest.fixture()
def buf():
    """Zeroed device memory for every argument, 4 KB each."""
    return torch.zeros(24, 4096, dtype=torch.uint8, device="cuda")


def each_misaligned(ctx, call, args, sizes):
    """call(*args) works; with the address of any argument in `sizes` (position: element's size) moved by half an
    element it is refused."""
    assert call(ctx.handle, *args) == TB_OK, lib.tb_last_error()
    for i, size in sizes.items():
        off = list(args)
        off[i] += size // 2
        assert call(ctx.handle, *off) == TB_ERR_INVALID, i
        assert b"misaligned" in lib.tb_last_error() or b"multiples of 16" in lib.tb_last_error(), i
    ctx.sync()


def test_product(ctx, buf):
    p = [b.data_ptr() for b in buf]
    args = (ROWS, N, COLS, p[0], COLS, p[1], p[2], COLS, p[3], p[4], 4, p[5], 0, N)
    each_misaligned(ctx, lib.tb_int8_gemm, args, {3: 16, 5: 4, 6: 16, 8: 4, 9: 4, 11: 4})


def test_connected(ctx, buf):
    p = [b.data_ptr() for b in buf]
    args = (ROWS, N, COLS, p[0], 1, COLS, p[2], COLS, p[3], p[4], 4, p[5], 2, N)
    each_misaligned(ctx, lib.tb_int8_connected_fwd, args, {3: 2, 6: 16, 8: 4, 9: 4, 11: 2})


def test_quantize(ctx, buf):
    p = [b.data_ptr() for b in buf]
    each_misaligned(ctx, lib.tb_quantize_rows, (ROWS, COLS, p[0], 0, COLS, p[1] + 1, COLS, p[2]), {2: 4, 7: 4})  # codes: any address


def test_logprobs(ctx, buf):
    p = [b.data_ptr() for b in buf]
    args = (ROWS, COLS, p[0], 2, COLS, p[1], 1.0, 4, *p[2:9])
    each_misaligned(ctx, lib.tb_token_logprobs_fwd, args, {2: 2, 5: 8, 8: 4, 9: 4, 10: 4, 11: 4, 12: 4, 13: 4, 14: 8})


def test_gradient(ctx, buf):
    p = [b.data_ptr() for b in buf]
    args = (ROWS, COLS, p[0], 0, COLS, p[1], 1.0, p[2], p[3], p[4], p[5], p[6], p[7], COLS)
    each_misaligned(ctx, lib.tb_token_logprobs_bwd, args, {2: 4, 5: 8, 7: 4, 8: 4, 9: 4, 10: 4, 11: 4, 12: 4})
