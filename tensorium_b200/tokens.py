"""The head of a network that answers with tokens: the connected layer on int8 weights and what a
program reads off its logits.

    quantize_rows             codes and a scale for each row (a token of x, an output channel of weights)
    int8_product              codes . codes with a scale for each token and channel, bias, activation
    int8_connected            the same from unquantized x, as a connected layer's forward
    token_logprobs            log probability of given tokens, entropy, most probable tokens
    token_logprobs_backward   gradient of the first two with respect to the logits

Tensors are float32, bfloat16 or float16 on the context's GPU, with any row stride; a last
dimension of stride 1 is asked for, not made.  Everything is launched on the context's stream: inputs
written on another one have to be finished or waited for there first.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import ACT, BF16_ELEM, F16_ELEM, F32_ELEM, check, lib
from .context import Context

_ELEM = {torch.float32: F32_ELEM, torch.bfloat16: BF16_ELEM, torch.float16: F16_ELEM}


class TokenLogprobs(NamedTuple):
    """Results of token_logprobs, a row each: float32, top_tokens int64 (None where not asked for).
    lse = row_max / temperature + log_sum; the gradient is taken from the two."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    lse: torch.Tensor
    row_max: torch.Tensor
    log_sum: torch.Tensor
    top_logprobs: Optional[torch.Tensor] = None
    top_tokens: Optional[torch.Tensor] = None


class _Stream:
    """Allocates results on the context's stream, and keeps the inputs' memory for it, where the
    calling thread's current torch stream is another one."""

    def __init__(self, ctx, inputs):
        self.guard = None
        raw = ctx.raw_stream
        if raw != torch._C._cuda_getCurrentRawStream(ctx.device):
            s = torch.cuda.ExternalStream(raw, device=ctx.torch_device)
            for t in inputs:
                if t is not None:
                    t.record_stream(s)
            self.guard = torch.cuda.stream(s)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _matrix(ctx, t, name, dtypes):
    """Row stride of a 2-D tensor of this context's GPU."""
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} is not one of {', '.join(map(str, dtypes))}")
    if t.dim() != 2:
        raise ValueError(f"{name}: 2 dimensions are wanted, not {t.dim()}")
    if not t.is_cuda or t.get_device() != ctx.device:
        raise ValueError(f"{name}: on {t.device}, not on the context's GPU {ctx.device}")
    rows, cols = t.shape
    stride, inner = t.stride()
    if cols > 1 and inner != 1:
        raise ValueError(f"{name}: the last dimension has stride {inner}, 1 is wanted")
    return stride if rows > 1 else max(stride, cols)


def _vector(ctx, t, name, dtype, n):
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: {n} values of {dtype} are wanted, not {tuple(t.shape)} of {t.dtype}")
    if not t.is_cuda or t.get_device() != ctx.device:
        raise ValueError(f"{name}: on {t.device}, not on the context's GPU {ctx.device}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name}: stride {t.stride(0)}, 1 is wanted")
    return t.data_ptr()


def _opt(ctx, t, name, dtype, n):
    return None if t is None else _vector(ctx, t, name, dtype, n)


def _activation(a) -> int:
    if isinstance(a, str):
        if a not in ACT:
            raise ValueError(f"activation {a!r} is not one of {', '.join(ACT)}")
        return ACT[a]
    return int(a)


_INT8 = (torch.int8,)
_FLOAT = tuple(_ELEM)


def _result(ctx, out, rows, cols, dtype):
    """(tensor, row stride) of a result: `out` checked, or a new tensor."""
    if out is None:
        return torch.empty((rows, cols), dtype=dtype, device=ctx.torch_device), cols
    stride = _matrix(ctx, out, "out", (dtype,))
    if out.shape[0] != rows or out.shape[1] != cols:
        raise ValueError(f"out: shape {tuple(out.shape)}, ({rows}, {cols}) is wanted")
    return out, stride


def quantize_rows(ctx: Context, x: torch.Tensor):
    """(codes, scales) of x [rows, cols]: codes int8 [rows, cols] in rows of whole 16 bytes (the
    layout that the product reads), scales float32 [rows]; x is about codes * scales[:, None]."""
    stride = _matrix(ctx, x, "x", _FLOAT)
    rows, cols = x.shape
    pitch = -(-cols // 16) * 16
    with _Stream(ctx, (x,)):
        codes = torch.empty((rows, pitch), dtype=torch.int8, device=ctx.torch_device)
        scales = torch.empty((rows,), dtype=torch.float32, device=ctx.torch_device)
    check(lib.tb_quantize_rows(ctx.handle, rows, cols, x.data_ptr(), _ELEM[x.dtype], stride, codes.data_ptr(),
                               pitch, scales.data_ptr()))
    return codes[:, :cols], scales


def int8_product(ctx: Context, a, a_scales, w, w_scales, bias=None, activation="linear",
                 dtype=torch.float32, out=None):
    """act((a . w^T) * a_scales[:, None] * w_scales + bias) of codes a [tokens, k] and w [channels, k],
    both int8 in rows of whole 16 bytes (as quantize_rows gives them), as `dtype` [tokens, channels]."""
    a_stride, w_stride = _matrix(ctx, a, "a", _INT8), _matrix(ctx, w, "w", _INT8)
    (m, k), (n, kw) = a.shape, w.shape
    if k != kw:
        raise ValueError(f"a has {k} columns and w {kw}")
    if dtype not in _ELEM:
        raise ValueError(f"dtype {dtype} is not one of {', '.join(map(str, _FLOAT))}")
    sa, sw = _vector(ctx, a_scales, "a_scales", torch.float32, m), _vector(ctx, w_scales, "w_scales", torch.float32, n)
    b = _opt(ctx, bias, "bias", torch.float32, n)
    with _Stream(ctx, (a, a_scales, w, w_scales, bias, out)):
        y, y_stride = _result(ctx, out, m, n, dtype)
    check(lib.tb_int8_gemm(ctx.handle, m, n, k, a.data_ptr(), _pitch(m, a_stride), sa, w.data_ptr(), _pitch(n, w_stride),
                           sw, b, _activation(activation), y.data_ptr(), _ELEM[dtype], y_stride))
    return y


def _pitch(rows, stride):
    return stride if rows > 1 else -(-stride // 16) * 16  # one row has no stride to keep


def int8_connected(ctx: Context, x, w, w_scales, bias=None, activation="linear", dtype=None, out=None):
    """The connected layer on int8 weights: every row of x [tokens, k] is quantized on the way in
    (quantize_rows) and multiplied with w [channels, k] (int8_product). dtype: x's unless given."""
    x_stride, w_stride = _matrix(ctx, x, "x", _FLOAT), _matrix(ctx, w, "w", _INT8)
    (m, k), (n, kw) = x.shape, w.shape
    if k != kw:
        raise ValueError(f"x has {k} columns and w {kw}")
    if dtype is None:
        dtype = x.dtype
    elif dtype not in _ELEM:
        raise ValueError(f"dtype {dtype} is not one of {', '.join(map(str, _FLOAT))}")
    sw, b = _vector(ctx, w_scales, "w_scales", torch.float32, n), _opt(ctx, bias, "bias", torch.float32, n)
    with _Stream(ctx, (x, w, w_scales, bias, out)):
        y, y_stride = _result(ctx, out, m, n, dtype)
    check(lib.tb_int8_connected_fwd(ctx.handle, m, n, k, x.data_ptr(), _ELEM[x.dtype], x_stride, w.data_ptr(),
                                    _pitch(n, w_stride), sw, b, _activation(activation), y.data_ptr(), _ELEM[dtype],
                                    y_stride))
    return y


def token_logprobs(ctx: Context, logits, tokens=None, top: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Of the softmax of logits / temperature, logits [rows, vocab]: the log probability of tokens
    (int64 [rows]; negative: none given, 0), the entropy, the log of the sum of exponentials and, with
    top > 0 (at most 32), the most probable tokens in descending order (equal logits: the lowest first)."""
    stride = _matrix(ctx, logits, "logits", _FLOAT)
    rows, vocab = logits.shape
    t = _opt(ctx, tokens, "tokens", torch.int64, rows)
    with _Stream(ctx, (logits, tokens)):
        logprobs, entropy, lse, row_max, log_sum = torch.empty((5, rows), dtype=torch.float32, device=ctx.torch_device).unbind()
        top_lp = top_tok = None
        if top > 0:
            top_lp = torch.empty((rows, top), dtype=torch.float32, device=ctx.torch_device)
            top_tok = torch.empty((rows, top), dtype=torch.int64, device=ctx.torch_device)
    check(lib.tb_token_logprobs_fwd(ctx.handle, rows, vocab, logits.data_ptr(), _ELEM[logits.dtype], stride, t, temperature,
                                    top, logprobs.data_ptr(), entropy.data_ptr(), lse.data_ptr(), row_max.data_ptr(), log_sum.data_ptr(),
                                    None if top_lp is None else top_lp.data_ptr(),
                                    None if top_tok is None else top_tok.data_ptr()))
    return TokenLogprobs(None if tokens is None else logprobs, entropy, lse, row_max, log_sum, top_lp, top_tok)


def token_logprobs_backward(ctx: Context, logits, tokens, forward: TokenLogprobs, grad_logprobs=None,
                            grad_entropy=None, temperature: float = 1.0, out=None):
    """Gradient with respect to the logits of sum(grad_logprobs * logprobs + grad_entropy * entropy),
    from token_logprobs' results on the same logits, tokens and temperature (float32 gradients, a row
    each; None: 0). out may be the logits themselves."""
    stride = _matrix(ctx, logits, "logits", _FLOAT)
    rows, vocab = logits.shape
    if grad_logprobs is not None and tokens is None:
        raise ValueError("grad_logprobs without tokens")
    t = _opt(ctx, tokens, "tokens", torch.int64, rows)
    f32 = torch.float32
    m, s = _vector(ctx, forward.row_max, "row_max", f32, rows), _vector(ctx, forward.log_sum, "log_sum", f32, rows)
    ent = _vector(ctx, forward.entropy, "entropy", f32, rows)
    gl, gh = _opt(ctx, grad_logprobs, "grad_logprobs", f32, rows), _opt(ctx, grad_entropy, "grad_entropy", f32, rows)
    with _Stream(ctx, (logits, tokens, forward.row_max, forward.log_sum, forward.entropy, grad_logprobs, grad_entropy, out)):
        d, d_stride = _result(ctx, out, rows, vocab, logits.dtype)
    check(lib.tb_token_logprobs_bwd(ctx.handle, rows, vocab, logits.data_ptr(), _ELEM[logits.dtype], stride, t, temperature,
                                    m, s, ent, gl, gh, d.data_ptr(), d_stride))
    return d
