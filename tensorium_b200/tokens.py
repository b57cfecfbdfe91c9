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

import importlib.util
from typing import Optional

import torch

from ._lib import ACT, BF16_ELEM, F16_ELEM, F32_ELEM, check, lib
from .build import FAST
from .context import Context


class _NoFast:
    """Stands for the extension where it was not built: no call is plain, all go through Python (10 to 18 us of
    host time instead of 5 to 7, the same kernels and results)."""

    @staticmethod
    def int8_connected(*args):
        return None

    token_logprobs = token_logprobs_backward = int8_connected


def _load_fast():
    if not FAST.exists():
        return _NoFast
    spec = importlib.util.spec_from_file_location(f"{__package__}._tokens_fast", FAST)
    try:
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except ImportError:
        return _NoFast
    return module


_fast = _load_fast()  # ordinary calls, checked and allocated outside Python

_current_stream = torch._C._cuda_getCurrentRawStream
_ELEM = {torch.float32: F32_ELEM, torch.bfloat16: BF16_ELEM, torch.float16: F16_ELEM}


class TokenLogprobs:
    """Results of token_logprobs, a row each, float32: logprobs (None without tokens), entropy, lse, row_max and
    log_sum (lse = row_max / temperature + log_sum; the gradient is taken from the two), and [rows, top]
    top_logprobs and top_tokens (int64; None where not asked for). The first five are rows of `stats`."""
    __slots__ = ("stats", "given", "top_logprobs", "top_tokens")

    def __init__(self, stats, given, top_logprobs=None, top_tokens=None):
        self.stats, self.given, self.top_logprobs, self.top_tokens = stats, given, top_logprobs, top_tokens

    @property
    def logprobs(self) -> Optional[torch.Tensor]:
        return self.stats[0] if self.given else None

    @property
    def entropy(self) -> torch.Tensor:
        return self.stats[1]

    @property
    def lse(self) -> torch.Tensor:
        return self.stats[2]

    @property
    def row_max(self) -> torch.Tensor:
        return self.stats[3]

    @property
    def log_sum(self) -> torch.Tensor:
        return self.stats[4]


def _refuse(ctx, t, name, dtypes):
    """Raises for a tensor that _matrix does not take, saying why."""
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} is not one of {', '.join(map(str, dtypes))}")
    if t.dim() != 2:
        raise ValueError(f"{name}: 2 dimensions are wanted, not {t.dim()}")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name}: on {t.device}, not on the context's GPU {ctx.device}")
    raise ValueError(f"{name}: the last dimension has stride {t.stride(1)}, 1 is wanted")


def _matrix(ctx, t, name, dtypes):
    """(rows, columns, row stride) of a 2-D tensor of this context's GPU."""
    shape = t.shape
    if t.dtype in dtypes and len(shape) == 2 and t.get_device() == ctx.device:
        rows, cols = shape
        stride, inner = t.stride()
        if inner == 1 or cols <= 1:
            return rows, cols, stride if rows > 1 else max(stride, cols)
    _refuse(ctx, t, name, dtypes)


def _vector(ctx, t, name, dtype, n):
    """Address of n contiguous values."""
    if t.dtype is dtype and t.shape == (n,) and t.get_device() == ctx.device and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype or t.shape != (n,):
        raise ValueError(f"{name}: {n} values of {dtype} are wanted, not {tuple(t.shape)} of {t.dtype}")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name}: on {t.device}, not on the context's GPU {ctx.device}")
    raise ValueError(f"{name}: stride {t.stride(0)}, 1 is wanted")


def _torch_stream(ctx):
    """The context's stream as torch's. ExternalStream(0) is not the legacy default stream: without an address
    torch makes a stream of its own."""
    raw = ctx.raw_stream
    return torch.cuda.ExternalStream(raw, device=ctx.torch_device) if raw else torch.cuda.default_stream(ctx.torch_device)


def _empty(ctx, shapes, dtypes, inputs):
    """New tensors for results. Where the calling thread's current torch stream is not the context's, they
    are allocated on the context's, and the inputs' memory is kept until it has passed this call."""
    if ctx.raw_stream == _current_stream(ctx.device):
        return [inputs[0].new_empty(s, dtype=d) for s, d in zip(shapes, dtypes)]
    stream = _torch_stream(ctx)
    for t in inputs:
        if t is not None:
            t.record_stream(stream)
    with torch.cuda.stream(stream):
        return [inputs[0].new_empty(s, dtype=d) for s, d in zip(shapes, dtypes)]


def _result(ctx, out, rows, cols, dtype, inputs):
    """(tensor, row stride) of a result: `out` checked, or a new tensor."""
    if out is None:
        return _empty(ctx, ((rows, cols),), (dtype,), inputs)[0], cols
    out_rows, out_cols, stride = _matrix(ctx, out, "out", (dtype,))
    if out_rows != rows or out_cols != cols:
        raise ValueError(f"out: shape {tuple(out.shape)}, ({rows}, {cols}) is wanted")
    _empty(ctx, (), (), (*inputs, out))
    return out, stride


def _activation(a) -> int:
    if isinstance(a, str):
        if a not in ACT:
            raise ValueError(f"activation {a!r} is not one of {', '.join(ACT)}")
        return ACT[a]
    return int(a)


_INT8 = (torch.int8,)


def quantize_rows(ctx: Context, x: torch.Tensor):
    """(codes, scales) of x [rows, cols]: codes int8 [rows, cols] in rows of whole 16 bytes (the
    layout that the product reads), scales float32 [rows]; x is about codes * scales[:, None]."""
    rows, cols, stride = _matrix(ctx, x, "x", _ELEM)
    pitch = -(-cols // 16) * 16
    codes, scales = _empty(ctx, ((rows, pitch), (rows,)), (torch.int8, torch.float32), (x,))
    check(lib.tb_quantize_rows(ctx.handle, rows, cols, x.data_ptr(), _ELEM[x.dtype], stride, codes.data_ptr(),
                               pitch, scales.data_ptr()))
    return codes[:, :cols], scales


def _pitch(rows, stride):
    return stride if rows > 1 else -(-stride // 16) * 16  # one row has no stride to keep


def int8_product(ctx: Context, a, a_scales, w, w_scales, bias=None, activation="linear",
                 dtype=torch.float32, out=None):
    """act((a . w^T) * a_scales[:, None] * w_scales + bias) of codes a [tokens, k] and w [channels, k],
    both int8 in rows of whole 16 bytes (as quantize_rows gives them), as `dtype` [tokens, channels]."""
    m, k, a_stride = _matrix(ctx, a, "a", _INT8)
    n, kw, w_stride = _matrix(ctx, w, "w", _INT8)
    if k != kw:
        raise ValueError(f"a has {k} columns and w {kw}")
    if dtype not in _ELEM:
        raise ValueError(f"dtype {dtype} is not one of {', '.join(map(str, _ELEM))}")
    sa, sw = _vector(ctx, a_scales, "a_scales", torch.float32, m), _vector(ctx, w_scales, "w_scales", torch.float32, n)
    b = None if bias is None else _vector(ctx, bias, "bias", torch.float32, n)
    y, y_stride = _result(ctx, out, m, n, dtype, (a, a_scales, w, w_scales, bias))
    check(lib.tb_int8_gemm(ctx.handle, m, n, k, a.data_ptr(), _pitch(m, a_stride), sa, w.data_ptr(), _pitch(n, w_stride),
                           sw, b, _activation(activation), y.data_ptr(), _ELEM[dtype], y_stride))
    return y


def int8_connected(ctx: Context, x, w, w_scales, bias=None, activation="linear", dtype=None, out=None):
    """The connected layer on int8 weights: every row of x [tokens, k] is quantized on the way in
    (quantize_rows) and multiplied with w [channels, k] (int8_product). dtype: x's unless given."""
    if dtype is None and out is None:
        y = _fast.int8_connected(ctx.handle.value, ctx.device, ctx.raw_stream, x, w, w_scales, bias, ACT.get(activation, activation))
        if y is not None:
            return y if y.__class__ is not int else check(y)
    m, k, x_stride = _matrix(ctx, x, "x", _ELEM)
    n, kw, w_stride = _matrix(ctx, w, "w", _INT8)
    if k != kw:
        raise ValueError(f"x has {k} columns and w {kw}")
    if dtype is None:
        dtype = x.dtype
    elif dtype not in _ELEM:
        raise ValueError(f"dtype {dtype} is not one of {', '.join(map(str, _ELEM))}")
    sw = _vector(ctx, w_scales, "w_scales", torch.float32, n)
    b = None if bias is None else _vector(ctx, bias, "bias", torch.float32, n)
    y, y_stride = _result(ctx, out, m, n, dtype, (x, w, w_scales, bias))
    check(lib.tb_int8_connected_fwd(ctx.handle, m, n, k, x.data_ptr(), _ELEM[x.dtype], x_stride, w.data_ptr(),
                                    _pitch(n, w_stride), sw, b, _activation(activation), y.data_ptr(), _ELEM[dtype],
                                    y_stride))
    return y


def token_logprobs(ctx: Context, logits, tokens=None, top: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Of the softmax of logits / temperature, logits [rows, vocab]: the log probability of tokens
    (int64 [rows]; negative: none given, 0), the entropy, the log of the sum of exponentials and, with
    top > 0 (at most 32), the most probable tokens in descending order (equal logits: the lowest first)."""
    r = _fast.token_logprobs(ctx.handle.value, ctx.device, ctx.raw_stream, logits, tokens, top, temperature)
    if r is not None:
        return TokenLogprobs(r[0], tokens is not None, r[1], r[2]) if r.__class__ is tuple else check(r)
    rows, vocab, stride = _matrix(ctx, logits, "logits", _ELEM)
    t = None if tokens is None else _vector(ctx, tokens, "tokens", torch.int64, rows)
    if top > 0:
        stats, top_lp, top_tok = _empty(ctx, ((5, rows), (rows, top), (rows, top)), (torch.float32, torch.float32, torch.int64), (logits, tokens))
        lp_at, tok_at = top_lp.data_ptr(), top_tok.data_ptr()
    else:
        stats, = _empty(ctx, ((5, rows),), (torch.float32,), (logits, tokens))
        top_lp = top_tok = lp_at = tok_at = None
    at, step = stats.data_ptr(), 4 * rows
    check(lib.tb_token_logprobs_fwd(ctx.handle, rows, vocab, logits.data_ptr(), _ELEM[logits.dtype], stride, t, temperature,
                                    top, at, at + step, at + 2 * step, at + 3 * step, at + 4 * step, lp_at, tok_at))
    return TokenLogprobs(stats, tokens is not None, top_lp, top_tok)


def token_logprobs_backward(ctx: Context, logits, tokens, forward: TokenLogprobs, grad_logprobs=None,
                            grad_entropy=None, temperature: float = 1.0, out=None):
    """Gradient with respect to the logits of sum(grad_logprobs * logprobs + grad_entropy * entropy),
    from token_logprobs' results on the same logits, tokens and temperature (float32 gradients, a row
    each; None: 0). out may be the logits themselves."""
    if out is None:
        d = _fast.token_logprobs_backward(ctx.handle.value, ctx.device, ctx.raw_stream, logits, tokens, forward.stats,
                                          grad_logprobs, grad_entropy, temperature)
        if d is not None:
            return d if d.__class__ is not int else check(d)
    rows, vocab, stride = _matrix(ctx, logits, "logits", _ELEM)
    if grad_logprobs is not None and tokens is None:
        raise ValueError("grad_logprobs without tokens")
    f32 = torch.float32
    t = None if tokens is None else _vector(ctx, tokens, "tokens", torch.int64, rows)
    gl = None if grad_logprobs is None else _vector(ctx, grad_logprobs, "grad_logprobs", f32, rows)
    gh = None if grad_entropy is None else _vector(ctx, grad_entropy, "grad_entropy", f32, rows)
    stats = forward.stats
    if stats.shape != (5, rows) or stats.get_device() != ctx.device:
        raise ValueError(f"forward: results of {stats.shape[1]} rows on {stats.device}, {rows} on GPU {ctx.device} are wanted")
    at, step = stats.data_ptr(), 4 * rows
    d, d_stride = _result(ctx, out, rows, vocab, logits.dtype, (logits, tokens, stats, grad_logprobs, grad_entropy))
    check(lib.tb_token_logprobs_bwd(ctx.handle, rows, vocab, logits.data_ptr(), _ELEM[logits.dtype], stride, t, temperature,
                                    at + 3 * step, at + 4 * step, at + step, gl, gh, d.data_ptr(), d_stride))
    return d
