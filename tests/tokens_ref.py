"""Plain implementations in 64 bits of the int8 connected layer and the token log probabilities, and
the error that the 32-bit kernels may have against them."""
import numpy as np

U = 2.0 ** -24                                    # half a unit in the last place of float32
HALF_ULP = {"float32": U, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # significands of 24, 8 and 11 bits
TINY = {"float32": 2.0 ** -126, "bfloat16": 2.0 ** -126, "float16": 2.0 ** -24}


def quantize(x):
    """(codes, scales) of rows: the definition's 32-bit operations, each rounded once (a product or
    quotient of two float32 taken in float64 and rounded to float32 is rounded correctly)."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x).all(1)
    amax = np.maximum(np.abs(np.where(np.isfinite(x), x, 0)).max(1), 2.0 ** -100)
    factor = (127.0 / amax).astype(np.float32).astype(np.float64)
    scales = (amax / 127.0).astype(np.float32)
    prod = (np.where(np.isfinite(x), x, 0) * factor[:, None]).astype(np.float32)
    codes = np.rint(prod).astype(np.int8)
    codes[bad] = 0
    scales[bad] = np.nan
    return codes, scales


ACTS = {
    "linear": lambda v: v,
    "relu": lambda v: np.where(v > 0, v, 0),
    "leaky": lambda v: np.where(v < 0, v * np.float64(np.float32(0.1)), v),
    "logistic": lambda v: 1 / (1 + np.exp(-v)),
    "elu": lambda v: np.where(v >= 0, v, np.expm1(v)),
    "hardtan": lambda v: np.clip(v, -1, 1),
}


def product(a, sa, w, sw, bias, act, out_type):
    """(y, how far a 32-bit epilogue may be off): the int32 sum is exact; its conversion, the two
    scale products, the bias and the activation are one rounding each, the output's type one more."""
    acc = np.asarray(a, np.float64) @ np.asarray(w, np.float64).T
    v = acc * (np.asarray(sa, np.float64)[:, None] * np.asarray(sw, np.float64))
    off = 3 * U * np.abs(v)
    if bias is not None:
        b = np.asarray(bias, np.float64)
        off = off + U * (np.abs(v) + np.abs(b))
        v = v + b
    y = ACTS[act](v)
    off = 1.01 * (off + 2 * U * np.abs(v))  # every activation here has a slope of at most 1
    return y, off + 1.01 * HALF_ULP[out_type] * (np.abs(y) + off) + TINY[out_type]


def logprobs(logits, tokens, temperature, top):
    """dict of logprobs, entropy, lse, top_tokens, top_logprobs and the whole log softmax."""
    l = np.asarray(logits, np.float64)
    rows, vocab = l.shape
    z = l / np.float64(np.float32(temperature))
    bad = (np.isnan(z) | (z == np.inf)).any(1)
    m = np.where(bad, 0, np.where(np.isnan(z), 0, z).max(1))
    empty = ~bad & (m == -np.inf)
    m = np.where(empty, 0, m)
    with np.errstate(all="ignore"):
        e = np.exp(z - m[:, None])
        lse = m + np.log(e.sum(1))
        lp = (z - m[:, None]) - np.log(e.sum(1))[:, None]  # z - lse loses log Z beside large logits
        p = np.exp(lp)
        h = -np.where(p > 0, p * lp, 0).sum(1)
    lse[empty], h[empty], lp[empty] = -np.inf, 0, -np.inf
    lse[bad], h[bad], lp[bad] = np.nan, np.nan, np.nan
    order = np.stack([np.lexsort((np.arange(vocab), -(r + 0.0)))[:top] for r in np.where(np.isnan(l), np.inf, l)]) if rows else np.zeros((0, top), int)
    tops = np.take_along_axis(lp, order, 1) if rows else np.zeros((0, top))
    order = np.where(bad[:, None], -1, order)
    out = {"entropy": h, "lse": lse, "row_max": np.where(bad, np.nan, np.where(empty, -np.inf, m)), "lp": lp, "top_tokens": order, "top_logprobs": tops}
    if tokens is not None:
        t = np.asarray(tokens)
        got = lp[np.arange(rows), np.clip(t, 0, vocab - 1)]
        out["logprobs"] = np.where(t >= vocab, np.nan, np.where(t < 0, np.where(bad, np.nan, 0), got))
    return out


def sum_off(vocab):
    """Relative error of the sum of exponentials in 32 bits: additions in chains of at most vocab / 128
    and a tree, each exponential off by (4 |argument| + 4) half units, arguments that matter under 32."""
    return (vocab / 128 + 32 + 4 * 32 + 4) * U


def logprob_off(lp, lse, vocab):
    with np.errstate(all="ignore"):
        return np.where(np.isfinite(lp), sum_off(vocab) + 4 * U * (np.abs(lp) + np.abs(np.log(vocab)) + 1), 0)


def entropy_off(h, vocab):
    # log Z - S / Z: both quotient's sums off by sum_off, S / Z as large as log(vocab) + H at most
    return np.where(np.isfinite(h), 3 * sum_off(vocab) * (1 + np.log(vocab)), 0)


def gradient(logits, tokens, temperature, a, b):
    """(d, how far off) of sum(a * logprob + b * entropy); a, b None for 0."""
    l = np.asarray(logits, np.float64)
    rows, vocab = l.shape
    r = logprobs(l, tokens, temperature, 0)
    lp, h = r["lp"], r["entropy"]
    p = np.exp(lp)
    t = np.full(rows, -1) if tokens is None or a is None else np.asarray(tokens)
    a = np.zeros(rows) if a is None else np.where(t >= 0, np.asarray(a, np.float64), 0)
    b = np.zeros(rows) if b is None else np.asarray(b, np.float64)
    with np.errstate(all="ignore"):
        inner = a[:, None] + np.where(p > 0, b[:, None] * (lp + h[:, None]), 0)
        parts = np.abs(a)[:, None] + np.where(p > 0, np.abs(b)[:, None] * (np.abs(lp) + np.abs(h)[:, None]), 0)
    hit = (t[:, None] == np.arange(vocab)) * a[:, None]
    T = np.float64(np.float32(temperature))
    d = (hit - p * inner) / T
    with np.errstate(all="ignore"):
        rel = sum_off(vocab) + 4 * U * (np.where(p > 0, np.abs(lp), 0) + np.log(vocab) + 2)
        off = (p * parts * (rel + 8 * U) + p * np.abs(b)[:, None] * (entropy_off(h, vocab)[:, None] + rel) + 4 * U * (np.abs(hit) + p * parts)) / T
    empty = r["lse"] == -np.inf
    d[empty], off[empty] = 0, 0
    bad = np.isnan(r["lse"]) | (t >= vocab)
    d[bad], off[bad] = np.nan, 0
    return d, off
