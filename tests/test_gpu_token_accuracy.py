"""How many digits the token log probabilities keep, over their launch forms: bounds from the terms of each row
instead of one for all, so that a lost bit shows.

With t the exponents of a row below its maximum (in nats), Z = sum e^t, H = ln Z - <t>, u = 2^-24, one rounding is off by at most u
of its result, and by 0.58 u (a uniform error's standard deviation) in the mean. What follows the sums: ln Z to 1 unit in the last
place (2 u), the quotient, its product with ln 2, the difference (u each of <t>, <t> and H). The exponent's constant is off
by 0.25 u, which moves H by that times the variance of t. The terms' own errors (2^-22 for the exponential) are independent, as are
the additions' in the chains that a sum is made of: they stay below u of Z and of <t> Z.
"""
import numpy as np
import pytest
import torch

from tensorium_b200 import tokens as K

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = 2.0 ** -24
# a warp to a row, two, four and eight; rows in parts; loads ahead of the sums; several rows to a warp
FORMS = [(2048, 32000), (4096, 6000), (512, 131072), (777, 50001), (150, 131075), (64, 50001), (700, 9001), (6000, 1000), (9000, 80)]


def rows_of(rows, vocab, dtype, surplus=None):
    """Flat to peaked rows; surplus: one token's logit is that many nats above the log of the others' sum."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = torch.randn(rows, vocab, device="cuda", generator=g)
    logits *= 1 + 3 * torch.rand(rows, 1, device="cuda", generator=g)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    if surplus:
        logits.scatter_(1, tokens[:, None], torch.logsumexp(logits, 1, keepdim=True) + surplus)
    return logits.to(TYPES[dtype]), tokens


def exact(logits, tokens):
    """(log probability, entropy, ln Z, <t>, variance of t) of each row, in 64 bits."""
    out = []
    for i in range(0, len(logits), 256):
        t = logits[i:i + 256].double()
        t = t - t.amax(1, keepdim=True)
        z = t.exp().sum(1)
        p = t.exp() / z[:, None]
        mean = (p * t).sum(1)
        lp = t.gather(1, tokens[i:i + 256, None])[:, 0] - z.log()
        out.append(torch.stack([lp, z.log() - mean, z.log(), mean, (p * t * t).sum(1) - mean * mean]))
    return torch.cat(out, 1).cpu().numpy()


def f64(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_entropy(ctx, rows, vocab, dtype):
    logits, tokens = rows_of(rows, vocab, dtype)
    _, h, log_z, mean, var = exact(logits, tokens)
    for top in (0, 5):
        r = K.token_logprobs(ctx, logits, tokens, top=top)
        off = np.abs(f64(r.entropy) - h) / (U * (log_z + np.abs(mean) + h + var / 4 + 1))
        assert np.sqrt(np.mean(off * off)) <= 1.25, np.sqrt(np.mean(off * off))
        assert off.max() <= 8, off.max()


@pytest.mark.parametrize("surplus", [13.0, 18.0, 30.0])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])  # half precision has no room for the second one's logit
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_rows_sure_of_their_token(ctx, rows, vocab, dtype, surplus):
    """Z is 1 and little: nothing before the sums' ends can be off by more than a few units of 1, and no log probability
    is above 0."""
    logits, tokens = rows_of(rows, vocab, dtype, surplus)
    lp, h, _, _, _ = exact(logits, tokens)
    for top in (0, 1, 5):
        r = K.token_logprobs(ctx, logits, tokens, top=top)
        assert (r.logprobs <= 0).all() and (r.log_sum >= 0).all() and (r.entropy >= 0).all()
        if top:
            assert (r.top_logprobs <= 0).all() and torch.equal(r.top_tokens[:, 0], tokens)
            assert not torch.isnan(torch.log1p(-r.top_logprobs.exp())).any()
        for got, ref in ((r.entropy, h), (r.logprobs, lp)):
            off = np.abs(f64(got) - ref)
            assert np.sqrt(np.mean(off * off)) <= 4 * U, np.sqrt(np.mean(off * off)) / U
            assert np.all(off <= 16 * U + 1e-4 * h), off.max() / U
