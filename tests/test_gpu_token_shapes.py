"""The token operators over the shapes that their launch rules tell apart: every number of warps to a row, rows in
parts, loads ahead; tiles of the product whole and shared out, pairs of CTAs on several tiles, few tokens with
fewer steps of k than warps. Larger than a 64-bit check of everything allows: samples of the rows and
columns are checked."""
import numpy as np
import pytest
import torch

import tokens_ref as R
from tensorium_b200 import tokens as K

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def f64(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab", [(5000, 3301), (5200, 6600), (3700, 2100), (1700, 9001), (800, 20003), (777, 50001), (700, 40000), (1200, 70000),
                                        (150, 30000), (90, 131072), (30, 131075), (296, 9000), (297, 9000), (2960, 1500), (2959, 1500)])
def test_logprobs(ctx, rows, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = torch.randn(rows, vocab, device="cuda", generator=g)
    logits *= 1 + 3 * torch.rand(rows, 1, device="cuda", generator=g)
    logits[rows // 2] = torch.where(torch.rand(vocab, device="cuda", generator=g) < 0.6, -torch.inf, logits[rows // 2])
    logits[rows // 3] = -torch.inf
    logits[rows // 4] = 0.25
    logits[rows - 2, : vocab - 3] = -torch.inf
    logits = logits.to(TYPES[dtype])
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    picks = sorted({0, 1, rows // 2, rows // 3, rows // 4, rows - 2, rows - 1, *np.random.default_rng(rows).integers(0, rows, 8).tolist()})
    e = R.logprobs(f64(logits[picks]), tokens[picks].cpu().numpy(), 0.9, 20)
    for top in (0, 1, 7, 20):
        r = K.token_logprobs(ctx, logits, tokens, top=top, temperature=0.9)
        for name, off in (("logprobs", R.logprob_off(e["logprobs"], e["lse"], vocab)), ("entropy", R.entropy_off(e["entropy"], vocab)),
                          ("lse", R.logprob_off(e["lse"], e["lse"], vocab))):
            got, ref = f64(getattr(r, name)[picks]), e[name]
            fin = np.isfinite(ref)
            assert np.array_equal(got[~fin], ref[~fin], equal_nan=True), (name, top)
            assert np.all(np.abs(got - ref)[fin] <= off[fin]), (name, top)
        if top:
            assert np.array_equal(r.top_tokens[picks].cpu().numpy(), e["top_tokens"][:, :top]), top
            # every row: in order, and no logit left out is above the last one taken
            vals = torch.gather(logits.float(), 1, r.top_tokens)
            assert torch.all(vals[:, 1:] <= vals[:, :-1])
            assert torch.all((logits.float() > vals[:, -1:]).sum(1) < top)
    assert torch.all(torch.isfinite(r.entropy)) and torch.all(r.entropy >= 0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [1, 3, 10, 33, 80, 128, 129, 255, 500, 511, 1000, 1003, 1024, 2040, 2048])
def test_short_rows(ctx, vocab, dtype):
    """Many rows that share warps: beside ordinary ones, rows of equal and of few different logits, masked but for a
    few columns or for none, with NaN and infinities, tokens not given or out of range."""
    rows = 10007
    g = torch.Generator(device="cuda").manual_seed(vocab)
    wide = torch.full((rows, vocab + 3), torch.nan, device="cuda", dtype=TYPES[dtype])
    logits = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(TYPES[dtype])
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    special = torch.arange(100, 112, device="cuda")
    logits[100] = 1.25
    logits[101] = -torch.inf
    logits[102] = -torch.inf
    logits[102, vocab // 2] = 4
    logits[103, vocab // 3] = torch.nan
    logits[104, vocab - 1] = torch.inf
    logits[105] = torch.finfo(TYPES[dtype]).min
    logits[106] = torch.where(torch.arange(vocab, device="cuda") % 3 == 1, 0.0, -0.0).to(TYPES[dtype])
    logits[107] = (torch.arange(vocab, device="cuda") // 9 % 4).to(TYPES[dtype])
    logits[108, ::2] = -torch.inf
    logits[109] = -torch.inf
    logits[109, -2:] = 0.5
    tokens[110], tokens[111] = -7, vocab
    logits[-1] = 2
    picks = sorted({*special.tolist(), 0, 1, rows - 2, rows - 1, *np.random.default_rng(1).integers(0, rows, 30).tolist()})
    wide[:, 1:vocab + 1] = logits
    e = R.logprobs(f64(logits[picks]), tokens[picks].cpu().numpy(), 1.1, min(8, vocab))
    for view in (logits, wide[:, 1:vocab + 1]):
        for top in sorted({0, 1, min(4, vocab), min(5, vocab), min(8, vocab)}):
            r = K.token_logprobs(ctx, view, tokens, top=top, temperature=1.1)
            pairs = [("logprobs", R.logprob_off(e["logprobs"], e["lse"], vocab)), ("entropy", R.entropy_off(e["entropy"], vocab)),
                     ("lse", R.logprob_off(e["lse"], e["lse"], vocab))]
            if top:
                assert np.array_equal(r.top_tokens[picks].cpu().numpy(), e["top_tokens"][:, :top]), top
                pairs.append(("top_logprobs", R.logprob_off(e["top_logprobs"], e["lse"][:, None], vocab)[:, :top]))
            for name, off in pairs:
                got, ref = f64(getattr(r, name)[picks]), e[name][:, :top] if name == "top_logprobs" else e[name]
                fin = np.isfinite(ref)
                assert np.array_equal(got[~fin], ref[~fin], equal_nan=True), (name, top)
                assert np.all(np.abs(got[fin] - ref[fin]) <= off[fin]), (name, top)


@pytest.mark.parametrize("m,n,k", [(17, 4096, 4096), (20, 130, 8192), (32, 16384, 1024), (40, 18944, 300), (64, 19000, 256), (100, 25000, 129), (128, 128, 131071),
                                   (129, 9000, 700), (200, 20000, 512), (300, 5000, 1000), (500, 2000, 3000), (600, 3700, 1111), (1500, 3300, 1111), (2048, 4096, 700),
                                   (3000, 257, 65), (5000, 1025, 400), (70000, 140, 33)])
def test_product(ctx, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    pitch = -(-k // 16) * 16

    def codes(rows):
        return torch.randint(-128, 128, (rows, pitch), device="cuda", dtype=torch.int8, generator=g)[:, :k]

    a, w = codes(m), codes(n)
    sa, sw = torch.rand(m, device="cuda", generator=g) + 0.1, torch.rand(n, device="cuda", generator=g) + 0.1
    bias = torch.randn(n, device="cuda", generator=g)
    y = K.int8_product(ctx, a, sa, w, sw, bias, "relu")
    assert torch.equal(y, K.int8_product(ctx, a, sa, w, sw, bias, "relu"))  # whatever the order of the shares
    rng = np.random.default_rng(1)
    rows = np.unique(np.r_[0, m - 1, rng.integers(0, m, 40)])
    cols = np.unique(np.r_[0, n - 1, rng.integers(0, n, 300)])
    ref, off = R.product(f64(a[rows]), f64(sa[rows]), f64(w[cols]), f64(sw[cols]), f64(bias[cols]), "relu", "float32")
    got = f64(y[rows][:, cols])
    assert np.all(np.abs(got - ref) <= off)
    # sums over whole rows and columns, in integers
    lin = K.int8_product(ctx, a, torch.ones_like(sa), w, torch.ones_like(sw))
    one = w.double().sum(0)
    assert torch.allclose(lin.double().sum(1), (a.double() * one).sum(1), rtol=0, atol=n * 2.0 ** 31 * 2.0 ** -24)


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16])
@pytest.mark.parametrize("n,k", [(5000, 64), (9000, 200), (20000, 16), (40, 70), (3000, 700), (16, 1), (33000, 130)])
def test_few_tokens(ctx, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = torch.randn(m, k, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randint(-127, 128, (n, -(-k // 16) * 16), device="cuda", dtype=torch.int8, generator=g)[:, :k]
    sw = torch.rand(n, device="cuda", generator=g) + 0.1
    y = K.int8_connected(ctx, x, w, sw, dtype=torch.float32)
    c, s = R.quantize(f64(x))
    ref, off = R.product(c, s, f64(w), f64(sw), None, "linear", "float32")
    assert np.all(np.abs(f64(y) - ref) <= off)
