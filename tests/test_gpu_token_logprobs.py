"""Token log probabilities, entropies, alternatives and their gradient against 64 bits."""
import numpy as np
import pytest
import torch

import tokens_ref as R
from tensorium_b200 import Context, TBError
from tensorium_b200 import tokens as K
from tensorium_b200.layers import TNNetState, TTokenLogprobsLayer

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def f64(t):
    return t.double().cpu().numpy()


def make(rows, vocab, dtype, seed, spread=4.0, masked=0.0):
    rng = np.random.default_rng(seed)
    l = rng.standard_normal((rows, vocab)) * rng.uniform(0.3, spread, (rows, 1))
    if masked:
        l[rng.random((rows, vocab)) < masked] = -np.inf
    t = torch.from_numpy(l.astype(np.float32)).to("cuda", TYPES[dtype])
    return t, torch.from_numpy(rng.integers(0, vocab, rows)).cuda()


def close(got, ref, off, what):
    got = f64(got)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = np.isfinite(ref)
    assert np.array_equal(got[~fin], ref[~fin], equal_nan=True), (what, got[~fin][:5], ref[~fin][:5])
    bad = ~(np.abs(got - np.where(fin, ref, 0)) <= off) & fin
    assert not bad.any(), (what, int(bad.sum()), [(tuple(i), got[tuple(i)], ref[tuple(i)], np.broadcast_to(off, ref.shape)[tuple(i)]) for i in np.argwhere(bad)[:4]])


def check(ctx, logits, tokens, top, temperature=1.0):
    vocab = logits.shape[1]
    r = K.token_logprobs(ctx, logits, tokens, top=top, temperature=temperature)
    e = R.logprobs(f64(logits), None if tokens is None else tokens.cpu().numpy(), temperature, top)
    close(r.entropy, e["entropy"], R.entropy_off(e["entropy"], vocab), "entropy")
    close(r.lse, e["lse"], R.logprob_off(e["lse"], e["lse"], vocab), "lse")
    if tokens is not None:
        close(r.logprobs, e["logprobs"], R.logprob_off(e["logprobs"], e["lse"], vocab), "logprobs")
    else:
        assert r.logprobs is None
    if top:
        assert np.array_equal(r.top_tokens.cpu().numpy(), e["top_tokens"]), "top_tokens"
        close(r.top_logprobs, e["top_logprobs"], R.logprob_off(e["top_logprobs"], e["lse"][:, None], vocab), "top_logprobs")
    else:
        assert r.top_tokens is None
    return r


VOCABS = [1, 2, 31, 33, 80, 255, 256, 257, 1000, 1023, 2049, 4097, 8191, 8192, 8200, 16500, 32000, 50001, 131072, 200003]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
def test_vocabularies(ctx, vocab, dtype):
    for rows, top in ((1, min(20, vocab)), (3, min(32, vocab)), (5, 0), (2, 1)):
        logits, tokens = make(rows, vocab, dtype, vocab + rows)
        check(ctx, logits, tokens, top)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 147, 300, 1000, 3001])
def test_rows(ctx, rows):
    for vocab, top in ((10, 3), (700, 5), (5003, 20)):
        logits, tokens = make(rows, vocab, "bfloat16", rows + vocab)
        check(ctx, logits, tokens, top, 0.7)


def test_many_rows(ctx):
    logits, tokens = make(70001, 11, "float16", 1)
    check(ctx, logits, tokens, 2)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 3.0, 100.0])
def test_temperature(ctx, temperature):
    logits, tokens = make(6, 9001, "float32", 3, spread=1.0)
    check(ctx, logits, tokens, 8, temperature)


@pytest.mark.parametrize("vocab", [20, 300, 3000, 40000, 131072])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_order_of_equal_logits(ctx, vocab, dtype):
    """Equal logits come lowest column first: constant rows, few values, signed zeros, rising and
    falling rows."""
    g = torch.Generator().manual_seed(1)
    few = torch.randint(-2, 3, (3, vocab), generator=g).float()
    zeros = torch.where(torch.rand(1, vocab, generator=g) < 0.5, 0.0, -0.0)
    ramp = torch.linspace(-30, 30, vocab)[None]
    steps = (torch.arange(vocab) // 7 % 50).float()[None] / 8
    logits = torch.cat([torch.full((1, vocab), 1.5), few, zeros, ramp, -ramp, steps, -steps]).to("cuda", TYPES[dtype])
    tokens = torch.zeros(logits.shape[0], dtype=torch.int64, device="cuda")
    check(ctx, logits, tokens, min(32, vocab))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [40, 1000, 5001, 131072])
def test_masked(ctx, vocab, dtype):
    """-infinity masks: half, nearly all (fewer columns left than alternatives), one left, none."""
    logits, tokens = make(9, vocab, dtype, 4, masked=0.5)
    logits[1] = -torch.inf
    logits[2] = -torch.inf
    logits[2, vocab // 2] = 3
    tokens[2] = vocab // 2
    logits[3] = -torch.inf
    logits[3, 3::7] = 0.5
    logits[4, :] = -torch.inf
    logits[4, vocab - 1] = -2
    logits[4, 1] = -5
    logits[5, : vocab - 5] = -torch.inf
    tokens[6] = -1
    tokens[7] = vocab + 5
    tokens[1] = 0
    check(ctx, logits, tokens, 32)
    check(ctx, logits, None, 3)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [33, 1000, 70000])
def test_lowest_value_masks(ctx, vocab, dtype):
    """Masks of the type's lowest finite value, alone and beside ordinary logits."""
    low = torch.finfo(TYPES[dtype]).min
    logits, tokens = make(5, vocab, dtype, 6)
    logits[0, ::2] = low
    logits[1] = low
    logits[2] = low
    logits[2, 7] = 1
    logits[3, 1:] = low
    tokens[2], tokens[3] = 7, 0
    tokens[0] = 1
    check(ctx, logits, tokens, 20)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [5, 900, 9000, 131072])
def test_nan_and_infinity(ctx, vocab, dtype):
    """A row with a NaN or +infinity anywhere is NaN throughout; its neighbours are not."""
    logits, tokens = make(10, vocab, dtype, 7)
    for row, (col, v) in enumerate([(0, torch.nan), (vocab - 1, torch.nan), (vocab // 2, torch.inf), (0, torch.inf), (vocab // 3, -torch.nan)]):
        logits[2 * row, col] = v
    logits[6, :] = torch.nan
    check(ctx, logits, tokens, 5)
    check(ctx, logits, tokens, 0)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_logits(ctx, dtype):
    """Values whose exponentials would overflow, and rows that rise over a wide range."""
    top = {"float32": 1e30, "bfloat16": 1e30, "float16": 6e4}[dtype]
    vocab = 6007
    logits, tokens = make(4, vocab, dtype, 8)
    logits[0] = torch.linspace(0, 5000, vocab)
    logits[1] = torch.linspace(5000, 0, vocab)
    logits[2] *= top / 20
    logits[3] += -800
    tokens[0], tokens[1] = vocab - 1, 0
    tokens[2] = logits[2].float().argmax()
    check(ctx, logits, tokens, 6)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [100, 1003, 20011])
def test_strides(ctx, vocab, dtype):
    """Rows at odd offsets inside a larger tensor whose other places hold NaN."""
    for lead, tail in ((1, 0), (3, 5), (8, 8), (0, 13)):
        big = torch.full((7, lead + vocab + tail), torch.nan, device="cuda", dtype=TYPES[dtype])
        logits, tokens = make(7, vocab, dtype, vocab + lead)
        big[:, lead:lead + vocab] = logits
        view = big[:, lead:lead + vocab]
        r = check(ctx, view, tokens, 7)
        gl, gh = torch.randn(7, device="cuda"), torch.randn(7, device="cuda")
        d = K.token_logprobs_backward(ctx, view, tokens, r, gl, gh)
        check_grad(d, view, tokens, 1.0, gl, gh)
        # out with another stride than the logits, with guards
        buf = torch.full((8, vocab + 3), 9.0, device="cuda", dtype=TYPES[dtype])
        d2 = K.token_logprobs_backward(ctx, view, tokens, r, gl, gh, out=buf[:7, 1:1 + vocab])
        assert torch.equal(d, d2)
        assert (buf[7] == 9).all() and (buf[:, 0] == 9).all() and (buf[:, 1 + vocab:] == 9).all()
        # in place
        d3 = K.token_logprobs_backward(ctx, view, tokens, r, gl, gh, out=view)
        assert d3.data_ptr() == view.data_ptr() and torch.equal(d, view)
        assert torch.isnan(big[:, :lead]).all() and torch.isnan(big[:, lead + vocab:]).all()


def check_grad(d, logits, tokens, temperature, gl, gh):
    dtype = str(logits.dtype).replace("torch.", "")
    ref, off = R.gradient(f64(logits), None if tokens is None else tokens.cpu().numpy(), temperature,
                          None if gl is None else f64(gl), None if gh is None else f64(gh))
    off = off + 1.01 * R.HALF_ULP[dtype] * (np.abs(np.where(np.isnan(ref), 0, ref)) + off) + R.TINY[dtype]
    close(d, ref, off, "gradient")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 80), (4, 1000), (130, 999), (3, 8193), (2, 50001), (1, 131072), (1000, 37)])
def test_gradient(ctx, rows, vocab, dtype):
    logits, tokens = make(rows, vocab, dtype, rows * vocab, masked=0.2 if vocab > 50 else 0)
    gl, gh = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    for temperature in (1.0, 0.6):
        r = K.token_logprobs(ctx, logits, tokens, temperature=temperature)
        for a, b in ((gl, gh), (gl, None), (None, gh), (None, None)):
            d = K.token_logprobs_backward(ctx, logits, tokens, r, a, b, temperature=temperature)
            check_grad(d, logits, tokens, temperature, a, b)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradient_of_odd_rows(ctx, dtype):
    """Empty rows, rows of NaN, tokens not given, out of range or masked, masks of the lowest value."""
    vocab = 3003
    logits, tokens = make(9, vocab, dtype, 12, masked=0.3)
    logits[0] = -torch.inf
    logits[1, 5] = torch.nan
    logits[2, 9] = torch.inf
    tokens[3] = -100
    tokens[4] = vocab
    logits[5, 17], tokens[5] = -torch.inf, 17
    logits[6] = torch.finfo(TYPES[dtype]).min
    logits[7, 1:] = torch.finfo(TYPES[dtype]).min
    r = K.token_logprobs(ctx, logits, tokens)
    gl, gh = torch.rand(9, device="cuda") + 0.5, torch.rand(9, device="cuda") + 0.5
    for a, b in ((gl, gh), (gl, None), (None, gh)):
        d = K.token_logprobs_backward(ctx, logits, tokens, r, a, b)
        check_grad(d, logits, tokens, 1.0, a, b)
    d = K.token_logprobs_backward(ctx, logits, tokens, r, gl, gh)
    assert (d[0] == 0).all()
    masked = torch.isneginf(logits[3])
    assert masked.any() and (d[3][masked] == 0).all()
    assert torch.isnan(d[1]).all() and torch.isnan(d[2]).all() and torch.isnan(d[4]).all()


def test_gradient_against_differences(ctx):
    """Central differences of the 64-bit loss: their own error is h^2 / 6 of a third derivative that the
    softmax keeps under 8 (|g| (1 + log vocab)) / T^3, and rounding of the loss over h."""
    rows, vocab, T, h = 3, 41, 0.8, 1e-4
    logits, tokens = make(rows, vocab, "float32", 21, spread=1.5)
    gl, gh = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    r = K.token_logprobs(ctx, logits, tokens, temperature=T)
    d = f64(K.token_logprobs_backward(ctx, logits, tokens, r, gl, gh, temperature=T))
    l, t, a, b = f64(logits), tokens.cpu().numpy(), f64(gl), f64(gh)

    def loss(x):
        e = R.logprobs(x, t, T, 0)
        return a * e["logprobs"] + b * e["entropy"]

    for j in range(vocab):
        step = np.zeros_like(l)
        step[:, j] = h
        diff = (loss(l + step) - loss(l - step)) / (2 * h)
        size = (np.abs(a) + np.abs(b)) * (1 + np.log(vocab)) / T ** 3
        assert np.all(np.abs(diff - d[:, j]) <= 8 * size * h * h + 1e-11 / h + 300 * R.U * size), j


def test_results_do_not_depend_on_neighbours(ctx):
    """A row alone and the same row among others: alternatives equal, sums within the bounds; the same call
    twice: the same bits."""
    logits, tokens = make(40, 30011, "bfloat16", 30)
    r = check(ctx, logits, tokens, 20)
    again = K.token_logprobs(ctx, logits, tokens, top=20)
    for name in ("logprobs", "entropy", "lse", "row_max", "log_sum", "top_logprobs", "top_tokens"):
        assert torch.equal(getattr(r, name), getattr(again, name))
    one = check(ctx, logits[7:8], tokens[7:8], 20)
    assert torch.equal(one.top_tokens[0], r.top_tokens[7])


def test_nothing(ctx):
    r = K.token_logprobs(ctx, torch.zeros(0, 50, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top=3)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 3)
    d = K.token_logprobs_backward(ctx, torch.zeros(0, 50, device="cuda"), None, r)
    assert d.shape == (0, 50)


def test_offsets_past_32_bits(ctx):
    """Rows whose elements lie more than 2^32 bytes and 2^31 elements from the first."""
    rows, vocab = 18000, 131072
    logits = torch.full((rows, vocab), -3.0, device="cuda", dtype=torch.bfloat16)
    last, tok = make(2, vocab, "bfloat16", 40)
    logits[-2:] = last
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    tokens[-2:] = tok
    r = K.token_logprobs(ctx, logits, tokens, top=4)
    few = check(ctx, last, tok, 4)
    assert torch.equal(few.top_tokens, r.top_tokens[-2:])
    assert r.top_tokens[0].tolist() == [0, 1, 2, 3]
    assert torch.allclose(r.entropy[:-2], torch.full_like(r.entropy[:-2], float(np.log(vocab))), rtol=0, atol=3 * R.sum_off(vocab) * 13)
    gl = torch.ones(rows, device="cuda")
    d = K.token_logprobs_backward(ctx, logits, tokens, r, gl, out=logits)
    assert abs(float(d[0, 0]) - (1 - 1 / vocab)) < 2.0 ** -8
    check_grad(d[-2:], last, tok, 1.0, gl[-2:], None)


def test_on_another_stream():
    side = torch.cuda.Stream()
    with Context(0, use_torch_stream=False) as c:
        c.set_stream(side)
        logits, tokens = make(5, 70001, "bfloat16", 41)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            check(c, logits, tokens, 9)
        r = K.token_logprobs(c, logits, tokens, top=9)  # called from the default stream
        side.synchronize()
        e = R.logprobs(f64(logits), tokens.cpu().numpy(), 1.0, 9)
        assert np.array_equal(r.top_tokens.cpu().numpy(), e["top_tokens"])


def test_in_a_graph():
    side = torch.cuda.Stream()
    with Context(0, use_torch_stream=False) as c:
        c.set_stream(side)
        logits, tokens = make(2, 50000, "bfloat16", 42)
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            r = K.token_logprobs(c, logits, tokens, top=12)
        for seed in (43, 44):
            new, tok = make(2, 50000, "bfloat16", seed)
            logits.copy_(new)
            tokens.copy_(tok)
            g.replay()
            torch.cuda.synchronize()
            e = R.logprobs(f64(logits), tok.cpu().numpy(), 1.0, 12)
            assert np.array_equal(r.top_tokens.cpu().numpy(), e["top_tokens"])
            close(r.logprobs, e["logprobs"], R.logprob_off(e["logprobs"], e["lse"], 50000), "logprobs")
        del g


def test_layer(ctx):
    logits, tokens = make(6, 500, "float32", 50)
    layer = TTokenLogprobsLayer(top=3, temperature=0.9).bind(ctx)
    r = layer.forward(TNNetState(logits), tokens)
    e = R.logprobs(f64(logits), tokens.cpu().numpy(), 0.9, 3)
    close(r.logprobs, e["logprobs"], R.logprob_off(e["logprobs"], e["lse"], 500), "logprobs")
    gl = torch.ones(6, device="cuda")
    check_grad(layer.backward(TNNetState(logits), tokens, gl), logits, tokens, 0.9, gl, None)


def test_refusals(ctx):
    logits, tokens = make(4, 100, "float32", 60)
    for kw, text in ((dict(top=33), "top over"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
                     (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"), (dict(top=-1), "top has to be")):
        with pytest.raises(TBError, match=text):
            K.token_logprobs(ctx, logits, tokens, **kw)
    with pytest.raises(TBError, match="top has to be"):
        K.token_logprobs(ctx, logits[:, :4].contiguous(), tokens, top=5)
    with pytest.raises(TBError, match="bad shape"):
        K.token_logprobs(ctx, logits[:, :0], tokens)
    with pytest.raises(TBError, match="row stride"):
        K.token_logprobs(ctx, torch.zeros(400, device="cuda").as_strided((4, 100), (50, 1)), tokens)
    for bad in (logits.double(), logits[0], logits.cpu(), logits.t()):
        with pytest.raises(ValueError):
            K.token_logprobs(ctx, bad, tokens)
    for bad in (tokens.int(), tokens[:3], tokens.cpu(), tokens[None]):
        with pytest.raises(ValueError):
            K.token_logprobs(ctx, logits, bad)
    r = K.token_logprobs(ctx, logits, tokens)
    gl = torch.ones(4, device="cuda")
    for kw in (dict(grad_logprobs=gl.double()), dict(grad_logprobs=gl[:2]), dict(grad_entropy=gl.expand(4, 4)[0:1, 0].expand(4)),
               dict(out=torch.zeros(4, 99, device="cuda")), dict(out=torch.zeros(4, 100, device="cuda").half())):
        with pytest.raises(ValueError):
            K.token_logprobs_backward(ctx, logits, tokens, r, **kw)
    with pytest.raises(ValueError):
        K.token_logprobs_backward(ctx, logits, None, r, gl)
    with pytest.raises(TBError, match="another row stride"):
        wide = torch.zeros(4, 120, device="cuda")
        K.token_logprobs_backward(ctx, wide[:, :50], tokens, r, out=wide.view(-1).as_strided((4, 50), (60, 1)))


def test_example(ctx):
    """examples/score_tokens.py: the int8 head and its scores against 64 bits."""
    import sys
    sys.path.insert(0, str(R.__file__).rsplit("/", 2)[0] + "/examples")
    import score_tokens
    hidden, weights, given, r, grad = score_tokens.main(["--rows", "9", "--hidden", "200", "--vocab", "1501", "--top", "4"])
    (cx, sx), (cw, sw) = R.quantize(f64(hidden)), R.quantize(f64(weights))
    y, _ = R.product(cx, sx, cw, sw, None, "linear", "bfloat16")
    logits = torch.from_numpy(y.astype(np.float32)).to(torch.bfloat16)
    e = R.logprobs(f64(logits), given.cpu().numpy(), 1.0, 4)
    # the logits' own rounding may fall either way: one unit in the last place of bfloat16 each
    assert np.all(np.abs(f64(r.logprobs) - e["logprobs"]) <= 2 * 2.0 ** -8 * (1 + np.abs(y).max(1)))
    assert grad.shape == (9, 1501) and abs(float(grad.float().sum())) < 9 * 1501 * 2.0 ** -9 / 9
