"""int8 connected layer: row quantization, the product and both in one call against 64 bits."""
import numpy as np
import pytest
import torch

import tokens_ref as R
from tensorium_b200 import Context, TBError
from tensorium_b200 import tokens as K
from tensorium_b200.layers import TInt8ConnectedLayer, TNNetState

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def inputs(rows, cols, dtype, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    return torch.from_numpy((scale * rng.standard_normal((rows, cols))).astype(np.float32)).to("cuda", TYPES[dtype])


def f64(t):
    return t.double().cpu().numpy()


def within(y, ref, off, what=""):
    y = f64(y)
    assert y.shape == ref.shape, (what, y.shape, ref.shape)
    assert np.array_equal(np.isnan(y), np.isnan(ref)), what
    bad = ~(np.abs(y - ref) <= off) & ~np.isnan(ref)
    assert not bad.any(), (what, int(bad.sum()), [(tuple(i), y[tuple(i)], ref[tuple(i)], off[tuple(i)]) for i in np.argwhere(bad)[:4]])


def padded_codes(rng, rows, cols, low=-127):
    """int8 rows of whole 16 bytes whose padding holds other values."""
    buf = rng.integers(low, 128, (rows, -(-cols // 16) * 16)).astype(np.int8)
    return torch.from_numpy(buf).cuda()[:, :cols]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (2, 129), (7, 1003), (300, 256), (1, 4096), (4, 8192), (2, 20001),
                                       (1, 40000), (1, 131071)])
def test_quantize_rows(ctx, rows, cols, dtype):
    x = inputs(rows, cols, dtype, rows * cols)
    if rows > 2:
        x[1] = 0
        x[2] *= 1e-4
    codes, scales = K.quantize_rows(ctx, x)
    c, s = R.quantize(f64(x))
    assert codes.stride(0) % 16 == 0 or rows == 1
    assert np.array_equal(codes.cpu().numpy(), c)
    assert np.array_equal(scales.cpu().numpy(), s)


def test_quantize_rows_extremes(ctx):
    x = torch.zeros(8, 100, device="cuda")
    x[0, 3] = torch.nan
    x[1, 99] = torch.inf
    x[2, 0] = -torch.inf
    x[3] = 1e-45          # below the floor: codes 0, finite scale
    x[4, :2] = torch.tensor([3e38, -3.4e38])
    x[5] = -0.0
    x[6, :5] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5])  # ties of rint go to even
    codes, scales = K.quantize_rows(ctx, x)
    c, s = R.quantize(f64(x))
    assert np.array_equal(codes.cpu().numpy(), c)
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
    assert codes[6, :5].tolist() == [127, 0, 2, 2, 0]


@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize_rows_strides(ctx, dtype):
    big = inputs(9, 700, dtype, 5)
    for view in (big[:, 1:602], big[::2, 8:520], big[2:3].expand(6, 700), big[:, :1]):
        codes, scales = K.quantize_rows(ctx, view)
        c, s = R.quantize(f64(view))
        assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(scales.cpu().numpy(), s)


SHAPES = [(1, 1, 1), (1, 5, 17), (2, 130, 64), (3, 64, 1003), (1, 4096, 4096), (4, 1000, 2048), (5, 257, 300), (8, 128, 16), (16, 384, 4096),
          (17, 255, 129), (33, 129, 1024), (64, 1024, 512), (65, 1000, 999), (128, 256, 128), (129, 257, 127), (200, 640, 5000), (257, 513, 96),
          (333, 4099, 1003), (512, 512, 1024), (1000, 300, 640), (2050, 1030, 272), (300, 16384, 80)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ctx, m, n, k):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, w = padded_codes(rng, m, k, -128), padded_codes(rng, n, k, -128)
    sa = torch.from_numpy(rng.uniform(0.01, 1, m).astype(np.float32)).cuda()
    sw = torch.from_numpy(rng.uniform(0.01, 1, n).astype(np.float32)).cuda()
    bias = torch.from_numpy(rng.standard_normal(n).astype(np.float32) * 100).cuda()
    for dtype, act, b in (("float32", "linear", None), ("bfloat16", "leaky", bias)):
        y = K.int8_product(ctx, a, sa, w, sw, b, act, TYPES[dtype])
        ref, off = R.product(f64(a), f64(sa), f64(w), f64(sw), None if b is None else f64(b), act, dtype)
        within(y, ref, off, (dtype, act))


def test_product_largest_sums(ctx):
    """k at its limit with every code -128: 131071 * 16384 is just inside int32."""
    for m in (1, 20, 150):
        a = torch.full((m, 131072), -128, dtype=torch.int8, device="cuda")[:, :131071]
        w = torch.full((130, 131072), -128, dtype=torch.int8, device="cuda")[:, :131071]
        w[1] = 127
        one = torch.ones(m, device="cuda")
        y = K.int8_product(ctx, a, one, w, torch.ones(130, device="cuda"))
        assert torch.all(y[:, 0] == float(np.float32(131071 * 16384)))
        assert torch.all(y[:, 1] == float(np.float32(-131071 * 128 * 127)))


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 16, 31, 32, 33, 48, 64, 100, 128, 160, 256, 300])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_connected_tokens(ctx, m, dtype):
    n, k = 515, 1040
    rng = np.random.default_rng(m)
    x, w = inputs(m, k, dtype, m, 3.0), padded_codes(rng, n, k)
    sw = torch.from_numpy(rng.uniform(1e-4, 1e-3, n).astype(np.float32)).cuda()
    bias = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).cuda()
    y = K.int8_connected(ctx, x, w, sw, bias, "leaky")
    assert y.dtype == x.dtype
    c, s = R.quantize(f64(x))
    ref, off = R.product(c, s, f64(w), f64(sw), f64(bias), "leaky", dtype)
    within(y, ref, off)
    # the same call again, and the two-step form: the same bits
    assert torch.equal(y, K.int8_connected(ctx, x, w, sw, bias, "leaky"))
    codes, scales = K.quantize_rows(ctx, x)
    assert torch.equal(y, K.int8_product(ctx, codes, scales, w, sw, bias, "leaky", x.dtype))


@pytest.mark.parametrize("m", [1, 3, 20, 300])
def test_connected_rows_in_long_and_odd_layers(ctx, m):
    for n, k in ((17, 20001), (4100, 33), (1, 4096), (131, 16400)):
        rng = np.random.default_rng(n)
        x, w = inputs(m, k, "bfloat16", n), padded_codes(rng, n, k)
        sw = torch.from_numpy(rng.uniform(1e-4, 1e-3, n).astype(np.float32)).cuda()
        c, s = R.quantize(f64(x))
        for dtype in ("float32", "bfloat16"):
            ref, off = R.product(c, s, f64(w), f64(sw), None, "linear", dtype)
            within(K.int8_connected(ctx, x, w, sw, dtype=TYPES[dtype]), ref, off, (n, k, dtype))


@pytest.mark.parametrize("act", ["linear", "relu", "logistic", "elu", "hardtan"])
@pytest.mark.parametrize("m", [1, 40, 260])
def test_connected_activations(ctx, act, m):
    rng = np.random.default_rng(3)
    x, w = inputs(m, 200, "float32", 4), padded_codes(rng, 300, 200)
    sw = torch.full((300,), 1e-3, device="cuda")
    c, s = R.quantize(f64(x))
    ref, off = R.product(c, s, f64(w), f64(sw), None, act, "float32")
    within(K.int8_connected(ctx, x, w, sw, activation=act), ref, off, act)


@pytest.mark.parametrize("m", [1, 4, 30, 140, 300])
def test_connected_row_of_nan(ctx, m):
    """A row with a NaN or an infinity is NaN; the others are as without it."""
    rng = np.random.default_rng(8)
    x, w = inputs(m, 333, "bfloat16", 9), padded_codes(rng, 200, 333)
    sw = torch.full((200,), 1e-3, device="cuda")
    clean = K.int8_connected(ctx, x, w, sw)
    for v in (torch.nan, torch.inf, -torch.inf):
        x2 = x.clone()
        x2[m // 2, 332] = v
        y = K.int8_connected(ctx, x2, w, sw)
        assert torch.isnan(y[m // 2]).all()
        keep = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("m", [1, 4, 24, 150, 300])
def test_connected_strides_and_guards(ctx, m):
    """Inputs and outputs that are parts of larger tensors, at odd offsets; nothing else is written."""
    n, k = 259, 301
    rng = np.random.default_rng(m)
    big = inputs(m, k + 9, "bfloat16", m)
    x = big[:, 3:3 + k]
    w = padded_codes(rng, n, k)
    sw = torch.from_numpy(rng.uniform(1e-4, 1e-3, n).astype(np.float32)).cuda()
    c, s = R.quantize(f64(x))
    ref, off = R.product(c, s, f64(w), f64(sw), None, "linear", "bfloat16")
    for lead, tail in ((0, 5), (1, 0), (8, 1)):
        buf = torch.full((m + 1, lead + n + tail), 77.0, device="cuda", dtype=torch.bfloat16)
        out = buf[:m, lead:lead + n]
        y = K.int8_connected(ctx, x, w, sw, out=out)
        assert y.data_ptr() == out.data_ptr()
        within(y, ref, off, (lead, tail))
        assert (buf[m] == 77).all() and (buf[:, :lead] == 77).all() and (buf[:, lead + n:] == 77).all()


def test_connected_nothing(ctx):
    w, sw = torch.zeros(4, 16, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    assert K.int8_connected(ctx, torch.zeros(0, 16, device="cuda"), w, sw).shape == (0, 4)
    assert K.int8_connected(ctx, torch.zeros(3, 16, device="cuda"), w[:0], sw[:0]).shape == (3, 0)
    codes, scales = K.quantize_rows(ctx, torch.zeros(0, 5, device="cuda"))
    assert codes.shape == (0, 5) and scales.shape == (0,)


def test_connected_on_another_stream():
    """A context on a side stream: the results, and memory that the caller frees at once, are safe."""
    side = torch.cuda.Stream()
    with Context(0, use_torch_stream=False) as c:
        c.set_stream(side)
        rng = np.random.default_rng(1)
        x, w = inputs(70, 512, "bfloat16", 2), padded_codes(rng, 300, 512)
        sw = torch.full((300,), 1e-3, device="cuda")
        cq, s = R.quantize(f64(x))
        ref, off = R.product(cq, s, f64(w), f64(sw), None, "linear", "bfloat16")
        side.wait_stream(torch.cuda.current_stream())
        ys = []
        for _ in range(20):
            own = x.clone()
            side.wait_stream(torch.cuda.current_stream())
            ys.append(K.int8_connected(c, own, w, sw))
            del own
            torch.full_like(x, 1e4)  # would land in the freed memory
        side.synchronize()
        for y in ys:
            within(y, ref, off)


def test_connected_in_a_graph(ctx):
    """One captured call (the workspace reserved first) replays on new inputs."""
    rng = np.random.default_rng(1)
    x, w = inputs(40, 512, "bfloat16", 2), padded_codes(rng, 300, 512)
    sw = torch.full((300,), 1e-3, device="cuda")
    out = torch.empty(40, 300, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    with Context(0, use_torch_stream=False) as c:
        c.set_stream(side)
        c.reserve(1 << 20)
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            K.int8_connected(c, x, w, sw, out=out)
        for seed in (5, 6):
            x.copy_(inputs(40, 512, "bfloat16", seed))
            g.replay()
            torch.cuda.synchronize()
            cq, s = R.quantize(f64(x))
            ref, off = R.product(cq, s, f64(w), f64(sw), None, "linear", "bfloat16")
            within(out, ref, off)
        del g


def test_layer(ctx):
    """TInt8ConnectedLayer is near the connected layer on the same float weights."""
    rng = np.random.default_rng(2)
    w, b = rng.standard_normal((70, 400)).astype(np.float32), rng.standard_normal(70).astype(np.float32)
    x = inputs(12, 400, "float32", 3)
    y = TInt8ConnectedLayer(400, 70, "leaky", w, b).bind(ctx).forward(TNNetState(x))
    (cx, sx), (cw, sw) = R.quantize(f64(x)), R.quantize(w)
    ref, off = R.product(cx, sx, cw, sw, b, "leaky", "float32")
    within(y, ref, off)
    full = R.ACTS["leaky"](f64(x) @ w.T.astype(np.float64) + b)
    assert np.linalg.norm(f64(y) - full) / np.linalg.norm(full) < 0.02  # two roundings to 1 / 254 of a row's largest


def test_refusals(ctx):
    w, sw = torch.zeros(8, 32, dtype=torch.int8, device="cuda"), torch.zeros(8, device="cuda")
    x = torch.zeros(2, 32, device="cuda")
    with pytest.raises(TBError, match="multiples of 16"):
        K.int8_connected(ctx, x[:, :31], w[:, 1:], sw)
    with pytest.raises(TBError, match="multiples of 16"):
        K.int8_connected(ctx, x[:, :24], torch.zeros(8, 24, dtype=torch.int8, device="cuda"), sw)
    with pytest.raises(TBError, match="multiples of 16"):
        K.int8_product(ctx, torch.zeros(2, 24, dtype=torch.int8, device="cuda"), sw[:2], w[:, :24], sw)
    with pytest.raises(TBError, match="overflow"):
        K.int8_connected(ctx, torch.zeros(1, 131072, device="cuda"), torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), sw[:1])
    with pytest.raises(TBError, match="bad shape"):
        K.int8_connected(ctx, x[:, :0], w[:, :0], sw)
    with pytest.raises(TBError, match="activation"):
        K.int8_connected(ctx, x, w, sw, activation=12)
    with pytest.raises(TBError, match="row stride"):
        K.int8_connected(ctx, x, w, sw, out=torch.zeros(16, device="cuda").as_strided((2, 8), (4, 1)))
    with pytest.raises(TBError, match="row stride"):
        K.quantize_rows(ctx, torch.zeros(40, device="cuda").as_strided((2, 32), (8, 1)))
    for bad in (dict(w_scales=sw[:7]), dict(w_scales=sw.double()), dict(bias=sw[:1]), dict(activation="swish"), dict(dtype=torch.float64),
                dict(out=torch.zeros(2, 9, device="cuda")), dict(out=torch.zeros(2, 8)), dict(out=torch.zeros(2, 8, device="cuda").half())):
        with pytest.raises(ValueError):
            K.int8_connected(ctx, x, w, **{"w_scales": sw, **bad})
    for bad in (x.double(), x[0], x.cpu(), x.t().contiguous().t(), x[:, :16]):
        with pytest.raises(ValueError):
            K.int8_connected(ctx, bad, w, sw)
    # a refused call leaves the context usable
    assert K.int8_connected(ctx, x, w, sw).shape == (2, 8)
