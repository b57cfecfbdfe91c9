"""Which stream the token operators' memory belongs to when the calling thread's current torch stream is not the
context's: results are allocated on the stream that writes them, and inputs are kept until it has read them."""
import contextlib
import types

import pytest
import torch

import tokens_ref as R
from tensorium_b200 import Context
from tensorium_b200 import tokens as K


class FakeInput:
    def __init__(self):
        self.recorded, self.made_on = [], []

    def record_stream(self, stream):
        self.recorded.append(stream)

    def new_empty(self, shape, dtype):
        return (shape, dtype, STREAM[-1])


STREAM = ["current"]


@pytest.mark.parametrize("raw,want", [(0, "default stream of cuda:0"), (4096, "stream at 4096 of cuda:0")])
def test_memory_goes_with_the_contexts_stream(monkeypatch, raw, want):
    """The legacy default stream has address 0, which no external stream can stand for."""
    @contextlib.contextmanager
    def on(stream):
        STREAM.append(stream)
        yield
        STREAM.pop()

    def external(address, device=None):
        assert address != 0, "torch makes a new stream where no address is given"
        return f"stream at {address} of {device}"

    monkeypatch.setattr(torch.cuda, "ExternalStream", external)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: f"default stream of {device}")
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(K, "_current_stream", lambda device: 77)
    ctx = types.SimpleNamespace(device=0, raw_stream=raw, torch_device=torch.device("cuda", 0))
    x = FakeInput()
    (shape, dtype, stream), = K._empty(ctx, ((3, 4),), (torch.float32,), (x, None))
    assert (shape, dtype, stream) == ((3, 4), torch.float32, want)
    assert x.recorded == [want]
    # a result that the caller gives is kept too
    assert K._empty(ctx, (), (), (x,)) == [] and x.recorded == [want, want]


def f64(t):
    return t.double().cpu().numpy()


@pytest.mark.gpu
def test_external_stream_of_a_context_on_the_default_stream():
    """The stream that memory is recorded on is the one that the context launches on."""
    with torch.cuda.stream(torch.cuda.default_stream(0)), Context(0) as c:
        assert c.raw_stream == 0
        assert K._torch_stream(c).cuda_stream == 0 and K._torch_stream(c) == torch.cuda.default_stream(0)
        side = torch.cuda.Stream()
        c.set_stream(side)
        assert K._torch_stream(c).cuda_stream == side.cuda_stream


@pytest.mark.gpu
def test_default_stream_context_under_a_side_stream():
    """Inputs freed and overwritten, and results dropped, at once, while the default stream is busy."""
    default, side = torch.cuda.default_stream(0), torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(70, 512, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randint(-127, 128, (300, 512), device="cuda", generator=g, dtype=torch.int8)
    sw = torch.full((300,), 1e-3, device="cuda")
    logits = 3 * torch.randn(70, 5000, device="cuda", generator=g)
    tokens = torch.randint(5000, (70,), device="cuda", generator=g)
    cq, s = R.quantize(f64(x))
    ref, off = R.product(cq, s, f64(w), f64(sw), None, "linear", "bfloat16")
    e = R.logprobs(f64(logits), tokens.cpu().numpy(), 1.0, 5)
    torch.cuda.synchronize()
    with torch.cuda.stream(default), Context(0) as c:
        kept = []
        for _ in range(20):
            with torch.cuda.stream(side):
                own, l = x.clone(), logits.clone()
                default.wait_stream(side)
                with torch.cuda.stream(default):
                    torch.cuda._sleep(200000)
                kept.append((K.int8_connected(c, own, w, sw), K.token_logprobs(c, l, tokens, top=5)))
                K.int8_connected(c, own, w, sw)  # dropped: its memory is the default stream's to give away
                K.token_logprobs(c, l, tokens, top=5)
                del own, l
                torch.full_like(x, 1e4)        # would land in the freed memory
                torch.full_like(logits, 1e4)
        torch.cuda.synchronize()
        for y, r in kept:
            assert (abs(f64(y) - ref) <= off).all()
            assert (r.top_tokens.cpu().numpy() == e["top_tokens"]).all()
            assert (abs(f64(r.logprobs) - e["logprobs"]) <= R.logprob_off(e["logprobs"], e["lse"], 5000)).all()
