"""The Python extension of the token operators saves host time and nothing else: without it the package imports, builds
and gives the same results."""
import os
import subprocess
import sys
import types

import pytest
import torch

from conftest import ROOT
from tensorium_b200 import build as B


def python(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)


def test_import_without_the_extension():
    r = python("""
import sys
sys.modules["tensorium_b200._tokens_fast"] = None  # an import of it raises ImportError
import tensorium_b200.layers, tensorium_b200.net
from tensorium_b200 import tokens
assert all(getattr(tokens._fast, f)(0, 0, 0) is None for f in ("int8_connected", "token_logprobs", "token_logprobs_backward"))
""")
    assert r.returncode == 0, r.stderr


def test_it_is_there_after_a_build():
    B.build()
    from tensorium_b200 import tokens
    assert tokens._fast.__name__.endswith("_tokens_fast")


@pytest.mark.parametrize("why", ["compiler fails", "no compiler"])
def test_library_builds_without_the_extension(monkeypatch, tmp_path, capsys, why):
    B.build()  # the library is there
    fast = tmp_path / "_tokens_fast.so"

    def run(*args, **kw):
        if why == "no compiler":
            raise FileNotFoundError("g++")
        return types.SimpleNamespace(returncode=1, stdout="", stderr="Python.h: No such file or directory")

    monkeypatch.setattr(B, "FAST", fast)
    monkeypatch.setattr(B.subprocess, "run", run)
    assert B.build() == B.LIB and B.LIB.exists()
    assert not fast.exists()
    assert "was not built" in capsys.readouterr().err
    # an older one is not left to stand beside a newer library
    fast.write_bytes(b"")
    os.utime(fast, (0, 0))
    assert B.build() == B.LIB and not fast.exists()


def test_another_torch_or_python_has_another_extension(monkeypatch):
    """One that was built for another C++ ABI is not loaded, nor taken for up to date."""
    assert B._fast_path() == B.FAST
    seen = {B.FAST}
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "99.1.0+cu990")
    seen.add(B._fast_path())
    monkeypatch.setattr(B.sysconfig, "get_config_var", lambda name: "cpython-399-x86_64-linux-gnu")
    seen.add(B._fast_path())
    assert len(seen) == 3

    def none(name):
        raise B.importlib.metadata.PackageNotFoundError(name)

    monkeypatch.setattr(B.importlib.metadata, "version", none)
    assert B._fast_path() not in seen


@pytest.mark.parametrize("content", [None, b"", b"not a library"])
def test_import_with_another_torchs_extension(tmp_path, content):
    """Only the file of this Python and torch counts, and one that does not load is passed over."""
    fast = tmp_path / "_tokens_fast.so"
    if content is not None:
        fast.write_bytes(content)
    r = python(f"""
import pathlib
from tensorium_b200 import build
build.FAST = pathlib.Path({str(fast)!r})
import tensorium_b200.layers, tensorium_b200.net
from tensorium_b200 import tokens
assert tokens._fast is tokens._NoFast
""")
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
def test_same_results_without_the_extension(ctx, monkeypatch):
    from tensorium_b200 import tokens as K
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(33, 500, device="cuda", generator=g)
    w, sw = K.quantize_rows(ctx, torch.randn(1200, 500, device="cuda", generator=g))
    bias = torch.randn(1200, device="cuda", generator=g)
    given = torch.randint(1200, (33,), device="cuda", generator=g)
    a, b = torch.randn(33, device="cuda", generator=g), torch.randn(33, device="cuda", generator=g)

    def all_of_it():
        y = K.int8_connected(ctx, x, w, sw, bias, "leaky")
        r = K.token_logprobs(ctx, y, given, top=6, temperature=0.8)
        d = K.token_logprobs_backward(ctx, y, given, r, a, b, temperature=0.8)
        assert K.token_logprobs(ctx, y).top_tokens is None
        return y, r.stats, r.top_logprobs, r.top_tokens, d

    one = all_of_it()
    monkeypatch.setattr(K, "_fast", K._NoFast)
    for p, q in zip(one, all_of_it()):
        assert p.dtype == q.dtype and p.shape == q.shape and torch.equal(p, q)
