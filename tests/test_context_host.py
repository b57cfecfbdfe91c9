"""The context's host code (csrc/ctx.cu) against a stand-in for the CUDA runtime that records what is called, on the CPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

from conftest import ROOT
from tensorium_b200 import build as B

CSRC = ROOT / "tensorium_b200" / "csrc"

# Streams are small numbers, device memory is host memory; calls on the legacy stream (0) have no order with the others.
FAKE = r'''
#include "ctx.cuh"
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>
#include <string>

static std::string calls;
static int fail_at = -1, count = 0;  // the call that fails
static int capturing = 0;
static size_t device_left = ~(size_t)0;
static std::set<void*> live;

static cudaError_t step(const char* what, cudaStream_t s) {
    calls += std::string(what) + ":" + std::to_string((int)(intptr_t)s) + " ";
    return count++ == fail_at ? cudaErrorUnknown : cudaSuccess;
}
extern "C" {
cudaError_t cudaStreamSynchronize(cudaStream_t s) { return step("sync", s); }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { memcpy(d, s, n); return step("copy", 0); }
cudaError_t cudaMemset(void* p, int v, size_t n) { memset(p, v, n); return step("set", 0); }
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t s) {
    cudaError_t e = step("set", s);
    if (e == cudaSuccess) memset(p, v, n);
    return e;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* c) {
    *c = capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
    return cudaSuccess;
}
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t n) {
    if (n > device_left) return cudaErrorMemoryAllocation;
    *p = malloc(n);
    live.insert(*p);
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
    if (live.erase(p)) free(p);
    return step("free", 0);
}
}
namespace tbi {
int fail(int code, const char*, ...) { return code; }
int cuda_fail(cudaError_t e, const char*) { return e == cudaErrorMemoryAllocation ? TB_ERR_OOM : TB_ERR_CUDA; }
}
#define CHECK(c) do { if (!(c)) { printf("line %d: %s (calls: %s)\n", __LINE__, #c, calls.c_str()); return 1; } } while (0)
'''


def run(tmp_path, body):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    cuda = Path(B.nvcc()).resolve().parent.parent / "include"
    src, exe = tmp_path / "main.cpp", tmp_path / "main"
    src.write_text(FAKE + "int main() {\n" + body + "\nreturn 0;\n}\n")
    r = subprocess.run(["g++", "-std=c++17", "-g", "-I", str(CSRC), "-I", str(cuda), "-x", "c++", str(CSRC / "ctx.cu"), str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


STATUS = r'''
    tb_ctx c;
    int status[4] = {}, cnt[8], side1[5], side2[3], st;
    auto dirty = [&](int s) {
        status[0] = s;
        for (int& v : cnt) v = 7;
        for (int& v : side1) v = 7;
        for (int& v : side2) v = 7;
        calls.clear();
        count = 0;
    };
    auto left = [&](auto& a) { int n = 0; for (int v : a) n += v != 0; return n; };
    c.stream = (cudaStream_t)5;
    c.d_status = status;
    c.tile_cnt = cnt, c.tile_cnt_len = 8;
    c.side_cnts = {{side1, 5}, {side2, 3}};
'''


def test_counters_are_cleared_before_the_next_launch(tmp_path):
    """After a kernel that gave up: every clear is on the context's stream, and has ended when the call returns."""
    run(tmp_path, STATUS + r'''
    dirty(931);
    CHECK(tbi::take_status(&c, &st) == TB_OK && st == 931);
    CHECK(calls == "sync:5 copy:0 set:5 set:5 set:5 set:5 sync:5 ");
    CHECK(!status[0] && !left(cnt) && !left(side1) && !left(side2));
    // nothing to clear: one wait, one read
    calls.clear();
    CHECK(tbi::take_status(&c, &st) == TB_OK && st == 0 && calls == "sync:5 copy:0 ");
''')


def test_a_clear_that_fails_is_reported(tmp_path):
    """... and the status stays, so that the next call tries again."""
    run(tmp_path, STATUS + r'''
    for (fail_at = 0; fail_at < 7; ++fail_at) {
        dirty(942);
        CHECK(tbi::take_status(&c, &st) == TB_ERR_CUDA);
        CHECK(fail_at == 6 || status[0] == 942);
    }
    dirty(942);
    CHECK(tbi::take_status(&c, &st) == TB_OK && st == 942 && !left(cnt) && !left(side2));
''')


WORKSPACE = r'''
    tb_ctx c;
    c.stream = (cudaStream_t)5;
    const size_t MB = 1 << 20;
    CHECK(tbi::ensure_workspace(&c, 3) == TB_OK && c.ws_bytes == MB && live.size() == 1);
    void* first = c.ws;
'''


def test_a_workspace_that_no_graph_uses_is_freed(tmp_path):
    run(tmp_path, WORKSPACE + r'''
    CHECK(tbi::ensure_workspace(&c, MB) == TB_OK && c.ws == first);
    calls.clear();
    CHECK(tbi::ensure_workspace(&c, MB + 1) == TB_OK && c.ws_bytes == 2 * MB && c.ws != first);
    CHECK(calls == "sync:5 free:0 " && live.size() == 1 && live.count(c.ws));
''')


def test_a_workspace_that_a_graph_may_use_is_kept(tmp_path):
    """A captured call holds the address; the graph is replayed after other calls have made the workspace grow."""
    run(tmp_path, WORKSPACE + r'''
    capturing = 1;
    CHECK(tbi::ensure_workspace(&c, 100) == TB_OK);
    CHECK(tbi::ensure_workspace(&c, 2 * MB) == TB_ERR_STATE && c.ws == first);
    capturing = 0;
    CHECK(tbi::ensure_workspace(&c, 2 * MB) == TB_OK && c.ws != first);
    CHECK(live.count(first) && c.ws_kept.size() == 1 && c.ws_kept[0] == first);
    // the new one is in no graph yet
    void* second = c.ws;
    CHECK(tbi::ensure_workspace(&c, 4 * MB) == TB_OK && !live.count(second) && live.size() == 2);
''')


def test_a_growth_that_fails_leaves_the_workspace(tmp_path):
    run(tmp_path, WORKSPACE + r'''
    device_left = 0;
    CHECK(tbi::ensure_workspace(&c, 5 * MB) == TB_ERR_OOM);
    CHECK(c.ws == first && c.ws_bytes == MB && live.count(first));
    device_left = ~(size_t)0;
    fail_at = count;  // the wait for queued work fails
    CHECK(tbi::ensure_workspace(&c, 5 * MB) == TB_ERR_CUDA);
    CHECK(c.ws == first && c.ws_bytes == MB && live.count(first) && live.size() == 1);
''')


@pytest.mark.gpu
def test_a_graph_is_replayed_after_the_workspace_has_grown():
    import torch

    import tokens_ref as R
    from tensorium_b200 import Context
    from tensorium_b200 import tokens as K
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(40, 512, device="cuda", generator=g)
    w = torch.randint(-127, 128, (300, 512), device="cuda", generator=g, dtype=torch.int8)
    sw = torch.full((300,), 1e-3, device="cuda")
    out = torch.empty(40, 300, device="cuda")
    side = torch.cuda.Stream()
    with Context(0, workspace_bytes=32 << 20, use_torch_stream=False) as c:
        c.set_stream(side)
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            K.int8_connected(c, x, w, sw, out=out)
        c.reserve(256 << 20)
        others = [torch.full((8 << 20,), 3.0, device="cuda") for _ in range(8)]  # would take the freed memory
        torch.cuda.synchronize()
        x.mul_(2).add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        f64 = lambda t: t.double().cpu().numpy()
        codes, scales = R.quantize(f64(x))
        ref, off = R.product(codes, scales, f64(w), f64(sw), None, "linear", "float32")
        assert (abs(f64(out) - ref) <= off).all()
        assert all((t == 3).all() for t in others)
        del graph
