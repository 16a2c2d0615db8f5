"""CPU checks of the decoding operators' host arithmetic: how rows are dealt out
to a grid (the launchers' own functions, built with the host compiler), and how
the Python entry points drive the context."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = '''
#include <vector>
#include "row_deal.cuh"
using namespace catnn::deal;
// CTAs of a grid; `rows`: what the workspace of the adjoint has of each weight sum, for `heads` heads.
extern "C" int grid(int sms, int64_t tokens, int groups, int per_sm, int runs, int64_t heads, int64_t* rows) {
    Deal d;
    *rows = adjoint_rows(sms, tokens, heads);
    return deal_out(sms, tokens, groups, per_sm, runs != 0, d);
}
// Whether the grid's warps have every group of every token, each once.
extern "C" int covers(int sms, int tokens, int groups, int per_sm, int runs) {
    Deal d;
    const int ctas = deal_out(sms, tokens, groups, per_sm, runs != 0, d);
    std::vector<int> seen((size_t)tokens * groups, 0);
    for (int w = 0; w < ctas * WARPS; ++w) {
        const Share s = share_of(d, w);
        for (int t = s.t0; t < s.t1; t += s.dt)
            for (int g = s.g0; g < s.g1; ++g) ++seen[(size_t)t * groups + g];
    }
    for (int n : seen)
        if (n != 1) return 0;
    return 1;
}
'''


@pytest.fixture(scope="module")
def deal(tmp_path_factory):
    d = tmp_path_factory.mktemp("deal")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "cat-nn-compiler_b200", "csrc"),
                    str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.grid.argtypes = [C.c_int, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int64, C.POINTER(C.c_int64)]
    lib.covers.argtypes = [C.c_int] * 5
    return lib


@pytest.mark.parametrize("sms", [148, 1, 132])
def test_a_grid_never_passes_its_limit(deal, sms):
    """Not even where one token has more row groups than the grid has warps;
    and the adjoint's workspace has a row for every CTA."""
    rows = C.c_int64()
    groups = sorted({1, 2, 5, 7, 20, 296, 2367, 2368, 2369, 2400, 3552, 3553, 4735, 9601, 16385, 32768}
                    | set(map(int, np.random.default_rng(sms).integers(1, 32769, 60))))
    for tokens in (1, 2, 3, 4, 8, 9, 63, 1000, 16384, 300_000, 0x7fff0000):
        for n in groups:
            for per_sm, runs in ((2, 0), (3, 0), (3, 1)):
                ctas = deal.grid(sms, tokens, n, per_sm, runs, n, C.byref(rows))  # at least as many heads as groups
                assert 1 <= ctas <= sms * per_sm, (tokens, n, per_sm, ctas)
                if per_sm == 2:
                    assert ctas <= rows.value, (tokens, n, ctas, rows.value)


def test_a_grid_has_every_row_once(deal):
    r = np.random.default_rng(0)
    cases = [(148, 1, 4735, 2, 0), (148, 1, 2401, 2, 0), (1, 1, 100, 2, 0), (1, 3, 33, 3, 1), (148, 16384, 5, 3, 0)]
    cases += [(int(r.choice([1, 4, 148])), int(np.exp(r.uniform(0, 8))), int(np.exp(r.uniform(0, 6))), int(r.integers(2, 4)),
               int(r.integers(0, 2))) for _ in range(200)]
    for c in cases:
        assert deal.covers(*c), c


def test_bind_sets_the_stream_every_time(monkeypatch):
    """The handle's stream is what the caller's is, whoever set it last: another
    thread between two calls, or a caller through the C ABI."""
    from types import SimpleNamespace

    import torch

    from catnn_b200 import _lib, ops
    handle = {"stream": None}
    now = {"stream": 0}

    def call(name, *args):
        if name == "catnn_ctx_set_stream":
            handle["stream"] = args[1].value or 0
        elif name == "catnn_ctx_create":
            args[1]._obj.value = 1234
        return 0
    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=now["stream"]))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: now["stream"], raising=False)
    ctx = ops.Context(0)
    for mine, other in ((0, 64), (64, 0), (64, 128), (128, 128)):
        now["stream"] = mine
        ctx.bind()
        assert handle["stream"] == mine
        handle["stream"] = other  # behind the context's back
        ctx.bind()
        assert handle["stream"] == mine


def test_the_stream_without_torchs_shortcut(monkeypatch):
    from types import SimpleNamespace

    import torch

    from catnn_b200 import ops
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=7 + device))
    assert ops._stream_of(1) == 8
