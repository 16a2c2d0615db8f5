"""CPU checks of the decoding operators: where a token of a paged cache lies
(the kernels' own index functions, built with the host compiler), and the
refusals that need no GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = '''
#include "paged_place.cuh"
extern "C" int position(const int32_t* lens, const int32_t* cu, int seqs, int t, int* seq) {
    return catnn::place::token_position(lens, cu, seqs, t, *seq);
}
extern "C" void positions(const int32_t* lens, const int32_t* cu, int seqs, int t0, int t1, int* out) {
    catnn::place::Token at;  // as a kernel's warp walks its rows
    for (int t = t0; t < t1; ++t) {
        at.move_to(lens, cu, seqs, t);
        out[t - t0] = at.position(t);
    }
}
extern "C" int64_t cache_at(const int32_t* table, int64_t seq, int pos, int page, int max_pages, int64_t pages, int hkv,
                            int hd) {
    return catnn::place::cache_index(table, seq, pos, page, max_pages, pages, hkv, hd);
}
'''


@pytest.fixture(scope="module")
def place(tmp_path_factory):
    d = tmp_path_factory.mktemp("place")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "cat-nn-compiler_b200", "csrc"), str(src), "-o",
                    str(so)], check=True)
    lib = C.CDLL(str(so))
    I32P = C.POINTER(C.c_int32)
    lib.position.argtypes = [I32P, I32P, C.c_int, C.c_int, I32P]
    lib.positions.argtypes = [I32P, I32P, C.c_int, C.c_int, C.c_int, I32P]
    lib.positions.restype = None
    lib.cache_at.argtypes = [I32P, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int64, C.c_int, C.c_int]
    lib.cache_at.restype = C.c_int64
    return lib


def ints(*v):
    return (C.c_int32 * max(1, len(v)))(*v)


def test_positions_of_ragged_new_tokens(place):
    cu, lens = [2, 5, 5, 6, 10], [7, 4, 1, 3]  # sequence 1 has no new token, 3 more than its length
    got = []
    for t in range(12):
        seq = C.c_int32(-7)
        p = place.position(ints(*lens), ints(*cu), 4, t, C.byref(seq))
        got.append((p, seq.value) if p >= 0 else p)
    # rows 0, 1 lie before the first sequence, 10, 11 behind the last; row 6 would be position -1
    assert got == [-1, -1, (4, 0), (5, 0), (6, 0), (0, 2), -1, (0, 3), (1, 3), (2, 3), -1, -1]


def test_positions_of_single_tokens_and_bad_starts(place):
    seq = C.c_int32()
    assert [place.position(ints(5, 0, -3, 1), None, 4, t, C.byref(seq)) for t in range(5)] == [4, -1, -1, 0, -1]
    assert place.position(ints(), ints(0), 0, 0, C.byref(seq)) == -1  # no sequences at all
    # starts that do not ascend name no sequence, and never an index out of [0, seqs)
    r = np.random.default_rng(0)
    for _ in range(2000):
        n = int(r.integers(1, 6))
        cu, lens = r.integers(-5, 15, n + 1), r.integers(-5, 40, n)
        t = int(r.integers(0, 20))
        seq = C.c_int32(0)
        p = place.position(ints(*map(int, lens)), ints(*map(int, cu)), n, t, C.byref(seq))
        assert p >= -1
        if p >= 0:
            assert 0 <= seq.value < n and cu[seq.value] <= t < cu[seq.value + 1]
            assert p == lens[seq.value] - (cu[seq.value + 1] - t)


def test_positions_of_a_walk(place):
    """A walk over rows, from anywhere, finds what a look-up of each finds."""
    r = np.random.default_rng(1)
    for _ in range(300):
        n = int(r.integers(1, 9))
        cu = np.concatenate([[0], np.cumsum(r.integers(0, 6, n))]) + int(r.integers(0, 3))
        lens = ints(*map(int, r.integers(-2, 12, n)))
        c = ints(*map(int, cu))
        t0, t1 = sorted(map(int, r.integers(0, 30, 2)))
        out = ints(*([0] * (t1 - t0)))
        place.positions(lens, c, n, t0, t1, out)
        seq = C.c_int32()
        assert list(out)[:t1 - t0] == [place.position(lens, c, n, t, C.byref(seq)) for t in range(t0, t1)]
    # lengths at the ends of their type do not wrap around
    big = 2 ** 31 - 1
    assert place.position(ints(-big - 1), ints(0, big), 1, 0, C.byref(seq)) == -1
    assert place.position(ints(big), ints(0, big), 1, big - 1, C.byref(seq)) == big - 1


@pytest.mark.parametrize("page", [1, 3, 16, 128])
def test_cache_index_stays_in_the_pool(place, page):
    r = np.random.default_rng(page)
    pages, hkv, hd, seqs, most = 9, 3, 40, 4, 5
    table = r.integers(-2, pages + 2, (seqs, most)).astype(np.int32)
    flat = ints(*map(int, table.reshape(-1)))
    for s in range(seqs):
        for pos in list(range(-2, page * most + 3)) + [2 ** 31 - 1]:
            at = place.cache_at(flat, s, pos, page, most, pages, hkv, hd)
            slot = pos // page
            ok = 0 <= slot < most and 0 <= table[s, slot] < pages
            assert (at >= 0) == ok
            if ok:
                assert at == (int(table[s, slot]) * hkv * page + pos % page) * hd
                assert at + (hkv - 1) * page * hd + hd <= pages * hkv * page * hd


def test_cache_index_passes_32_bits(place):
    assert place.cache_at(ints(2_000_000), 0, 15, 16, 1, 2_000_001, 8, 128) == (2_000_000 * 8 * 16 + 15) * 128 > 2 ** 34


# ------------------------------------------------------------------ refusals before any kernel
def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_refusals_without_a_gpu():
    from catnn_b200 import ops
    from catnn_b200.errors import DTypeMismatch, InvalidArgument, ShapeMismatch
    q, k, w = z(2, 3, 4, 8), z(2, 3, 2, 8), z(8)
    for bad, err in (((q, z(2, 3, 2, 6), w, w), ShapeMismatch), ((q, z(2, 4, 2, 8), w, w), ShapeMismatch),
                     ((q[0], k[0], w, w), ShapeMismatch), ((q, k.bfloat16(), w, w), DTypeMismatch),
                     ((q, k, w, w), InvalidArgument)):  # the last is right but not on a GPU
        with pytest.raises(err):
            ops.qk_norm_rope(*bad, 1e4)
        with pytest.raises(err):
            ops.qk_norm_rope_backward(*bad, bad[0], bad[1], 1e4)
    with pytest.raises(ShapeMismatch):
        ops.qk_norm_rope(q, k, w, w, 1e4, positions=i(3, 2))
    with pytest.raises(ShapeMismatch):
        ops.qk_norm_rope_backward(q, k, w, w, k, k, 1e4)
    cache, table, lens = z(5, 2, 4, 8), i(3, 2), i(3)
    t3, kk = z(3, 4, 8), z(3, 2, 8)
    ops_append = [((t3, kk, z(3, 2, 6), cache, cache, table, lens), {}, ShapeMismatch),
                  ((z(2, 4, 8), kk, kk, cache, cache, table, lens), {}, ShapeMismatch),
                  ((t3, kk, kk, z(5, 3, 4, 8), cache, table, lens), {}, ShapeMismatch),
                  ((t3, kk, kk, z(5, 2, 4, 16)[..., ::2], z(5, 2, 4, 16)[..., ::2], table, lens), {}, InvalidArgument),
                  ((t3, kk, kk, cache.bfloat16(), cache, table, lens), {}, DTypeMismatch),
                  ((t3, kk, kk, cache, cache, table.long(), lens), {}, DTypeMismatch),
                  ((t3, kk, kk, cache, cache, table, i(4)), {}, ShapeMismatch),
                  ((z(2, 4, 8), z(2, 2, 8), z(2, 2, 8), cache, cache, table, lens), {}, ShapeMismatch),
                  ((t3, kk, kk, cache, cache, table, lens), {"cu_tokens": i(3)}, ShapeMismatch),
                  ((t3, kk, kk, cache, cache, table, lens), {"wq": w}, InvalidArgument),
                  ((t3, kk, kk, cache, cache, table, lens), {}, InvalidArgument)]
    for args, kw, err in ops_append:
        with pytest.raises(err):
            ops.kv_append(*args, 1e4, **kw)
    for args, err in (((z(3, 3, 8), cache, cache, table, lens), ShapeMismatch), ((z(2, 4, 8), cache, cache, table, lens),
                      ShapeMismatch), ((t3, cache, cache, table, i(3, 1)), ShapeMismatch),
                      ((t3.bfloat16(), cache, cache, table, lens), DTypeMismatch),
                      ((t3, cache, cache, table, lens), InvalidArgument)):
        with pytest.raises(err):
            ops.paged_attention(*args)
    x, gate, w1, w2 = z(3, 8), z(8, 4), z(4, 8, 16), z(4, 16, 8)
    for args, err in (((x, gate, w1, w1, w1, 2), ShapeMismatch), ((x, z(8, 5), w1, w1, w2, 2), ShapeMismatch),
                      ((x, gate, w1, w1, w2, 5), ShapeMismatch), ((x, gate, w1, w1, w2, 0), ShapeMismatch),
                      ((z(65, 8), gate, w1, w1, w2, 2), ShapeMismatch), ((x, gate.bfloat16(), w1, w1, w2, 2), DTypeMismatch),
                      ((x, gate, w1, w1, w2.transpose(1, 2).contiguous().transpose(1, 2), 2), InvalidArgument),
                      ((x, gate, w1, w1, w2, 2), InvalidArgument)):
        with pytest.raises(err):
            ops.moe_few(*args)


def test_token_strides():
    from catnn_b200.errors import InvalidArgument
    from catnn_b200.ops import _rows
    qkv = z(2, 3, 48)
    assert _rows(qkv[..., :32].unflatten(-1, (4, 8)), "q") == 48
    assert _rows(z(2, 3, 4, 8), "q") == 32
    assert _rows(qkv[:, :1, 32:40].unflatten(-1, (1, 8)), "q") == 144  # one token a sequence
    assert _rows(qkv[:1, :1, :8].unflatten(-1, (1, 8)), "q") == 8
    for bad in (qkv[:, ::2, :32].unflatten(-1, (4, 8)), z(2, 3, 8, 4).transpose(-1, -2), z(2, 4, 3, 8).transpose(1, 2)):
        with pytest.raises(InvalidArgument):
            _rows(bad, "q")
