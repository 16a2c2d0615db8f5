"""The decoding operators where their first tests did not look: sizes at which
a grid or a workspace reaches its limit, infinities and NaN on every path,
lengths beyond a table, waits that run out, captured layers. Tolerances are
counted in roundings as in test_gpu_decode.py."""
import ctypes as C
import math

import pytest
import torch

from test_gpu_decode import BF, D, EPS, F32, U, inv_rms, own_rounding, pair_size, qk_inputs, rand, gen, turn, u, within

pytestmark = pytest.mark.gpu

from catnn_b200 import _lib, ops  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _load():
    import catnn_b200
    catnn_b200.load()


@pytest.mark.parametrize("dtype,h,hkv,hd", [(BF, 2400, 1, 256), (F32, 2500, 3, 128), (BF, 9600, 1, 64), (BF, 4000, 735, 136)])
def test_qk_norm_rope_backward_of_a_token_with_more_heads_than_the_grid_has_warps(dtype, h, hkv, hd):
    """The workspace has the size that is asked for, and nothing behind it changes."""
    _, q, k, wq, wk = qk_inputs(h, dtype, 1, 1, h, hkv, hd, False)
    _, gq, gk, _, _ = qk_inputs(h + 1, dtype, 1, 1, h, hkv, hd, False)
    pos = torch.tensor([[77]], dtype=torch.int32, device="cuda")
    ctx = ops.context(q.device)
    n = C.c_size_t()
    _lib.call("catnn_qk_norm_rope_bwd_workspace", ctx.handle, 1, 1, h, hkv, hd, C.byref(n))
    assert n.value % 4 == 0
    guard = 1 << 18
    ws = torch.full((n.value // 4 + guard,), -12345.0, device="cuda")
    dq, dk, dwq, dwk = torch.empty_like(q), torch.empty_like(k), torch.empty_like(wq), torch.empty_like(wk)
    _lib.call("catnn_qk_norm_rope_bwd", ctx.bind(), q.data_ptr(), h * hd, k.data_ptr(), hkv * hd, wq.data_ptr(), wk.data_ptr(),
              pos.data_ptr(), gq.data_ptr(), h * hd, gk.data_ptr(), hkv * hd, dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(),
              dwk.data_ptr(), 1, 1, h, hkv, hd, 1e5, EPS, 1 if dtype == BF else 0, ws.data_ptr(), n.value)
    assert bool((ws[n.value // 4:] == -12345.0).all()), "what lies behind the workspace"
    for dx, dw, x, w, dy, what in ((dq, dwq, q, wq, gq, "q"), (dk, dwk, k, wk, gk, "k")):
        x, w, dy = x.double(), w.double(), dy.double()
        r, t = inv_rms(x), turn(dy, pos, 1e5, inverse=True)
        xh, tw, size = x * r, t * w, pair_size(dy)
        ref = r * (tw - xh * (tw * xh).mean(-1, keepdim=True))
        # the counts of test_qk_norm_rope_backward
        scale = r * (size * w.abs() + xh.abs() * (size * w.abs() * xh.abs()).mean(-1, keepdim=True))
        within(dx, ref, own_rounding(ref, dtype) * (1 + 1e-3) + 64 * u * scale, f"d{what}")
        within(dw, (t * xh).flatten(0, 2).sum(0), 192 * u * (size * xh.abs()).flatten(0, 2).sum(0), f"dw{what}")
