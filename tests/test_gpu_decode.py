"""The decoding operators and the per-head query/key norm on the GPU, against
plain implementations in 64 bits.

Tolerances are counted in roundings. u = 2^-24 is half a step of fp32, U = 2^-8
half a step of bf16, both relative to the rounded value. Each bound below is
U·|result| for a bf16 result's own rounding plus a count of fp32 roundings
times the sum of the magnitudes that enter; the counts stand at each check.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from catnn_b200 import _lib, ops  # noqa: E402
from catnn_b200.errors import InvalidArgument, ShapeMismatch, Unsupported  # noqa: E402

u, U = 2.0 ** -24, 2.0 ** -8
F32, BF = torch.float32, torch.bfloat16
D = torch.float64
EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def _load():
    import catnn_b200
    catnn_b200.load()


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, ref, bound, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    over = err - bound
    assert not torch.isnan(got).any() and bool((over <= 0).all()), (
        f"{what}: {int((over > 0).sum())} of {ref.numel()} out of bounds, worst by {float(over.max()):.3e} "
        f"(error {float(err.max()):.3e}, value {float(ref.abs().max()):.3e})")


def own_rounding(ref, dtype):
    return ref.abs() * (U if dtype == BF else 0.0)


# ------------------------------------------------------------------ references in 64 bits
def turn(x, pos, theta, inverse=False):
    """Pairs (2i, 2i+1) of x [..., heads, hd] turned by pos·theta^(-2i/hd)."""
    hd = x.shape[-1]
    f = theta ** (-torch.arange(0, hd, 2, dtype=D, device=x.device) / hd)
    ang = (pos.double()[..., None] * f)[..., None, :] * (-1 if inverse else 1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()), -1).flatten(-2)


def pair_size(x):
    """|x_2i| + |x_2i+1| at both places of each pair."""
    s = x.abs().unflatten(-1, (-1, 2)).sum(-1)
    return torch.stack((s, s), -1).flatten(-2)


def inv_rms(x):
    return (x.square().mean(-1, keepdim=True) + EPS).rsqrt()


def norm_turn(x, w, pos, theta):
    x = x.double()
    y = x if w is None else x * inv_rms(x) * w.double()
    return turn(y, pos, theta), pair_size(y)


def qk_inputs(seed, dtype, b, s, h, hkv, hd, packed, scale=1.0):
    g = gen(seed)
    if packed:
        qkv = rand(g, b, s, (h + 2 * hkv) * hd, dtype=dtype, scale=scale)
        q = qkv[..., :h * hd].unflatten(-1, (h, hd))
        k = qkv[..., h * hd:(h + hkv) * hd].unflatten(-1, (hkv, hd))
    else:
        q, k = rand(g, b, s, h, hd, dtype=dtype, scale=scale), rand(g, b, s, hkv, hd, dtype=dtype, scale=scale)
    return g, q, k, 1 + rand(g, hd, scale=0.3), 1 + rand(g, hd, scale=0.3)


QK = [  # b, s, h, hkv, hd, packed
    (1, 1, 1, 1, 64, False), (2, 37, 4, 2, 64, True), (1, 5, 16, 4, 128, True), (3, 33, 6, 2, 80, False),
    (2, 9, 3, 3, 96, True), (1, 700, 5, 1, 32, False), (1, 3, 2, 1, 256, True), (2, 4, 3, 1, 2, False),
    (1, 6, 5, 2, 30, True), (1, 2, 2, 2, 254, False), (1, 17, 7, 7, 16, False), (2, 8, 2, 1, 8, True), (5, 1, 4, 4, 48, True),
    (2, 3001, 16, 4, 128, True), (1, 2500, 19, 3, 96, False)]  # warps with many tokens, tokens of several batches of rows


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("b,s,h,hkv,hd,packed", QK)
def test_qk_norm_rope(b, s, h, hkv, hd, packed, dtype):
    g, q, k, wq, wk = qk_inputs(b * 1000 + s + hd, dtype, b, s, h, hkv, hd, packed)
    far = torch.randint(-5, 200_000, (b, s), generator=g, device="cuda", dtype=torch.int32)
    for theta, pos in ((1e4, None), (1e6, far)):
        at = torch.arange(s, device="cuda").expand(b, s) if pos is None else pos
        got = ops.qk_norm_rope(q, k, wq, wk, theta, EPS, pos)
        for y, x, w, what in ((got[0], q, wq, "q"), (got[1], k, wk, "k")):
            ref, size = norm_turn(x, w, at, theta)
            # sum of squares, division, root: <= 24 roundings (half of them reach r); two products; angle and sine:
            # 4 in fp32, 11 for bf16's hardware sine; the turn: 3
            assert y.is_contiguous() and y.dtype == dtype
            within(y, ref, own_rounding(ref, dtype) * (1 + 1e-3) + 64 * u * size, f"{what} theta {theta}")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("b,s,h,hkv,hd,packed", QK)
def test_qk_norm_rope_backward(b, s, h, hkv, hd, packed, dtype):
    g, q, k, wq, wk = qk_inputs(b * 1000 + s + hd, dtype, b, s, h, hkv, hd, packed)
    _, gq, gk, _, _ = qk_inputs(7 + hd, dtype, b, s, h, hkv, hd, not packed)
    pos = torch.randint(0, 9000, (b, s), generator=g, device="cuda", dtype=torch.int32)
    theta = 1e5
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(q, k, wq, wk, gq, gk, theta, EPS, pos)
    again = ops.qk_norm_rope_backward(q, k, wq, wk, gq, gk, theta, EPS, pos)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dwq, dwk), again)), "the same bits on every call"
    for dx, dw, x, w, dy, what in ((dq, dwq, q, wq, gq, "q"), (dk, dwk, k, wk, gk, "k")):
        x, w, dy = x.double(), w.double(), dy.double()
        r, t = inv_rms(x), turn(dy, pos, theta, inverse=True)
        xh, tw, size = x * r, t * w, pair_size(dy)
        ref = r * (tw - xh * (tw * xh).mean(-1, keepdim=True))
        # as forward, and the second sum over hd: <= 64 roundings of the terms that enter
        scale = r * (size * w.abs() + xh.abs() * (size * w.abs() * xh.abs()).mean(-1, keepdim=True))
        within(dx, ref, own_rounding(ref, dtype) * (1 + 1e-3) + 64 * u * scale, f"d{what}")
        # at these sizes a sum passes <= 128 additions (a lane's rows, 8 warps, CTAs / 32, 32 row groups)
        within(dw, (t * xh).flatten(0, 2).sum(0), 192 * u * (size * xh.abs()).flatten(0, 2).sum(0), f"dw{what}")


def test_qk_norm_rope_gradient_by_differences():
    """The adjoint against central differences of the forward's own formula:
    the gradient of <y, c> along a random direction, in 64 bits, and against
    torch's autograd of the same formula."""
    _, q, k, wq, wk = qk_inputs(5, F32, 2, 7, 4, 2, 64, False)
    _, cq, ck, _, _ = qk_inputs(6, F32, 2, 7, 4, 2, 64, False)
    pos = torch.arange(7, device="cuda", dtype=torch.int32).expand(2, 7).contiguous()
    grads = ops.qk_norm_rope_backward(q, k, wq, wk, cq, ck, 1e4, EPS, pos)

    def f(a, b, c, d):
        return (norm_turn(a, c, pos, 1e4)[0] * cq.double()).sum() + (norm_turn(b, d, pos, 1e4)[0] * ck.double()).sum()
    at = [t.double() for t in (q, k, wq, wk)]
    g = gen(9)
    for i in range(4):
        d = torch.randn(at[i].shape, generator=g, device="cuda", dtype=D)
        h = 1e-5
        num = (f(*[t + h * d if j == i else t for j, t in enumerate(at)])
               - f(*[t - h * d if j == i else t for j, t in enumerate(at)])) / (2 * h)
        ours = (grads[i].double() * d).sum()
        # differences: h² third derivatives (~1e-9 of the sum of magnitudes) and 1e-16/h rounding; ours: 192 roundings
        size = float((grads[i].double() * d).abs().sum())
        assert abs(float(num - ours)) <= 1e-8 * size + 192 * u * size * 4, (i, float(num), float(ours))
    leaves = [t.clone().requires_grad_() for t in at]
    for got, ref in zip(grads, torch.autograd.grad(f(*leaves), leaves)):
        assert float((got.double() - ref).norm() / ref.norm()) < 64 * u


def test_qk_norm_rope_edges():
    w = torch.ones(64, device="cuda")
    # zero rows: r = eps^-1/2, output and every gradient but r·g·w vanish
    z = torch.zeros(1, 3, 2, 64, device="cuda")
    y, _ = ops.qk_norm_rope(z, z, w, w, 1e4)
    assert not y.any()
    one = torch.ones_like(z)
    dq, _, dwq, _ = ops.qk_norm_rope_backward(z, z, w, w, one, one, 1e4)
    within(dq, turn(one.double(), torch.arange(3, device="cuda")[None], 1e4, inverse=True) * EPS ** -0.5,
           torch.full_like(dq, 64 * u * 2 * EPS ** -0.5, dtype=D), "dx of a zero row")
    assert not dwq.any()
    # no tokens
    e = torch.empty(0, 5, 2, 64, device="cuda")
    assert ops.qk_norm_rope(e, e, w, w, 1e4)[0].shape == (0, 5, 2, 64)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(e, e, w, w, e, e, 1e4)
    assert dq.shape == e.shape and not dwq.any() and not dwk.any()
    # one token's NaN stays in its own head
    q = torch.randn(1, 4, 3, 64, device="cuda")
    q[0, 1, 2, 5] = float("nan")
    y, _ = ops.qk_norm_rope(q, q, w, w, 1e4)
    bad = torch.isnan(y).any(-1)
    assert bad[0, 1, 2] and int(bad.sum()) == 1
    # rows that no 16-byte access can take
    base = torch.randn(1 + 6 * 2 * 64, device="cuda")
    q = base[1:].view(1, 6, 2, 64)
    ref, size = norm_turn(q, w, torch.arange(6, device="cuda")[None], 1e4)
    within(ops.qk_norm_rope(q, q, w, w, 1e4)[0], ref, 64 * u * size, "misaligned rows")
    # the same call in place, through the C ABI
    x, x2 = torch.randn(2, 5, 3, 64, device="cuda"), torch.randn(2, 5, 3, 64, device="cuda")
    want = ops.qk_norm_rope(x, x2, w, w, 1e4)
    _lib.call("catnn_qk_norm_rope_fwd", ops.context(x.device).bind(), x.data_ptr(), 192, x2.data_ptr(), 192, w.data_ptr(),
              w.data_ptr(), None, x.data_ptr(), x2.data_ptr(), 2, 5, 3, 3, 64, 1e4, EPS, 0)
    assert torch.equal(x, want[0]) and torch.equal(x2, want[1])


def test_qk_norm_rope_is_rmsnorm_then_rope():
    """The two operators that it stands beside, one after the other."""
    for dtype in (F32, BF):
        _, q, k, wq, wk = qk_inputs(3, dtype, 2, 50, 4, 2, 64, False)
        y, _ = ops.qk_norm_rope(q, k, wq, wk, 1e4, EPS)
        two = ops.rope(ops.rmsnorm(q, wq, EPS), 1e4)
        _, size = norm_turn(q, wq, torch.arange(50, device="cuda")[None], 1e4)
        # the pair of calls rounds in between: U on each element of a pair, then both round the result
        bound = (3 * U if dtype == BF else 0) * size + 128 * u * size
        within(y, two.double(), bound, "rmsnorm + rope")


# ------------------------------------------------------------------ paged cache
def make_cache(g, dtype, lens, hkv, hd, page, spare=2, fill=None):
    need = [-(-max(n, 0) // page) for n in lens]
    most, total = max(need + [1]), sum(need)
    pool = total + spare
    kc, vc = rand(g, pool, hkv, page, hd, dtype=dtype), rand(g, pool, hkv, page, hd, dtype=dtype)
    ids = torch.randperm(pool, generator=g, device="cuda")[:total].int().cpu()
    table = torch.full((len(lens), most), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    if fill is not None:  # everything that no sequence holds
        held = torch.zeros(pool, page, dtype=torch.bool)
        for i, n in enumerate(lens):
            for j in range(n):
                held[table[i, j // page], j % page] = True
        kc.transpose(1, 2)[~held.cuda()] = fill
        vc.transpose(1, 2)[~held.cuda()] = fill
    return kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def gather(cache, table, b, lo, n):
    page = cache.shape[2]
    j = torch.arange(lo, n, device="cuda")
    return cache[table[b].long()[j // page], :, j % page]  # [n - lo, hkv, hd]


APPEND = [  # lens with the new tokens, new tokens, h, hkv, hd, page
    ([5], [1], 4, 2, 64, 16), ([1], [1], 1, 1, 64, 1), ([40, 3, 17, 16], [40, 3, 1, 16], 4, 4, 64, 16),
    ([100, 7, 33], [3, 0, 33], 8, 2, 128, 24), ([20, 20], [5, 20], 3, 1, 80, 8), ([9, 2], [9, 1], 2, 2, 30, 4),
    ([300], [300], 5, 5, 96, 128), ([12, 31, 7], [12, 30, 2], 2, 1, 256, 5)]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lens,new,h,hkv,hd,page", APPEND)
def test_kv_append(lens, new, h, hkv, hd, page, dtype, norm):
    g = gen(sum(lens) + hd)
    kc, vc, table, ln = make_cache(g, dtype, lens, hkv, hd, page)
    behind = 3  # rows of no sequence
    t = sum(new) + behind
    qkv = rand(g, t, (h + 2 * hkv) * hd, dtype=dtype)
    q, k, v = (x.unflatten(-1, (-1, hd)) for x in qkv.split([h * hd, hkv * hd, hkv * hd], -1))
    wq, wk = (1 + rand(g, hd, scale=0.3), 1 + rand(g, hd, scale=0.3)) if norm else (None, None)
    cu = torch.tensor([0] + new).cumsum(0).int().cuda()
    k0, v0 = kc.clone(), vc.clone()
    qo = ops.kv_append(q, k, v, kc, vc, table, ln, 1e5, cu_tokens=cu, wq=wq, wk=wk, eps=EPS, check=True)
    where = torch.tensor([p for n, m in zip(lens, new) for p in range(n - m, n)] + [0] * behind, device="cuda")
    qr, qs = norm_turn(q, wq, where, 1e5)
    kr, ks = norm_turn(k, wk, where, 1e5)
    qr[sum(new):] = qs[sum(new):] = 0
    within(qo, qr, own_rounding(qr, dtype) * (1 + 1e-3) + 64 * u * qs, "queries")
    row = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for j in range(n - m, n):
            p, s = int(table[b, j // page]), j % page
            within(kc[p, :, s], kr[row], own_rounding(kr[row], dtype) * (1 + 1e-3) + 64 * u * ks[row], "keys")
            assert torch.equal(vc[p, :, s], v[row])
            k0[p, :, s], v0[p, :, s] = kc[p, :, s], vc[p, :, s]
            row += 1
    assert torch.equal(kc, k0) and torch.equal(vc, v0), "every other slot stays as it was"
    # without queries the cache gets the same bits
    k1, v1 = k0.clone(), v0.clone()
    assert ops.kv_append(None, k, v, k1, v1, table, ln, 1e5, cu_tokens=cu, wq=wq, wk=wk, eps=EPS) is None
    assert torch.equal(k1, kc) and torch.equal(v1, vc)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_kv_append_long_prompts(dtype):
    """Prompts of thousands of rows, of which a warp walks many, across
    sequence ends, sequences without new tokens and page ends."""
    g = gen(44)
    new = [1999, 0, 3, 1500, 1, 0, 777]
    lens = [n + m for n, m in zip(new, [0, 40, 13, 2, 500, 0, 31])]
    h, hkv, hd, page = 16, 4, 128, 24
    kc, vc, table, ln = make_cache(g, dtype, lens, hkv, hd, page)
    t = sum(new)
    qkv = rand(g, t + 5, (h + 2 * hkv) * hd, dtype=dtype)
    q, k, v = (x.unflatten(-1, (-1, hd)) for x in qkv.split([h * hd, hkv * hd, hkv * hd], -1))
    w = 1 + rand(g, 2, hd, scale=0.3)
    cu = torch.tensor([0] + new).cumsum(0).int().cuda()
    k0, v0 = kc.clone(), vc.clone()
    qo = ops.kv_append(q, k, v, kc, vc, table, ln, 1e6, cu_tokens=cu, wq=w[0], wk=w[1], eps=EPS, check=True)
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(new)]).cuda()
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).cuda()
    at = (table[seq, pos // page].long(), slice(None), pos % page)
    kr, ks = norm_turn(k[:t], w[1], pos, 1e6)
    qr, qs = norm_turn(q[:t], w[0], pos, 1e6)
    within(kc[at], kr, own_rounding(kr, dtype) * (1 + 1e-3) + 64 * u * ks, "keys")
    within(qo[:t], qr, own_rounding(qr, dtype) * (1 + 1e-3) + 64 * u * qs, "queries")
    assert torch.equal(vc[at], v[:t]) and not qo[t:].any()
    k0[at], v0[at] = kc[at], vc[at]
    assert torch.equal(kc, k0) and torch.equal(vc, v0), "every other slot stays as it was"


def test_kv_append_one_token_each_and_idle_sequences():
    g = gen(4)
    kc, vc, table, ln = make_cache(g, BF, [7, 0, 33, -2, 16], 2, 64, 16)
    q, k, v = rand(g, 5, 4, 64, dtype=BF), rand(g, 5, 2, 64, dtype=BF), rand(g, 5, 2, 64, dtype=BF)
    q[1] = float("nan")  # an idle row's leftovers
    k0, v0 = kc.clone(), vc.clone()
    qo = ops.kv_append(q, k, v, kc, vc, table, ln, 1e4, check=True)
    assert not qo[1].any() and not qo[3].any() and torch.equal(vc[table[4, 0], :, 15], v[4])
    cu = torch.arange(6, dtype=torch.int32, device="cuda")
    assert torch.equal(qo, ops.kv_append(q, k, v, k0, v0, table, ln, 1e4, cu_tokens=cu))
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_kv_append_pages_that_are_not_there():
    """Positions without a page are left out; check=True says so, and an
    unchecked call before it does not."""
    g = gen(5)
    kc, vc, table, ln = make_cache(g, F32, [20, 20], 1, 64, 16)
    table[0, 1], table[1, 1] = -1, kc.shape[0]
    k0, v0 = kc.clone(), vc.clone()
    q, k = rand(g, 2, 1, 64), rand(g, 2, 1, 64)
    ops.kv_append(q, k, k, kc, vc, table, ln, 1e4)
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    with pytest.raises(ShapeMismatch, match="no page"):
        ops.kv_append(q, k, k, kc, vc, table, ln, 1e4, check=True)
    ln[:] = 1000  # beyond the table
    with pytest.raises(ShapeMismatch, match="no page"):
        ops.kv_append(q, k, k, kc, vc, table, ln, 1e4, check=True)
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    ln[:] = 3
    ops.kv_append(q, k, k, kc, vc, table, ln, 1e4)
    ops.kv_append(q, k, k, kc, vc, table, ln, 1e4, check=True)
    # no sequences, no pages, no tokens
    e = torch.empty(0, 1, 64, device="cuda")
    none = torch.empty(0, 1, 16, 64, device="cuda")
    assert ops.kv_append(e, e, e, none, none, table[:0], ln[:0], 1e4).shape == (0, 1, 64)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not ops.kv_append(q, k, k, kc, vc, table[:0], ln[:0], 1e4, cu_tokens=zero).any()


def attention_ref(q, kc, vc, table, lens, window):
    b, h, hd = q.shape
    hkv = kc.shape[1]
    o, lse = torch.zeros(b, h, hd, dtype=D, device="cuda"), torch.full((b, h), -math.inf, dtype=D, device="cuda")
    mean, spread = torch.zeros_like(o), torch.zeros(b, h, dtype=D, device="cuda")
    for i, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        lo = max(0, n - window) if window else 0
        k, v = gather(kc, table, i, lo, n).double(), gather(vc, table, i, lo, n).double()
        qq = q[i].double().view(hkv, h // hkv, hd)
        s = torch.einsum("ngd,jnd->ngj", qq, k) / math.sqrt(hd)
        p = torch.softmax(s, -1)
        o[i] = torch.einsum("ngj,jnd->ngd", p, v).reshape(h, hd)
        mean[i] = torch.einsum("ngj,jnd->ngd", p, v.abs()).reshape(h, hd)
        lse[i] = torch.logsumexp(s, -1).reshape(h)
        spread[i] = (torch.einsum("ngd,jnd->ngj", qq.abs(), k.abs()).amax(-1) / math.sqrt(hd)).reshape(h)
    return o.view(b, h * hd), lse, mean.view(b, h * hd), spread


def check_attention(q, kc, vc, table, lens, window, o, lse):
    dtype, (b, h, hd) = q.dtype, q.shape
    ref, rl, mean, spread = attention_ref(q, kc, vc, table, lens, window)
    # a score passes <= hd + 8 fp32 roundings of its products' magnitudes and moves its weight by as much, in numerator
    # and sum; the weights are held in the cache's type for the second product (bf16: U each, so up to U·Σp|v|);
    # exponential, sums in tiles and joins: <= 64 + len/64 roundings
    n = float(lens.max()) if b else 0
    score = (2 * (hd + 8) * u * spread)[:, :, None].expand(b, h, hd).reshape(b, h * hd)
    bound = own_rounding(ref, dtype) * (1 + 1e-3) + (score + (64 + n / 64) * u + (U if dtype == BF else 0)) * mean
    within(o, ref, bound, "o")
    empty = lens <= 0
    assert bool((lse[empty] == -math.inf).all()) and not o[empty].any()
    within(lse[~empty], rl[~empty], ((hd + 8) * u * spread + (64 + n / 64) * u + 4 * u * rl.abs())[~empty], "lse")


PAGED = [  # lens, h, hkv, hd, page, window
    ([1], 1, 1, 64, 16, 0), ([1, 0, 2], 4, 2, 64, 16, 0), ([17, 300, 16, 15, 64], 4, 4, 64, 16, 0),
    ([1000, 1, 63], 16, 4, 128, 16, 0), ([129, 5], 8, 1, 128, 32, 0), ([77], 10, 2, 96, 24, 0), ([50, 90], 6, 2, 80, 1, 0),
    ([200, 4096], 16, 1, 64, 64, 0), ([333, 20], 40, 2, 64, 16, 0), ([40, 41], 3, 3, 7, 8, 0), ([65], 4, 2, 32, 128, 0),
    ([500, 3, 99, 0], 4, 2, 64, 16, 100), ([500], 8, 2, 128, 16, 1), ([2000, 31], 2, 1, 16, 5, 777), ([260], 9, 3, 120, 16, 33),
    ([0, 0], 2, 1, 64, 16, 0), (list(range(0, 64)), 2, 2, 64, 8, 0)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lens,h,hkv,hd,page,window", PAGED)
def test_paged_attention(lens, h, hkv, hd, page, window, dtype):
    g = gen(sum(lens) + h + hd)
    # slots that no sequence holds are NaN: past an end, in other pages
    kc, vc, table, ln = make_cache(g, dtype, lens, hkv, hd, page, fill=math.nan)
    if window:  # and so are the positions that left the window
        for i, n in enumerate(lens):
            for j in range(max(0, n - window)):
                kc[table[i, j // page], :, j % page] = vc[table[i, j // page], :, j % page] = math.nan
    wide = rand(g, len(lens), (h + 2 * hkv) * hd, dtype=dtype)
    q = wide[:, :h * hd].unflatten(-1, (h, hd))
    o, lse = ops.paged_attention(q, kc, vc, table, ln, window or None, check=True)
    assert o.shape == (len(lens), h * hd) and o.dtype == dtype
    check_attention(q, kc, vc, table, ln, window, o, lse)
    again = ops.paged_attention(q.contiguous(), kc, vc, table, ln, window)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1]), "the same bits on every call"


@pytest.mark.parametrize("dtype,n,h,hkv,hd,page", [(BF, 30011, 16, 4, 128, 16), (F32, 20001, 8, 2, 64, 64),
                                                   (BF, 70000, 2, 1, 64, 16)])
def test_paged_attention_long(dtype, n, h, hkv, hd, page):
    g = gen(n)
    lens = [n, 5, n // 3]
    kc, vc, table, ln = make_cache(g, dtype, lens, hkv, hd, page)
    q = rand(g, 3, h, hd, dtype=dtype)
    o, lse = ops.paged_attention(q, kc, vc, table, ln)
    check_attention(q, kc, vc, table, ln, 0, o, lse)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_paged_attention_many_short_sequences(dtype):
    """More sequences than one warp's scan counts at once, many of them empty."""
    g = gen(9)
    b, page, hd = 20_000, 16, 16
    lens = torch.randint(-3, 45, (b,), generator=g, device="cuda").int()
    table = torch.randperm(b * 3, generator=g, device="cuda")[:b * 3].int().view(b, 3).contiguous()
    kc, vc = rand(g, b * 3, 1, page, hd, dtype=dtype), rand(g, b * 3, 1, page, hd, dtype=dtype)
    q = rand(g, b, 2, hd, dtype=dtype)
    o, lse = ops.paged_attention(q, kc, vc, table, lens, check=True)
    k, v = (x[table.long()].view(b, 3 * page, hd).double() for x in (kc, vc))
    s = q.double() @ k.transpose(1, 2) / math.sqrt(hd)
    out = torch.arange(3 * page, device="cuda") >= lens[:, None]
    p = torch.softmax(s.masked_fill(out[:, None], -math.inf), -1).nan_to_num(0.0)
    ref, mean = (p @ v).reshape(b, -1), (p @ v.abs()).reshape(b, -1)
    spread = float((q.double().abs() @ k.abs().transpose(1, 2)).amax()) / math.sqrt(hd)
    within(o, ref, own_rounding(ref, dtype) * (1 + 1e-3)
           + (2 * (hd + 8) * u * spread + 64 * u + (U if dtype == BF else 0)) * mean, "o")
    assert bool((lse[lens <= 0] == -math.inf).all()) and torch.isfinite(lse[lens > 0]).all()


def test_paged_attention_large_scores():
    """Scores of hundreds that rise and fall along the sequence: the running
    maximum moves, and what came before it all but vanishes."""
    for dtype in (F32, BF):
        g = gen(1)
        kc, vc, table, ln = make_cache(g, dtype, [700, 90], 2, 64, 16)
        ramp = torch.linspace(-30, 30, 700, device="cuda")
        for j in range(700):
            kc[table[0, j // 16], :, j % 16] *= ramp[j].to(dtype)
        q = rand(g, 2, 8, 64, dtype=dtype, scale=4.0)
        o, lse = ops.paged_attention(q, kc, vc, table, ln)
        check_attention(q, kc, vc, table, ln, 0, o, lse)
        # a NaN key shows in its own sequence and heads, and in no other
        kc[table[0, 3], 1, 2, 0] = math.nan
        o2, _ = ops.paged_attention(q, kc, vc, table, ln)
        assert torch.isnan(o2[0, 4 * 64:]).all() and torch.equal(o2[0, :4 * 64], o[0, :4 * 64]) and torch.equal(o2[1], o[1])


def test_paged_attention_infinite_scores():
    """Keys whose score is -inf take no weight; a sequence of nothing else gets
    zeros and -inf, as one of length zero does."""
    for dtype in (F32, BF):
        g = gen(2)
        kc, vc, table, ln = make_cache(g, dtype, [100, 40], 1, 64, 16)
        q = rand(g, 2, 2, 64, dtype=dtype).abs() + 0.5
        clean = ops.paged_attention(q, kc, vc, table, ln)
        for j in range(40):
            kc[table[1, j // 16], :, j % 16] = -math.inf
        kc[table[0, 0], :, 3] = -math.inf
        o, lse = ops.paged_attention(q, kc, vc, table, ln)
        assert not o[1].any() and bool((lse[1] == -math.inf).all())
        keep = [j for j in range(100) if j != 3]
        k = torch.stack([kc[table[0, j // 16], 0, j % 16] for j in keep]).double()
        v = torch.stack([vc[table[0, j // 16], 0, j % 16] for j in keep]).double()
        p = torch.softmax(q[0].double() @ k.T / 8, -1)
        bound = (p @ v).abs() * U + (2 * U if dtype == BF else 4000 * u) * (p @ v.abs())
        within(o[0].view(2, 64), p @ v, bound, "o without the -inf key")
        assert not torch.equal(o[0], clean[0][0])


def test_paged_attention_pages_that_are_not_there():
    for dtype in (F32, BF):
        g = gen(3)
        kc, vc, table, ln = make_cache(g, dtype, [64, 48], 2, 64, 16)
        q = rand(g, 2, 4, 64, dtype=dtype)
        good = ops.paged_attention(q, kc, vc, table, ln)
        bad = table.clone()
        bad[0, 3] = 10 ** 6  # its last page
        o, _ = ops.paged_attention(q, kc, vc, bad, ln)
        short = ln.clone()
        short[0] = 48
        check_attention(q, kc, vc, table, short, 0, o, ops.paged_attention(q, kc, vc, table, short)[1])
        assert torch.equal(o[1], good[0][1])
        with pytest.raises(ShapeMismatch, match="no page"):
            ops.paged_attention(q, kc, vc, bad, ln, check=True)
        long = ln.clone()
        long[1] = 2 ** 31 - 1  # beyond the table: its 64 positions of which the last page is not there
        with pytest.raises(ShapeMismatch, match="no page"):
            ops.paged_attention(q, kc, vc, table, long, check=True)
        ops.paged_attention(q, kc, vc, table, ln, check=True)
        # a pool without pages, a table without columns
        none = torch.empty(0, 2, 16, 64, device="cuda", dtype=dtype)
        for t, c in ((table, none), (table[:, :0].contiguous(), kc)):
            o, lse = ops.paged_attention(q, c, c, t, ln)
            assert not o.any() and bool((lse == -math.inf).all())
        assert ops.paged_attention(q[:0], kc, vc, table[:0], ln[:0])[0].shape == (0, 256)


def test_paged_attention_offsets_past_32_bits():
    """A pool of more than 2^32 elements; the sequence's pages lie at its end."""
    pages, hkv, page, hd = 2 ** 32 // (8 * 64 * 128) + 40, 8, 64, 128
    if torch.cuda.mem_get_info()[0] < 5 * pages * hkv * page * hd:
        pytest.skip("not enough device memory")
    kc = torch.empty(pages, hkv, page, hd, dtype=BF, device="cuda")
    vc = torch.empty_like(kc)
    g = gen(8)
    kc[-5:], vc[-5:] = rand(g, 5, hkv, page, hd, dtype=BF), rand(g, 5, hkv, page, hd, dtype=BF)
    table = torch.arange(pages - 5, pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    ln = torch.tensor([290], dtype=torch.int32, device="cuda")
    q, k, v = rand(g, 1, 16, hd, dtype=BF), rand(g, 1, hkv, hd, dtype=BF), rand(g, 1, hkv, hd, dtype=BF)
    qr = ops.kv_append(q, k, v, kc, vc, table, ln, 1e6, check=True)
    assert torch.equal(vc[table[0, 4], :, 289 % 64], v[0])
    o, lse = ops.paged_attention(qr, kc, vc, table, ln)
    check_attention(qr, kc, vc, table, ln, 0, o, lse)


def test_paged_attention_refusals():
    g = gen(6)
    kc, vc, table, ln = make_cache(g, F32, [9], 1, 136, 16)
    with pytest.raises(Unsupported):
        ops.paged_attention(rand(g, 1, 2, 136), kc, vc, table, ln)
    kc, vc, table, ln = make_cache(g, F32, [9], 2, 64, 16)
    q = rand(g, 1, 2, 64)
    o, lse = torch.empty(1, 128, device="cuda"), torch.empty(1, 2, device="cuda")
    h = ops.context(q.device).bind()

    def call(**kw):
        a = dict(q=q.data_ptr(), stride=128, k=kc.data_ptr(), v=vc.data_ptr(), table=table.data_ptr(), lens=ln.data_ptr(),
                 o=o.data_ptr(), lse=lse.data_ptr(), seqs=1, h=2, hkv=2, hd=64, pages=kc.shape[0], page=16, most=1, window=0,
                 dtype=0, ws=None, n=0, check=0)
        a.update(kw)
        _lib.call("catnn_paged_attention_fwd", h, *a.values())
    for kw, err in (({"q": None}, InvalidArgument), ({"seqs": -1}, ShapeMismatch), ({"hkv": 0}, ShapeMismatch),
                    ({"h": 3}, ShapeMismatch), ({"page": 0}, ShapeMismatch), ({"page": 2 ** 20, "most": 2 ** 12}, ShapeMismatch),
                    ({"page": 2 ** 31 - 1}, ShapeMismatch),
                    ({"pages": -1}, ShapeMismatch), ({"seqs": 2, "stride": 8}, ShapeMismatch),
                    ({"seqs": 2 ** 31 - 1}, ShapeMismatch)):
        with pytest.raises(err):
            call(**kw)


# ------------------------------------------------------------------ MoE for a few tokens
def moe_inputs(seed, dtype, t, hid, mid, e):
    g = gen(seed)
    return (rand(g, t, hid, dtype=dtype), rand(g, hid, e, dtype=dtype, scale=hid ** -0.5),
            rand(g, e, hid, mid, dtype=dtype, scale=hid ** -0.5), rand(g, e, hid, mid, dtype=dtype, scale=hid ** -0.5),
            rand(g, e, mid, hid, dtype=dtype, scale=mid ** -0.5))


def moe_ref(x, gate, w1, w3, w2, k):
    """-> y, and the magnitudes of its terms: those that a rounding of the
    pre-activations reaches, and those that a rounding of h reaches."""
    x, logits = x.double(), (x.double() @ gate.double())
    sel, idx = torch.sort(logits, dim=-1, descending=True, stable=True)
    if logits.shape[1] > k and len(x):  # no choice may hang on the last bits of fp32 sums, but for ties that are exact
        gap = sel[:, k - 1] - sel[:, k]
        assert not ((gap > 0) & (gap < 1e-5)).any(), "the test's inputs: choose another seed"
    sel, idx = sel[:, :k], idx[:, :k]
    w = torch.softmax(sel, -1)
    y, pre, hh, act = (torch.zeros_like(x) for _ in range(4))
    for t in range(len(x)):
        for j in range(k):
            i = int(idx[t, j])
            a, c = x[t] @ w1[i].double(), x[t] @ w3[i].double()
            aa, cc = x[t].abs() @ w1[i].double().abs(), x[t].abs() @ w3[i].double().abs()
            s = a * torch.sigmoid(a)
            w2i = w2[i].double()
            y[t] += w[t, j] * ((s * c) @ w2i)
            pre[t] += w[t, j] * ((1.1 * aa * c.abs() + s.abs() * cc) @ w2i.abs())  # |silu'| <= 1.1
            hh[t] += w[t, j] * ((s * c).abs() @ w2i.abs())
    return y, pre, hh


def check_moe(args, k, y):
    x, gate, w1, w3, w2 = args
    ref, pre, hh = moe_ref(*args, k)
    hid, mid = w1.shape[1:]
    dtype = x.dtype
    # a and c: hid products added in fp32, y: mid of them; the router's weights: hid products in the logit, whose error
    # (hid·u·|x||gate|, up to about 2·hid·u here) moves a weight by as much; exponentials and the join: 32.
    # bf16 holds h in bf16 for the second product: U on each of its terms.
    bound = own_rounding(ref, dtype) * (1 + 1e-3) + (hid + 32) * u * pre + (mid + 4 * hid + 64) * u * hh
    if dtype == BF:
        bound = bound + U * hh
    within(y, ref, bound, "y")
    if ref.numel():
        # the roundings of h and of y are independent: rms U/sqrt(3) of their own terms, here allowed twice that
        rel = float((y.double() - ref).norm() / ref.norm())
        assert rel <= (2 * U if dtype == BF else 2e-6), rel


MOE = [  # t, hidden, mid, e, k
    (1, 64, 128, 8, 2), (1, 1024, 512, 8, 2), (2, 256, 512, 8, 2), (3, 8, 8, 2, 1), (7, 256, 512, 8, 2), (8, 72, 200, 4, 4),
    (9, 264, 136, 16, 2), (16, 512, 1000, 32, 4), (17, 128, 128, 1, 1), (33, 256, 384, 8, 3), (64, 512, 256, 8, 2),
    (64, 64, 64, 4, 1), (5, 33, 47, 3, 2), (2, 1, 1, 2, 2), (40, 136, 72, 32, 8), (64, 24, 1032, 2, 2), (6, 2056, 520, 4, 2),
    (33, 1024, 72, 32, 2), (12, 1280, 136, 20, 3), (8, 1024, 264, 32, 2), (5, 2048, 64, 6, 1), (1, 72, 3000, 30, 1)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("t,hid,mid,e,k", MOE)
def test_moe_few(t, hid, mid, e, k, dtype):
    args = moe_inputs(t * 100 + hid, dtype, t, hid, mid, e)
    y = ops.moe_few(*args, k)
    assert y.shape == args[0].shape and y.dtype == dtype
    check_moe(args, k, y)
    assert torch.equal(y, ops.moe_few(*args, k)), "the same bits on every call"


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("t", [4, 9, 13, 16, 17, 29, 33, 37, 52, 64])
@pytest.mark.parametrize("hid,mid", [(136, 72), (264, 128), (320, 3200), (2056, 72)])
def test_moe_few_every_token_on_every_expert(t, hid, mid, dtype):
    """The tokens of an expert at every way to split them, in few tiles and in many."""
    args = moe_inputs(t * 10 + hid, dtype, t, hid, mid, 3)
    check_moe(args, 3, ops.moe_few(*args, 3))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_moe_few_ties_and_crowds(dtype):
    """Equal logits go to the lower experts; all tokens on one pair of experts."""
    x, gate, w1, w3, w2 = moe_inputs(11, dtype, 64, 128, 128, 8)
    check_moe((x, torch.zeros_like(gate), w1, w3, w2), 2, ops.moe_few(x, torch.zeros_like(gate), w1, w3, w2, 2))
    steep = torch.zeros_like(gate)
    steep[0] = torch.arange(8, device="cuda").to(dtype)
    x[:, 0] = 1.0
    check_moe((x, steep, w1, w3, w2), 2, ops.moe_few(x, steep, w1, w3, w2, 2))
    same = gate.clone()
    same[:, 5] = same[:, 2]  # exact ties between 2 and 5
    check_moe((x, same, w1, w3, w2), 3, ops.moe_few(x, same, w1, w3, w2, 3))
    z = torch.zeros_like(x)
    assert not ops.moe_few(z, gate, w1, w3, w2, 2).any()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_moe_few_keeps_tokens_apart(dtype):
    """A token's NaN, or an expert's that no other token takes, stays there;
    a token's result does not hang on the company it comes in."""
    x, gate, w1, w3, w2 = moe_inputs(12, dtype, 12, 128, 264, 8)
    y = ops.moe_few(x, gate, w1, w3, w2, 2)
    bad = x.clone()
    bad[4] = math.nan
    y2 = ops.moe_few(bad, gate, w1, w3, w2, 2)
    others = [i for i in range(12) if i != 4]
    assert torch.equal(y2[others], y[others]) and torch.isnan(y2[4]).all()
    idx = torch.sort(x.double() @ gate.double(), dim=-1, descending=True, stable=True)[1][:, :2]
    for e in range(8):
        uses = (idx == e).any(1)
        if uses.any() and not uses.all():
            wb = w1.clone()
            wb[e] = math.inf
            y3 = ops.moe_few(x, gate, wb, w3, w2, 2)
            assert torch.equal(y3[~uses], y[~uses]) and not torch.isfinite(y3[uses]).any()


def test_moe_few_beside_moe_and_refusals():
    """The block for many tokens gives the same layer."""
    for dtype in (F32, BF):
        args = moe_inputs(13, dtype, 48, 256, 512, 8)
        y, big = ops.moe_few(*args, 2), ops.moe(*args, 2)
        assert float((y.float() - big.float()).norm() / big.float().norm()) <= (2 * U if dtype == BF else 4e-6)
    assert ops.moe_few(args[0][:0], *args[1:], 2).shape == (0, 256)
    assert ops.moe_few(args[0].view(4, 12, 256), *args[1:], 2).shape == (4, 12, 256)
    x, gate, w1, w3, w2 = args
    h = ops.context(x.device).bind()
    y = torch.empty_like(x)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")

    def call(T=48, hid=256, mid=512, e=8, k=2, dt=1, p=ws.data_ptr(), n=ws.numel(), x=x.data_ptr()):
        _lib.call("catnn_moe_few_fwd", h, x, gate.data_ptr(), w1.data_ptr(), w3.data_ptr(), w2.data_ptr(), y.data_ptr(), T, hid,
                  mid, e, k, dt, p, n)
    call()
    for kw, err in (({"T": 65}, ShapeMismatch), ({"T": -1}, ShapeMismatch), ({"k": 9}, ShapeMismatch), ({"e": 33}, ShapeMismatch),
                    ({"n": 16}, InvalidArgument), ({"p": ws.data_ptr() + 64}, InvalidArgument), ({"p": None}, InvalidArgument),
                    ({"x": None}, InvalidArgument), ({"hid": 0}, ShapeMismatch), ({"x": y.data_ptr()}, InvalidArgument)):
        with pytest.raises(err):
            call(**kw)


# ------------------------------------------------------------------ together, as a decoder uses them
class Layer:
    """A layer of the decoder that the trainer trains: RMSNorm, GQA + RoPE,
    residual, RMSNorm, MoE, residual."""

    def __init__(self, dtype, hid=256, h=4, hkv=2, hd=64, mid=512, e=8, seed=21):
        g = gen(seed)
        self.h, self.hkv, self.hd, self.theta = h, hkv, hd, 1e4
        self.n1, self.n2 = 1 + rand(g, hid, scale=0.1), 1 + rand(g, hid, scale=0.1)
        self.wq, self.wk, self.wv = (rand(g, hid, n * hd, dtype=dtype, scale=hid ** -0.5) for n in (h, hkv, hkv))
        self.wqkv = torch.cat((self.wq, self.wk, self.wv), 1).contiguous()
        self.wo = rand(g, h * hd, hid, dtype=dtype, scale=(h * hd) ** -0.5)
        self.experts = moe_inputs(seed, dtype, 1, hid, mid, e)[1:]

    def whole(self, x):
        """All positions at once, with the operators for whole sequences."""
        y = ops.add(x, ops.gqa(ops.rmsnorm(x, self.n1), self.wq, self.wk, self.wv, self.wo, self.h, self.hkv, self.theta))
        return ops.add(y, ops.moe(ops.rmsnorm(y, self.n2), *self.experts, 2))

    def step(self, x, kc, vc, table, lens, cu=None, few=True):
        """x [T, hid]: new tokens of several sequences; one each without cu."""
        q, k, v = (t.unflatten(-1, (-1, self.hd)) for t in ops.gemm(ops.rmsnorm(x, self.n1), self.wqkv).split(
            [self.h * self.hd, self.hkv * self.hd, self.hkv * self.hd], -1))
        q = ops.kv_append(q, k, v, kc, vc, table, lens, self.theta, cu_tokens=cu)
        if cu is not None:
            return q
        o, _ = ops.paged_attention(q, kc, vc, table, lens)
        y = ops.add(x, ops.gemm(o, self.wo))
        return ops.add(y, ops.moe_few(ops.rmsnorm(y, self.n2), *self.experts, 2))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_decoding_a_layer_matches_whole_sequences(dtype):
    layer = Layer(dtype)
    g = gen(22)
    b, s, prompt, page = 3, 40, 21, 16
    x = rand(g, b, s, 256, dtype=dtype)
    want = layer.whole(x)
    pool = b * 3 + 1
    kc = torch.full((pool, 2, page, 64), math.nan, device="cuda", dtype=dtype)
    vc = kc.clone()
    table = torch.randperm(pool, generator=g, device="cuda")[:b * 3].int().view(b, 3).contiguous()
    lens = torch.full((b,), prompt, dtype=torch.int32, device="cuda")
    cu = torch.arange(b + 1, device="cuda", dtype=torch.int32) * prompt
    layer.step(x[:, :prompt].reshape(-1, 256).contiguous(), kc, vc, table, lens, cu=cu)
    for t in range(prompt, s):
        lens += 1
        y = layer.step(x[:, t].contiguous(), kc, vc, table, lens)
        ref = want[:, t].double()
        rel = float((y.double() - ref).norm() / ref.norm())
        # fp32: sums of up to 512 terms in other orders, through four products; bf16: nine bf16 roundings on each side
        # (norms, QKV, rotation, P, o, sums, h, y), of which a routing weight moves with the residual's
        assert rel <= (2e-5 if dtype == F32 else 6 * U), (t, rel)


def test_decoding_captured_and_replayed():
    """One decoding step as a CUDA graph whose tokens and lengths change
    between replays, beside a second graph of the same operators on other
    buffers and eager calls in between: nothing that they use is shared."""
    layer = Layer(BF)
    g = gen(23)

    def setup(b):
        kc, vc, table, lens = make_cache(g, BF, [60] * b, 2, 64, 16)
        lens[:] = torch.arange(b, device="cuda") * 7 + 3
        return [rand(g, b, 256, dtype=BF), kc, vc, table, lens]
    runs = []
    for b in (5, 2):
        st = setup(b)
        layer.step(*st)  # sizes what the framework's own operators keep
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                q = ops.kv_append(*(st[0].view(b, 4, 64), st[0][:, :128].view(b, 2, 64), st[0][:, 128:].view(b, 2, 64)), st[1],
                                  st[2], st[3], st[4], 1e4)
                o, lse = ops.paged_attention(q, *st[1:])
                y = ops.moe_few(o, *layer.experts, 2)
        torch.cuda.current_stream().wait_stream(side)
        runs.append((st, graph, (q, o, lse, y)))
    for r in range(4):
        for st, graph, out in runs:
            st[0].copy_(rand(g, *st[0].shape, dtype=BF))
            st[4] += 1
        for st, graph, out in runs:
            graph.replay()
        got = [[t.clone() for t in out] + [st[1].clone(), st[2].clone()] for st, graph, out in runs]
        for (st, graph, out), have in zip(runs, got):
            b = len(st[0])
            q = ops.kv_append(st[0].view(b, 4, 64), st[0][:, :128].view(b, 2, 64), st[0][:, 128:].view(b, 2, 64), *st[1:], 1e4)
            o, lse = ops.paged_attention(q, *st[1:])
            want = [q, o, lse, ops.moe_few(o, *layer.experts, 2), st[1], st[2]]
            assert all(torch.equal(x, y) for x, y in zip(have, want)), r


def test_two_streams_at_once():
    """The same operators on two streams, whose kernels may overlap."""
    layer = Layer(BF)
    g = gen(24)
    sets = []
    for i in range(2):
        kc, vc, table, lens = make_cache(g, BF, [900 + i, 30, 411], 2, 64, 16)
        sets.append((rand(g, 3, 4, 64, dtype=BF), kc, vc, table, lens))
    x, w = rand(g, 4, 300, 4, 64, dtype=BF), torch.ones(64, device="cuda")
    want = []
    for q, *cache in sets:
        o, lse = ops.paged_attention(q, *cache)
        want.append((o, lse, ops.moe_few(o, *layer.experts, 2), *ops.qk_norm_rope_backward(x, x, w, w, x, x, 1e4)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for r in range(10):
        for i, (q, *cache) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                o, lse = ops.paged_attention(q, *cache)
                outs[i].append((o, lse, ops.moe_few(o, *layer.experts, 2), *ops.qk_norm_rope_backward(x, x, w, w, x, x, 1e4)))
    torch.cuda.synchronize()
    for i in range(2):
        for got in outs[i]:
            assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


def test_training_with_the_norm_inside_a_graph():
    """Forward and adjoint captured while an eager result of the same inputs lives."""
    _, q, k, wq, wk = qk_inputs(31, BF, 2, 60, 4, 2, 64, True)
    _, gq, gk, _, _ = qk_inputs(32, BF, 2, 60, 4, 2, 64, False)
    eager = (*ops.qk_norm_rope(q, k, wq, wk, 1e4), *ops.qk_norm_rope_backward(q, k, wq, wk, gq, gk, 1e4))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (*ops.qk_norm_rope(q, k, wq, wk, 1e4), *ops.qk_norm_rope_backward(q, k, wq, wk, gq, gk, 1e4))
    ops.qk_norm_rope(q, k, wq, wk, 1e6)  # another base in between
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, eager))
