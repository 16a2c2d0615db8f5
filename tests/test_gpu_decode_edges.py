"""The decoding operators where their first tests did not look: sizes at which
a grid or a workspace reaches its limit, infinities and NaN on every path,
lengths beyond a table, waits that run out, captured layers. Tolerances are
counted in roundings as in test_gpu_decode.py."""
import ctypes as C
import math

import pytest
import torch

from test_gpu_decode import (BF, EPS, F32, Layer, U, check_attention, check_moe, gather, gen, inv_rms, make_cache, moe_inputs,
                             own_rounding, pair_size, qk_inputs, rand, turn, u, within)

pytestmark = pytest.mark.gpu

from catnn_b200 import _lib, ops  # noqa: E402
from catnn_b200.train import MoeConfig, MoeTrainer, init_params, packed_layout  # noqa: E402
from catnn_b200.errors import DeviceTimeout, InvalidArgument, ShapeMismatch  # noqa: E402


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


# ------------------------------------------------------------------ infinities and NaN, on every path
#: dtype, head size, whether the caches start off a 16-byte boundary: tensor cores, FMA, and any size and alignment
PATHS = [(BF, 64, False), (F32, 64, False), (BF, 7, False), (F32, 7, False), (BF, 64, True), (F32, 64, True)]


def off_boundary(t):
    """t's values in memory that starts one element off a 16-byte boundary."""
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = room[1:].view(t.shape)
    out.copy_(t)
    return out


def plain_attention(q, kc, vc, table, n):
    """softmax(q·Kᵀ/√hd)·V of sequence 0 in 64 bits, with what infinities and NaN make of it."""
    h, hd, hkv = q.shape[1], q.shape[2], kc.shape[1]
    k, v = gather(kc, table, 0, 0, n).double(), gather(vc, table, 0, 0, n).double()
    s = torch.einsum("ngd,jnd->ngj", q[0].double().view(hkv, h // hkv, hd), k) / math.sqrt(hd)
    return torch.einsum("ngj,jnd->ngd", torch.softmax(s, -1), v).reshape(-1), torch.logsumexp(s, -1).reshape(-1)


@pytest.mark.parametrize("dtype,hd,off", PATHS)
@pytest.mark.parametrize("what", ["query", "first key", "early key", "late key", "every key", "value", "value of no weight",
                                  "infinite score"])
def test_paged_attention_shows_nan_on_every_path(what, dtype, hd, off):
    """A NaN shows in the heads that meet it, in every kernel, wherever it stands, and in no others."""
    g = gen(71)
    kc, vc, table, ln = make_cache(g, dtype, [300, 40], 2, hd, 16)
    q = rand(g, 2, 4, hd, dtype=dtype).abs() + 0.25

    def put(cache, j, value):  # into kv head 0 of sequence 0
        cache[table[0, j // 16], 0, j % 16] = value
    if what == "query":
        q[0, 0, hd - 1] = math.nan
    elif what == "every key":
        for j in range(300):
            put(kc, j, math.nan)
    elif what == "value":
        put(vc, 123, math.nan)
    elif what == "value of no weight":
        put(kc, 123, -math.inf)
        put(vc, 123, math.inf)
    elif what == "infinite score":
        put(kc, 5, math.inf)
    else:
        put(kc, {"first key": 0, "early key": 9, "late key": 299}[what], math.nan)
    if off:
        kc, vc = off_boundary(kc), off_boundary(vc)
    o, lse = ops.paged_attention(q, kc, vc, table, ln)
    ref, rl = plain_attention(q, kc, vc, table, 300)
    assert torch.equal(torch.isnan(o[0]), torch.isnan(ref)) and torch.isnan(ref).any() and not torch.isnan(ref).all()
    if what != "infinite score":  # there the largest score alone is known to be infinite
        assert torch.equal(torch.isnan(lse[0]), torch.isnan(rl))
    assert torch.isfinite(o[1]).all() and torch.isfinite(lse[1]).all()


@pytest.mark.parametrize("dtype,hd,off", PATHS)
def test_paged_attention_infinite_scores_on_every_path(dtype, hd, off):
    """Scores of -inf take no weight, wherever they stand; a sequence of nothing else gets zeros and -inf."""
    g = gen(72)
    kc, vc, table, ln = make_cache(g, dtype, [100, 40], 1, hd, 16)
    q = rand(g, 2, 2, hd, dtype=dtype).abs() + 0.5
    gone = [0, 1, 8, 40, 99]
    for b, js in ((0, gone), (1, range(40))):
        for j in js:
            kc[table[b, j // 16], :, j % 16] = -math.inf
    if off:
        kc, vc = off_boundary(kc), off_boundary(vc)
    o, lse = ops.paged_attention(q, kc, vc, table, ln)
    assert not o[1].any() and bool((lse[1] == -math.inf).all())
    keep = torch.tensor([j for j in range(100) if j not in gone], device="cuda")
    k, v = gather(kc, table, 0, 0, 100)[keep, 0].double(), gather(vc, table, 0, 0, 100)[keep, 0].double()
    s = q[0].double() @ k.T / math.sqrt(hd)
    p = torch.softmax(s, -1)
    # the counts of check_attention: a score's roundings twice, 66 of the sums, P in bf16
    spread = float((q[0].double().abs() @ k.abs().T).amax()) / math.sqrt(hd)
    mean = p @ v.abs()
    within(o[0].view(2, hd), p @ v, own_rounding(p @ v, dtype) * (1 + 1e-3)
           + (2 * (hd + 8) * u * spread + 66 * u + (U if dtype == BF else 0)) * mean, "o")


@pytest.mark.parametrize("dtype,hd,off", PATHS)
def test_paged_attention_windows_beyond_the_table(dtype, hd, off):
    """A sequence longer than its table: the positions of its window that the
    table does not hold are left out, and none before the window comes in for them."""
    g = gen(73)
    kc, vc, table, _ = make_cache(g, dtype, [64, 64, 64, 64], 2, hd, 16)
    q = rand(g, 4, 4, hd, dtype=dtype)
    if off:
        kc, vc = off_boundary(kc), off_boundary(vc)
    ln = torch.tensor([1000, 70, 64, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    o, lse = ops.paged_attention(q, kc, vc, table, ln, window=16)
    assert not o[0].any() and not o[3].any() and bool((lse[[0, 3]] == -math.inf).all())
    # positions 54 to 63 of sequence 1: what a length of 64 attends to with a window of 10
    held = torch.full_like(ln, 64)
    short, sl = ops.paged_attention(q, kc, vc, table, held, window=10)
    check_attention(q[1:2], kc, vc, table[1:2], held[1:2], 10, o[1:2], lse[1:2])
    check_attention(q[1:2], kc, vc, table[1:2], held[1:2], 10, short[1:2], sl[1:2])
    check_attention(q[2:3], kc, vc, table[2:3], held[2:3], 16, o[2:3], lse[2:3])
    with pytest.raises(ShapeMismatch, match="no page"):
        ops.paged_attention(q, kc, vc, table, ln, window=16, check=True)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("t,hid,mid,e", [(1, 128, 128, 8), (7, 128, 136, 8), (12, 136, 128, 6), (40, 256, 128, 32), (5, 24, 40, 8),
                                         (3, 130, 66, 5)])
def test_moe_few_experts_shut_off(t, hid, mid, e, dtype):
    """Experts whose logit is -inf, or the type's lowest value, are taken by
    nobody; an infinite row of x leaves the other rows as they are."""
    x, gate, w1, w3, w2 = moe_inputs(74 + hid, dtype, t, hid, mid, e)
    x[:, 0] = 1.0
    for low in (-math.inf, torch.finfo(dtype).min):
        for shut in ([0], [e - 1], [0, 2, 3]):
            off = gate.clone()
            off[0, shut] = low
            y = ops.moe_few(x, off, w1, w3, w2, 2)
            clean = gate.clone()
            clean[0, shut] = -1e4  # far below every other logit
            check_moe((x, clean, w1, w3, w2), 2, y)
    if t > 1:
        y = ops.moe_few(x, gate, w1, w3, w2, 2)
        bad = x.clone()
        bad[1, 5] = math.inf
        y2 = ops.moe_few(bad, gate, w1, w3, w2, 2)
        others = [i for i in range(t) if i != 1]
        assert torch.equal(y2[others], y[others]) and not torch.isfinite(y2[1]).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("t,hid,mid,e,k", [(3, 128, 128, 8, 1), (5, 128, 136, 8, 2), (20, 136, 128, 32, 3), (4, 24, 40, 8, 2)])
def test_moe_few_infinite_rows(t, hid, mid, e, k, dtype):
    """A row with an infinity has infinite logits, whose softmax is NaN; so is
    a row of NaN. Neither reaches another row."""
    x, gate, w1, w3, w2 = moe_inputs(78 + hid, dtype, t, hid, mid, e)
    y = ops.moe_few(x, gate, w1, w3, w2, k)
    x[1, 7], x[2, 9], x[2, 11] = math.inf, -math.inf, math.nan
    y2 = ops.moe_few(x, gate, w1, w3, w2, k)
    others = [i for i in range(t) if i not in (1, 2)]
    assert torch.isnan(y2[1:3]).all() and torch.equal(y2[others], y[others])


# ------------------------------------------------------------------ waits that run out
@pytest.mark.parametrize("dtype,t,hid,mid,e", [(BF, 1, 1024, 1024, 8), (BF, 8, 512, 1024, 32), (BF, 64, 1024, 3584, 8),
                                               (F32, 3, 256, 512, 8), (F32, 12, 1024, 1024, 8), (F32, 50, 1024, 3584, 4)])
def test_moe_few_reports_a_wait_that_runs_out(dtype, t, hid, mid, e):
    """With no patience at all the kernels give up before their tiles are there:
    their rows are NaN, the check says so once, and neither another operator nor
    the next call is the worse for it."""
    args = moe_inputs(75, dtype, t, hid, mid, e)
    good = ops.moe_few(*args, 2, check=True)
    a, b = rand(gen(76), 300, 256, dtype=BF), rand(gen(77), 256, 300, dtype=BF)
    product = ops.gemm(a, b)
    h = ops.context(args[0].device).bind()
    _lib.call("catnn_moe_few_set_timeout_ms", h, 0)
    try:
        y = ops.moe_few(*args, 2)
        assert torch.equal(ops.gemm(a, b), product)
        assert torch.isnan(y).any() and bool((torch.isnan(y) | (y == good)).all())
        with pytest.raises(DeviceTimeout):
            _lib.call("catnn_moe_few_check", h)
        _lib.call("catnn_moe_few_check", h)
        with pytest.raises(DeviceTimeout):
            ops.moe_few(*args, 2, check=True)
    finally:
        _lib.call("catnn_moe_few_set_timeout_ms", h, 2000)
    assert torch.equal(ops.moe_few(*args, 2, check=True), good)
    for ms in (-1, 2 ** 40):
        with pytest.raises(InvalidArgument):
            _lib.call("catnn_moe_few_set_timeout_ms", h, ms)


# ------------------------------------------------------------------ captured calls and what the context keeps
def outgrow(dtype):
    """Calls whose split sums and temporaries are larger than all before them."""
    for k in (2 ** 14, 2 ** 16):
        a = torch.ones(1024, k, dtype=BF, device="cuda")
        assert float(ops.gemm(a, a, trans_b=True)[0, 0]) == k
    big = moe_inputs(81, dtype, 3000, 256, 512, 8)
    return ops.moe(*big, 2)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_captured_layer_outlives_larger_calls(dtype):
    """A whole layer of a decoding step as a graph, products with split sums
    among it, replayed after eager calls that outgrow the context's memory."""
    layer = Layer(dtype, hid=1024, h=16, hkv=4, mid=1024, seed=82)
    g = gen(83)
    kc, vc, table, lens = make_cache(g, dtype, [60] * 5, 4, 64, 16)
    lens[:] = torch.arange(5, device="cuda") * 7 + 3
    x = rand(g, 5, 1024, dtype=dtype)
    layer.step(x, kc, vc, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer.step(x, kc, vc, table, lens)
        with torch.cuda.graph(graph, stream=side):
            y = layer.step(x, kc, vc, table, lens)
    torch.cuda.current_stream().wait_stream(side)
    for r in range(4):
        if r:
            assert torch.isfinite(outgrow(dtype).float()).all()
            torch.cuda.synchronize()
        x.copy_(rand(g, 5, 1024, dtype=dtype))
        lens += 1
        graph.replay()
        got = (y.clone(), kc.clone(), vc.clone())
        want = (layer.step(x, kc, vc, table, lens), kc, vc)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), r


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_captured_rotation_keeps_its_angles(dtype):
    """A captured rope after eager calls of other lengths and bases."""
    g = gen(84)
    x = rand(g, 2, 100, 4, 64, dtype=dtype)
    y = torch.empty_like(x)
    want = ops.rope(x.clone(), 1e4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y.copy_(x)
        ops.rope(y, 1e4)
    for s, theta in ((100, 1e6), (3000, 1e4), (7, 1e4), (100, 1e5)):
        ops.rope(rand(g, 1, s, 4, 64, dtype=dtype), theta)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    long = rand(g, 1, 4096, 4, 64, dtype=dtype)
    free = torch.cuda.mem_get_info()[0]
    for _ in range(40):  # tables that no capture holds are not kept
        ops.rope(x, 1e5)
        ops.rope(long, 1e4)
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] < 32 * 2 ** 20


def test_a_captured_training_step_outlives_larger_calls():
    """The trainer's graph, replayed after eager calls that outgrow the memory
    and change the table that its capture was given."""
    cfg = MoeConfig.make(1024, 256, 512, 2, 4, 4, 8, 2, batch=2, seq=128, rope_theta=1e6, dtype=BF, optimizer="adam", lr=1e-3)
    params = init_params(cfg, 85)
    tok = torch.randint(0, 1024, (256,), generator=gen(85), device="cuda", dtype=torch.int32)
    a, b = MoeTrainer(cfg), MoeTrainer(cfg)
    a.set_params(params)
    b.set_params(params)
    b.set_graphs(True)
    la, lb = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
    for i in range(6):
        a.step(tok, update=True, loss_out=la)
        b.step(tok, update=True, loss_out=lb)
        torch.cuda.synchronize()
        assert torch.equal(la, lb), i
        if i > 2:  # captured by now
            outgrow(BF)
            ops.rope(rand(gen(i), 1, 50 + i, 4, 64, dtype=BF), 1e4)
    assert torch.equal(a.params(), b.params())
    a.close()
    b.close()


# ------------------------------------------------------------------ a trained decoder
def decoder_weights(trainer):
    """The weights of a trainer's packed vector, as the operators take them."""
    cfg, at, p = trainer.cfg, packed_layout(trainer.cfg), trainer.params()
    h, f, e, hd = cfg.hidden, cfg.mid, cfg.experts, cfg.hidden // cfg.heads

    def take(start, *shape):
        return p[start:start + math.prod(shape)].view(*shape)
    layers = []
    for i in range(cfg.layers):
        base = at["layer0"] + i * at["layer_stride"]
        w = {n: take(base + at[n], *s) for n, s in (
            ("rms_attn", (h,)), ("wq", (h, h)), ("wk", (h, cfg.kv_heads * hd)), ("wv", (h, cfg.kv_heads * hd)), ("wo", (h, h)),
            ("rms_moe", (h,)), ("gate", (h, e)), ("w1", (e, h, f)), ("w3", (e, h, f)), ("w2", (e, f, h)))}
        w = {n: t if n.startswith("rms") or cfg.dtype == 0 else t.to(BF) for n, t in w.items()}
        w["wqkv"] = torch.cat((w["wq"], w["wk"], w["wv"]), 1).contiguous()
        layers.append({n: t.contiguous() for n, t in w.items()})
    return take(0, cfg.vocab, h), layers, take(at["final_norm"], h), take(at["lm_head"], cfg.vocab, h)


def test_decoding_with_a_trainers_weights():
    """Prompts in one go, then token by token, against the activations of the
    trainer's own pass over the whole sequences."""
    b, s, prompt, page = 3, 40, 23, 16
    cfg = MoeConfig.make(512, 256, 512, 2, 4, 2, 8, 2, batch=b, seq=s, dtype=F32, optimizer="adam", lr=1e-3)
    tr = MoeTrainer(cfg)
    tr.set_params(init_params(cfg, 86, std=0.05))
    tok = torch.randint(0, 512, (b, s), generator=gen(86), device="cuda", dtype=torch.int32)
    for _ in range(3):
        tr.step(tok.view(-1), update=True)
    tr.step(tok.view(-1), update=False)
    want = tr.activation("xf").view(b, s, 256).double()
    for i in range(2):  # no choice of experts may hang on the last bits
        sel = tr.activation("router_logits", i).sort(-1, descending=True)[0]
        assert float((sel[:, 1] - sel[:, 2]).min()) > 1e-5, "the test's inputs: choose another seed"
    embed, layers, norm, _ = decoder_weights(tr)
    h, hkv, hd, eps, theta = 4, 2, 64, cfg.rms_eps, cfg.rope_theta
    pools = [(torch.empty(9, hkv, page, hd, device="cuda"), torch.empty(9, hkv, page, hd, device="cuda")) for _ in layers]
    table = torch.randperm(9, generator=gen(87), device="cuda").int().view(b, 3).contiguous()
    lens = torch.full((b,), prompt, dtype=torch.int32, device="cuda")
    cu = torch.arange(b + 1, device="cuda", dtype=torch.int32) * prompt

    def forward(x, cu=None):
        for w, (kc, vc) in zip(layers, pools):
            q, k, v = (t.unflatten(-1, (-1, hd)) for t in ops.gemm(ops.rmsnorm(x, w["rms_attn"], eps), w["wqkv"]).split(
                [h * hd, hkv * hd, hkv * hd], -1))
            q = ops.kv_append(q, k, v, kc, vc, table, lens, theta, cu_tokens=cu, check=True)
            if cu is None:
                o, _ = ops.paged_attention(q, kc, vc, table, lens, check=True)
            else:  # prompts of one length: their keys rotated once more, for the attention of whole sequences
                k, v = (t.reshape(b, prompt, hkv, hd).contiguous() for t in (k, v))
                o, _ = ops.attention_core(q.view(b, prompt, h, hd), ops.rope(k, theta), v)
                o = o.view(b * prompt, h * hd)
            x = ops.add(x, ops.gemm(o, w["wo"]))
            y = ops.rmsnorm(x, w["rms_moe"], eps)
            moe = ops.moe_few(y, *(w[n] for n in ("gate", "w1", "w3", "w2")), 2) if len(y) <= 64 else \
                ops.moe(y, *(w[n] for n in ("gate", "w1", "w3", "w2")), 2)
            x = ops.add(x, moe)
        return ops.rmsnorm(x, norm, eps)

    def close(got, ref, what):
        # as test_decoding_a_layer_matches_whole_sequences: 2e-5 a layer, once more for the final norm
        rel = float((got.double() - ref).norm() / ref.norm())
        assert rel <= 6e-5, (what, rel)
    close(forward(embed[tok[:, :prompt].reshape(-1).long()], cu).view(b, prompt, 256), want[:, :prompt], "prompts")
    for t in range(prompt, s):
        lens += 1
        close(forward(embed[tok[:, t].long()]), want[:, t], t)
    tr.close()
