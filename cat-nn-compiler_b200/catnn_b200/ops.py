"""Functional operators over device tensors, one per C-ABI entry point.

PyTorch is used only as the device allocator and stream source: every
computation below is a kernel of libcatnn_b200 launched on the current
torch stream of the tensor's device. Inputs must be contiguous CUDA
tensors; float32 selects the fp32 parity path and bfloat16 the
tensor-core path (norm weights, losses, router weights and optimizer state
stay float32).
"""
import ctypes as C

import torch

from . import _lib
from .errors import DTypeMismatch, InvalidArgument, ShapeMismatch

F32, BF16, TF32 = 0, 1, 2
ACT = {"none": 0, None: 0, "relu": 1, "gelu": 2}


def _stream_of(device):
    """The handle of torch's current stream, without the object round it where
    torch offers that (a call's host side 2.0 -> 0.6 us)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw else torch.cuda.current_stream(device).cuda_stream


class Context:
    """One libcatnn_b200 context per device (catnn_ctx_create)."""

    def __init__(self, device):
        self.device = device
        h = C.c_void_p()
        _lib.call("catnn_ctx_create", int(device), C.byref(h))
        self.handle = h
        self._workspace = {}

    def bind(self):
        # set on every call: another thread, or a caller of the C ABI, may have set another one since
        _lib.call("catnn_ctx_set_stream", self.handle, C.c_void_p(_stream_of(self.device)))
        return self.handle

    def workspace(self, name, *sizes):
        """(workspace, bytes) that `name`'s _workspace function asks for, from
        torch's allocator (so it belongs to the current stream, or to the
        graph being captured); (None, 0) where it asks for none. The size is
        kept, not the memory."""
        n = self._workspace.get((name, sizes))
        if n is None:
            v = C.c_size_t()
            _lib.call(name, self.handle, *sizes, C.byref(v))
            n = self._workspace[(name, sizes)] = int(v.value)
        return (torch.empty(n, dtype=torch.uint8, device=self.device), n) if n else (None, 0)

    def launch_count(self):
        v = C.c_uint64()
        _lib.call("catnn_ctx_launch_count", self.handle, C.byref(v))
        return int(v.value)

    def synchronize(self):
        _lib.call("catnn_ctx_synchronize", self.handle)


_CTX = {}


def context(device=None):
    if device is None:
        device = torch.cuda.current_device()
    if isinstance(device, torch.device):
        device = device.index if device.index is not None else torch.cuda.current_device()
    if device not in _CTX:
        _CTX[device] = Context(device)
    return _CTX[device]


def _h(t):
    return context(t.device).bind()


def _p(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise InvalidArgument("catnn_b200 operators take CUDA tensors")
    if not t.is_contiguous():
        raise InvalidArgument("catnn_b200 operators take contiguous tensors")
    return C.c_void_p(t.data_ptr())


def _dt(t):
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise DTypeMismatch(f"unsupported dtype {t.dtype}")


def _same(*ts):
    d = ts[0].dtype
    for t in ts[1:]:
        if t is not None and t.dtype != d:
            raise DTypeMismatch(f"{d} vs {t.dtype}")


def _f32(t, what):
    if t is not None and t.dtype != torch.float32:
        raise DTypeMismatch(f"{what} must be float32")


# ------------------------------------------------------------------ dense
def gemm(a, b, trans_a=False, trans_b=False, out=None, out_dtype=None, bias=None, act="none", accumulate=False,
         tf32=False):
    """C = act(op(a)·op(b) + bias) (+C). tf32=True multiplies fp32 a, b on
    the tensor cores as TF32 (fp32 accumulation) instead of the fp32 path."""
    _same(a, b)
    if tf32 and a.dtype != torch.float32:
        raise DTypeMismatch("tf32 gemm takes fp32 operands")
    M, K = (a.shape[1], a.shape[0]) if trans_a else (a.shape[0], a.shape[1])
    Kb, N = (b.shape[1], b.shape[0]) if trans_b else (b.shape[0], b.shape[1])
    if K != Kb:
        raise ShapeMismatch(f"gemm K {K} vs {Kb}")
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype or a.dtype, device=a.device)
    _f32(bias, "bias")
    _lib.call("catnn_gemm", _h(a), int(trans_a), int(trans_b), M, N, K, _p(a), a.shape[1], _p(b), b.shape[1], _p(out),
              N, TF32 if tf32 else _dt(a), _dt(out), _p(bias), ACT[act], int(accumulate))
    return out


def linear(x, w, b=None, act="none"):
    """cpu::linear (cpu.rs:135): y = act(x @ w + b), w [in, out]."""
    _same(x, w)
    _f32(b, "bias")
    k = x.shape[-1]
    if w.dim() != 2 or w.shape[0] != k:
        raise ShapeMismatch(f"linear K {k} vs {tuple(w.shape)}")
    n = w.shape[1]
    m = x.numel() // max(k, 1)
    y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    _lib.call("catnn_linear_fwd", _h(x), _p(x), _p(w), _p(b), _p(y), m, k, n, ACT[act], _dt(x))
    return y


def linear_backward(x, w, dy, need_dx=True, need_dw=True, need_db=True):
    """adjoint::linear_backward (adjoint.rs:35) -> (dx, dw, db)."""
    _same(x, w, dy)
    k, n = w.shape
    m = x.numel() // k
    dx = torch.empty_like(x) if need_dx else None
    dw = torch.empty_like(w) if need_dw else None
    db = torch.empty(n, dtype=torch.float32, device=x.device) if need_db else None
    _lib.call("catnn_linear_bwd", _h(x), _p(x), _p(w), _p(dy), _p(dx), _p(dw), _p(db), m, k, n, _dt(x))
    return dx, dw, db


def lm_head(x, w):
    """moe::lm_head (moe.rs:325): x @ w.T, w [vocab, hidden]."""
    _same(x, w)
    v, h = w.shape
    rows = x.numel() // h
    y = torch.empty(*x.shape[:-1], v, dtype=x.dtype, device=x.device)
    _lib.call("catnn_lm_head_fwd", _h(x), _p(x), _p(w), _p(y), rows, h, v, _dt(x))
    return y


def lm_head_backward(x, w, dy):
    _same(x, w, dy)
    v, h = w.shape
    rows = x.numel() // h
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    _lib.call("catnn_lm_head_bwd", _h(x), _p(x), _p(w), _p(dy), _p(dx), _p(dw), rows, h, v, _dt(x))
    return dx, dw


# ------------------------------------------------------------------ elementwise
def _unary(name, x):
    y = torch.empty_like(x)
    _lib.call(name, _h(x), _p(x), _p(y), x.numel(), _dt(x))
    return y


def relu(x):
    return _unary("catnn_relu_fwd", x)


def gelu(x):
    return _unary("catnn_gelu_fwd", x)


def relu_backward(x, dy):
    _same(x, dy)
    if x.numel() != dy.numel():
        raise ShapeMismatch("relu grad")
    dx = torch.empty_like(x)
    _lib.call("catnn_relu_bwd", _h(x), _p(x), _p(dy), _p(dx), x.numel(), _dt(x))
    return dx


def gelu_backward(x, dy):
    _same(x, dy)
    dx = torch.empty_like(x)
    _lib.call("catnn_gelu_bwd", _h(x), _p(x), _p(dy), _p(dx), x.numel(), _dt(x))
    return dx


def add(a, b):
    """cpu::add (cpu.rs:80): same length, or b broadcast over the last dim."""
    _same(a, b)
    if b.numel() != a.numel():
        last = a.shape[-1] if a.dim() else a.numel()
        if b.numel() != last:
            raise ShapeMismatch(f"add {tuple(a.shape)} vs {tuple(b.shape)}")
    y = torch.empty_like(a)
    _lib.call("catnn_add", _h(a), _p(a), _p(b), _p(y), a.numel(), b.numel(), _dt(a))
    return y


def mul(a, b):
    _same(a, b)
    if a.numel() != b.numel():
        raise ShapeMismatch("mul length")
    y = torch.empty_like(a)
    _lib.call("catnn_mul", _h(a), _p(a), _p(b), _p(y), a.numel(), _dt(a))
    return y


# ------------------------------------------------------------------ softmax / losses
def softmax_last(x):
    y = torch.empty_like(x)
    last = x.shape[-1] if x.dim() else 1
    _lib.call("catnn_softmax_fwd", _h(x), _p(x), _p(y), x.numel() // max(last, 1), last, _dt(x))
    return y


def softmax_backward(y, dy):
    _same(y, dy)
    dx = torch.empty_like(y)
    last = y.shape[-1]
    _lib.call("catnn_softmax_bwd", _h(y), _p(y), _p(dy), _p(dx), y.numel() // last, last, _dt(y))
    return dx


def cross_entropy(logits, targets, check=True):
    """adjoint::cross_entropy (adjoint.rs:123) -> (loss scalar tensor, dlogits)."""
    if targets.dtype != torch.int32 and targets.dtype != torch.uint32:
        targets = targets.to(torch.int32)
    last = logits.shape[-1]
    rows = logits.numel() // last
    if targets.numel() != rows:
        raise ShapeMismatch("ce targets")
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    d = torch.empty_like(logits)
    _lib.call("catnn_xent_fwdbwd", _h(logits), _p(logits), _p(targets.contiguous()), rows, last, _p(loss), _p(d),
              _dt(logits), int(check))
    return loss, d


def mse_loss(pred, target):
    _f32(pred, "pred")
    _f32(target, "target")
    if pred.numel() != target.numel():
        raise ShapeMismatch("mse")
    loss = torch.empty((), dtype=torch.float32, device=pred.device)
    d = torch.empty_like(pred)
    _lib.call("catnn_mse_fwdbwd", _h(pred), _p(pred), _p(target), pred.numel(), _p(loss), _p(d))
    return loss, d


# ------------------------------------------------------------------ norms
def layer_norm(x, gamma, beta, eps=1e-5):
    last = x.shape[-1]
    if gamma.numel() != last or beta.numel() != last:
        raise ShapeMismatch("ln gamma/beta length")
    _f32(gamma, "gamma")
    _f32(beta, "beta")
    y = torch.empty_like(x)
    _lib.call("catnn_layernorm_fwd", _h(x), _p(x), _p(gamma), _p(beta), _p(y), x.numel() // last, last, eps, _dt(x))
    return y


def layer_norm_backward(x, gamma, dy, eps=1e-5):
    last = x.shape[-1]
    if gamma.numel() != last or dy.numel() != x.numel():
        raise ShapeMismatch("layernorm grad")
    dx = torch.empty_like(x)
    dg = torch.empty(last, dtype=torch.float32, device=x.device)
    db = torch.empty(last, dtype=torch.float32, device=x.device)
    _lib.call("catnn_layernorm_bwd", _h(x), _p(x), _p(gamma), _p(dy), _p(dx), _p(dg), _p(db), x.numel() // last, last,
              eps, _dt(x))
    return dx, dg, db


def rmsnorm(x, w, eps=1e-5):
    last = x.shape[-1]
    if w.numel() != last:
        raise ShapeMismatch("rmsnorm weight")
    _f32(w, "rmsnorm weight")
    y = torch.empty_like(x)
    _lib.call("catnn_rmsnorm_fwd", _h(x), _p(x), _p(w), _p(y), x.numel() // last, last, eps, _dt(x))
    return y


def rmsnorm_backward(x, w, dy, eps=1e-5):
    last = x.shape[-1]
    if w.numel() != last:
        raise ShapeMismatch("rmsnorm w")
    dx = torch.empty_like(x)
    dw = torch.empty(last, dtype=torch.float32, device=x.device)
    _lib.call("catnn_rmsnorm_bwd", _h(x), _p(x), _p(w), _p(dy), _p(dx), _p(dw), x.numel() // last, last, eps, _dt(x))
    return dx, dw


# ------------------------------------------------------------------ embedding
def _ids(ids):
    if ids.dtype not in (torch.int32, torch.uint32):
        ids = ids.to(torch.int32)
    return ids.contiguous()


def embedding(ids, table):
    """moe::embedding (moe.rs:34): raises ShapeMismatch on id >= vocab."""
    ids = _ids(ids)
    v, h = table.shape
    y = torch.empty(*ids.shape, h, dtype=table.dtype, device=table.device)
    _lib.call("catnn_embedding_fwd", _h(table), _p(ids), ids.numel(), _p(table), v, h, _p(y), _dt(table))
    return y


def embedding_backward(ids, dy, vocab):
    """adjoint::embedding_backward (adjoint.rs:195): fp32 [vocab, hidden]."""
    ids = _ids(ids)
    h = dy.shape[-1]
    dw = torch.empty(vocab, h, dtype=torch.float32, device=dy.device)
    _lib.call("catnn_embedding_bwd", _h(dy), _p(ids), ids.numel(), _p(dy), _p(dw), vocab, h, _dt(dy))
    return dw


# ------------------------------------------------------------------ attention
def rope(x, theta, inverse=False):
    """In-place RoPE on x [B,S,heads,hd] (moe.rs:47; inverse = adjoint.rs:454)."""
    b, s, hh, hd = x.shape
    _lib.call("catnn_rope", _h(x), _p(x), b, s, hh, hd, float(theta), int(inverse), _dt(x))
    return x


def attention_core(q, k, v, causal=True, window=None):
    """q [B,S,H,hd], k/v [B,S,Hkv,hd] -> (o [B,S,H*hd], lse [B,H,S])."""
    _same(q, k, v)
    b, s, h, hd = q.shape
    hkv = k.shape[2]
    o = torch.empty(b, s, h * hd, dtype=q.dtype, device=q.device)
    lse = torch.empty(b, h, s, dtype=torch.float32, device=q.device)
    _lib.call("catnn_attention_fwd", _h(q), _p(q), _p(k), _p(v), _p(o), _p(lse), b, s, h, hkv, hd, int(causal),
              int(window or 0), _dt(q))
    return o, lse


def attention_core_backward(q, k, v, o, lse, dout, causal=True, window=None):
    b, s, h, hd = q.shape
    hkv = k.shape[2]
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    _lib.call("catnn_attention_bwd", _h(q), _p(q), _p(k), _p(v), _p(o), _p(lse), _p(dout), _p(dq), _p(dk), _p(dv), b, s,
              h, hkv, hd, int(causal), int(window or 0), _dt(q))
    return dq, dk, dv


def attention(x, wq, wk, wv, wo, n_heads, causal=False):
    """cpu::attention (cpu.rs:235); causal=True adds the j <= i mask."""
    _same(x, wq, wk, wv, wo)
    b, s, d = x.shape
    if d % n_heads:
        raise ShapeMismatch("attention head split")
    y = torch.empty_like(x)
    _lib.call("catnn_mha_fwd", _h(x), _p(x), _p(wq), _p(wk), _p(wv), _p(wo), _p(y), b, s, d, n_heads, int(causal), _dt(x))
    return y


def attention_backward(x, wq, wk, wv, wo, dy, n_heads, causal=False):
    """attention_backward (adjoint.rs:582) -> (dx, dwq, dwk, dwv, dwo)."""
    b, s, d = x.shape
    outs = [torch.empty_like(t) for t in (x, wq, wk, wv, wo)]
    _lib.call("catnn_mha_bwd", _h(x), _p(x), _p(wq), _p(wk), _p(wv), _p(wo), _p(dy), *[_p(o) for o in outs], b, s, d,
              n_heads, int(causal), _dt(x))
    return tuple(outs)


def gqa(x, wq, wk, wv, wo, n_heads, n_kv, theta, window=None):
    """moe::gqa (moe.rs:64): causal GQA with RoPE and optional window."""
    _same(x, wq, wk, wv, wo)
    b, s, d = x.shape
    hd = wq.shape[1] // n_heads
    y = torch.empty(b, s, wo.shape[1], dtype=x.dtype, device=x.device)
    _lib.call("catnn_gqa_fwd", _h(x), _p(x), _p(wq), _p(wk), _p(wv), _p(wo), _p(y), b, s, d, n_heads, n_kv, hd,
              float(theta), int(window or 0), _dt(x))
    return y


def gqa_backward(x, wq, wk, wv, wo, dy, n_heads, n_kv, theta, window=None):
    """gqa_backward (adjoint.rs:287) -> (dx, dwq, dwk, dwv, dwo)."""
    b, s, d = x.shape
    hd = wq.shape[1] // n_heads
    outs = [torch.empty_like(t) for t in (x, wq, wk, wv, wo)]
    _lib.call("catnn_gqa_bwd", _h(x), _p(x), _p(wq), _p(wk), _p(wv), _p(wo), _p(dy), *[_p(o) for o in outs], b, s, d,
              n_heads, n_kv, hd, float(theta), int(window or 0), _dt(x))
    return tuple(outs)


# ------------------------------------------------------------------ MoE
def router_topk(logits, k):
    """lens::moe::topk_softmax per row -> (idx int32 [T,k], w fp32 [T,k])."""
    _f32(logits, "logits")
    t, e = logits.shape
    idx = torch.empty(t, k, dtype=torch.int32, device=logits.device)
    w = torch.empty(t, k, dtype=torch.float32, device=logits.device)
    _lib.call("catnn_router_topk", _h(logits), _p(logits), t, e, k, _p(idx), _p(w))
    return idx, w


def moe_permute_map(idx, n_experts, align=1):
    """Stable counting sort of (token, slot) pairs by expert."""
    t, k = idx.shape
    dev = idx.device
    cap = t * k + n_experts * (align - 1)
    counts = torch.empty(n_experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    row_of = torch.empty(t * k, dtype=torch.int32, device=dev)
    src_of = torch.empty(cap, dtype=torch.int32, device=dev)
    _lib.call("catnn_moe_permute_map", _h(idx), _p(idx.contiguous()), t, n_experts, k, align, _p(counts), _p(offsets),
              _p(row_of), _p(src_of))
    return counts, offsets, row_of, src_of


def moe_permute(x, src_of, k):
    rows = src_of.numel()
    h = x.shape[-1]
    xp = torch.empty(rows, h, dtype=x.dtype, device=x.device)
    _lib.call("catnn_moe_permute", _h(x), _p(x), _p(src_of), rows, h, k, _p(xp), _dt(x))
    return xp


def moe_unpermute(yp, row_of, w, tokens, k):
    h = yp.shape[-1]
    y = torch.empty(tokens, h, dtype=yp.dtype, device=yp.device)
    _lib.call("catnn_moe_unpermute", _h(yp), _p(yp), _p(row_of), _p(w), tokens, k, h, _p(y), _dt(yp))
    return y


def grouped_gemm(a, b, offsets, trans_b=False, out=None, out_dtype=None):
    """Per-expert GEMM over expert-sorted rows (catnn_grouped_gemm):
    rows [off[g], off[g+1]) of a [rows, K] times b[g] ([K,N], or [N,K] with trans_b)."""
    _same(a, b)
    rows, k = a.shape
    g = b.shape[0]
    n = b.shape[1] if trans_b else b.shape[2]
    if out is None:
        out = torch.empty(rows, n, dtype=out_dtype or a.dtype, device=a.device)
    _lib.call("catnn_grouped_gemm", _h(a), int(trans_b), rows, n, k, g, _p(offsets), _p(a), _p(b), _p(out), _dt(a),
              _dt(out))
    return out


def interleave_w13(w1s, w3s):
    """[E, hidden, 2·mid] with each expert's w1 and w3 columns interleaved in
    blocks of 128 (the layout of the fused SwiGLU expert GEMMs)."""
    E, h, F = w1s.shape
    if F % 128:
        raise ShapeMismatch("interleaved w13: mid must be a multiple of 128")
    return torch.stack((w1s.reshape(E, h, F // 128, 128), w3s.reshape(E, h, F // 128, 128)), 3).reshape(E, h, 2 * F)


def moe_expert_swiglu(x, w13, offsets):
    """ac = x·w13 and h = silu(a)·c per expert group, the SwiGLU in the GEMM
    epilogue (catnn_moe_expert_swiglu_fwd; bf16). Returns (ac, h)."""
    _same(x, w13)
    rows, hidden = x.shape
    E, _, F2 = w13.shape
    ac = torch.empty(rows, F2, dtype=x.dtype, device=x.device)
    h = torch.empty(rows, F2 // 2, dtype=x.dtype, device=x.device)
    _lib.call("catnn_moe_expert_swiglu_fwd", _h(x), _p(x), _p(w13), _p(offsets), rows, hidden, F2 // 2, E, _p(ac), _p(h))
    return ac, h


def moe_expert_swiglu_backward(dy, w2, ac, offsets):
    """dac = [da | dc] from dh = dy·w2ᵀ per expert group and the saved ac
    (catnn_moe_expert_swiglu_bwd; bf16)."""
    _same(dy, w2, ac)
    rows, hidden = dy.shape
    E, F, _ = w2.shape
    dac = torch.empty(rows, 2 * F, dtype=dy.dtype, device=dy.device)
    _lib.call("catnn_moe_expert_swiglu_bwd", _h(dy), _p(dy), _p(w2), _p(ac), _p(offsets), rows, hidden, F, E, _p(dac))
    return dac


def swiglu(x, w1, w3, w2):
    """moe::swiglu (moe.rs:159)."""
    _same(x, w1, w3, w2)
    h = x.shape[-1]
    t = x.numel() // h
    mid = w1.shape[1]
    y = torch.empty_like(x)
    _lib.call("catnn_swiglu_fwd", _h(x), _p(x), _p(w1), _p(w3), _p(w2), _p(y), t, h, mid, _dt(x))
    return y


def swiglu_backward(x, w1, w3, w2, dy):
    """swiglu_backward (adjoint.rs:217) -> (dx, dw1, dw3, dw2)."""
    h = x.shape[-1]
    t = x.numel() // h
    mid = w1.shape[1]
    outs = [torch.empty_like(a) for a in (x, w1, w3, w2)]
    _lib.call("catnn_swiglu_bwd", _h(x), _p(x), _p(w1), _p(w3), _p(w2), _p(dy), *[_p(o) for o in outs], t, h, mid, _dt(x))
    return tuple(outs)


def moe(x, gate, w1s, w3s, w2s, top_k):
    """moe::moe (moe.rs:197); expert weights stacked [E, ...]."""
    _same(x, gate, w1s, w3s, w2s)
    h = x.shape[-1]
    t = x.numel() // h
    e, _, mid = w1s.shape
    y = torch.empty_like(x)
    _lib.call("catnn_moe_fwd", _h(x), _p(x), _p(gate), _p(w1s), _p(w3s), _p(w2s), _p(y), t, h, mid, e, top_k, _dt(x))
    return y


def moe_backward(x, gate, w1s, w3s, w2s, dy, top_k):
    """moe_backward (adjoint.rs:471) -> (dx, dgate, dw1s, dw3s, dw2s)."""
    h = x.shape[-1]
    t = x.numel() // h
    e, _, mid = w1s.shape
    outs = [torch.empty_like(a) for a in (x, gate, w1s, w3s, w2s)]
    _lib.call("catnn_moe_bwd", _h(x), _p(x), _p(gate), _p(w1s), _p(w3s), _p(w2s), _p(dy), *[_p(o) for o in outs], t, h, mid,
              e, top_k, _dt(x))
    return tuple(outs)


# ------------------------------------------------------------------ decoding
# A decoding step calls these with next to nothing to compute, so what the
# host spends on a call counts: shapes are unpacked once and compared as numbers.
def _on(t, *others):
    """All of one call's tensors lie on one CUDA device; its context."""
    d = t.get_device()
    if d < 0:
        raise InvalidArgument("catnn_b200 operators take CUDA tensors")
    for o in others:
        if o is not None and o.get_device() != d:
            raise InvalidArgument(f"tensors on {t.device} and {o.device}")
    return _CTX.get(d) or context(d)


def _rows(t, what):
    """Elements between the tokens of t [..., heads, hd], whose heads must be
    dense and whose tokens evenly spaced: a tensor of its own, or a column
    block of the rows that one QKV product writes."""
    *lead, heads, hd = t.shape
    if t.is_contiguous() or t.numel() == 0:
        return heads * hd
    *st, per_head, per_value = t.stride()
    if (hd > 1 and per_value != 1) or (heads > 1 and per_head != hd):
        raise InvalidArgument(f"{what}: a token's heads must be dense")
    token, span = heads * hd, None  # span: stride of the next outer dimension that is evenly spaced
    while lead:
        n, step = lead.pop(), st.pop()
        if n == 1:
            continue
        if span is None:
            token = step
        elif step != span:
            raise InvalidArgument(f"{what}: tokens must be evenly spaced")
        span = step * n
    return token


def _dense_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _i32(t, what):
    if t.dtype != torch.int32:
        raise DTypeMismatch(f"{what} must be int32")
    if not t.is_contiguous():
        raise InvalidArgument(f"{what} must be contiguous")
    return t.data_ptr()


def _weight(w, hd, what):
    if w.dtype != torch.float32:
        raise DTypeMismatch(f"{what} must be float32")
    if w.numel() != hd or w.dim() != 1 or not w.is_contiguous():
        raise ShapeMismatch(f"{what} must be a dense [{hd}] vector")
    return w.data_ptr()


def _qk(q, k, what):
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[0] != ks[0] or qs[1] != ks[1] or qs[3] != ks[3]:
        raise ShapeMismatch(f"{what}: q {tuple(qs)}, k {tuple(ks)}")
    if q.dtype != k.dtype:
        _same(q, k)
    b, s, h, hd = qs
    return b, s, h, ks[2], hd


def _positions(positions, b, s, what):
    if positions is None:
        return None
    if tuple(positions.shape) != (b, s):
        raise ShapeMismatch(f"{what}: positions {tuple(positions.shape)}")
    return _i32(positions, "positions")


def qk_norm_rope(q, k, wq, wk, theta, eps=1e-5, positions=None):
    """RMS norm of every head of q [B,S,H,hd] and k [B,S,Hkv,hd] with the
    weights wq, wk [hd] (fp32), then the rotation of its pairs to its position,
    in one pass -> (q', k'), dense. positions int32 [B,S]; None: 0..S-1. q and k
    may be column blocks of packed QKV rows."""
    b, s, h, hkv, hd = _qk(q, k, "qk_norm_rope")
    pos = _positions(positions, b, s, "qk_norm_rope")
    ctx = _on(q, k, wq, wk, positions)
    qo, ko = _dense_like(q), _dense_like(k)
    _lib.call("catnn_qk_norm_rope_fwd", ctx.bind(), q.data_ptr(), _rows(q, "q"), k.data_ptr(), _rows(k, "k"),
              _weight(wq, hd, "wq"), _weight(wk, hd, "wk"), pos, qo.data_ptr(), ko.data_ptr(), b, s, h, hkv, hd, theta, eps,
              _dt(q))
    return qo, ko


def qk_norm_rope_backward(q, k, wq, wk, dq_out, dk_out, theta, eps=1e-5, positions=None):
    """Adjoint of qk_norm_rope from its inputs and the gradients of its
    results -> (dq, dk, dwq, dwk); dwq and dwk are summed in a fixed order."""
    b, s, h, hkv, hd = _qk(q, k, "qk_norm_rope backward")
    pos = _positions(positions, b, s, "qk_norm_rope backward")
    if dq_out.shape != q.shape or dk_out.shape != k.shape:
        raise ShapeMismatch(f"qk_norm_rope backward: dq_out {tuple(dq_out.shape)}, dk_out {tuple(dk_out.shape)}")
    _same(q, dq_out, dk_out)
    ctx = _on(q, k, wq, wk, positions, dq_out, dk_out)
    ws, n = ctx.workspace("catnn_qk_norm_rope_bwd_workspace", b, s, h, hkv, hd)
    dq, dk, dwq, dwk = _dense_like(q), _dense_like(k), torch.empty_like(wq), torch.empty_like(wk)
    _lib.call("catnn_qk_norm_rope_bwd", ctx.bind(), q.data_ptr(), _rows(q, "q"), k.data_ptr(), _rows(k, "k"),
              _weight(wq, hd, "wq"), _weight(wk, hd, "wk"), pos, dq_out.data_ptr(), _rows(dq_out, "dq_out"),
              dk_out.data_ptr(), _rows(dk_out, "dk_out"), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(),
              b, s, h, hkv, hd, theta, eps, _dt(q), ws.data_ptr() if n else None, n)
    return dq, dk, dwq, dwk


def _cache(k_cache, v_cache, page_table, seq_lens, hkv, hd, like, what):
    """Checks a paged cache -> (pages, page size), (sequences, table columns), table, lengths."""
    ks, ts = k_cache.shape, page_table.shape
    if len(ks) != 4 or v_cache.shape != ks or ks[1] != hkv or ks[3] != hd:
        raise ShapeMismatch(f"{what}: caches {tuple(ks)}, {tuple(v_cache.shape)} for {hkv} heads of {hd}")
    if len(ts) != 2 or seq_lens.dim() != 1 or seq_lens.numel() != ts[0]:
        raise ShapeMismatch(f"{what}: page table {tuple(ts)}, lengths {tuple(seq_lens.shape)}")
    _same(like, k_cache, v_cache)
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise InvalidArgument(f"{what}: caches must be contiguous")
    return (ks[0], ks[2]), ts, _i32(page_table, "page_table"), _i32(seq_lens, "seq_lens")


def kv_append(q, k, v, k_cache, v_cache, page_table, seq_lens, theta, cu_tokens=None, wq=None, wk=None, eps=1e-5,
              check=False):
    """Appends the keys and values of new tokens to a paged cache, in place,
    and returns their rotated queries [T,H,hd] (None for q None).

    q [T,H,hd], k and v [T,Hkv,hd] (column blocks of packed QKV rows, or
    tensors of their own); caches [pages,Hkv,page,hd]; page_table int32
    [seqs,max_pages]; seq_lens int32 [seqs], with the new tokens; cu_tokens
    int32 [seqs+1]: where each sequence's new tokens begin among the T rows,
    None for one new token each. wq, wk (fp32 [hd]): per-head RMS norm before
    the rotation. Rows of no sequence are not appended (their queries are
    zero); slots without a page are not written, which check=True
    (synchronizing) reports as a ShapeMismatch. No two rows may name the same
    slot."""
    ks = k.shape
    if len(ks) != 3 or v.shape != ks:
        raise ShapeMismatch(f"kv_append: k {tuple(ks)}, v {tuple(v.shape)}")
    t, hkv, hd = ks
    (pages, page), (seqs, most), table, lens = _cache(k_cache, v_cache, page_table, seq_lens, hkv, hd, k, "kv_append")
    _same(k, v, q)
    h, qo, qp, q_rows, qop = 0, None, None, 0, None
    if q is not None:
        qs = q.shape
        if len(qs) != 3 or qs[0] != t or qs[2] != hd:
            raise ShapeMismatch(f"kv_append: q {tuple(qs)}, k {tuple(ks)}")
        h, qp, q_rows = qs[1], q.data_ptr(), _rows(q, "q")
    cu = None
    if cu_tokens is not None:
        if cu_tokens.dim() != 1 or cu_tokens.numel() != seqs + 1:
            raise ShapeMismatch(f"kv_append: cu_tokens {tuple(cu_tokens.shape)} for {seqs} sequences")
        cu = _i32(cu_tokens, "cu_tokens")
    elif t != seqs:
        raise ShapeMismatch(f"kv_append: {t} rows for {seqs} sequences without cu_tokens")
    if (wq is None) != (wk is None):
        raise InvalidArgument("kv_append: both norm weights or neither")
    wqp, wkp = (None, None) if wq is None else (_weight(wq, hd, "wq"), _weight(wk, hd, "wk"))
    ctx = _on(k, q, v, k_cache, v_cache, page_table, seq_lens, cu_tokens, wq, wk)
    if q is not None:
        qo = _dense_like(q)
        qop = qo.data_ptr()
    _lib.call("catnn_kv_append", ctx.bind(), qp, q_rows, k.data_ptr(), _rows(k, "k"), v.data_ptr(), _rows(v, "v"), wqp, wkp,
              qop, k_cache.data_ptr(), v_cache.data_ptr(), table, lens, cu, t, seqs, h, hkv, hd, pages, page, most, theta, eps,
              _dt(k), check)
    return qo


def paged_attention(q, k_cache, v_cache, page_table, seq_lens, window=None, check=False):
    """Attention of one new token of each sequence, q [seqs,H,hd], against its
    cached positions, the last of which is its own (append first)
    -> (o [seqs,H*hd], lse [seqs,H]). Caches, table and lengths as in
    kv_append; a sequence of length 0 gets zeros and -inf."""
    qs, ks = q.shape, k_cache.shape
    hkv = ks[1] if len(ks) == 4 else 0
    if len(qs) != 3 or hkv < 1 or qs[1] % hkv:
        raise ShapeMismatch(f"paged_attention: q {tuple(qs)} for {hkv} kv heads")
    b, h, hd = qs
    (pages, page), (seqs, most), table, lens = _cache(k_cache, v_cache, page_table, seq_lens, hkv, hd, q, "paged_attention")
    if seqs != b:
        raise ShapeMismatch(f"paged_attention: {b} queries, {seqs} sequences")
    ctx = _on(q, k_cache, v_cache, page_table, seq_lens)
    dt = _dt(q)
    ws, n = ctx.workspace("catnn_paged_attention_workspace", b, h, hkv, hd, dt)
    o, lse = q.new_empty(b, h * hd), torch.empty(b, h, dtype=torch.float32, device=q.device)
    _lib.call("catnn_paged_attention_fwd", ctx.bind(), q.data_ptr(), _rows(q, "q"), k_cache.data_ptr(), v_cache.data_ptr(),
              table, lens, o.data_ptr(), lse.data_ptr(), b, h, hkv, hd, pages, page, most, window or 0, dt,
              ws.data_ptr() if n else None, n, check)
    return o, lse


def moe_few(x, gate, w1s, w3s, w2s, top_k, check=False):
    """moe() for at most 64 rows of x (more are refused: moe() takes them), in
    two kernels that read each chosen expert's weights once; expert weights
    stacked [E, ...]. That is for hidden and mid of at least 64, multiples of 8
    (fp32: 4), and operands on 16-byte boundaries; other calls are computed by
    kernels that take 1 ms and more where these take 20 to 170 us. check=True
    (synchronizing) reports a bounded wait that ran out, in this call or one
    since the last check, as a DeviceTimeout; its rows are NaN."""
    _same(x, gate, w1s, w3s, w2s)
    ws1 = w1s.shape
    hid = x.shape[-1]
    if len(ws1) != 3 or ws1[1] != hid:
        raise ShapeMismatch(f"moe_few: x {tuple(x.shape)}, w1s {tuple(ws1)}")
    e, _, mid = ws1
    if w3s.shape != ws1 or tuple(w2s.shape) != (e, mid, hid) or tuple(gate.shape) != (hid, e):
        raise ShapeMismatch(f"moe_few: gate {tuple(gate.shape)}, w1s {tuple(ws1)}, w3s {tuple(w3s.shape)}, "
                            f"w2s {tuple(w2s.shape)}")
    if not (x.is_contiguous() and gate.is_contiguous() and w1s.is_contiguous() and w3s.is_contiguous()
            and w2s.is_contiguous()):
        raise InvalidArgument("catnn_b200 operators take contiguous tensors")
    t = x.numel() // max(hid, 1)
    if t > 64 or not 1 <= top_k <= e <= 32:
        raise ShapeMismatch(f"moe_few: {t} rows (at most 64), top {top_k} of {e} experts (at most 32)")
    dt = _dt(x)
    ctx = _on(x, gate, w1s, w3s, w2s)
    ws, n = ctx.workspace("catnn_moe_few_workspace", t, hid, mid, e, top_k, dt)
    y = torch.empty_like(x)
    _lib.call("catnn_moe_few_fwd", ctx.bind(), x.data_ptr(), gate.data_ptr(), w1s.data_ptr(), w3s.data_ptr(),
              w2s.data_ptr(), y.data_ptr(), t, hid, mid, e, top_k, dt, ws.data_ptr() if n else None, n)
    if check:
        _lib.call("catnn_moe_few_check", ctx.handle)
    return y


# ------------------------------------------------------------------ optimizers
def sgd_(p, g, lr, shadow=None):
    """Sgd::put in place (optim.rs:32): p -= lr * g."""
    _f32(p, "param")
    _f32(g, "grad")
    if p.numel() != g.numel():
        raise ShapeMismatch("sgd put")
    _lib.call("catnn_sgd", _h(p), _p(p), _p(g), p.numel(), float(lr), _p(shadow))
    return p


def adam_(p, g, m, v, t, lr, beta1=0.9, beta2=0.999, eps=1e-8, shadow=None):
    """Adam::put in place (optim.rs:95) at step count t (>= 1)."""
    _f32(p, "param")
    if not (p.numel() == g.numel() == m.numel() == v.numel()):
        raise ShapeMismatch("adam shapes")
    _lib.call("catnn_adam", _h(p), _p(p), _p(g), _p(m), _p(v), p.numel(), int(t), float(lr), float(beta1), float(beta2),
              float(eps), _dt(g), _p(shadow))
    return p


# ------------------------------------------------------------------ MLP step
def mlp_step(w1, b1, w2, b2, x, labels=None, y_mse=None):
    """train::mlp_step (train.rs:71) -> (loss tensor, dw1, db1, dw2, db2)."""
    batch, din = x.shape
    hid, dout = w1.shape[1], w2.shape[1]
    ce = labels is not None
    loss = torch.empty((), dtype=torch.float32, device=x.device)
    dw1, db1, dw2, db2 = (torch.empty_like(t) for t in (w1, b1, w2, b2))
    lab = _ids(labels) if ce else None
    _lib.call("catnn_mlp_step", _h(x), _p(w1), _p(b1), _p(w2), _p(b2), _p(x), _p(lab), _p(y_mse), int(ce), batch, din, hid,
              dout, _p(loss), _p(dw1), _p(db1), _p(dw2), _p(db2))
    return loss, dw1, db1, dw2, db2


def checksum(x):
    """FNV-1a over the f32 bits (tensor.rs:279), computed on the device."""
    _f32(x, "checksum input")
    v = C.c_uint64()
    _lib.call("catnn_checksum_f32", _h(x), _p(x), x.numel(), C.byref(v))
    return int(v.value)


# ------------------------------------------------------------------ kernel resources
class KernelShape(C.Structure):
    """catnn_kernel_shape (include/catnn_b200.h)."""
    _fields_ = [(n, C.c_int64) for n in ("rows", "width", "inner", "batch", "seq", "heads", "head_dim")]


class KernelResource(C.Structure):
    """catnn_kernel_resource (include/catnn_b200.h): KernelResource of
    crates/catnn-compile/src/kernel/resource.rs:28-44, measured."""
    _fields_ = [("kernel", C.c_char * 192), ("file", C.c_char * 32), ("registers_per_thread", C.c_int32),
                ("max_threads_per_block", C.c_int32), ("static_smem_bytes", C.c_int64),
                ("dynamic_smem_bytes", C.c_int64), ("local_bytes_per_thread", C.c_int64), ("grid", C.c_uint32 * 3),
                ("block", C.c_uint32 * 3), ("launch_arg_bytes", C.c_int64), ("code_bytes", C.c_int64),
                ("code_estimated", C.c_int32), ("binary_version", C.c_int32)]


def kernel_describe(op, dtype=torch.bfloat16, device=None, rows=0, width=0, inner=0, batch=0, seq=0, heads=0,
                    head_dim=0):
    """The resource record of the kernel that runs IR op `op` (resource::describe,
    resource.rs:159), as a dict."""
    shape = KernelShape(rows, width, inner, batch, seq, heads, head_dim)
    out = KernelResource()
    h = context(device).bind()
    _lib.call("catnn_kernel_describe", h, op.encode(), BF16 if dtype == torch.bfloat16 else F32, C.byref(shape),
              C.byref(out))
    d = {f: getattr(out, f) for f, _ in KernelResource._fields_}
    d["kernel"], d["file"] = out.kernel.decode(), out.file.decode()
    d["grid"], d["block"] = list(out.grid), list(out.block)
    return d
