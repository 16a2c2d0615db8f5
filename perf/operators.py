"""What is measured of the decoding operators and of the per-head query/key norm.

The cases cover the four operators that take a trained decoder from its
training step to answering with it:

- ``qk_norm_rope`` and its adjoint: RMS norm of every query and key head with
  the position rotation in the same pass (training and prompt processing),
- ``kv_append``: new keys and values rotated into a paged cache, the queries
  of the same tokens rotated beside them,
- ``paged_attention``: one new token of each sequence against the paged cache,
- ``moe_few``: a whole mixture-of-experts layer for a few tokens.

``run`` computes them in elementary torch operations, or, with ``own``, by the
calls of ``catnn_b200.ops``. Sizes are those of the Mixtral-style decoder
(hidden 1024, 16 heads of 64, 8 experts of 3584, top 2, 2048 positions) and of
the tiny one (hidden 256, 512, 4 heads), or generic ones beside them.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-5
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
_ops = None


def _own():
    global _ops
    if _ops is None:
        at = os.path.abspath("cat-nn-compiler_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        from catnn_b200 import ops
        _ops = ops
    return _ops


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of one sequence: what a decoding loop pays per layer, all latency
        {"name": "qk_fwd_one_token", "op": "qk_fwd", "dtype": "bf16", "b": 1, "s": 1, "h": 16, "hkv": 4, "hd": 64,
         "theta": 1e6, "packed": True, "positions": True},
        # a layer of the training step: 8 sequences of 2048 read out of the packed QKV rows
        {"name": "qk_fwd_train", "op": "qk_fwd", "dtype": "bf16", "b": 8, "s": 2048, "h": 16, "hkv": 4, "hd": 64,
         "theta": 1e6, "packed": True, "positions": False},
        # its adjoint
        {"name": "qk_bwd_train", "op": "qk_bwd", "dtype": "bf16", "b": 8, "s": 2048, "h": 16, "hkv": 4, "hd": 64,
         "theta": 1e6, "packed": True, "positions": False},
        # the fp32 parity path at a head size that is no power of two
        {"name": "qk_bwd_odd_f32", "op": "qk_bwd", "dtype": "f32", "b": 3, "s": 333, "h": 6, "hkv": 2, "hd": 80,
         "theta": 1e4, "packed": False, "positions": True},
        # one token of each of 32 sequences, as a decoding step appends them
        {"name": "append_decode", "op": "append", "dtype": "bf16", "seqs": 32, "new": 1, "past": 2000, "spread": 5,
         "h": 16, "hkv": 4, "hd": 64, "page": 16, "theta": 1e6, "norm": False},
        # prompts of 8 requests entering the cache, with the per-head norm
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "seqs": 8, "new": 2047, "past": 300, "spread": 7,
         "h": 16, "hkv": 4, "hd": 128, "page": 32, "theta": 1e6, "norm": True},
        # a single chat at the trained length, a key/value head to every query head
        {"name": "paged_one_chat", "op": "paged", "dtype": "bf16", "seqs": 1, "len": 2047, "spread": 1, "h": 16,
         "hkv": 16, "hd": 64, "page": 16, "window": 0},
        # a serving batch of ragged lengths
        {"name": "paged_batch", "op": "paged", "dtype": "bf16", "seqs": 64, "len": 6000, "spread": 3, "h": 16, "hkv": 4,
         "hd": 128, "page": 16, "window": 0},
        # two long documents on the fp32 path
        {"name": "paged_long_f32", "op": "paged", "dtype": "f32", "seqs": 2, "len": 40001, "spread": 2, "h": 8,
         "hkv": 2, "hd": 64, "page": 64, "window": 0},
        # one token through a layer of the decoder: two of eight experts
        {"name": "moe_one_token", "op": "moe", "dtype": "bf16", "t": 1, "hidden": 1024, "mid": 3584, "e": 8, "k": 2},
        # a decoding batch: every expert has some of the 64 tokens
        {"name": "moe_64_tokens", "op": "moe", "dtype": "bf16", "t": 64, "hidden": 1024, "mid": 3584, "e": 8, "k": 2},
        # the tiny decoder on the fp32 path
        {"name": "moe_tiny_f32", "op": "moe", "dtype": "f32", "t": 7, "hidden": 256, "mid": 512, "e": 8, "k": 2},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


#: the most bytes a drawn case of an operator moves: a little under its largest listed case
_MOST = {"qk_fwd": 80e6, "qk_bwd": 120e6, "append": 150e6, "paged": 4e8, "moe": 1.7e8}


def draw(rng):
    """Heads, head sizes, lengths, pages and batches over the ranges of the listed cases."""
    op = rng.choice(["qk_fwd", "qk_bwd", "append", "paged", "moe"])
    while True:
        c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f32"])}
        hkv = rng.choice([1, 2, 3, 4, 8, 16])
        group = rng.choice([1, 1, 2, 4, 5, 8])
        heads = {"h": hkv * group, "hkv": hkv, "hd": rng.choice([32, 64, 64, 80, 96, 128, 128])}
        if op in ("qk_fwd", "qk_bwd"):
            c.update(heads, b=_log(rng, 1, 16), s=_log(rng, 1, 4096), theta=rng.choice([1e4, 1e6]),
                     packed=rng.random() < 0.5, positions=rng.random() < 0.5)
        elif op == "append":
            c.update(heads, seqs=_log(rng, 1, 64), new=_log(rng, 1, 2048), past=_log(rng, 1, 4000),
                     spread=rng.randrange(1000), page=rng.choice([1, 8, 16, 24, 32, 64, 128]),
                     theta=rng.choice([1e4, 1e6]), norm=rng.random() < 0.5)
        elif op == "paged":
            c.update(heads, seqs=_log(rng, 1, 128), len=_log(rng, 1, 40000), spread=rng.randrange(1000),
                     page=rng.choice([1, 8, 16, 24, 32, 64, 128]), window=rng.choice([0, 0, 0, 100, 1000]))
        else:
            c.update(t=_log(rng, 1, 64), hidden=8 * _log(rng, 8, 256), mid=8 * _log(rng, 8, 448),
                     e=rng.choice([2, 4, 8, 8, 16, 32]), k=rng.choice([1, 2, 2, 4]))
            c["k"] = min(c["k"], c["e"])
        if work(c)["bytes"] <= _MOST[op] and _held(c) <= 1e9:
            return c


def _held(c):
    """Bytes of a case's inputs, its unread ones (cache pages, experts that no token takes) among them."""
    if c["op"] == "moe":
        return c["e"] * 3 * c["hidden"] * c["mid"] * SIZE[c["dtype"]]
    if c["op"] in ("append", "paged"):
        return 2 * sum(_lens(c)) * c["hkv"] * c["hd"] * SIZE[c["dtype"]]
    return 0


def _news(c):
    """How many tokens each sequence appends: ragged around c['new'] (1 stays 1)."""
    r = random.Random(c["spread"])
    return [max(1, c["new"] - r.randrange(c["new"] // 2 + 1)) for _ in range(c["seqs"])]


def _lens(c):
    """Length of each sequence, from nearly nothing to the case's largest, which is there."""
    r = random.Random(c["spread"] + 1)
    if c["op"] == "append":
        return [n + r.randrange(c["past"] + 1) for n in _news(c)]
    return [c["len"]] + [max(1, round(c["len"] * r.random())) for _ in range(c["seqs"] - 1)]


def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] in ("qk_fwd", "qk_bwd"):
        n = c["b"] * c["s"] * (c["h"] + c["hkv"]) * c["hd"]
        pos = 4 * c["b"] * c["s"] if c["positions"] else 0
        if c["op"] == "qk_fwd":
            return {"bytes": 2 * n * e + pos + 8 * c["hd"], "flops": 8 * n}
        return {"bytes": 3 * n * e + pos + 16 * c["hd"], "flops": 20 * n}
    if c["op"] == "append":
        n = sum(_news(c)) * (c["h"] + 2 * c["hkv"]) * c["hd"]
        return {"bytes": 2 * n * e + 4 * sum(_news(c)) // max(1, c["page"]), "flops": 8 * n}
    if c["op"] == "paged":
        lens = [min(n, c["window"]) if c["window"] else n for n in _lens(c)]
        keys, rows = sum(lens), c["seqs"] * c["h"] * c["hd"]
        return {"bytes": 2 * keys * c["hkv"] * c["hd"] * e + 2 * rows * e + 4 * c["seqs"] * c["h"] + 4 * keys // c["page"],
                "flops": 4 * keys * c["h"] * c["hd"]}
    # of E experts, T tokens that take k each reach this many on average
    used = c["e"] * (1 - (1 - c["k"] / c["e"]) ** c["t"])
    weights = 3 * c["hidden"] * c["mid"]
    return {"bytes": used * weights * e + c["hidden"] * c["e"] * e + 2 * c["t"] * c["hidden"] * e,
            "flops": 2 * c["t"] * (c["k"] * weights + c["hidden"] * c["e"])}


# ------------------------------------------------------------------ inputs
def _rand(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[c["dtype"]]
    s = {"case": c}
    if c["op"] in ("qk_fwd", "qk_bwd"):
        b, n, h, hkv, hd = c["b"], c["s"], c["h"], c["hkv"], c["hd"]
        if c["packed"]:  # the rows that one QKV product writes
            qkv = _rand(g, b, n, (h + 2 * hkv) * hd, dtype=dt)
            s["q"] = qkv[..., :h * hd].unflatten(-1, (h, hd))
            s["k"] = qkv[..., h * hd:(h + hkv) * hd].unflatten(-1, (hkv, hd))
        else:
            s["q"], s["k"] = _rand(g, b, n, h, hd, dtype=dt), _rand(g, b, n, hkv, hd, dtype=dt)
        s["wq"] = 1 + _rand(g, hd, dtype=torch.float32, scale=0.2)
        s["wk"] = 1 + _rand(g, hd, dtype=torch.float32, scale=0.2)
        s["positions"] = None
        if c["positions"]:  # each sequence goes on from where it stands
            start = torch.randint(0, 4096, (b, 1), generator=g, device="cuda", dtype=torch.int32)
            s["positions"] = start + torch.arange(n, device="cuda", dtype=torch.int32)
        if c["op"] == "qk_bwd":
            s["dq"], s["dk"] = _rand(g, b, n, h, hd, dtype=dt), _rand(g, b, n, hkv, hd, dtype=dt)
        return s
    if c["op"] == "moe":
        t, hid, mid, e = c["t"], c["hidden"], c["mid"], c["e"]
        s["x"] = _rand(g, t, hid, dtype=dt)
        s["gate"] = _rand(g, hid, e, dtype=dt, scale=hid ** -0.5)
        s["w1"] = _rand(g, e, hid, mid, dtype=dt, scale=hid ** -0.5)
        s["w3"] = _rand(g, e, hid, mid, dtype=dt, scale=hid ** -0.5)
        s["w2"] = _rand(g, e, mid, hid, dtype=dt, scale=mid ** -0.5)
        return s
    # the cache: every sequence's pages lie anywhere in the pool, and what is in them past a sequence's end is stale
    seqs, h, hkv, hd, page = c["seqs"], c["h"], c["hkv"], c["hd"], c["page"]
    lens = _lens(c)
    order = list(range(seqs))
    random.Random(seed).shuffle(order)
    lens = [lens[i] for i in order]
    need = [-(-n // page) for n in lens]
    most, total = max(need), sum(need)
    pool = total + 3
    s["k_cache"] = _rand(g, pool, hkv, page, hd, dtype=dt)
    s["v_cache"] = _rand(g, pool, hkv, page, hd, dtype=dt)
    ids = torch.randperm(pool, generator=g, device="cuda")[:total].to(torch.int32).cpu()
    table = torch.full((seqs, most), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    s["table"] = table.cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    if c["op"] == "paged":
        s["q"] = _rand(g, seqs, h, hd, dtype=dt)
        return s
    news = _news(c)
    news = [news[i] for i in order]
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    s["cu"] = torch.tensor(cu, dtype=torch.int32).cuda()
    qkv = _rand(g, cu[-1], (h + 2 * hkv) * hd, dtype=dt)
    s["q"] = qkv[:, :h * hd].unflatten(-1, (h, hd))
    s["k"] = qkv[:, h * hd:(h + hkv) * hd].unflatten(-1, (hkv, hd))
    s["v"] = qkv[:, (h + hkv) * hd:].unflatten(-1, (hkv, hd))
    s["wq"] = 1 + _rand(g, hd, dtype=torch.float32, scale=0.2) if c["norm"] else None
    s["wk"] = 1 + _rand(g, hd, dtype=torch.float32, scale=0.2) if c["norm"] else None
    return s


# ------------------------------------------------------------------ plain forms
def _angles(pos, hd, theta):
    """cos and sin of pos·theta^(-2i/hd): angles of far positions in 64 bits."""
    i = torch.arange(hd // 2, device=pos.device, dtype=torch.float64)
    a = pos.double().unsqueeze(-1) * theta ** (-2 * i / hd)
    return torch.cos(a).float().unsqueeze(-2), torch.sin(a).float().unsqueeze(-2)


def _rotate(x, cos, sin):
    """Pairs (2i, 2i + 1) of x [..., heads, hd] turned by their angles."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _positions(s):
    q = s["q"]
    return s["positions"] if s["positions"] is not None else torch.arange(q.shape[1], device=q.device).expand(q.shape[:2])


def _plain_qk_fwd(s):
    cos, sin = _angles(_positions(s), s["case"]["hd"], s["case"]["theta"])
    return [_rotate(_normed(x, w), cos, sin).to(x.dtype) for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"]))]


def _plain_norm_adjoint(x, w, dy, cos, sin):
    g = _rotate(dy.float(), cos, -sin)
    xf = x.float()
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    xhat = xf * r
    gw = g * w
    dx = r * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * xhat).flatten(0, -2).sum(0, dtype=torch.float64).float()


def _plain_qk_bwd(s):
    cos, sin = _angles(_positions(s), s["case"]["hd"], s["case"]["theta"])
    dq, dwq = _plain_norm_adjoint(s["q"], s["wq"], s["dq"], cos, sin)
    dk, dwk = _plain_norm_adjoint(s["k"], s["wk"], s["dk"], cos, sin)
    return [dq, dk, dwq, dwk]


def _plain_append(s):
    c, cu, lens = s["case"], s["cu"], s["lens"]
    t = torch.arange(s["q"].shape[0], device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], t, right=True)
    pos = lens[seq] - cu[1:][seq] + t
    cos, sin = _angles(pos, c["hd"], c["theta"])
    page = s["table"][seq, (pos // c["page"]).long()].long()[:, None]
    at = (pos % c["page"]).long()[:, None]
    head = torch.arange(c["hkv"], device=cu.device)[None]
    s["k_cache"][page, head, at] = _rotate(_normed(s["k"], s["wk"]), cos, sin).to(s["k"].dtype)
    s["v_cache"][page, head, at] = s["v"]
    return [_rotate(_normed(s["q"], s["wq"]), cos, sin).to(s["q"].dtype), s["k_cache"], s["v_cache"]]


def _plain_paged(s):
    c, q, lens = s["case"], s["q"], s["lens"]
    b, h, hd = q.shape
    pages = s["table"].clamp(min=0).long()
    k = s["k_cache"][pages].transpose(1, 2).flatten(2, 3).float()  # [b, hkv, keys, hd]
    v = s["v_cache"][pages].transpose(1, 2).flatten(2, 3).float()
    scores = q.float().view(b, c["hkv"], -1, hd) @ k.transpose(-1, -2) / math.sqrt(hd)
    j = torch.arange(k.shape[2], device=q.device)
    seen = j < lens[:, None]
    if c["window"]:
        seen &= j >= lens[:, None] - c["window"]
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill(~seen.transpose(-1, -2), 0.0)
    o = (p / total) @ v
    return [o.reshape(b, h * hd).to(q.dtype), (top + torch.log(total)).reshape(b, h)]


def _plain_moe(s):
    c, x = s["case"], s["x"]
    xf = x.float()
    logits = x.double() @ s["gate"].double()  # which experts a token takes can hang on the last bits
    sel, idx = torch.sort(logits, dim=-1, descending=True, stable=True)
    sel, idx = sel[:, :c["k"]], idx[:, :c["k"]]
    p = torch.exp(sel - sel[:, :1])
    w = (p / p.sum(-1, keepdim=True)).float()
    if c["t"] * c["k"] <= c["e"]:  # fewer (token, expert) pairs than experts: the pairs' own weights
        xs = xf[:, None, None, :]
        a = (xs @ s["w1"][idx].float())
        h = a / (1 + torch.exp(-a)) * (xs @ s["w3"][idx].float())
        y = (w[:, :, None] * (h @ s["w2"][idx].float()).squeeze(2)).sum(1)
        return y.to(x.dtype)
    a = torch.matmul(xf, s["w1"].float())  # every expert on every token [e, t, mid]
    h = a / (1 + torch.exp(-a)) * torch.matmul(xf, s["w3"].float())
    y = torch.matmul(h, s["w2"].float())  # [e, t, hidden]
    t = torch.arange(c["t"], device=x.device)[:, None]
    return (w[:, :, None] * y[idx, t]).sum(1).to(x.dtype)


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        ops = _ops or _own()
        if op == "qk_fwd":
            return ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], c["theta"], EPS, s["positions"])
        if op == "qk_bwd":
            return ops.qk_norm_rope_backward(s["q"], s["k"], s["wq"], s["wk"], s["dq"], s["dk"], c["theta"], EPS,
                                             s["positions"])
        if op == "append":
            q = ops.kv_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], c["theta"],
                              cu_tokens=s["cu"], wq=s["wq"], wk=s["wk"], eps=EPS)
            return [q, s["k_cache"], s["v_cache"]]
        if op == "paged":
            return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], window=c["window"])
        return ops.moe_few(s["x"], s["gate"], s["w1"], s["w3"], s["w2"], c["k"])
    return {"qk_fwd": _plain_qk_fwd, "qk_bwd": _plain_qk_bwd, "append": _plain_append, "paged": _plain_paged,
            "moe": _plain_moe}[op](s)


# ------------------------------------------------------------------ 64 bits
def _turned(x, pos, theta):
    """x [..., heads, hd] as complex numbers times e^(i·angle)."""
    hd = x.shape[-1]
    f = torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device),
                  -torch.arange(0, hd, 2, dtype=torch.float64, device=x.device) / hd)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device).expand(*pos.shape, hd // 2),
                       pos.double()[..., None] * f)
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], hd // 2, 2).contiguous())
    return torch.view_as_real(z * turn[..., None, :]).reshape(x.shape)


def _unit(x, w):
    return x if w is None else x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * w


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("qk_fwd", "qk_bwd"):
        n = s["q"].shape[1]
        pos = s["positions"] if c["positions"] else torch.arange(n, device="cuda")[None].repeat(c["b"], 1)
        ins = [s[n].double().contiguous().requires_grad_(c["op"] == "qk_bwd") for n in ("q", "k", "wq", "wk")]
        out = [_turned(_unit(ins[0], ins[2]), pos, c["theta"]), _turned(_unit(ins[1], ins[3]), pos, c["theta"])]
        if c["op"] == "qk_fwd":
            return out
        return list(torch.autograd.grad(out, ins, [s["dq"].double(), s["dk"].double()]))
    if c["op"] == "append":
        cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"].tolist()
        seq, where = [], []
        for b in range(c["seqs"]):
            new = cu[b + 1] - cu[b]
            where += range(lens[b] - new, lens[b])
            seq += [b] * new
        slot = torch.tensor([table[b][p // c["page"]] * c["page"] + p % c["page"] for b, p in zip(seq, where)],
                            device="cuda")
        pos = torch.tensor(where, device="cuda")
        caches = []
        for name, new in (("k_cache", _turned(_unit(s["k"].double(), s["wk"]), pos, c["theta"])),
                          ("v_cache", s["v"].double())):
            rows = s[name].double().transpose(1, 2).reshape(-1, c["hkv"], c["hd"])
            rows[slot] = new
            caches.append(rows.reshape(-1, c["page"], c["hkv"], c["hd"]).transpose(1, 2).contiguous())
        return [_turned(_unit(s["q"].double(), s["wq"]), pos, c["theta"])] + caches
    if c["op"] == "paged":
        outs, lses = [], []
        for b, n in enumerate(s["lens"].tolist()):
            lo = max(0, n - c["window"]) if c["window"] else 0
            j = torch.arange(lo, n, device="cuda")
            page, at = s["table"][b].long()[j // c["page"]], j % c["page"]
            k, v = (s[m][page, :, at].double() for m in ("k_cache", "v_cache"))  # [keys, hkv, hd]
            q = s["q"][b].double().reshape(c["hkv"], -1, c["hd"])
            z = torch.einsum("ngd,jnd->ngj", q, k) * c["hd"] ** -0.5
            outs.append(torch.einsum("ngj,jnd->ngd", torch.softmax(z, -1), v).reshape(-1))
            lses.append(torch.logsumexp(z, -1).reshape(-1))
        return [torch.stack(outs), torch.stack(lses)]
    x, y = s["x"].double(), []
    logits = (x @ s["gate"].double()).cpu().tolist()
    for t, row in enumerate(logits):
        take = sorted(range(c["e"]), key=lambda i: (-row[i], i))[:c["k"]]
        w = torch.softmax(torch.tensor([row[i] for i in take], dtype=torch.float64), 0).tolist()
        y.append(sum(g * ((torch.nn.functional.silu(x[t] @ s["w1"][i].double()) * (x[t] @ s["w3"][i].double()))
                          @ s["w2"][i].double()) for g, i in zip(w, take)))
    return torch.stack(y)
