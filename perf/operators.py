"""Performance cases of the attention's training operators: a sliding window with sink tokens, a
learned relative position bias by buckets, counter-based dropout (on the attention's probabilities
and in the residual add), each with its gradients.

A case is a dict of plain values.
  kind "attn":     lens (sequence lengths as text, comma separated), H, Hkv (head dim 64, bf16),
                   wl, wr (window to the left and right, -1: unlimited), sinks, pos ("none",
                   "alibi" or "buckets"), buckets, far (the bias's largest distance), p (dropout
                   probability of the attention's probabilities), train (forward and backward)
  kind "residual": n, d, dtype ("bf16" | "f32"), p, alpha (forward and backward)

Inputs are drawn on the GPU from the seed: queries, keys, values and gradients N(0, 1) (the size
that normalised activations and projections of a trained model have), bias tables N(0, 1) in bf16, the
type of every other parameter of a bf16 model.
"""
from __future__ import annotations

import math

import numpy as np
import torch
import torch.nn.functional as F

own = False

DEV = "cuda:0"
SCALE = 0.125
M32 = 0xFFFFFFFF


def _attn(name, lens, H=12, Hkv=12, wl=-1, wr=-1, sinks=0, pos="none", buckets=32, far=128,
          p=0.0, train=False):
    c = dict(kind="attn", lens=lens, H=H, Hkv=Hkv, wl=wl, wr=wr, sinks=sinks, pos=pos,
             buckets=buckets, far=far, p=p, train=train)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # inference on one short fragment through a local encoder: latency
        _attn("window_query_77", "77", wl=64, wr=64, sinks=4),
        # inference on a packed batch of eight windows with local attention
        _attn("window_packed_8x4550", ",".join(["4550"] * 8), wl=512, wr=512, sinks=16,
              pos="alibi"),
        # a training micro-step on ragged genes, grouped key/value heads, a one-sided window
        _attn("window_train_ragged", "1100,31,2048,777,1,640,1499,95", Hkv=4, wl=256, wr=0,
              sinks=8, train=True),
        # a training step on one long locus with a wide window
        _attn("window_train_1x9000", "9000", wl=1024, wr=1024, sinks=64, train=True),
        # inference on one gene with the learned bias
        _attn("buckets_gene_777", "777", pos="buckets"),
        # training on short genes with the learned bias: most blocks lie near the diagonal
        _attn("buckets_train_16x512", ",".join(["512"] * 16), pos="buckets", train=True),
        # training on two whole windows with the learned bias
        _attn("buckets_train_2x4550", "4550,4550", pos="buckets", train=True),
        # the encoder's training batch: eight packed windows, ALiBi, every key visible
        _attn("alibi_train_8x4550", ",".join(["4550"] * 8), pos="alibi", train=True),
        # a training micro-step with dropout on the attention's probabilities
        _attn("dropout_train_4x1100", "1100,1100,1100,1100", pos="alibi", p=0.1, train=True),
        # all of it together on packed sequences of mixed length
        _attn("local_train_packed", "2750,1333,4097,1024,1820", wl=384, wr=384, sinks=16,
              pos="buckets", p=0.1, train=True),
        # the residual add of one gene in fp32
        dict(name="residual_gene_777", kind="residual", n=777, d=768, dtype="f32", p=0.1,
             alpha=1.0),
        # the residual add of a packed training batch (the second layer's depth scaling)
        dict(name="residual_packed_36400", kind="residual", n=36400, d=768, dtype="bf16", p=0.1,
             alpha=1.0 / math.sqrt(2.0)),
    ]


# the pairs (key, query) of all heads that the largest listed case computes
_MOST_PAIRS = 12 * 8 * 4550 * 4550


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.2:
        return dict(kind="residual", n=_log_int(rng, 48, 36400),
                    d=rng.choice([128, 256, 512, 768, 768, 770, 127]),
                    dtype=rng.choice(["bf16", "bf16", "f32"]), p=rng.choice([0.05, 0.1, 0.3]),
                    alpha=rng.choice([1.0, 1.0 / math.sqrt(rng.randint(2, 12))]))
    op = rng.choice(["window", "window", "buckets", "dropout", "all", "alibi"])
    H, Hkv = rng.choice([(12, 12), (12, 12), (12, 4), (8, 1), (4, 2)])
    top = _log_int(rng, 33, 9000)
    lens = [rng.randint(max(1, top // 3), top) for _ in range(rng.randint(1, 8))]
    if op in ("dropout", "all"):
        lens = [min(n, 3000) for n in lens]
    while H * sum(n * n for n in lens) > _MOST_PAIRS:
        lens.pop()
    wl = wr = -1
    sinks = 0
    if op in ("window", "all"):
        wl, wr = rng.choice([(1, 1), (1, 1), (1, 0), (0, 1), (1, -1), (-1, 0)])
        wl, wr = (w * _log_int(rng, 16, 2048) if w > 0 else w for w in (wl, wr))
        sinks = rng.choice([0, 1, 4, 16, 64, 100])
    pos = {"window": rng.choice(["none", "alibi"]), "buckets": "buckets", "all": "buckets",
           "dropout": rng.choice(["none", "alibi"]), "alibi": "alibi"}[op]
    buckets, far = rng.choice([(32, 128), (32, 128), (16, 64), (64, 512), (8, 20), (32, 1000)])
    return _attn(None, ",".join(map(str, lens)), H, Hkv, wl, wr, sinks, pos, buckets, far,
                 rng.choice([0.05, 0.1, 0.25]) if op in ("dropout", "all") else 0.0,
                 rng.random() < 0.7)


# ---- inputs ---------------------------------------------------------------------------------

def _lens(case):
    return [int(v) for v in case["lens"].split(",")]


def _slopes(n):
    """ALiBi's head slopes (Press et al., 2022)."""
    def pow2(m):
        return [2.0 ** (-8.0 * (i + 1) / m) for i in range(m)]
    m = 1 << (n.bit_length() - 1)
    return pow2(m) if m == n else pow2(m) + pow2(2 * m)[0::2][: n - m]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    st = dict(case=case, seed=(int(seed) * 0x9E3779B97F4A7C15 + 1) & ((1 << 62) - 1))
    if case["kind"] == "residual":
        dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        shape = (case["n"], case["d"])
        st.update(x=randn(*shape, dtype=dt).requires_grad_(True),
                  residual=randn(*shape, dtype=dt).requires_grad_(True),
                  dout=randn(*shape, dtype=dt))
        return st
    lens = _lens(case)
    T, H, Hkv, train = sum(lens), case["H"], case["Hkv"], case["train"]
    st["q"] = randn(T, H, 64).requires_grad_(train)
    st["k"] = randn(T, Hkv, 64).requires_grad_(train)
    st["v"] = randn(T, Hkv, 64).requires_grad_(train)
    st["dout"] = randn(T, H, 64) if train else None
    st["cu"] = torch.tensor(np.cumsum([0] + lens), device=DEV, dtype=torch.int32)
    st["lens"] = lens
    st["slopes"] = (torch.tensor(_slopes(H), device=DEV, dtype=torch.float32)
                    if case["pos"] == "alibi" else None)
    st["table"] = (randn(case["buckets"], H).requires_grad_(train)
                   if case["pos"] == "buckets" else None)
    return st


# ---- the framework's operators --------------------------------------------------------------

def _run_own(st):
    c = st["case"]
    if c["kind"] == "residual":
        from genet5_amd import residual
        out = residual.dropout_add(st["x"], st["residual"], c["p"], alpha=c["alpha"],
                                   seed=st["seed"])
        dx, dres = torch.autograd.grad(out, (st["x"], st["residual"]), st["dout"])
        return dict(out=out.detach(), dx=dx, dresidual=dres)
    from genet5_amd import attention
    top = max(st["lens"])
    with torch.set_grad_enabled(c["train"]):
        out = attention.flash_attn_varlen_func(
            st["q"], st["k"], st["v"], st["cu"], st["cu"], top, top, dropout_p=c["p"],
            softmax_scale=SCALE, window_size=(c["wl"], c["wr"]), alibi_slopes=st["slopes"],
            sink_tokens=c["sinks"], relative_bias=st["table"], max_distance=c["far"],
            dropout_seed=st["seed"])
    if not c["train"]:
        return dict(out=out)
    names = ["q", "k", "v"] + (["table"] if st["table"] is not None else [])
    grads = torch.autograd.grad(out, [st[n] for n in names], st["dout"])
    return dict(out=out.detach(), **{"d" + n: g for n, g in zip(names, grads)})


# ---- the plain form -------------------------------------------------------------------------

def _bucket_starts(buckets, far):
    """The smallest distance of each of a side's buckets after the first, in whole numbers: among
    the side's `half` buckets the first e = half / 2 hold one distance each; bucket e + s starts at
    the smallest n with (n / e)^(half - e) >= (far / e)^s."""
    half = buckets // 2
    e = half // 2
    starts = list(range(1, e + 1))
    for s in range(1, half - e):
        n = int(e * (far / e) ** (s / (half - e))) - 1
        while n ** (half - e) * e ** s < far ** s * e ** (half - e):
            n += 1
        starts.append(n)
    return starts


def _bucket_table(L, buckets, far):
    """Bucket of each distance j - i from -(L - 1) to L - 1."""
    rel = torch.arange(-(L - 1), L, device=DEV)
    starts = torch.tensor(_bucket_starts(buckets, far), device=DEV)
    side = (rel.abs()[:, None] >= starts).sum(1)
    return torch.where(rel > 0, side + buckets // 2, side)


def _mix(x):
    """The 32-bit finaliser of MurmurHash3 on int64 tensors that hold 32-bit words."""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & M32
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & M32
    return x ^ (x >> 16)


def _kept(rows, cols, seed, p):
    """(keep mask [*rows, cols], scale): row r's key is mix(mix(r ^ low) + high) of the seed's two
    words; columns 2c and 2c + 1 take the low and the high half of mix(key + c golden)."""
    thr = int(p * 65536 + 0.5)
    key = _mix((_mix((rows & M32) ^ (seed & M32)) + (seed >> 32)) & M32)
    c = torch.arange((cols + 1) // 2, device=rows.device, dtype=torch.int64)
    bits = _mix((key.unsqueeze(-1) + c * 0x9E3779B9) & M32)
    r = torch.stack((bits & 0xFFFF, bits >> 16), dim=-1).flatten(-2)[..., :cols]
    return r >= thr, 65536.0 / (65536 - thr)


def _plain_sequence(st, a, b, h0, h1, out, grads):
    """One sequence (tokens a to b), query heads h0 to h1 (the same number for each key head)."""
    c = st["case"]
    L, n = b - a, h1 - h0
    rep = c["H"] // c["Hkv"]
    kv = [h // rep for h in range(h0, h1)]
    q = st["q"].detach()[a:b, h0:h1].float().transpose(0, 1).contiguous()
    k = st["k"].detach()[a:b, kv].float().transpose(0, 1).contiguous()
    v = st["v"].detach()[a:b, kv].float().transpose(0, 1).contiguous()
    pos = torch.arange(L, device=DEV)
    rel = pos[None, :] - pos[:, None]
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) * SCALE
    if st["slopes"] is not None:
        s -= st["slopes"][h0:h1, None, None] * rel.abs()
    if st["table"] is not None:
        lut = _bucket_table(L, c["buckets"], c["far"])
        s += st["table"].detach()[:, h0:h1].float().t()[:, lut[rel + L - 1]]
    if c["wl"] >= 0 or c["wr"] >= 0:
        seen = torch.ones_like(rel, dtype=torch.bool)
        if c["wl"] >= 0:
            seen &= rel >= -c["wl"]
        if c["wr"] >= 0:
            seen &= rel <= c["wr"]
        seen |= pos[None, :] < c["sinks"]
        s.masked_fill_(~seen, -math.inf)
    s -= s.amax(-1, keepdim=True)
    prob = s.exp_()
    prob /= prob.sum(-1, keepdim=True)
    dropped = prob
    if c["p"] > 0:
        rows = (a + pos)[None, :] * c["H"] + torch.arange(h0, h1, device=DEV)[:, None]
        keep, up = _kept(rows, L, st["seed"], c["p"])
        mult = keep.float() * up
        dropped = prob * mult
    out[a:b, h0:h1] = torch.bmm(dropped, v).transpose(0, 1).to(out.dtype)
    if grads is None:
        return
    do = st["dout"][a:b, h0:h1].float().transpose(0, 1).contiguous()
    grads["v"][a:b] += torch.zeros_like(grads["v"][a:b]).index_add_(
        1, torch.tensor(kv, device=DEV),
        torch.bmm(dropped.transpose(1, 2).contiguous(), do).transpose(0, 1))
    ds = torch.bmm(do, v.transpose(1, 2).contiguous())
    if c["p"] > 0:
        ds *= mult
    ds -= (ds * prob).sum(-1, keepdim=True)
    ds *= prob
    grads["q"][a:b, h0:h1] = torch.bmm(ds, k).transpose(0, 1) * SCALE
    grads["k"][a:b] += torch.zeros_like(grads["k"][a:b]).index_add_(
        1, torch.tensor(kv, device=DEV),
        torch.bmm(ds.transpose(1, 2).contiguous(), q).transpose(0, 1) * SCALE)
    if st["table"] is not None:
        # sums along the diagonals: rows flipped, each shifted by one more column
        diag = F.pad(ds.flip(1), (0, L)).flatten(1)[:, : L * (2 * L - 1)]
        diag = diag.view(n, L, 2 * L - 1).sum(1, dtype=torch.float64)
        grads["table"][:, h0:h1].index_add_(0, lut, diag.t().contiguous())


def _run_plain(st):
    c = st["case"]
    if c["kind"] == "residual":
        x, r, do = (st[n].detach().float() for n in ("x", "residual", "dout"))
        keep, up = _kept(torch.arange(c["n"], device=DEV), c["d"], st["seed"], c["p"])
        m = keep.float() * (up * c["alpha"])
        dt = st["x"].dtype
        return dict(out=(r + x * m).to(dt), dx=(do * m).to(dt), dresidual=do.to(dt))
    T, H, Hkv = st["q"].shape[0], c["H"], c["Hkv"]
    out = torch.empty(T, H, 64, dtype=torch.bfloat16, device=DEV)
    grads = None
    if c["train"]:
        grads = dict(q=torch.zeros(T, H, 64, device=DEV), k=torch.zeros(T, Hkv, 64, device=DEV),
                     v=torch.zeros(T, Hkv, 64, device=DEV))
        if st["table"] is not None:
            grads["table"] = torch.zeros(c["buckets"], H, device=DEV, dtype=torch.float64)
    a = 0
    for L in st["lens"]:
        step = max(1, min(H, (1 << 28) // (L * L)))
        for h0 in range(0, H, step):
            _plain_sequence(st, a, a + L, h0, min(H, h0 + step), out, grads)
        a += L
    if grads is None:
        return dict(out=out)
    return dict(out=out, **{"d" + n: g.to(torch.bfloat16) for n, g in grads.items()})


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- work -----------------------------------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    for L in _lens(case):
        i = np.arange(L)
        lo = np.maximum(i - case["wl"], 0) if case["wl"] >= 0 else np.zeros(L, int)
        hi = np.minimum(i + case["wr"], L - 1) if case["wr"] >= 0 else np.full(L, L - 1)
        total += int((hi - lo + 1 + np.minimum(lo, min(case["sinks"], L))).sum())
        total += int(np.maximum(min(case["sinks"], L) - 1 - hi, 0).sum())
    return total


def work(case):
    if case["kind"] == "residual":
        e = case["n"] * case["d"] * (2 if case["dtype"] == "bf16" else 4)
        return dict(bytes=5 * e, flops=5 * case["n"] * case["d"])
    T, H, Hkv = sum(_lens(case)), case["H"], case["Hkv"]
    q, kv = T * H * 128, T * Hkv * 128
    table = case["buckets"] * H * 4 if case["pos"] == "buckets" else 0
    pairs = _pairs(case) * H
    if not case["train"]:
        return dict(bytes=2 * q + 2 * kv + table, flops=4 * 64 * pairs)
    return dict(bytes=4 * q + 4 * kv + 2 * table, flops=14 * 64 * pairs)


# ---- the definition in 64 bits --------------------------------------------------------------

def _words(rows, cols, seed):
    """The generator on the host in 32-bit words: 16 bits for each column of each row."""
    def fin(x):
        for shift, mul in ((16, 0x85EBCA6B), (13, 0xC2B2AE35)):
            x = (x ^ (x >> np.uint32(shift))) * np.uint32(mul)
        return x ^ (x >> np.uint32(16))
    key = fin(fin(rows.astype(np.uint32) ^ np.uint32(seed & M32)) + np.uint32(seed >> 32))
    step = np.arange((cols + 1) // 2, dtype=np.uint32) * np.uint32(0x9E3779B9)
    w = fin(key[:, None] + step[None, :])
    both = np.empty((len(rows), 2 * w.shape[1]), dtype=np.uint16)
    both[:, 0::2] = w
    both[:, 1::2] = w >> np.uint32(16)
    return both[:, :cols]


def _far_bucket(n, half, far):
    """Bucket of distance n on one side, by logarithms with an integer check of the border."""
    e = half // 2
    if n < e:
        return n
    s = int(math.log(n / e) / math.log(far / e) * (half - e) + 0.5)
    while s > 0 and (n ** (half - e)) * e ** s < far ** s * e ** (half - e):
        s -= 1
    return min(half - 1, e + s)


def exact(case, seed):
    st = prepare(case, seed)
    with np.errstate(over="ignore"):
        if case["kind"] == "residual":
            if case["n"] * case["d"] > 1 << 28:
                return None
            thr = round(case["p"] * 65536)
            w = _words(np.arange(case["n"]), case["d"], st["seed"])
            m = torch.from_numpy(w >= thr).to(DEV).double() * (65536 / (65536 - thr)
                                                               * case["alpha"])
            x, r, do = (st[n].detach().double() for n in ("x", "residual", "dout"))
            return dict(out=r + m * x, dx=m * do, dresidual=do)
        if case["p"] > 0 and case["H"] * sum(n * n for n in _lens(case)) > 1 << 29:
            return None
        return _exact_attn(case, st)


def _exact_attn(case, st):
    H, rep = case["H"], case["H"] // case["Hkv"]
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    dtab = torch.zeros(case["buckets"], H, dtype=torch.float64, device=DEV)
    thr = round(case["p"] * 65536)
    half = case["buckets"] // 2
    start = 0
    for L in _lens(case):
        sl = slice(start, start + L)
        i = torch.arange(L, device=DEV)[:, None]
        j = torch.arange(L, device=DEV)[None, :]
        hidden = torch.zeros(L, L, dtype=torch.bool, device=DEV)
        if case["wl"] >= 0:
            hidden |= j < i - case["wl"]
        if case["wr"] >= 0:
            hidden |= j > i + case["wr"]
        hidden &= j >= case["sinks"]
        dist = (j - i).abs()
        if case["pos"] == "buckets":
            side = torch.tensor([_far_bucket(n, half, case["far"]) for n in range(L)], device=DEV)
            which = side[dist] + half * (j > i)
        for h in range(H):
            g = h // rep
            qh, kh, vh = (t.contiguous() for t in (q[sl, h], k[sl, g], v[sl, g]))
            t = qh @ kh.t().contiguous() / 8
            if case["pos"] == "alibi":
                t = t - float(st["slopes"][h]) * dist
            elif case["pos"] == "buckets":
                t = t + st["table"].detach()[:, h].double()[which]
            p = torch.softmax(t.masked_fill(hidden, -math.inf), dim=1)
            del t
            m = 1.0
            if case["p"] > 0:
                rows = (start + np.arange(L)) * H + h
                m = torch.from_numpy(_words(rows, L, st["seed"]) >= thr).to(DEV) * (
                    65536 / (65536 - thr))
            out[sl, h] = (p * m) @ vh
            if not case["train"]:
                continue
            do = st["dout"][sl, h].double()
            dv[sl, g] += (p * m).t().contiguous() @ do
            ds = (do @ vh.t().contiguous()) * m
            ds = p * (ds - (do * out[sl, h]).sum(1, keepdim=True))
            dq[sl, h] = ds @ kh / 8
            dk[sl, g] += ds.t().contiguous() @ qh / 8
            if case["pos"] == "buckets":
                for b in range(case["buckets"]):
                    dtab[b, h] += torch.where(which == b, ds, 0.0).sum()
        start += L
    if not case["train"]:
        return dict(out=out)
    res = dict(out=out, dq=dq, dk=dk, dv=dv)
    if case["pos"] == "buckets":
        res["dtable"] = dtab
    return res
