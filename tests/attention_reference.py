"""The attention with window, sinks, bucketed position bias and dropout in 64 bits, with its
gradients, and element by element how far a computation in bf16 and fp32 may be from them.

Roundings counted (u = 2^-8, half a step of bf16; SLACK for everything kept in fp32):
  P enters the output product as bf16:    u sum_j |m P v|
  out is rounded once:                    u |out|
  delta = dO . out is formed from that out, so it is off by at most sum_d |dO_d| err(out_d)
  P enters the value gradient as bf16:    u sum_i |m P dO|
  dS carries delta's error times P, and enters the products as bf16: u |dS|
  each gradient is rounded once to its type
SLACK: a score of 64 products summed in fp32 is off by at most 64 2^-24 sum |q_d k_d| scale,
which for the sizes used here (sum |q_d k_d| scale < 25) is below 1e-4, and a probability by
that factor; the sums of up to 2^11 terms add 2^11 2^-24 = 1.2e-4 at most.  2.5e-4 covers both.
"""
import math

import numpy as np
import torch

U = 2.0 ** -8
SLACK = 2.5e-4


def fmix32(x):
    x = x ^ (x >> np.uint32(16))
    x = x * np.uint32(0x85EBCA6B)
    x = x ^ (x >> np.uint32(13))
    x = x * np.uint32(0xC2B2AE35)
    return x ^ (x >> np.uint32(16))


def keep_mask(rows, cols, seed, p):
    """(bool [len(rows), cols], scale) of g5moe_dropout."""
    with np.errstate(over="ignore"):
        rows = np.asarray(rows, dtype=np.uint64).astype(np.uint32)
        key = fmix32(fmix32(rows ^ np.uint32(seed & 0xFFFFFFFF)) + np.uint32(seed >> 32))
        c = np.arange(cols, dtype=np.uint32)
        bits = fmix32(key[:, None] + (c >> np.uint32(1)) * np.uint32(0x9E3779B9))
    r = np.where(c & 1, bits >> np.uint32(16), bits & np.uint32(0xFFFF))
    thr = min(65536, int(math.floor(p * 65536 + 0.5)))
    return r >= thr, (65536.0 / (65536 - thr) if thr < 65536 else 0.0)


def bucket(rel, num_buckets, max_distance):
    """The bucket of key - query position, one number at a time, in whole numbers."""
    half = num_buckets // 2
    e = half // 2
    n = min(abs(rel), max_distance)
    b = n
    if n >= e:
        b = e
        while b + 1 < half and (n ** (half - e) * e ** (b + 1 - e)
                                >= max_distance ** (b + 1 - e) * e ** (half - e)):
            b += 1
    return b + half if rel > 0 else b


def visible(L, window, sinks):
    i, j = np.arange(L)[:, None], np.arange(L)[None, :]
    wl, wr = window
    seen = np.ones((L, L), dtype=bool)
    if wl >= 0:
        seen &= j >= i - wl
    if wr >= 0:
        seen &= j <= i + wr
    return torch.from_numpy(seen | (j < sinks))


def attention(q, k, v, cu, scale, dout=None, window=(-1, -1), sinks=0, slopes=None, table=None,
              max_distance=128, p=0.0, seed=0):
    """dict of out, lse and, with dout, dq, dk, dv (and dtable), each with its bound under
    "<name>_tol".  Tensors of any float type on any device, results in float64 on the CPU."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    T, H, D = q.shape
    Hkv = k.shape[1]
    rep = H // Hkv
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)
    r = dict(out=z(T, H, D), out_tol=z(T, H, D), lse=z(H, T))
    if dout is not None:
        dout = dout.detach().double().cpu()
        for n, h in (("dq", H), ("dk", Hkv), ("dv", Hkv)):
            r[n], r[n + "_tol"] = z(T, h, D), z(T, h, D)
        if table is not None:
            r["dtable"], r["dtable_tol"] = z(*table.shape), z(*table.shape)
    for a, b in zip(cu[:-1], cu[1:]):
        L = b - a
        if L <= 0:
            continue
        seen = visible(L, window, sinks)
        rel = torch.arange(L)[None, :] - torch.arange(L)[:, None]
        if table is not None:
            lut = torch.tensor([bucket(n, table.shape[0], max_distance)
                                for n in range(-(L - 1), L)])
            which = lut[rel + L - 1]
        for h in range(H):
            g = h // rep
            qh, kh, vh = q[a:b, h], k[a:b, g], v[a:b, g]
            t = qh @ kh.T * scale
            if slopes is not None:
                t = t - float(slopes[h]) * rel.abs().double()
            if table is not None:
                t = t + table.detach().double().cpu()[which, h]
            t = t.masked_fill(~seen, -math.inf)
            m = t.amax(1, keepdim=True)
            m = torch.where(m == -math.inf, torch.zeros_like(m), m)
            e = torch.exp(t - m)
            s = e.sum(1, keepdim=True)
            P = torch.where(s > 0, e / s.clamp_min(1e-300), torch.zeros_like(e))
            r["lse"][h, a:b] = torch.where(s > 0, m + torch.log(s), -math.inf)[:, 0]
            mult = torch.ones((), dtype=torch.float64)
            if p > 0:
                keep, up = keep_mask((a + np.arange(L)) * H + h, L, seed, p)
                mult = torch.from_numpy(keep).double() * up
            Pm = P * mult
            out = Pm @ vh
            err = U * out.abs() + (U + SLACK) * (Pm @ vh.abs())
            r["out"][a:b, h], r["out_tol"][a:b, h] = out, err
            if dout is None:
                continue
            do = dout[a:b, h]
            derr = (do.abs() * err).sum(1, keepdim=True)
            dP = (do @ vh.T) * mult
            delta = (do * out).sum(1, keepdim=True)
            dS = P * (dP - delta)
            size = P * ((do.abs() @ vh.abs().T) * mult + (do.abs() * out.abs()).sum(1, keepdim=True))
            eS = P * derr + SLACK * size           # of dS in fp32
            eB = eS + U * (dS.abs() + eS)          # of dS in bf16
            r["dv"][a:b, g] += Pm.T @ do
            r["dv_tol"][a:b, g] += (U + SLACK) * (Pm.T @ do.abs())
            r["dq"][a:b, h] = dS @ kh * scale
            r["dq_tol"][a:b, h] = eB @ kh.abs() * abs(scale)
            r["dk"][a:b, g] += dS.T @ qh * scale
            r["dk_tol"][a:b, g] += eB.T @ qh.abs() * abs(scale)
            if table is not None:
                for x in range(table.shape[0]):
                    at = which == x
                    r["dtable"][x, h] += dS[at].sum()
                    r["dtable_tol"][x, h] += eS[at].sum() + SLACK * dS[at].abs().sum()
    for n in ("dq", "dk", "dv"):
        if n in r:
            r[n + "_tol"] += U * (r[n].abs() + r[n + "_tol"]) + 1e-30
    if "dtable" in r and table.dtype == torch.bfloat16:
        r["dtable_tol"] += U * (r["dtable"].abs() + r["dtable_tol"])
    return r


def check(got, ref, name, what=""):
    """Every element of got within its bound of ref[name]."""
    g = got.detach().double().cpu()
    over = (g - ref[name]).abs() - ref[name + "_tol"]
    worst = ((g - ref[name]).abs() / (ref[name + "_tol"] + 1e-30)).max().item() if g.numel() else 0
    print(f"  {what} {name}: largest error {worst:.3f} of its bound", flush=True)
    assert not torch.isnan(g).any(), (what, name, "NaN")
    assert over.max().item() <= 0 if g.numel() else True, (what, name, worst)
