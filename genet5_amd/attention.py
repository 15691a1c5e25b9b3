"""Varlen bidirectional attention on the HIP kernels of libg5moe.so: ALiBi or a learned
bucketed position bias, a sliding window with sink tokens, dropout, and the backward.

Reference interface: GeneT5's FlashAttention (lib/blocks/_flash_att.py:15-98)
calls flash-attn's

    flash_attn_varlen_func(q, k, v, cu_seqlens_q=cu, cu_seqlens_k=cu,
                           max_seqlen_q=L, max_seqlen_k=L, dropout_p=p,
                           softmax_scale=1/sqrt(head_dim), causal=False)   (:76-88)
    flash_attn_func(q, k, v, dropout_p=p, softmax_scale=..., causal=False)  (:90-96)

with q [total, H, D] (varlen) or [B, L, H, D], GQA through fewer key/value
heads (:49-58).  This module keeps those two functions' signatures (and
flash-attn's `alibi_slopes` argument: bias[h, i, j] = -slope_h * |i - j| on
sequence-local positions) and a `FlashAttention`-shaped module whose
`forward(hidden_states, cu_seqlens=None, max_seqlen=None)` returns
`(out, None)` like the reference's.

Beyond flash-attn's arguments: `sink_tokens` (first tokens of each sequence that stay
visible outside the window), `relative_bias` with `max_distance` (a learned bias
[num_buckets, heads] over bucketed relative positions) and `dropout_seed`.

Supported: bf16, head_dim 64, self-attention, forward and backward.  Anything else
raises; there is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn as nn

from . import _lib, ops
from .ops import _check_device, _ptr, _stream

HEAD_DIM = 64


def alibi_slopes(n_heads: int) -> List[float]:
    """Head slopes of Press et al. (2022), "Train Short, Test Long": a geometric
    sequence starting at 2^(-8/n) for n a power of two; otherwise the slopes of
    the nearest lower power of two followed by every other slope of twice that
    count."""
    def pow2(n):
        start = 2.0 ** (-8.0 / n)
        return [start ** (i + 1) for i in range(n)]
    if n_heads & (n_heads - 1) == 0:
        return pow2(n_heads)
    m = 1 << int(math.floor(math.log2(n_heads)))
    return pow2(m) + pow2(2 * m)[0::2][: n_heads - m]


def _check_qkv(t: torch.Tensor, name: str, total: int, heads: int, dev: torch.device) -> None:
    if t.device == dev and t.dtype == torch.bfloat16 and t.shape == (total, heads, HEAD_DIM):
        st = t.stride()
        if st[2] == 1 and st[0] % 8 == 0 and st[1] % 8 == 0 and st[0] >= 0 and st[1] >= 0 \
                and t.data_ptr() % 16 == 0:
            return
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} has dtype {t.dtype}; the attention kernel takes bfloat16")
    if t.dim() != 3 or tuple(t.shape) != (total, heads, HEAD_DIM):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({total}, {heads}, "
                         f"{HEAD_DIM})")
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.stride(0) < 0 \
            or t.stride(1) < 0:
        raise ValueError(f"{name}: head dims must be contiguous and the token/head strides "
                         f"multiples of 8 elements (strides {t.stride()})")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")


def attn_varlen_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    cu_seqlens: torch.Tensor, max_seqlen: int, softmax_scale: float,
                    alibi_slopes: Optional[torch.Tensor] = None, return_lse: bool = False,
                    key_bounds: bool = True):
    """g5moe_attn_varlen_fwd on the current stream.  q [T, H, 64], k/v [T, Hkv, 64]
    bf16 (head dims contiguous, other strides free); cu_seqlens int32 [n + 1] on
    the GPU; alibi_slopes fp32 [H] or None.  Returns out [T, H, 64] (and the
    natural-log softmax_lse [H, T] fp32 when return_lse).

    key_bounds: give the kernel a workspace for per-64-key-block norm maxima (one
    pre-pass over k).  With them it (a) leaves out, under ALiBi, the key blocks whose
    probabilities are provably below 2^-64 of each row's largest (a key-norm bound
    against the ALiBi distance), and (b) uses a fixed per-query reference maximum
    instead of the online running maximum where the bounds keep every score term
    within 32 of zero (base 2).  The result equals the plain online computation over
    every block (key_bounds=False) to fp32 rounding of the probabilities.  Calls without
    alibi_slopes and with max_seqlen <= 2,048 leave the pre-pass out (nothing to skip, and
    it costs about what the other loop gains)."""
    dev = _check_device(q)
    T, H = q.shape[0], q.shape[1]
    Hkv = k.shape[1] if k.dim() == 3 else -1
    _check_qkv(q, "q", T, H, dev)
    _check_qkv(k, "k", T, Hkv, dev)
    _check_qkv(v, "v", T, Hkv, dev)
    if H % Hkv:
        raise ValueError(f"key/value heads {Hkv} must divide query heads {H}")
    if cu_seqlens.device != dev or cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 \
            or cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous int32 vector [n_seqs + 1] on "
                         f"{dev}")
    if alibi_slopes is not None:
        if alibi_slopes.device != dev or alibi_slopes.dtype != torch.float32 \
                or tuple(alibi_slopes.shape) != (H,) or not alibi_slopes.is_contiguous():
            raise ValueError(f"alibi_slopes must be a contiguous float32 [{H}] tensor on {dev}")
    # ops.ROW_PAD rows of slack after the output, so that the output projection's
    # grouped GEMM (ops.linear) reads it in place
    out = torch.empty((T + ops.ROW_PAD, H, HEAD_DIM), dtype=torch.bfloat16, device=dev)[:T]
    lse = torch.empty((H, T), dtype=torch.float32, device=dev) if return_lse else None
    shape = _lib.AttnShape(
        cu_seqlens.numel() - 1, int(max_seqlen), T, H, Hkv, HEAD_DIM, 0,
        q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        out.stride(0), out.stride(1))
    ws = None
    if key_bounds:
        ws = torch.empty(_lib.attn_workspace_size(T, H, Hkv, HEAD_DIM), dtype=torch.uint8,
                         device=dev)
    _lib.call("g5moe_attn_varlen_fwd", _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(cu_seqlens),
              _ptr(alibi_slopes), ctypes.c_float(softmax_scale), _ptr(lse), _ptr(ws),
              ctypes.byref(shape), _stream(dev))
    return (out, lse) if return_lse else out


@torch.library.custom_op("g5moe::attn_varlen_fwd", mutates_args=())
def _attn_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
             max_seqlen: int, softmax_scale: float, alibi_slopes: Optional[torch.Tensor],
             return_lse: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, softmax_lse [H, T]) with return_lse, else (out, an empty [0] tensor): the
    kernel keeps the fp32 row sums lse needs only when it is asked for."""
    if return_lse:
        return attn_varlen_fwd(q, k, v, cu_seqlens, max_seqlen, softmax_scale, alibi_slopes,
                               return_lse=True)
    out = attn_varlen_fwd(q, k, v, cu_seqlens, max_seqlen, softmax_scale, alibi_slopes)
    return out, out.new_empty((0,), dtype=torch.float32)


@_attn_op.register_fake
def _(q, k, v, cu_seqlens, max_seqlen, softmax_scale, alibi_slopes, return_lse):
    T, H, D = q.shape
    lse_shape = (H, T) if return_lse else (0,)
    return q.new_empty((T, H, D)), q.new_empty(lse_shape, dtype=torch.float32)


def _no_backward(ctx, *grads):
    raise NotImplementedError("g5moe::attn_varlen_fwd has no backward (inference kernel)")


_attn_op.register_autograd(_no_backward)


# ---- window, sinks, bucketed position bias, dropout, backward -------------------------

MAX_BIAS_DISTANCE = 1024
_INT32_MAX = 2 ** 31 - 1


@functools.lru_cache(maxsize=64)
def _bucket_starts(num_buckets: int, max_distance: int) -> Tuple[int, ...]:
    """The smallest distance of each bucket of one side after the first, in whole numbers.
    Of a side's half = num_buckets / 2 buckets the first e = half / 2 hold one distance
    each; bucket e + s starts at the smallest n with (n / e)^(half - e) >= (D / e)^s, i.e.
    log(n / e) / log(D / e) (half - e) >= s without rounding."""
    half = num_buckets // 2
    e = half // 2
    starts = list(range(1, e + 1))
    for s in range(1, half - e):
        lo, hi = starts[-1], max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid ** (half - e) * e ** s >= max_distance ** s * e ** (half - e):
                hi = mid
            else:
                lo = mid + 1
        starts.append(lo)
    return tuple(starts)


def _check_buckets(num_buckets: int, max_distance: int) -> None:
    if num_buckets < 4 or num_buckets % 2:
        raise ValueError(f"num_buckets {num_buckets} must be even and at least 4 (half of them "
                         "for keys after the query)")
    if not num_buckets // 4 < max_distance <= MAX_BIAS_DISTANCE:
        raise ValueError(f"max_distance {max_distance} must exceed num_buckets / 4 = "
                         f"{num_buckets // 4} and be at most {MAX_BIAS_DISTANCE}")


def relative_buckets(num_buckets: int, max_distance: int,
                     device: Optional[torch.device] = None) -> torch.Tensor:
    """int32 [2 * max_distance + 1]: the bucket of each relative position r = key - query
    from -max_distance to max_distance; positions farther away share the ends' buckets.
    Keys after the query (r > 0) use the upper half of the buckets.  With half =
    num_buckets / 2 and e = half / 2, distances below e have a bucket each, distance n >= e
    is in bucket e + floor(log(n / e) / log(max_distance / e) (half - e)), half - 1 at most
    (exact at the borders, whatever a logarithm rounds to)."""
    _check_buckets(num_buckets, max_distance)
    starts = torch.tensor(_bucket_starts(num_buckets, max_distance))
    n = torch.arange(max_distance + 1)
    side = torch.searchsorted(starts, n, right=True)
    out = torch.cat([side.flip(0), side[1:] + num_buckets // 2])
    return out.to(torch.int32).to(device) if device is not None else out.to(torch.int32)


_BUCKETS: dict = {}


def _buckets_on(num_buckets: int, max_distance: int, device: torch.device) -> torch.Tensor:
    """relative_buckets on `device`, built once per device and pair of numbers and kept (a
    captured graph may read it from then on)."""
    key = (num_buckets, max_distance, device)
    t = _BUCKETS.get(key)
    if t is None:
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the bucket table of a relative bias is built by the first call "
                               "with its sizes: run one before capturing a graph")
        t = relative_buckets(num_buckets, max_distance, device)
        if device.type == "cuda":
            torch.cuda.current_stream(device).synchronize()  # used on any stream from now on
        _BUCKETS[key] = t
    return t


def _check_cu(cu_seqlens: torch.Tensor, dev: torch.device) -> None:
    if cu_seqlens.device != dev or cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 \
            or cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous int32 vector [n_seqs + 1] on "
                         f"{dev}")


def _options(window_left: int, window_right: int, sink_tokens: int, dropout_p: float, seed: int,
             bias: Optional[torch.Tensor], max_distance: int) -> _lib.AttnOptions:
    o = _lib.AttnOptions(window_left, window_right, sink_tokens, 0, 0, 0,
                         _lib.make_dropout(dropout_p, seed), 0)
    if bias is not None:
        o.bias_buckets = bias.shape[0]
        o.bias_distance = max_distance
        o.bias_dtype = ops._dtype_code(bias.dtype)
    return o


def _check_position(alibi_slopes: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                    max_distance: int, H: int, dev: torch.device) -> None:
    if alibi_slopes is not None:
        if alibi_slopes.device != dev or alibi_slopes.dtype != torch.float32 \
                or tuple(alibi_slopes.shape) != (H,) or not alibi_slopes.is_contiguous():
            raise ValueError(f"alibi_slopes must be a contiguous float32 [{H}] tensor on {dev}")
        if bias is not None:
            raise ValueError("alibi_slopes and relative_bias exclude each other")
    if bias is not None:
        if bias.device != dev:
            raise ValueError(f"relative_bias is on {bias.device}, expected {dev}")
        if bias.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"relative_bias has dtype {bias.dtype}; it must be bfloat16 or "
                            "float32")
        if bias.dim() != 2 or bias.shape[1] != H:
            raise ValueError(f"relative_bias has shape {tuple(bias.shape)}, expected "
                             f"(num_buckets, {H})")
        _check_buckets(bias.shape[0], max_distance)


def attn_local_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                   max_seqlen: int, softmax_scale: float,
                   alibi_slopes: Optional[torch.Tensor] = None,
                   relative_bias: Optional[torch.Tensor] = None, max_distance: int = 128,
                   window_size: Tuple[int, int] = (-1, -1), sink_tokens: int = 0,
                   dropout_p: float = 0.0, dropout_seed: int = 0, return_lse: bool = False,
                   for_backward: bool = False):
    """g5moe_attn_local_fwd on the current stream: attention over the visible keys with an
    optional position bias and dropout.  Tensors as attn_varlen_fwd takes them;
    relative_bias [num_buckets, H] bf16 or fp32.  Returns out [T, H, 64]; (out, softmax_lse
    [H, T] fp32) with return_lse; with for_backward (out, softmax_lse, out_low, key_norms),
    which attn_bwd takes.  Rows behind the last sequence are zeros in out."""
    dev = _check_device(q)
    T, H = q.shape[0], q.shape[1]
    Hkv = k.shape[1] if k.dim() == 3 else -1
    _check_qkv(q, "q", T, H, dev)
    _check_qkv(k, "k", T, Hkv, dev)
    _check_qkv(v, "v", T, Hkv, dev)
    if Hkv < 1 or H % Hkv:
        raise ValueError(f"key/value heads {Hkv} must divide query heads {H}")
    _check_cu(cu_seqlens, dev)
    _check_position(alibi_slopes, relative_bias, max_distance, H, dev)
    bias = None if relative_bias is None else relative_bias.contiguous()
    buckets = None if bias is None else _buckets_on(bias.shape[0], max_distance, dev)
    n_seqs, max_seqlen = cu_seqlens.numel() - 1, int(max_seqlen)
    empty = n_seqs == 0 or max_seqlen <= 0   # nothing is launched
    out = (torch.zeros if empty else torch.empty)((T + ops.ROW_PAD, H, HEAD_DIM),
                                                  dtype=torch.bfloat16, device=dev)[:T]
    lse = out_low = None
    if return_lse or for_backward:
        lse = torch.empty((H, T), dtype=torch.float32, device=dev)
    if for_backward:
        out_low = torch.empty((T, H, HEAD_DIM), dtype=torch.bfloat16, device=dev)
    shape = _lib.AttnShape(n_seqs, max_seqlen, T, H, Hkv, HEAD_DIM, 0, q.stride(0), q.stride(1),
                           k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0),
                           out.stride(1))
    opts = _options(*window_size, sink_tokens, dropout_p, dropout_seed, bias, max_distance)
    ws = None
    if alibi_slopes is not None or (bias is None and dropout_p == 0 and max(window_size) < 0):
        # for the key norms: ALiBi's reach, the bounds of long calls without any option
        ws = torch.empty(_lib.attn_workspace_size(T, H, Hkv, HEAD_DIM), dtype=torch.uint8,
                         device=dev)
    ops._call_on(dev, "g5moe_attn_local_fwd", _ptr(q), _ptr(k), _ptr(v), _ptr(out),
                 _ptr(cu_seqlens), _ptr(alibi_slopes), _ptr(bias), _ptr(buckets),
                 ctypes.c_float(softmax_scale), _ptr(lse), _ptr(out_low), _ptr(ws),
                 ctypes.byref(opts), ctypes.byref(shape), _stream(dev))
    if for_backward:
        return out, lse, out_low, ws if alibi_slopes is not None and not empty else None
    return (out, lse) if return_lse else out


def attn_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
             out: torch.Tensor, softmax_lse: torch.Tensor, cu_seqlens: torch.Tensor,
             max_seqlen: int, softmax_scale: float,
             alibi_slopes: Optional[torch.Tensor] = None,
             relative_bias: Optional[torch.Tensor] = None, max_distance: int = 128,
             window_size: Tuple[int, int] = (-1, -1), sink_tokens: int = 0,
             dropout_p: float = 0.0, dropout_seed: int = 0, bias_grad: bool = True,
             out_low: Optional[torch.Tensor] = None, key_norms: Optional[torch.Tensor] = None):
    """g5moe_attn_bwd on the current stream: (dq, dk, dv, d_relative_bias) of a forward with
    these arguments, from its out and softmax_lse; d_relative_bias is None without a table
    or with bias_grad = False.  out_low: the forward's (attn_local_fwd, for_backward), what the
    rounding of out left over, without which the gradients carry its error.  key_norms: the
    forward's, which the call would otherwise form again under ALiBi.  Rows behind the last
    sequence are zeros."""
    dev = _check_device(q)
    T, H = q.shape[0], q.shape[1]
    Hkv = k.shape[1] if k.dim() == 3 else -1
    _check_qkv(q, "q", T, H, dev)
    _check_qkv(k, "k", T, Hkv, dev)
    _check_qkv(v, "v", T, Hkv, dev)
    _check_qkv(out, "out", T, H, dev)
    _check_qkv(dout, "dout", T, H, dev)
    if Hkv < 1 or H % Hkv:
        raise ValueError(f"key/value heads {Hkv} must divide query heads {H}")
    _check_cu(cu_seqlens, dev)
    _check_position(alibi_slopes, relative_bias, max_distance, H, dev)
    ops._require(softmax_lse, "softmax_lse", (H, T), torch.float32, dev)
    if out_low is not None:
        ops._require(out_low, "out_low", (T, H, HEAD_DIM), torch.bfloat16, dev)
    if key_norms is not None and (
            key_norms.device != dev or key_norms.dtype != torch.uint8
            or key_norms.numel() < _lib.attn_workspace_size(T, H, Hkv, HEAD_DIM)):
        raise ValueError("key_norms must be what attn_local_fwd returned for this call")
    return _attn_bwd(dout, q, k, v, out, softmax_lse, out_low, cu_seqlens, alibi_slopes,
                     relative_bias, key_norms, (int(max_seqlen), softmax_scale, max_distance,
                                                *window_size, sink_tokens, dropout_p),
                     dropout_seed, bias_grad)


@functools.lru_cache(maxsize=256)
def _bwd_workspace_size(opts: tuple, dropout_p: float, sizes: tuple) -> int:
    o = _lib.AttnOptions(*opts[:6], _lib.make_dropout(dropout_p, 0), 0)
    s = _lib.AttnShape(*sizes)
    n = ctypes.c_size_t(0)
    _lib.call("g5moe_attn_bwd_workspace_size", ctypes.byref(o), ctypes.byref(s), ctypes.byref(n))
    return int(n.value)


def _attn_bwd(dout, q, k, v, out, softmax_lse, out_low, cu_seqlens, alibi_slopes, relative_bias,
              key_norms, call, dropout_seed, bias_grad):
    """attn_bwd on arguments that have been checked (saved by a forward)."""
    max_seqlen, softmax_scale, max_distance, wl, wr, sink_tokens, dropout_p = call
    dev = q.device
    T, H, Hkv = q.shape[0], q.shape[1], k.shape[1]
    bias = None if relative_bias is None else relative_bias.contiguous()
    buckets = None if bias is None else _buckets_on(bias.shape[0], max_distance, dev)
    n_seqs = cu_seqlens.numel() - 1
    empty = n_seqs == 0 or max_seqlen <= 0 or T == 0   # nothing is launched
    new = torch.zeros if empty else torch.empty
    dq, dk, dv = (new((T, h, HEAD_DIM), dtype=torch.bfloat16, device=dev) for h in (H, Hkv, Hkv))
    dbias = None
    if bias is not None and bias_grad:
        dbias = (torch.zeros_like if empty else torch.empty_like)(bias)
    if empty:
        return dq, dk, dv, dbias
    sizes = (n_seqs, max_seqlen, T, H, Hkv, HEAD_DIM, 0)
    shape = _lib.AttnShape(*sizes, *q.stride()[:2], *k.stride()[:2], *v.stride()[:2],
                           *out.stride()[:2])
    gshape = _lib.AttnShape(*sizes, *dq.stride()[:2], *dk.stride()[:2], *dv.stride()[:2],
                            *dout.stride()[:2])
    opts = _options(wl, wr, sink_tokens, dropout_p, dropout_seed, bias, max_distance)
    ws = torch.empty(_bwd_workspace_size(
        (wl, wr, sink_tokens, opts.bias_buckets, opts.bias_distance, opts.bias_dtype), dropout_p,
        sizes), dtype=torch.uint8, device=dev)
    ops._call_on(dev, "g5moe_attn_bwd", _ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out),
                 _ptr(out_low), _ptr(softmax_lse), _ptr(cu_seqlens), _ptr(alibi_slopes),
                 _ptr(bias), _ptr(buckets), ctypes.c_float(softmax_scale), _ptr(dq), _ptr(dk),
                 _ptr(dv), _ptr(dbias), _ptr(key_norms), _ptr(ws), ctypes.byref(opts),
                 ctypes.byref(shape), ctypes.byref(gshape), _stream(dev))
    return dq, dk, dv, dbias


def _draw_seed() -> int:
    """A dropout seed from torch's default CPU generator (torch.manual_seed reproduces it)."""
    return int(torch.randint(0, 2 ** 62, (1,)).item())


def _bwd_call(need_bias, dout, q, k, v, out, lse, low, cu, slopes, bias, norms, call, seed):
    """attn_bwd with dout brought into a form the kernel reads."""
    st = dout.stride()
    if dout.dtype != torch.bfloat16 or st[2] != 1 or st[0] % 8 or st[1] % 8 \
            or dout.data_ptr() % 16:
        dout = dout.to(torch.bfloat16).contiguous()
    return _attn_bwd(dout, q, k, v, out, lse, low, cu, slopes, bias, norms, call, seed, need_bias)


class _AttnFunction(torch.autograd.Function):
    """The differentiable attention of eager programs (a traced one records the custom op
    below, whose dispatch costs more host time per call)."""

    @staticmethod
    def forward(ctx, q, k, v, bias, cu, max_seqlen, scale, slopes, max_distance, wl, wr, sinks,
                p, seed):
        out, lse, low, norms = attn_local_fwd(q, k, v, cu, max_seqlen, scale, slopes, bias,
                                              max_distance, (wl, wr), sinks, p, seed,
                                              for_backward=True)
        ctx.save_for_backward(q, k, v, out, lse, low, cu, slopes, bias, norms)
        ctx.call = (max_seqlen, scale, max_distance, wl, wr, sinks, p)
        ctx.seed = seed
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @ops._once_differentiable
    def backward(ctx, dout, _dlse):
        none = (None,) * 14
        if dout is None:
            return none
        need = ctx.needs_input_grad
        grads = _bwd_call(need[3], dout, *ctx.saved_tensors, ctx.call, ctx.seed)
        return tuple(g if n else None for g, n in zip(grads, need)) + none[4:]


@torch.library.custom_op("g5moe::attn_local", mutates_args=())
def _attn_local_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                   max_seqlen: int, softmax_scale: float, alibi_slopes: Optional[torch.Tensor],
                   relative_bias: Optional[torch.Tensor], max_distance: int, window_left: int,
                   window_right: int, sink_tokens: int, dropout_p: float,
                   dropout_seed: Optional[int], for_backward: bool
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(out, softmax_lse [H, T], for_backward: out_low, else an empty tensor, the dropout seed
    as host int64 [1]).  With dropout and no seed the op draws one per call, so a compiled
    program draws anew each time."""
    seed = 0
    if dropout_p > 0:
        seed = _draw_seed() if dropout_seed is None else dropout_seed
    out, lse, *saved = attn_local_fwd(q, k, v, cu_seqlens, max_seqlen, softmax_scale,
                                      alibi_slopes, relative_bias, max_distance,
                                      (window_left, window_right), sink_tokens, dropout_p, seed,
                                      return_lse=True, for_backward=for_backward)
    low = saved[0] if for_backward else q.new_empty((0,))
    return out, lse, low, torch.tensor([seed], dtype=torch.int64)


@_attn_local_op.register_fake
def _(q, k, v, cu_seqlens, max_seqlen, softmax_scale, alibi_slopes, relative_bias, max_distance,
      window_left, window_right, sink_tokens, dropout_p, dropout_seed, for_backward):
    T, H, D = q.shape
    return (q.new_empty((T, H, D)), q.new_empty((H, T), dtype=torch.float32),
            q.new_empty((T, H, D) if for_backward else (0,)),
            torch.empty((1,), dtype=torch.int64, device="cpu"))


@torch.library.custom_op("g5moe::attn_local_backward", mutates_args=())
def _attn_local_bwd_op(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       out: torch.Tensor, lse: torch.Tensor, out_low: torch.Tensor,
                       cu_seqlens: torch.Tensor, max_seqlen: int, softmax_scale: float,
                       alibi_slopes: Optional[torch.Tensor],
                       relative_bias: Optional[torch.Tensor], max_distance: int,
                       window_left: int, window_right: int, sink_tokens: int, dropout_p: float,
                       seed: torch.Tensor, bias_grad: bool
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv, d_relative_bias or an empty tensor)."""
    dq, dk, dv, db = _bwd_call(bias_grad, dout, q, k, v, out, lse, out_low, cu_seqlens,
                               alibi_slopes, relative_bias, None,
                               (max_seqlen, softmax_scale, max_distance, window_left,
                                window_right, sink_tokens, dropout_p), int(seed[0]))
    return dq, dk, dv, q.new_empty((0,)) if db is None else db


@_attn_local_bwd_op.register_fake
def _(dout, q, k, v, out, lse, out_low, cu_seqlens, max_seqlen, softmax_scale, alibi_slopes,
      relative_bias, max_distance, window_left, window_right, sink_tokens, dropout_p, seed,
      bias_grad):
    grads = tuple(t.new_empty(t.shape) for t in (q, k, v))
    if relative_bias is None or not bias_grad:
        return grads + (q.new_empty((0,)),)
    return grads + (relative_bias.new_empty(relative_bias.shape),)


def _local_setup(ctx, inputs, output):
    (q, k, v, cu, max_seqlen, scale, slopes, bias, max_distance, wl, wr, sinks, p, _, _) = inputs
    out, lse, low, seed = output
    ctx.save_for_backward(q, k, v, out, lse, low, cu, slopes, bias, seed)
    ctx.call = (max_seqlen, scale, max_distance, wl, wr, sinks, p)
    ctx.mark_non_differentiable(lse, low, seed)
    ctx.set_materialize_grads(False)


def _local_backward(ctx, dout, _dlse, _dlow, _dseed):
    grads = [None] * 15
    if dout is not None:
        q, k, v, out, lse, low, cu, slopes, bias, seed = ctx.saved_tensors
        max_seqlen, scale, max_distance, wl, wr, sinks, p = ctx.call
        need = ctx.needs_input_grad
        dq, dk, dv, db = _attn_local_bwd_op(dout, q, k, v, out, lse, low, cu, max_seqlen,
                                            scale, slopes, bias, max_distance, wl, wr, sinks, p,
                                            seed, need[7])
        for i, g in ((0, dq), (1, dk), (2, dv), (7, db)):
            if need[i]:
                grads[i] = g
    return tuple(grads)


_attn_local_op.register_autograd(_local_backward, setup_context=_local_setup)


def _unsupported(causal, window_size):
    if causal:
        raise NotImplementedError("causal attention is not supported (GeneT5's encoder is "
                                  "bidirectional); window_size=(-1, 0) leaves out the keys "
                                  "after each query")
    if len(tuple(window_size)) != 2 or any(int(w) != w or w < -1 for w in window_size):
        raise ValueError(f"window_size {window_size!r} must be two integers >= -1 (-1: no limit "
                         "on that side)")


def flash_attn_varlen_func(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                           dropout_p=0.0, softmax_scale=None, causal=False,
                           window_size=(-1, -1), alibi_slopes=None, deterministic=False,
                           return_attn_probs=False, *, sink_tokens=0, relative_bias=None,
                           max_distance=128, dropout_seed=None):
    """flash-attn's varlen entry point over the HIP kernels (self-attention: the
    query and key segmentations must be the same).  Returns out [T, H, D], or
    (out, softmax_lse, None) with return_attn_probs.  Differentiable in q, k, v and
    relative_bias; every result is deterministic.

    window_size (left, right): query i sees the keys i - left .. i + right of its sequence
    (-1: no limit), and with sink_tokens = n its first n tokens always.  relative_bias
    [num_buckets, H] (bf16 or fp32) is added to the scaled scores by the bucket of
    key - query (relative_buckets); it excludes alibi_slopes.  dropout_p drops
    probabilities after the softmax by the counter-based mask of g5moe_dropout; without
    dropout_seed (a non-negative integer below 2^63) the 64-bit seed is drawn from torch's
    CPU generator, one per call (fixed at capture in a HIP graph)."""
    _unsupported(causal, window_size)
    if not 0.0 <= dropout_p <= 1.0:
        raise ValueError(f"dropout_p {dropout_p} is not in [0, 1]")
    if sink_tokens < 0:
        raise ValueError(f"sink_tokens {sink_tokens} must be >= 0")
    if dropout_seed is not None and not 0 <= int(dropout_seed) < 2 ** 63:
        raise ValueError(f"dropout_seed {dropout_seed} is not in [0, 2^63)")
    if cu_seqlens_k is not cu_seqlens_q and not torch.equal(cu_seqlens_k, cu_seqlens_q):
        raise NotImplementedError("cu_seqlens_k must equal cu_seqlens_q (self-attention)")
    if max_seqlen_q is None:
        max_seqlen_q = int((cu_seqlens_q[1:] - cu_seqlens_q[:-1]).max().item()) \
            if cu_seqlens_q.numel() > 1 else 0
    if max_seqlen_k is not None and max_seqlen_k != max_seqlen_q:
        raise NotImplementedError("max_seqlen_k must equal max_seqlen_q (self-attention)")
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    if dropout_p and q.device.type != "cuda":
        raise NotImplementedError("attention dropout runs on the GPU only (dropout_p must be 0 "
                                  f"on {q.device})")
    # beyond every position is as good as unlimited
    wl, wr, sink_tokens, max_seqlen_q = (min(int(x), _INT32_MAX) for x in
                                         (*window_size, sink_tokens, max_seqlen_q))
    leaves = (q, k, v) if relative_bias is None else (q, k, v, relative_bias)
    grad = torch.is_grad_enabled() and any(t.requires_grad for t in leaves)
    lse = None
    if not grad and wl < 0 and wr < 0 and relative_bias is None and dropout_p == 0:
        out, lse = _attn_op(q, k, v, cu_seqlens_q, int(max_seqlen_q), float(softmax_scale),
                            alibi_slopes, bool(return_attn_probs))
    elif torch.compiler.is_compiling():
        out, lse, _, _ = _attn_local_op(
            q, k, v, cu_seqlens_q, int(max_seqlen_q), float(softmax_scale), alibi_slopes,
            relative_bias, int(max_distance), wl, wr, int(sink_tokens), float(dropout_p),
            None if dropout_seed is None else int(dropout_seed), grad)
    else:
        seed = 0
        if dropout_p > 0:
            seed = _draw_seed() if dropout_seed is None else int(dropout_seed)
        if grad:
            out, lse = _AttnFunction.apply(
                q, k, v, relative_bias, cu_seqlens_q, int(max_seqlen_q), float(softmax_scale),
                alibi_slopes, int(max_distance), wl, wr, int(sink_tokens), float(dropout_p), seed)
        else:
            out = attn_local_fwd(
                q, k, v, cu_seqlens_q, int(max_seqlen_q), float(softmax_scale), alibi_slopes,
                relative_bias, int(max_distance), (wl, wr), int(sink_tokens), float(dropout_p),
                seed, return_lse=bool(return_attn_probs))
            if return_attn_probs:
                out, lse = out
    return (out, lse, None) if return_attn_probs else out


_CU_CACHE: dict = {}


def _uniform_cu_seqlens(batch: int, seqlen: int, device: torch.device) -> torch.Tensor:
    if torch.compiler.is_compiling():
        return torch.arange(batch + 1, dtype=torch.int32, device=device) * seqlen
    # by stream, so that its use follows its making without a synchronisation
    key = (batch, seqlen, device, _stream(device) if device.type == "cuda" else None)
    cu = _CU_CACHE.get(key)
    if cu is None:
        cu = torch.arange(batch + 1, dtype=torch.int32, device=device) * seqlen
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            return cu  # the graph's own: written by its replays only
        # kept: a captured graph may read it from now on
        _CU_CACHE[key] = cu
    return cu


def flash_attn_func(q, k, v, dropout_p=0.0, softmax_scale=None, causal=False,
                    window_size=(-1, -1), alibi_slopes=None, deterministic=False,
                    return_attn_probs=False, *, sink_tokens=0, relative_bias=None,
                    max_distance=128, dropout_seed=None):
    """flash-attn's fixed-length entry point: q [B, L, H, D], k/v [B, L, Hkv, D]; the other
    arguments as in flash_attn_varlen_func."""
    B, L = q.shape[0], q.shape[1]
    cu = _uniform_cu_seqlens(B, L, q.device)
    res = flash_attn_varlen_func(q.reshape(B * L, *q.shape[2:]), k.reshape(B * L, *k.shape[2:]),
                                 v.reshape(B * L, *v.shape[2:]), cu, cu, L, L, dropout_p,
                                 softmax_scale, causal, window_size, alibi_slopes, deterministic,
                                 return_attn_probs, sink_tokens=sink_tokens,
                                 relative_bias=relative_bias, max_distance=max_distance,
                                 dropout_seed=dropout_seed)
    if return_attn_probs:
        out, lse, _ = res
        return out.view(B, L, *out.shape[1:]), lse, None
    return res.view(B, L, *res.shape[1:])


@dataclass
class FlashAttentionConfig:
    """Fields of the reference's FlashAttentionConfig (lib/blocks/_flash_att.py:15-30)
    plus `alibi` (slopes of Press et al. per head when True), `sink_tokens` (first tokens that
    stay visible outside window_size) and `num_buckets` (> 0: a learned position bias
    [num_buckets, num_heads] over distances up to max_distance, in ALiBi's place)."""
    embed_dim: int = 768
    num_heads: int = 12
    num_kv_heads: int = None
    head_dim: int = None
    dropout: float = 0.0
    window_size: tuple = (-1, -1)
    alibi: bool = True
    sink_tokens: int = 0
    num_buckets: int = 0
    max_distance: int = 128

    def __post_init__(self):
        if self.num_buckets:
            _check_buckets(self.num_buckets, self.max_distance)
            self.alibi = False
        if self.num_kv_heads is None:
            self.num_kv_heads = self.num_heads
        if self.head_dim is None:
            self.head_dim = self.embed_dim // self.num_heads


class FlashAttention(nn.Module):
    """Bidirectional attention with optional varlen packing and ALiBi, mirroring
    the reference's FlashAttention (lib/blocks/_flash_att.py:38-98): bias-free
    q/k/v/o projections, GQA, softmax scale 1/sqrt(head_dim); forward returns
    (out, None).  The config's window, sinks and learned bias apply in training and in
    inference; in training mode its dropout applies to the probabilities and to the output."""

    def __init__(self, config: FlashAttentionConfig):
        super().__init__()
        if config.head_dim != HEAD_DIM:
            raise NotImplementedError(f"head_dim {config.head_dim}: the kernel supports "
                                      f"{HEAD_DIM}")
        if config.num_heads % config.num_kv_heads:
            raise ValueError("num_kv_heads must divide num_heads")
        self.config = config
        self.embed_dim = config.embed_dim
        self.num_heads = config.num_heads
        self.num_kv_heads = config.num_kv_heads
        self.head_dim = config.head_dim
        self.kv_dim = config.head_dim * config.num_kv_heads
        self.softmax_scale = 1.0 / math.sqrt(self.head_dim)
        self.q = nn.Linear(config.embed_dim, config.num_heads * self.head_dim, bias=False)
        self.k = nn.Linear(config.embed_dim, self.kv_dim, bias=False)
        self.v = nn.Linear(config.embed_dim, self.kv_dim, bias=False)
        self.o = nn.Linear(config.num_heads * self.head_dim, config.embed_dim, bias=False)
        self.dropout = nn.Dropout(config.dropout)
        # a row per bucket, a column per head; zeros: no bias until it is learned
        self.relative_bias = nn.Parameter(
            torch.zeros(config.num_buckets, config.num_heads)) if config.num_buckets else None
        # fp32 slopes kept outside the module's buffers, so that casting the model
        # to bf16 does not round them
        self._slopes = alibi_slopes(config.num_heads) if config.alibi else None
        self._slopes_dev: dict = {}

    def alibi_slopes(self, device: torch.device) -> Optional[torch.Tensor]:
        """The per-head slopes as a float32 tensor on `device` (None without ALiBi)."""
        if self._slopes is None:
            return None
        t = self._slopes_dev.get(device)
        if t is None:
            t = torch.tensor(self._slopes, dtype=torch.float32, device=device)
            self._slopes_dev[device] = t
        return t

    def qkv_weight(self) -> torch.Tensor:
        """[H*hd + 2*Hkv*hd, D] concatenation of the q, k and v weights, rebuilt when
        any of them changes."""
        key = tuple((p.data_ptr(), p._version, p.dtype) for p in
                    (self.q.weight, self.k.weight, self.v.weight))
        if getattr(self, "_qkv_key", None) != key:
            self._qkv = torch.cat([self.q.weight, self.k.weight, self.v.weight]).detach()
            self._qkv_key = key
        return self._qkv

    def _fused_projections(self, hidden_states: torch.Tensor) -> bool:
        """In inference (no gradient) with bf16 on the GPU, q, k and v come from one
        product and o from another on the grouped GEMM (ops.linear), faster than
        three nn.Linear calls at GeneT5's shapes; the module's parameters, outputs'
        shapes and meaning are unchanged (values differ from nn.Linear's only by the
        bf16 rounding of a different fp32 summation order)."""
        D = hidden_states.shape[-1]
        nq = self.num_heads * self.head_dim + 2 * self.kv_dim
        proj = (self.q, self.k, self.v, self.o)
        # the fused products know a weight and nothing else: a replaced projection (a
        # bias, an adapter) keeps its own forward
        if not all(type(m) is nn.Linear and m.bias is None for m in proj):
            return False
        weights = [m.weight for m in proj]
        needs_grad = torch.is_grad_enabled() and (
            hidden_states.requires_grad or any(w.requires_grad for w in weights)
            or (self.relative_bias is not None and self.relative_bias.requires_grad))
        return (not needs_grad and hidden_states.is_cuda
                and hidden_states.dtype == torch.bfloat16
                and all(w.dtype == torch.bfloat16 for w in weights)
                and D % 64 == 0 and D >= 128 and nq % 128 == 0 and D % 128 == 0
                and self.num_heads * self.head_dim >= 128)

    def forward(self, hidden_states, cu_seqlens=None, max_seqlen=None):
        B, L, _ = hidden_states.shape
        fused = self._fused_projections(hidden_states)
        if fused:
            hq = self.num_heads * self.head_dim
            qkv = ops.linear(hidden_states.reshape(B * L, -1), self.qkv_weight())
            q = qkv[:, :hq].view(B * L, self.num_heads, self.head_dim)
            k = qkv[:, hq:hq + self.kv_dim].view(B * L, self.num_kv_heads, self.head_dim)
            v = qkv[:, hq + self.kv_dim:].view(B * L, self.num_kv_heads, self.head_dim)
        else:
            q = self.q(hidden_states).view(B * L, self.num_heads, self.head_dim)
            k = self.k(hidden_states).view(B * L, self.num_kv_heads, self.head_dim)
            v = self.v(hidden_states).view(B * L, self.num_kv_heads, self.head_dim)
        drop_p = self.dropout.p if self.training else 0.0
        if cu_seqlens is None:
            cu_seqlens = _uniform_cu_seqlens(B, L, hidden_states.device)
            max_seqlen = L
        out = flash_attn_varlen_func(q, k, v, cu_seqlens, cu_seqlens, max_seqlen, max_seqlen,
                                     dropout_p=drop_p, softmax_scale=self.softmax_scale,
                                     causal=False, window_size=self.config.window_size,
                                     alibi_slopes=self.alibi_slopes(hidden_states.device),
                                     sink_tokens=self.config.sink_tokens,
                                     relative_bias=self.relative_bias,
                                     max_distance=self.config.max_distance)
        if fused:
            out = ops.linear(out.reshape(B * L, self.num_heads * self.head_dim),
                             self.o.weight).view(B, L, -1)
        else:
            out = self.o(out.reshape(B, L, self.num_heads * self.head_dim))
        return self.dropout(out), None
