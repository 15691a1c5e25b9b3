"""Residual add with counter-based dropout on the HIP kernel of libg5moe.so.

Reference: `hidden_states + dropout(ff_output) * alpha` of EncoderBlock.forward
(lib/blocks/encoder.py:89).  The mask is a hash of (seed, row, column) as in the expert
layer's dropout (g5moe_dropout in include/g5moe.h), formed again in the backward and never
stored; torch's Philox stream is not reproduced.  There is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib, ops
from .ops import _check_device, _ptr, _stream


def _draw_seed() -> int:
    return int(torch.randint(0, 2 ** 62, (1,)).item())


def _launch(name: str, x2: torch.Tensor, residual: Optional[torch.Tensor], p: float, alpha: float,
            seed: int) -> torch.Tensor:
    dev = _check_device(x2)
    out = torch.empty_like(x2)
    if x2.numel() == 0:
        return out
    drop = _lib.make_dropout(p, seed)
    tensors = (_ptr(x2), _ptr(out)) if residual is None else (_ptr(x2), _ptr(residual), _ptr(out))
    ops._call_on(dev, name, *tensors, ctypes.byref(drop), ctypes.c_float(alpha), x2.shape[0],
                 x2.shape[1], ops._dtype_code(x2.dtype), _stream(dev))
    return out


class _DropoutAdd(torch.autograd.Function):
    """The operator in eager programs (a traced one records the custom op below, whose
    dispatch costs more host time per call)."""

    @staticmethod
    def forward(ctx, x, residual, p, alpha, seed):
        ctx.call = (p, alpha, seed)
        ctx.set_materialize_grads(False)
        return _launch("g5moe_dropout_add", x, residual, p, alpha, seed)

    @staticmethod
    @ops._once_differentiable
    def backward(ctx, dout):
        if dout is None:
            return None, None, None, None, None
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _launch("g5moe_dropout_add_backward", dout.contiguous(), None, *ctx.call)
        return dx, dout if ctx.needs_input_grad[1] else None, None, None, None


@torch.library.custom_op("g5moe::dropout_add", mutates_args=())
def _dropout_add_op(x: torch.Tensor, residual: torch.Tensor, p: float, alpha: float,
                    seed: Optional[int]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, the seed as host int64 [1]); without a seed one is drawn per call from torch's
    CPU generator."""
    s = 0
    if p > 0:
        s = _draw_seed() if seed is None else seed
    return (_launch("g5moe_dropout_add", x, residual, p, alpha, s),
            torch.tensor([s], dtype=torch.int64))


@_dropout_add_op.register_fake
def _(x, residual, p, alpha, seed):
    return torch.empty_like(x), torch.empty((1,), dtype=torch.int64, device="cpu")


@torch.library.custom_op("g5moe::dropout_add_backward", mutates_args=())
def _dropout_add_bwd_op(dout: torch.Tensor, p: float, alpha: float,
                        seed: torch.Tensor) -> torch.Tensor:
    return _launch("g5moe_dropout_add_backward", dout, None, p, alpha, int(seed[0]))


@_dropout_add_bwd_op.register_fake
def _(dout, p, alpha, seed):
    return torch.empty_like(dout)


def _setup(ctx, inputs, output):
    _, _, ctx.p, ctx.alpha, _ = inputs
    ctx.save_for_backward(output[1])
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _backward(ctx, dout, _dseed):
    if dout is None:
        return None, None, None, None, None
    dx = None
    if ctx.needs_input_grad[0]:
        dx = _dropout_add_bwd_op(dout.contiguous(), ctx.p, ctx.alpha, ctx.saved_tensors[0])
    return dx, dout if ctx.needs_input_grad[1] else None, None, None, None


_dropout_add_op.register_autograd(_backward, setup_context=_setup)


def dropout_add(x: torch.Tensor, residual: torch.Tensor, p: float, alpha: float = 1.0,
                training: bool = True, seed: Optional[int] = None) -> torch.Tensor:
    """residual + alpha * dropout(x, p): [..., d] bf16 or fp32, both of one shape and dtype.
    Differentiable in x and residual.  training = False leaves the dropout out.  Without
    `seed` (a non-negative integer below 2^63) the mask's seed is drawn from torch's CPU
    generator, one per call (fixed at capture in a HIP graph).  Rows are the flattened
    leading dimensions, so a mask belongs to (seed, row, column) whatever their split."""
    dev = _check_device(x)
    if residual.device != dev:
        raise ValueError(f"residual is on {residual.device}, expected {dev}")
    if residual.dtype != x.dtype:
        raise TypeError(f"residual has dtype {residual.dtype}, x {x.dtype}")
    ops._dtype_code(x.dtype)
    if x.dim() < 1 or residual.shape != x.shape:
        raise ValueError(f"x has shape {tuple(x.shape)} and residual {tuple(residual.shape)}; "
                         "they must be equal and have a last dimension")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} is not in [0, 1]")
    if seed is not None and not 0 <= int(seed) < 2 ** 63:
        raise ValueError(f"seed {seed} is not in [0, 2^63)")
    d = x.shape[-1]
    if x.numel() == 0:
        return residual + x * alpha
    p, alpha = float(p) if training else 0.0, float(alpha)
    x2, r2 = x, residual
    if x.dim() != 2 or not (x.is_contiguous() and residual.is_contiguous()):
        x2, r2 = x.reshape(-1, d).contiguous(), residual.reshape(-1, d).contiguous()
    if torch.compiler.is_compiling():
        out, _ = _dropout_add_op(x2, r2, p, alpha, None if seed is None else int(seed))
    else:
        if seed is None:
            seed = _draw_seed() if p > 0 else 0
        out = _DropoutAdd.apply(x2, r2, p, alpha, int(seed))
    return out if x2 is x else out.view(x.shape)
