"""`torch.library` registration of the operator: ``torch.ops.neogemm.linear(x, w)`` and the
out-variant ``torch.ops.neogemm.linear_out(x, w, out)``.

The reference exposes one in-place, column-major, default-stream function (nemgemmV03.cu:343,383).
Its layout is already that of ``torch.nn.Linear`` without bias - y = x @ W^T with W stored [N, K]
(benchmark.py:10-11,18) - so the same kernel serves as a module drop-in for the decode-shaped
MLP projections.  Registering it as a custom op gives it a fake (meta) implementation, so shape
inference and tracing tools see through it; the real implementation calls the C ABI on torch's
current stream.  There is no CPU implementation: calling it with CPU tensors raises.
"""
from __future__ import annotations

import math

import torch

from . import ops as _ops

_LIB_NAME = "neogemm"


def _check(x: torch.Tensor, weight: torch.Tensor) -> None:
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError("linear expects x[..., K] and weight[N, K]")
    if x.shape[-1] != weight.shape[1]:
        raise ValueError(f"K mismatch: x has {x.shape[-1]}, weight has {weight.shape[1]}")
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("linear expects bfloat16 tensors")


@torch.library.custom_op(f"{_LIB_NAME}::linear", mutates_args=())
def linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    _check(x, weight)
    return _ops.linear(x, weight)


@linear.register_fake
def _(x, weight):
    _check(x, weight)
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op(f"{_LIB_NAME}::linear_out", mutates_args=("out",))
def linear_out(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor) -> None:
    _check(x, weight)
    x2 = x.reshape(-1, x.shape[-1])
    if x2.size(1) > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    out2 = out.view(-1, weight.shape[0])
    _ops.matmul(x2, weight, out=out2)


@linear_out.register_fake
def _(x, weight, out):
    _check(x, weight)
    if tuple(out.shape) != (*x.shape[:-1], weight.shape[0]):
        raise ValueError("out has the wrong shape")
    return None


class NeoLinear(torch.nn.Module):
    """Bias-free ``nn.Linear`` whose forward is the B200 kernel (inference only: no autograd
    formula is registered)."""

    def __init__(self, in_features: int, out_features: int, device=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.weight = torch.nn.Parameter(
            torch.empty(out_features, in_features, dtype=torch.bfloat16, device=device),
            requires_grad=False)
        torch.nn.init.normal_(self.weight, std=in_features ** -0.5)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return torch.ops.neogemm.linear(x, self.weight)


# ----------------------------------------------------------------------------------------------
# Products grouped by expert, with their gradients
# ----------------------------------------------------------------------------------------------
def _check_grouped(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> None:
    if x.dim() != 2 or weight.dim() != 3 or offsets.dim() != 1:
        raise ValueError("grouped_linear expects x[T, K], weight[groups, N, K] and offsets[groups + 1]")
    if x.shape[1] != weight.shape[2]:
        raise ValueError(f"K mismatch: x has {x.shape[1]}, weight has {weight.shape[2]}")
    if offsets.shape[0] != weight.shape[0] + 1:
        raise ValueError(f"{weight.shape[0]} matrices need {weight.shape[0] + 1} offsets, got "
                         f"{offsets.shape[0]}")
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("grouped_linear expects bfloat16 tensors")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    groups, rows, width = weight.shape
    if groups > MAX_GROUPS:
        raise ValueError(f"at most {MAX_GROUPS} groups, got {groups}")
    # The kernels read weights in place (a copy per call is nobody's wish): from 16 bytes on.
    if weight.numel() > 0 and (
            weight.storage_offset() % 8 != 0 or (width > 1 and weight.stride(2) != 1) or
            (rows > 1 and (weight.stride(1) % 8 != 0 or weight.stride(1) < width)) or
            (groups > 1 and (weight.stride(0) % 8 != 0 or weight.stride(0) == 0))):
        raise ValueError("weight must have contiguous rows that start on multiples of 8 values, and a matrix "
                         f"per group: shape {tuple(weight.shape)} has strides {tuple(weight.stride())}, "
                         f"offset {weight.storage_offset()}")


MAX_GROUPS = 1024


def _readable(t: torch.Tensor) -> torch.Tensor:
    """A matrix in a layout that the kernels read: contiguous rows that start on 16 bytes."""
    step = 16 // t.element_size()
    if (t.shape[1] <= 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0 and (
            t.shape[0] <= 1 or (t.stride(0) % step == 0 and t.stride(0) >= t.shape[1])):
        return t
    rows, width = t.shape
    return t.new_empty((rows, (width + step - 1) // step * step))[:, :width].copy_(t)


@torch.library.custom_op(f"{_LIB_NAME}::grouped_linear", mutates_args=())
def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """y[t] = x[t] @ weight[e]^T for the rows of group e (``ops.grouped_matmul``); differentiable in
    ``x`` and ``weight``.  Rows of no group are zero, and so are their gradients.  ``x`` may have any
    layout (it is copied if its rows are not contiguous or do not start on 16 bytes); ``weight`` is read in
    place, so its rows start on multiples of 8 values."""
    _check_grouped(x, weight, offsets)
    return _ops.grouped_matmul(_readable(x), weight, offsets)


@grouped_linear.register_fake
def _(x, weight, offsets):
    _check_grouped(x, weight, offsets)
    return x.new_empty((x.shape[0], weight.shape[1]))


@torch.library.custom_op(f"{_LIB_NAME}::grouped_linear_dx", mutates_args=())
def _grouped_linear_dx(dy: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return _ops.grouped_matmul_dx(_readable(dy), weight, offsets)


@_grouped_linear_dx.register_fake
def _(dy, weight, offsets):
    return dy.new_empty((dy.shape[0], weight.shape[2]))


@torch.library.custom_op(f"{_LIB_NAME}::grouped_linear_dw", mutates_args=())
def _grouped_linear_dw(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return _ops.grouped_matmul_dw(_readable(dy), _readable(x), offsets)


@_grouped_linear_dw.register_fake
def _(dy, x, offsets):
    return dy.new_empty((offsets.shape[0] - 1, dy.shape[1], x.shape[1]))


def _grouped_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _grouped_backward(ctx, dy):
    x, weight, offsets = ctx.saved_tensors
    dx = _grouped_linear_dx(dy, weight, offsets) if ctx.needs_input_grad[0] else None
    dw = _grouped_linear_dw(dy, x, offsets) if ctx.needs_input_grad[1] else None
    return dx, dw, None


grouped_linear.register_autograd(_grouped_backward, setup_context=_grouped_setup)


class NeoGroupedLinear(torch.nn.Module):
    """One bias-free linear layer per group (expert, at most 1024): rows sorted by group in, rows out,
    trainable.  ``in_features`` is a multiple of 8."""

    def __init__(self, groups: int, in_features: int, out_features: int, device=None):
        super().__init__()
        if in_features % 8 != 0:
            raise ValueError(f"in_features must be a multiple of 8, got {in_features}")
        if groups > MAX_GROUPS:
            raise ValueError(f"at most {MAX_GROUPS} groups, got {groups}")
        self.groups, self.in_features, self.out_features = groups, in_features, out_features
        self.weight = torch.nn.Parameter(
            torch.empty(groups, out_features, in_features, dtype=torch.bfloat16, device=device))
        torch.nn.init.normal_(self.weight, std=in_features ** -0.5)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        return torch.ops.neogemm.grouped_linear(x, self.weight, offsets)


# ----------------------------------------------------------------------------------------------
# Linear layers with weights held in MXFP4 (inference)
# ----------------------------------------------------------------------------------------------
def _check_mxfp4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, dims: int) -> None:
    if x.dim() < 1 or codes.dim() != dims or (dims == 3 and x.dim() != 2):
        raise ValueError(f"expected x[{'..., ' if dims == 2 else 'T, '}K] and codes of {dims} dimensions")
    width = 2 * codes.shape[-1]
    if x.shape[-1] != width:
        raise ValueError(f"K mismatch: x has {x.shape[-1]}, weight has {width}")
    if width % 64 != 0:
        raise ValueError(f"K must be a multiple of 64, got {width}")
    if x.dtype not in (torch.bfloat16, torch.float32) or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError("expected x in bfloat16 or float32, codes and scales in uint8")
    want = (*codes.shape[:-2], (codes.shape[-2] + 127) // 128, (width + 127) // 128, 32, 4, 4)
    if tuple(scales.shape) != want:
        raise ValueError(f"scales of codes {tuple(codes.shape)} must be {want}, got {tuple(scales.shape)}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError("codes and scales must be contiguous")


def _check_mxfp4_grouped(x, codes, scales, offsets) -> None:
    _check_mxfp4_linear(x, codes, scales, 3)
    if offsets.dim() != 1 or offsets.shape[0] != codes.shape[0] + 1:
        raise ValueError(f"{codes.shape[0]} matrices need a vector of {codes.shape[0] + 1} offsets, got shape "
                         f"{tuple(offsets.shape)}")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    if codes.shape[0] > MAX_GROUPS:
        raise ValueError(f"at most {MAX_GROUPS} groups, got {codes.shape[0]}")


@torch.library.custom_op(f"{_LIB_NAME}::mxfp4_linear", mutates_args=())
def mxfp4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """y = x @ W^T with x[..., K] (any layout) quantised to MXFP4 on the way and W[N, K] held in it; bf16
    result.  K is a multiple of 64."""
    _check_mxfp4_linear(x, codes, scales, 2)
    x2 = _readable(x.reshape(math.prod(x.shape[:-1]), x.shape[-1]))
    y = _ops.matmul_mxfp4(_ops.quantize_mxfp4(x2), _ops.MxFp4(codes, scales))
    return y.reshape(*x.shape[:-1], codes.shape[0])


@mxfp4_linear.register_fake
def _(x, codes, scales):
    _check_mxfp4_linear(x, codes, scales, 2)
    return x.new_empty((*x.shape[:-1], codes.shape[0]), dtype=torch.bfloat16)


@torch.library.custom_op(f"{_LIB_NAME}::mxfp4_grouped_linear", mutates_args=())
def mxfp4_grouped_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                         offsets: torch.Tensor) -> torch.Tensor:
    """``grouped_linear`` with x quantised to MXFP4 on the way and the weights held in it."""
    _check_mxfp4_grouped(x, codes, scales, offsets)
    return _ops.grouped_matmul_mxfp4(_ops.quantize_mxfp4(_readable(x)), _ops.MxFp4(codes, scales), offsets)


@mxfp4_grouped_linear.register_fake
def _(x, codes, scales, offsets):
    _check_mxfp4_grouped(x, codes, scales, offsets)
    return x.new_empty((x.shape[0], codes.shape[1]), dtype=torch.bfloat16)


class NeoLinearMxFp4(torch.nn.Module):
    """Bias-free linear layer (or one per group, from a [groups, N, K] weight) whose weight is held in
    MXFP4, 17/32 of a byte per value, and whose input is quantised on the way in.  K is a multiple of 64.
    Inference only."""

    def __init__(self, weight: torch.Tensor):
        super().__init__()
        if weight.dim() not in (2, 3) or weight.shape[-1] % 64 != 0:
            raise ValueError(f"expected a weight [N, K] or [groups, N, K] with K a multiple of 64, got shape "
                             f"{tuple(weight.shape)}")
        weight = weight.detach().contiguous()
        q = _ops.quantize_mxfp4(weight if weight.data_ptr() % 16 == 0 else weight.clone())
        self.register_buffer("codes", q.codes)
        self.register_buffer("scales", q.scales)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor | None = None) -> torch.Tensor:
        if self.codes.dim() == 3:
            if offsets is None:
                raise ValueError("a layer per group needs the groups' offsets")
            return torch.ops.neogemm.mxfp4_grouped_linear(x, self.codes, self.scales, offsets)
        return torch.ops.neogemm.mxfp4_linear(x, self.codes, self.scales)
