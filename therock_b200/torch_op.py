"""`torch.library` bindings: `torch.ops.therock_b200.fused_moe` and the operators an expert layer is
built from (`grouped_matmul`, `matmul_block128`, `silu_mul`, with their gradients registered).

The ops have fake (meta) implementations, so they can sit inside traced / compiled graphs, and
their CUDA implementations only enqueue kernels on the current stream (no host sync), so they can
be captured in a CUDA graph.  The workspace comes from torch's caching allocator, which is
graph-pool aware."""
from __future__ import annotations

from typing import Optional

import torch

from . import api, ops


@torch.library.custom_op("therock_b200::fused_moe", mutates_args=(), device_types="cuda")
def fused_moe_op(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk_ids: torch.Tensor,
                 topk_weight: torch.Tensor, w1_scale: Optional[torch.Tensor] = None,
                 w2_scale: Optional[torch.Tensor] = None, quant: str = "none") -> torch.Tensor:
    traits = api.FusedMoeTraits(prec_w="bf16" if quant == "none" else "fp8", quant=quant)
    args = api.FusedMoeArgs(a=x, g=w1, d=w2, topk_ids=topk_ids, topk_weight=topk_weight,
                            g_scale=w1_scale, d_scale=w2_scale)
    return api.fused_moe(traits, args)


@fused_moe_op.register_fake
def _(x, w1, w2, topk_ids, topk_weight, w1_scale=None, w2_scale=None, quant="none"):
    return torch.empty_like(x)


@torch.library.custom_op("therock_b200::route", mutates_args=(), device_types="cuda")
def route_op(logits: torch.Tensor, topk: int, mode: str = "softmax") -> tuple[torch.Tensor, torch.Tensor]:
    return api.route(logits, topk, mode)


@route_op.register_fake
def _(logits, topk, mode="softmax"):
    T = logits.shape[0]
    return (torch.empty(T, topk, dtype=torch.int32, device=logits.device),
            torch.empty(T, topk, dtype=torch.float32, device=logits.device))


# ----------------------------------------------------------------------------- the parts of an expert layer
# The fake implementations refuse what the operators refuse by type, shape and layout.
def _fake_grouped(rows, weight, offsets, dim):
    torch._check(rows.dim() == 2 and weight.dim() == 3 and offsets.dim() == 1, lambda: "rows must be a matrix, weight [groups, n, k], offsets [groups + 1]")
    torch._check(rows.dtype in ops._DTYPE and weight.dtype == rows.dtype and offsets.dtype == torch.int32,
                 lambda: "rows and weight must both be bfloat16 or both float16, offsets int32")
    torch._check(rows.shape[1] == weight.shape[dim], lambda: "rows and weight do not fit each other")
    torch._check(offsets.shape[0] == weight.shape[0] + 1, lambda: "offsets must have one more element than there are groups")
    _fake_widths(weight.shape[1], weight.shape[2])
    _fake_dense(weight, offsets)


def _fake_widths(*widths):
    for n in widths:
        torch._check(n > 0, lambda: "a width must not be zero")
        torch._check(n % 8 == 0, lambda: "n, k and width must be multiples of 8")


def _fake_dense(*tensors):
    for t in tensors:
        torch._check(t.is_contiguous(), lambda: "tensors must be contiguous")


def _fake_silu(gu, row_weight):
    torch._check(gu.dim() == 2 and gu.dtype in ops._DTYPE, lambda: "gu must be [rows, 2 * width] in bfloat16 or float16")
    torch._check(gu.shape[1] % 2 == 0, lambda: "gu must be [rows, 2 * width]")
    _fake_widths(gu.shape[1] // 2)
    _fake_dense(gu)
    if row_weight is not None:
        torch._check(row_weight.dim() == 1 and row_weight.dtype == torch.float32, lambda: "row_weight must be float32 [rows]")
        torch._check(row_weight.shape[0] == gu.shape[0], lambda: "row_weight must be float32 [rows]")
        _fake_dense(row_weight)


@torch.library.custom_op("therock_b200::grouped_matmul", mutates_args=(), device_types="cuda")
def grouped_matmul_op(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return ops.grouped_matmul(x, weight, offsets)


@grouped_matmul_op.register_fake
def _(x, weight, offsets):
    _fake_grouped(x, weight, offsets, 2)
    _fake_dense(x)
    return x.new_empty(x.shape[0], weight.shape[1])


@torch.library.custom_op("therock_b200::grouped_matmul_dgrad", mutates_args=(), device_types="cuda")
def grouped_matmul_dgrad_op(dy: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return ops.grouped_matmul_dgrad(ops._for_kernel(dy), weight, offsets)


@grouped_matmul_dgrad_op.register_fake
def _(dy, weight, offsets):
    _fake_grouped(dy, weight, offsets, 1)
    return dy.new_empty(dy.shape[0], weight.shape[2])


@torch.library.custom_op("therock_b200::grouped_matmul_wgrad", mutates_args=(), device_types="cuda")
def grouped_matmul_wgrad_op(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return ops.grouped_matmul_wgrad(ops._for_kernel(dy), x, offsets)


@grouped_matmul_wgrad_op.register_fake
def _(dy, x, offsets):
    torch._check(dy.dim() == 2 and x.dim() == 2 and offsets.dim() == 1, lambda: "dy must be [rows, n], x [rows, k], offsets [groups + 1]")
    torch._check(x.dtype in ops._DTYPE and dy.dtype == x.dtype and offsets.dtype == torch.int32,
                 lambda: "dy and x must both be bfloat16 or both float16, offsets int32")
    torch._check(dy.shape[0] == x.shape[0], lambda: "dy and x must have the same rows")
    torch._check(offsets.shape[0] >= 2, lambda: "offsets must be int32 [groups + 1]")
    _fake_widths(dy.shape[1], x.shape[1])
    _fake_dense(x, offsets)
    return dy.new_empty(offsets.shape[0] - 1, dy.shape[1], x.shape[1])


def _check_capture(t):
    """A captured backward pass must not reach a node of the default stream (torch_binding.cpp)."""
    if type(t) is torch.Tensor or type(t) is torch.nn.Parameter:
        with torch.cuda.device(t.device):
            ops._native().check_capture()


def _grouped_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _grouped_backward(ctx, dy):
    x, weight, offsets = ctx.saved_tensors
    _check_capture(x)
    return (grouped_matmul_dgrad_op(dy, weight, offsets) if ctx.needs_input_grad[0] else None,
            grouped_matmul_wgrad_op(dy, x, offsets) if ctx.needs_input_grad[1] else None, None)


grouped_matmul_op.register_autograd(_grouped_backward, setup_context=_grouped_setup)


@torch.library.custom_op("therock_b200::matmul_block128", mutates_args=(), device_types="cuda")
def matmul_block128_op(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                       quant: str = "block128") -> torch.Tensor:
    return ops.matmul_block128(a, a_scale, w, w_scale, quant)


@matmul_block128_op.register_fake
def _(a, a_scale, w, w_scale, quant="block128"):
    torch._check(quant in ops._BLOCK_QUANT, lambda: f"quant must be one of {ops._BLOCK_QUANT}")
    torch._check(a.dtype in ops._E4M3 and w.dtype in ops._E4M3 and w_scale.dtype == torch.float32, lambda: "a and w must be e4m3, w_scale float32")
    torch._check(a_scale.dtype == torch.uint8 or (a_scale.dtype == torch.float32 and quant == "block128"), lambda: "a_scale must be as quantise_rows returns it")
    torch._check(a.dim() == 2 and w.dim() == 2 and a_scale.dim() == 2 and w_scale.dim() == 2, lambda: "a, a_scale, w and w_scale must be matrices")
    torch._check(a.shape[1] == w.shape[1], lambda: "a must be [m, k] and w [n, k]")
    torch._check(a.shape[1] > 0 and w.shape[0] > 0, lambda: "n and k must not be zero")
    torch._check(a.shape[1] % 128 == 0, lambda: "k must be a multiple of 128")
    blocks = a.shape[1] // 128
    row_bytes = 4 * blocks if quant == "block128" else (blocks + 3) // 4 * 4
    torch._check(a_scale.shape[0] == a.shape[0], lambda: "a_scale must have a's rows")
    torch._check(a_scale.shape[1] * a_scale.element_size() == row_bytes, lambda: "a_scale must be as quantise_rows returns it")
    torch._check(w_scale.shape[0] == (w.shape[0] + 127) // 128, lambda: "w_scale must be [ceil(n / 128), k / 128]")
    torch._check(w_scale.shape[1] == blocks, lambda: "w_scale must be [ceil(n / 128), k / 128]")
    _fake_dense(a, a_scale, w, w_scale)
    return a.new_empty(a.shape[0], w.shape[0], dtype=torch.bfloat16)


@torch.library.custom_op("therock_b200::silu_mul", mutates_args=(), device_types="cuda")
def silu_mul_op(gu: torch.Tensor, row_weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    return ops.silu_mul(gu, row_weight)


@silu_mul_op.register_fake
def _(gu, row_weight=None):
    _fake_silu(gu, row_weight)
    return gu.new_empty(gu.shape[0], gu.shape[1] // 2)


@torch.library.custom_op("therock_b200::silu_mul_backward", mutates_args=(), device_types="cuda")
def silu_mul_backward_op(gu: torch.Tensor, dy: torch.Tensor, row_weight: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    dgu, dweight = ops.silu_mul_backward(gu, ops._for_kernel(dy), row_weight)
    return dgu, gu.new_empty(0, dtype=torch.float32) if dweight is None else dweight


@silu_mul_backward_op.register_fake
def _(gu, dy, row_weight=None):
    _fake_silu(gu, row_weight)
    torch._check(dy.dim() == 2 and dy.dtype == gu.dtype, lambda: "dy must be [rows, width] of gu's type")
    torch._check(dy.shape[0] == gu.shape[0], lambda: "dy must be [rows, width] of gu's type")
    torch._check(2 * dy.shape[1] == gu.shape[1], lambda: "dy must be [rows, width] of gu's type")
    return torch.empty_like(gu), gu.new_empty(0 if row_weight is None else gu.shape[0], dtype=torch.float32)


def _silu_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _silu_backward(ctx, dy):
    gu, row_weight = ctx.saved_tensors
    _check_capture(gu)
    dgu, dweight = silu_mul_backward_op(gu, dy, row_weight)
    return dgu, None if row_weight is None else dweight


silu_mul_op.register_autograd(_silu_backward, setup_context=_silu_setup)
