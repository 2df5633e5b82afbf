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
@torch.library.custom_op("therock_b200::grouped_matmul", mutates_args=(), device_types="cuda")
def grouped_matmul_op(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return ops.grouped_matmul(x, weight, offsets)


@grouped_matmul_op.register_fake
def _(x, weight, offsets):
    return x.new_empty(x.shape[0], weight.shape[1])


@torch.library.custom_op("therock_b200::grouped_matmul_dgrad", mutates_args=(), device_types="cuda")
def grouped_matmul_dgrad_op(dy: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return ops.grouped_matmul_dgrad(ops._for_kernel(dy), weight, offsets)


@grouped_matmul_dgrad_op.register_fake
def _(dy, weight, offsets):
    return dy.new_empty(dy.shape[0], weight.shape[2])


@torch.library.custom_op("therock_b200::grouped_matmul_wgrad", mutates_args=(), device_types="cuda")
def grouped_matmul_wgrad_op(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return ops.grouped_matmul_wgrad(ops._for_kernel(dy), x, offsets)


@grouped_matmul_wgrad_op.register_fake
def _(dy, x, offsets):
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
    return a.new_empty(a.shape[0], w.shape[0], dtype=torch.bfloat16)


@torch.library.custom_op("therock_b200::silu_mul", mutates_args=(), device_types="cuda")
def silu_mul_op(gu: torch.Tensor, row_weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    return ops.silu_mul(gu, row_weight)


@silu_mul_op.register_fake
def _(gu, row_weight=None):
    return gu.new_empty(gu.shape[0], gu.shape[1] // 2)


@torch.library.custom_op("therock_b200::silu_mul_backward", mutates_args=(), device_types="cuda")
def silu_mul_backward_op(gu: torch.Tensor, dy: torch.Tensor, row_weight: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    dgu, dweight = ops.silu_mul_backward(gu, ops._for_kernel(dy), row_weight)
    return dgu, gu.new_empty(0, dtype=torch.float32) if dweight is None else dweight


@silu_mul_backward_op.register_fake
def _(gu, dy, row_weight=None):
    return torch.empty_like(gu), gu.new_empty(0 if row_weight is None else gu.shape[0], dtype=torch.float32)


def _silu_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _silu_backward(ctx, dy):
    gu, row_weight = ctx.saved_tensors
    _check_capture(gu)
    dgu, dweight = silu_mul_backward_op(gu, dy, row_weight)
    return dgu, None if row_weight is None else dweight


silu_mul_op.register_autograd(_silu_backward, setup_context=_silu_setup)
