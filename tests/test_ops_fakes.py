"""The registered operators on tensors without data: shapes and types of the results, and refusals of what
the operators refuse, as a traced or compiled program meets them.  Needs no GPU."""
import pytest
import torch

import therock_b200.torch_op  # noqa: F401

NS = torch.ops.therock_b200
BF, F8, F32, I32, U8 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.int32, torch.uint8


def meta(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


def offsets(groups):
    return meta(groups + 1, dtype=I32)


@pytest.mark.parametrize("call,shape,dtype", [
    (lambda: NS.grouped_matmul(meta(5, 64), meta(3, 96, 64), offsets(3)), (5, 96), BF),
    (lambda: NS.grouped_matmul(meta(0, 64), meta(3, 96, 64), offsets(3)), (0, 96), BF),
    (lambda: NS.grouped_matmul(meta(5, 64, dtype=torch.half), meta(3, 96, 64, dtype=torch.half), offsets(3)), (5, 96), torch.half),
    (lambda: NS.grouped_matmul_dgrad(meta(5, 96), meta(3, 96, 64), offsets(3)), (5, 64), BF),
    (lambda: NS.grouped_matmul_dgrad(meta(1, 1).expand(5, 96), meta(3, 96, 64), offsets(3)), (5, 64), BF),
    (lambda: NS.grouped_matmul_wgrad(meta(5, 96), meta(5, 64), offsets(3)), (3, 96, 64), BF),
    (lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(5, 2, dtype=F32), meta(70, 256, dtype=U8), meta(1, 2, dtype=F32)), (5, 70), BF),
    (lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(5, 8, dtype=U8), meta(70, 256, dtype=F8), meta(1, 2, dtype=F32)), (5, 70), BF),
    (lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(5, 4, dtype=U8), meta(130, 256, dtype=F8), meta(2, 2, dtype=F32), "block128_ue8m0"), (5, 130), BF),
    (lambda: NS.silu_mul(meta(5, 48)), (5, 24), BF),
    (lambda: NS.silu_mul(meta(5, 48), meta(5, dtype=F32)), (5, 24), BF),
    (lambda: NS.silu_mul_backward(meta(5, 48), meta(5, 24))[0], (5, 48), BF),
    (lambda: NS.silu_mul_backward(meta(5, 48), meta(5, 24), meta(5, dtype=F32))[1], (5,), F32),
])
def test_results(call, shape, dtype):
    out = call()
    assert tuple(out.shape) == shape and out.dtype == dtype


@pytest.mark.parametrize("call", [
    lambda: NS.grouped_matmul(meta(5, 64, dtype=F32), meta(3, 96, 64, dtype=F32), offsets(3)),
    lambda: NS.grouped_matmul(meta(5, 64, dtype=torch.half), meta(3, 96, 64), offsets(3)),
    lambda: NS.grouped_matmul(meta(5, 60), meta(3, 96, 60), offsets(3)),
    lambda: NS.grouped_matmul(meta(5, 64), meta(3, 90, 64), offsets(3)),
    lambda: NS.grouped_matmul(meta(5, 72), meta(3, 96, 64), offsets(3)),
    lambda: NS.grouped_matmul(meta(5, 64), meta(3, 96, 64), offsets(2)),
    lambda: NS.grouped_matmul(meta(5, 64), meta(3, 96, 64), meta(4, dtype=torch.int64)),
    lambda: NS.grouped_matmul(meta(64, 5).mT, meta(3, 96, 64), offsets(3)),
    lambda: NS.grouped_matmul(meta(5, 64), meta(3, 64, 96).mT, offsets(3)),
    lambda: NS.grouped_matmul(meta(64), meta(3, 96, 64), offsets(3)),
    lambda: NS.grouped_matmul_dgrad(meta(5, 64), meta(3, 96, 64), offsets(3)),
    lambda: NS.grouped_matmul_wgrad(meta(5, 96), meta(4, 64), offsets(3)),
    lambda: NS.grouped_matmul_wgrad(meta(5, 96), meta(5, 60), offsets(3)),
    lambda: NS.grouped_matmul_wgrad(meta(5, 96), meta(5, 64), offsets(0)),
    lambda: NS.matmul_block128(meta(5, 200, dtype=F8), meta(5, 1, dtype=F32), meta(70, 200, dtype=F8), meta(1, 1, dtype=F32)),
    lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(5, 2, dtype=F32), meta(70, 256, dtype=F8), meta(1, 2, dtype=F32), "token_channel"),
    lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(5, 2, dtype=F32), meta(70, 256, dtype=F8), meta(1, 2, dtype=F32), "block128_ue8m0"),
    lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(5, 4, dtype=U8), meta(70, 256, dtype=F8), meta(1, 2, dtype=F32)),
    lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(4, 2, dtype=F32), meta(70, 256, dtype=F8), meta(1, 2, dtype=F32)),
    lambda: NS.matmul_block128(meta(5, 256, dtype=F8), meta(5, 2, dtype=F32), meta(130, 256, dtype=F8), meta(1, 2, dtype=F32)),
    lambda: NS.matmul_block128(meta(5, 256), meta(5, 2, dtype=F32), meta(70, 256, dtype=F8), meta(1, 2, dtype=F32)),
    lambda: NS.silu_mul(meta(5, 48, dtype=F32)),
    lambda: NS.silu_mul(meta(5, 40)),
    lambda: NS.silu_mul(meta(5, 49)),
    lambda: NS.silu_mul(meta(5, 0)),
    lambda: NS.silu_mul(meta(5, 48), meta(4, dtype=F32)),
    lambda: NS.silu_mul(meta(5, 48), meta(5)),
    lambda: NS.silu_mul(meta(48, 5).mT),
    lambda: NS.silu_mul_backward(meta(5, 48), meta(5, 48)),
    lambda: NS.silu_mul_backward(meta(5, 48), meta(5, 24, dtype=torch.half)),
])
def test_refusals(call):
    with pytest.raises(RuntimeError):
        call()
