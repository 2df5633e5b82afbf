"""What the parts of an expert layer refuse, checked without a GPU: the C-ABI's argument checks come
before any CUDA call, the Python wrappers raise before they reach the library."""
import pytest
import torch

from therock_b200 import build


@pytest.fixture(scope="module")
def lib():
    build.build()
    from therock_b200 import ops
    return ops._bound()


P = 4096          # an aligned address nothing dereferences: every call below is refused first


@pytest.mark.parametrize("kw,code,text", [
    (dict(offsets=None), -1, b"offsets"),
    (dict(rows=-1), -1, b"bad dimensions"),
    (dict(groups=0), -1, b"bad dimensions"),
    (dict(n=0), -1, b"bad dimensions"),
    (dict(dtype=1), -2, b"bf16 and f16"),
    (dict(groups=1025), -2, b"1024"),
    (dict(n=100), -2, b"multiples of 8"),
    (dict(k=4), -2, b"multiples of 8"),
    (dict(rows=1 << 40), -2, b"too large"),
    (dict(groups=1024, n=1 << 20, k=1 << 20), -2, b"too large"),
    (dict(x=None), -1, b"required"),
    (dict(out=None), -1, b"required"),
    (dict(x=P + 8), -1, b"aligned"),
    (dict(out=P + 2), -1, b"aligned"),
])
def test_grouped_matmul_refuses(lib, kw, code, text):
    a = dict(x=P, w=P, offsets=P, rows=4, groups=2, n=64, k=64, dtype=0, transpose=0, out=P)
    a.update(kw)
    assert lib.fmoe_grouped_matmul(a["x"], a["w"], a["offsets"], a["rows"], a["groups"], a["n"], a["k"], a["dtype"],
                                   a["transpose"], a["out"], None, None) == code
    assert text in lib.fmoe_last_error()
    # the gradient of the weights takes the same dimensions: dy for w, dw for out
    assert lib.fmoe_grouped_matmul_wgrad(a["w"], a["x"], a["offsets"], a["rows"], a["groups"], a["n"], a["k"], a["dtype"],
                                         a["out"], None, None) == code
    assert text in lib.fmoe_last_error()


def test_grouped_matmul_without_rows_launches_nothing(lib):
    assert lib.fmoe_grouped_matmul(None, None, P, 0, 2, 64, 64, 0, 0, None, None, None) == 0
    assert lib.fmoe_grouped_matmul(P, P, P, 4, 2, 64, 64, 0, 2, P, None, None) == -1
    assert b"transpose_w" in lib.fmoe_last_error()


@pytest.mark.parametrize("kw,code,text", [
    (dict(quant=0), -1, b"block mode"), (dict(quant=1), -1, b"block mode"),
    (dict(m=-1), -1, b"bad dimensions"), (dict(n=0), -1, b"bad dimensions"), (dict(k=0), -1, b"bad dimensions"),
    (dict(k=192), -2, b"multiple of 128"), (dict(m=1 << 40), -2, b"too large"),
    (dict(a=None), -1, b"required"), (dict(w_scale=None), -1, b"required"),
    (dict(a=P + 1), -1, b"aligned"), (dict(w=P + 8), -1, b"aligned"), (dict(out=P + 2), -1, b"aligned"), (dict(a_scale=P + 1), -1, b"aligned"),
])
def test_matmul_block128_refuses(lib, kw, code, text):
    a = dict(a=P, a_scale=P, w=P, w_scale=P, m=3, n=40, k=256, quant=2, out=P)
    a.update(kw)
    assert lib.fmoe_matmul_block128(a["a"], a["a_scale"], a["w"], a["w_scale"], a["m"], a["n"], a["k"], a["quant"], a["out"],
                                    None, None) == code
    assert text in lib.fmoe_last_error()


def test_silu_mul_refuses(lib):
    assert lib.fmoe_silu_mul(None, None, 3, 64, 0, P, None) == -1
    assert lib.fmoe_silu_mul(P, None, 3, 64, 1, P, None) == -2
    assert lib.fmoe_silu_mul(P, None, 3, 60, 0, P, None) == -2
    assert lib.fmoe_silu_mul(P, None, -3, 64, 0, P, None) == -1
    assert lib.fmoe_silu_mul(P + 8, None, 3, 64, 0, P, None) == -1
    assert lib.fmoe_silu_mul(P, None, 3, 64, 0, None, None) == -1
    assert lib.fmoe_silu_mul(None, None, 0, 64, 0, None, None) == 0
    assert lib.fmoe_silu_mul_quantise(P, None, 3, 64, 0, 3, P, P, None) == -2        # not a multiple of 128
    assert lib.fmoe_silu_mul_quantise(P, None, 3, 128, 0, 1, P, P, None) == -1       # not a block mode
    assert lib.fmoe_silu_mul_quantise(P, None, 3, 128, 0, 3, P, None, None) == -1
    assert lib.fmoe_silu_mul_quantise(P, None, 3, 128, 0, 3, P + 4, P, None) == -1
    assert lib.fmoe_silu_mul_backward(P, P, P, 3, 64, 0, P, None, None) == -1        # weight without its gradient
    assert lib.fmoe_silu_mul_backward(P, None, None, 3, 64, 0, P, None, None) == -1
    assert lib.fmoe_silu_mul_backward(P, None, P + 8, 3, 64, 0, P, None, None) == -1


def test_wrappers_refuse_host_tensors(lib):
    import therock_b200 as M
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(2, 64, 64, dtype=torch.bfloat16)
    off = torch.tensor([0, 2, 4], dtype=torch.int32)
    q = torch.zeros(4, 128, dtype=torch.uint8)
    for call in (lambda: M.grouped_matmul(x, w, off), lambda: M.grouped_matmul_dgrad(x, w, off),
                 lambda: M.grouped_matmul_wgrad(x, x, off), lambda: M.silu_mul(x), lambda: M.silu_mul_backward(x, x),
                 lambda: M.silu_mul_quantise(x, "block128"), lambda: M.silu_mul_quantise(x, "none"),
                 lambda: M.matmul_block128(q, torch.zeros(4, 1), q, torch.zeros(1, 1)),
                 lambda: M.matmul_block128(q, torch.zeros(4, 1), q, torch.zeros(1, 1), quant="token_channel")):
        with pytest.raises(M.FmoeError):
            call()


def test_pointers_below_their_types_alignment_are_refused(lib):
    assert lib.fmoe_grouped_matmul(P, P, P + 2, 4, 2, 64, 64, 0, 0, P, None, None) == -1
    assert lib.fmoe_grouped_matmul(P, P, P, 4, 2, 64, 64, 0, 0, P, P + 1, None) == -1
    assert lib.fmoe_grouped_matmul_wgrad(P, P, P + 1, 4, 2, 64, 64, 0, P, None, None) == -1
    assert lib.fmoe_grouped_matmul_wgrad(P, P, P, 4, 2, 64, 64, 0, P, P + 2, None) == -1
    assert lib.fmoe_matmul_block128(P, P, P, P, 3, 40, 256, 2, P, P + 2, None) == -1
    assert lib.fmoe_silu_mul(P, P + 2, 3, 64, 0, P, None) == -1
    assert lib.fmoe_silu_mul_quantise(P, P + 1, 3, 128, 0, 3, P, P, None) == -1
    assert lib.fmoe_silu_mul_backward(P, P + 2, P, 3, 64, 0, P, P, None) == -1
    assert lib.fmoe_silu_mul_backward(P, P, P, 3, 64, 0, P, P + 2, None) == -1
    assert b"aligned" in lib.fmoe_last_error()


def test_sizes_past_32_bits_are_refused(lib):
    from therock_b200 import ops
    with pytest.raises(ops.FmoeError):
        ops._sizes(8, 2 ** 32 + 8)
    ops._sizes(2 ** 31 - 1)
