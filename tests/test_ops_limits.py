"""Sizes at the ends of 32 bits: what the kernels' index arithmetic cannot hold is refused before any CUDA
call.  Needs no GPU: nothing is launched, and a size that passes ends at the missing device."""
import pytest

from therock_b200 import build

P = 4096          # an aligned address nothing dereferences
MOST = 0x7fffff00
MOST_ROWS = 0x7f000000


@pytest.fixture(scope="module")
def lib():
    build.build()
    from therock_b200 import ops
    return ops._bound()


def _grouped(lib, rows, groups, n, k, transpose):
    if transpose == 2:
        return lib.fmoe_grouped_matmul_wgrad(P, P, P, rows, groups, n, k, 0, P, None, None)
    return lib.fmoe_grouped_matmul(P, P, P, rows, groups, n, k, 0, transpose, P, None, None)


@pytest.mark.parametrize("transpose", [0, 1, 2])
@pytest.mark.parametrize("rows,n,k", [(MOST_ROWS + 1, 8, 8), (2 ** 31 - 256, 8, 8), (1, MOST + 8, 8), (1, 8, MOST + 8), (1, 2 ** 31 - 8, 8), (1, 8, 2 ** 31 - 8)])
def test_grouped_products_past_their_indices(lib, rows, n, k, transpose):
    assert _grouped(lib, rows, 1, n, k, transpose) == -2
    assert b"too large" in lib.fmoe_last_error()


@pytest.mark.parametrize("m,n", [(1, MOST + 1), (1, 2 ** 31 - 1), (MOST + 1, 8)])
def test_e4m3_products_past_their_indices(lib, m, n):
    for quant in (2, 3):
        assert lib.fmoe_matmul_block128(P, P, P, P, m, n, 128, quant, P, None, None) == -2
        assert b"too large" in lib.fmoe_last_error()


def test_the_index_arithmetic_of_the_largest_sizes_that_pass():
    """The expressions of grouped.cuh and grouped.cu that add to a size, in 64 bits, against what 32 hold."""
    top = 2 ** 31 - 1
    chunks = -(-MOST_ROWS // 256)
    assert MOST_ROWS + 256 - 1 <= top                    # pieces of 256 rows
    assert MOST_ROWS + chunks - 1 <= top                 # rows of equal pieces
    assert (chunks - 1) * ((-(-MOST_ROWS // chunks) + 31) // 32 * 32) <= top
    assert MOST_ROWS + 64 + 128 <= top                   # a stage's and a half's last row
    assert MOST + 256 - 1 <= top and -(-MOST // 256) * 256 - 1 <= top
