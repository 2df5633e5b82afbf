"""What describe_matmul_block128 refuses and answers without a GPU."""
import ctypes

import pytest

from therock_b200 import build


@pytest.fixture(scope="module")
def ops():
    build.build()
    from therock_b200 import ops
    return ops


@pytest.mark.parametrize("m,n,k,quant", [(-1, 40, 256, 2), (3, 0, 256, 2), (3, 40, 0, 2), (3, 40, 192, 3), (1 << 40, 40, 256, 2), (3, 40, 256, 0), (3, 40, 256, 1)])
def test_sizes_that_the_product_refuses(ops, m, n, k, quant):
    lib, info = ops._bound(), ops._MatmulInfo()
    info.kernel = 9
    assert lib.fmoe_describe_matmul_block128(m, n, k, quant, ctypes.byref(info)) == lib.fmoe_matmul_block128(4096, 4096, 4096, 4096, m, n, k, quant, 4096, None, None) < 0
    assert info.kernel == 0
    assert lib.fmoe_describe_matmul_block128(3, 40, 256, 2, None) == -1


def test_no_rows_run_nothing(ops):
    assert ops.describe_matmul_block128(0, 40, 256) == {"kernel": "none", "rows_per_tile": 0, "cols_per_tile": 0, "k_split": 0}
    with pytest.raises(ops.FmoeError):
        ops.describe_matmul_block128(3, 40, 256, "token_channel")
    with pytest.raises(ops.FmoeError):
        ops.describe_matmul_block128(3, 2 ** 32 + 40, 256)
