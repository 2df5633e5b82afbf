"""What ptxas reports for the operators' kernels, read from the build's logs.

The e4m3 product with f32 scales hands registers from its thin warps to the warps that promote: the shares must
not exceed what the block is launched with, or setmaxnreg.inc would wait for ever, so the kernel has to be
compiled for exactly 128.  It also runs at the edge of its budget and spills a few bytes; more than now is a change
that costs its speed.  No other kernel spills."""
import os
import re

import pytest

from tests.test_kernel_resources import _kernels
from therock_b200 import build


@pytest.fixture(scope="module")
def kernels():
    build.build()
    out = {}
    for name in ("grouped", "block_matmul", "silu"):
        with open(os.path.join(build.OBJ_DIR, name + ".o.log")) as f:
            out.update(_kernels(f.read()))
    return out


def test_registers_of_the_kernel_that_hands_them_on(kernels):
    promote = {n: v for n, v in kernels.items() if "fmoe_matmul_block128_kernel" in n}
    assert len(promote) == 2
    text = open(os.path.join(build.CSRC, "block_matmul.cuh")).read()
    thin, issue, fat = (int(re.search(rf"{k} = (\d+)", text).group(1)) for k in ("kBmmThinRegs", "kBmmIssueRegs", "kBmmFatRegs"))
    for name, (stores, loads, registers) in promote.items():
        assert registers == 128 and 128 * (thin + issue) + 256 * fat <= 512 * registers, name
        assert stores <= 32 and loads <= 64, (name, stores, loads)


def test_the_other_kernels_do_not_spill(kernels):
    others = {n: v for n, v in kernels.items() if "fmoe_matmul_block128_kernel" not in n}
    for part, count in (("fmoe_grouped_rows_kernel", 4), ("fmoe_grouped_wgrad_kernel", 2), ("block128_hw_kernel", 2),
                        ("block128_small_kernel", 6), ("silu_mul", 4)):
        assert sum(part in n for n in others) >= count, part
    for name, (stores, loads, _) in others.items():
        assert stores == 0 and loads == 0, (name, stores, loads)
