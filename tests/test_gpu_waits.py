"""Bounded waits in the operators' kernels, in a build whose limit the host sets (fmoe_set_wait_limit).
Each test runs in a process of its own, which loads that build in place of the product library."""
import os
import subprocess
import sys

import pytest

from therock_b200 import build

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PRELUDE = """
import ctypes, torch, therock_b200 as M
d = "cuda:0"
lib = M.lib()
lib.fmoe_set_wait_limit.argtypes = [ctypes.c_int64]
def limit(cycles):
    assert lib.fmoe_set_wait_limit(cycles) == 0
def whole(*shape):
    return torch.randint(-1, 2, shape, device=d, dtype=torch.int8)
torch.manual_seed(0)
"""


def run(text):
    lib = build.build(wait_limit_switch=True)
    r = subprocess.run([sys.executable, "-c", PRELUDE + text], capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env={**os.environ, "FMOE_B200_LIBRARY": lib})
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout[-1000:] + r.stderr[-2000:]


def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right():
    """With no time at all to wait every kernel gives up: the call returns, the caller's word or the
    library's holds the code, reading the library's clears it, and the same call is right afterwards."""
    run("""
off = torch.tensor([0, 40, 40, 300], dtype=torch.int32, device=d)
x, w, dy = whole(300, 512).bfloat16(), whole(3, 320, 512).bfloat16(), whole(300, 320).bfloat16()
xs, os_, dys = x[:4], off.clamp(max=4), dy[:4]
e4 = lambda *s: whole(*s).float().to(torch.float8_e4m3fn)
calls = {"y": (0x500, lambda o: M.grouped_matmul(x, w, off)), "dx": (0x500, lambda o: M.grouped_matmul_dgrad(dy, w, off)),
         "dw": (0x500, lambda o: M.grouped_matmul_wgrad(dy, x, off)), "few y": (0x500, lambda o: M.grouped_matmul(xs, w, os_)),
         "few dw": (0x500, lambda o: M.grouped_matmul_wgrad(dys, xs, os_))}
for quant in ("block128", "block128_ue8m0"):
    for m, n, k in ((1, 63, 2048), (17, 2304, 4096), (130, 640, 1920), (250, 4999, 384), (1030, 7743, 128), (2304, 18432, 1280)):
        a, b = e4(m, k), e4(n, k)
        sa = torch.ones(m, k // 128, device=d) if quant == "block128" else torch.full((m, (k // 128 + 3) // 4 * 4), 127, dtype=torch.uint8, device=d)
        sb = torch.ones((n + 127) // 128, k // 128, device=d)
        calls[quant, m, n, k] = (0x600, lambda o, a=a, sa=sa, b=b, sb=sb, q=quant: M.matmul_block128(a, sa, b, sb, q))
assert M.operator_status(d) == 0
for name, (code, call) in calls.items():
    want = call(None)
    assert M.operator_status(d) == 0, name
    for _ in range(3):
        limit(0)
        call(None)
        got = M.operator_status(d)
        assert got & ~0xff == code and got & 0xff, (name, hex(got))
        assert M.operator_status(d) == 0, name
        limit(4000000000)
        assert torch.equal(call(None), want), name
    assert M.operator_status(d) == 0, name
# a word of the caller's: the library's own stays clear, and the code stays until the caller clears it
from therock_b200 import ops
word = torch.zeros(1, dtype=torch.int32, device=d)
out = torch.empty(300, 320, dtype=torch.bfloat16, device=d)
def direct():
    assert ops._bound().fmoe_grouped_matmul(x.data_ptr(), w.data_ptr(), off.data_ptr(), 300, 3, 320, 512, 0, 0, out.data_ptr(),
                                            word.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
limit(0)
direct()
assert int(word) & ~0xff == 0x500 and M.operator_status(d) == 0
limit(4000000000)
code = int(word)
direct()
assert int(word) == code and torch.equal(out, M.grouped_matmul(x, w, off))
print("done")
""")
