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


def test_a_tile_may_take_longer_than_a_wait():
    """A wait for a whole tile covers all of its contraction: its limit grows with the stages, so a sum
    over any number of rows is finished.  Here one stage may take 0.1 ms and a tile takes more than that.
    Small whole numbers, so every sum is exact."""
    run("""
def same(out, ref):
    assert torch.equal(out, ref.to(out.dtype)), (out.double() - ref).abs().max()
def dots(a, b):
    return sum((a[..., i:i + 65536].double() @ b[..., i:i + 65536].double().mT) for i in range(0, a.shape[-1], 65536))
long = 1 << 20
limit(200000)
for rows in (long, long - 3):
    x, dy = whole(rows, 8).bfloat16(), whole(rows, 8).bfloat16()
    off = torch.tensor([0, 5, rows], dtype=torch.int32, device=d)
    dw = M.grouped_matmul_wgrad(dy, x, off)
    assert M.operator_status(d) == 0
    same(dw[1], dots(dy[5:].mT, x[5:].mT))
off = torch.tensor([0, 40], dtype=torch.int32, device=d)
x, w = whole(40, long).bfloat16(), whole(1, 8, long).bfloat16()
y = M.grouped_matmul(x, w, off)
assert M.operator_status(d) == 0
same(y, dots(x, w[0]))
wt = w[0].mT.contiguous()[None]
dx = M.grouped_matmul_dgrad(x, wt, off)
assert M.operator_status(d) == 0
same(dx, dots(x, w[0]))
del x, w, wt
byte = lambda t: ((t == 1) * 0x38 + (t == -1) * 0xb8).to(torch.uint8)      # 1 and -1 in e4m3
m, n, k = 8192, 4096, 1 << 17
a, b = torch.cat([byte(whole(1024, k)) for _ in range(m // 1024)]), torch.cat([byte(whole(1024, k)) for _ in range(n // 1024)])
ones = lambda *s: torch.ones(*s, device=d)
at = torch.tensor([0, 1, 127, 128, 4095, 4096, m - 1], device=d)
value = lambda t: t.view(torch.float8_e4m3fn).float()
ref = dots(value(a[at]), value(b))
for quant, sa in (("block128_ue8m0", torch.full((m, k // 128), 127, dtype=torch.uint8, device=d)), ("block128", ones(m, k // 128))):
    out = M.matmul_block128(a, sa, b, ones(n // 128, k // 128), quant)
    assert M.operator_status(d) == 0, quant
    same(out[at], ref)
print("done")
""")
