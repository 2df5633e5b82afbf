"""The parts of an expert layer against plain 64-bit implementations.

Tolerances, element by element.  A product's operands are exact in 32 bits and its sum of K terms
is built from at most K additions, each off by at most 2^-23 of the sum of magnitudes S; the result is
rounded once (half a step, eps / 2 of its type, of the value):
    |out - ref| <= eps/2 |ref| + (K + 8) 2^-23 S      (+ half the smallest subnormal of float16)
The gated activation: __expf is off by at most 2 + 1.173 |g| units in the last place (2^-23), the
reciprocal by one, and at most eight further 32-bit operations follow, so every factor is within
d(g) = (12 + 1.173 |g|) 2^-23 of its value."""
import pytest
import torch

import therock_b200 as M
from therock_b200 import api

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(out, ref, slack):
    """out == ref up to one rounding to out's type plus `slack`, element by element."""
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[out.dtype]
    bound = half_step(out.dtype) * (ref.abs() + slack) + slack + tiny
    diff = (out.double() - ref).abs()
    bad = ~(diff <= bound)
    assert not bool(bad.any()), (int(bad.sum()), float((diff - bound).nan_to_num(nan=1e30).max()))


def offsets_of(sizes, head=0):
    ends = [head]
    for s in sizes:
        ends.append(ends[-1] + s)
    return torch.tensor(ends, dtype=torch.int32, device=DEV)


def grouped_reference(x, w, dy, lo_hi):
    """y, dx, dw and the sums of magnitudes of each, in 64 bits."""
    xd, wd = x.double(), w.double()
    G, N, K = w.shape
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(xd), torch.zeros_like(wd)
    sy, sdx, sdw = torch.zeros_like(y), torch.zeros_like(dx), torch.zeros_like(dw)
    for g, (lo, hi) in enumerate(lo_hi):
        if lo >= hi:
            continue
        xg, dg, wg = xd[lo:hi], dy[lo:hi].double(), wd[g]
        y[lo:hi], sy[lo:hi] = xg @ wg.T, xg.abs() @ wg.abs().T
        dx[lo:hi], sdx[lo:hi] = dg @ wg, dg.abs() @ wg.abs()
        dw[g], sdw[g] = dg.T @ xg, dg.abs().T @ xg.abs()
    return (y, sy), (dx, sdx), (dw, sdw)


def ranges_of(offsets, rows):
    """The rows of each group as the documentation says: a running maximum clamped to [0, rows]."""
    o = offsets.tolist()
    out, run = [], min(max(o[0], 0), rows)
    for e in o[1:]:
        end = max(run, min(max(e, 0), rows))
        out.append((run, end))
        run = end
    return out


SIZES = [
    [1], [0, 1], [5, 0, 0, 3], [31, 32, 33], [255, 256, 257], [64, 15, 16, 17, 1, 48, 0],
    [700], [513, 2, 1025], [0, 0, 0], [3] * 40,
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nk", [(8, 8), (72, 136), (256, 64), (264, 520), (1000, 328)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s[:7])))
def test_grouped_matmul_and_gradients(sizes, nk, dtype):
    n, k = nk
    gen = torch.Generator(device=DEV)
    gen.manual_seed(17)
    rows = sum(sizes) + 3
    x = torch.randn(rows, k, device=DEV, generator=gen).to(dtype)
    w = (torch.randn(len(sizes), n, k, device=DEV, generator=gen) * 0.1).to(dtype)
    dy = torch.randn(rows, n, device=DEV, generator=gen).to(dtype)
    off = offsets_of(sizes, head=1)
    # rows of no group hold what must not be seen
    for t in (x, dy):
        t[0] = float("nan")
        t[-2:] = float("inf")
    x.requires_grad_()
    w.requires_grad_()
    y = M.grouped_matmul(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    torch.cuda.synchronize()
    (ry, sy), (rdx, sdx), (rdw, sdw) = grouped_reference(x.detach(), w.detach(), dy, ranges_of(off, rows))
    close(y.detach(), ry, (k + 8) * U * sy)
    close(dx, rdx, (n + 8) * U * sdx)
    close(dw, rdw, (max(sizes) + 8) * U * sdw)
    assert M.operator_status(DEV) == 0


@pytest.mark.parametrize("offsets", [[0, 9, 4, 20], [-7, 3, 3, 500], [40, 40, 40, 40], [30, 10, 35, 12], [2 ** 31 - 1, -2 ** 31, 0, 5]])
def test_any_offsets_are_safe(offsets):
    rows, n, k = 40, 96, 200
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    x, dy = (torch.randn(rows, c, device=DEV, generator=gen).bfloat16() for c in (k, n))
    w = torch.randn(3, n, k, device=DEV, generator=gen).bfloat16()
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    (ry, sy), (rdx, sdx), (rdw, sdw) = grouped_reference(x, w, dy, ranges_of(off, rows))
    close(M.grouped_matmul(x, w, off), ry, (k + 8) * U * sy)
    close(M.grouped_matmul_dgrad(dy, w, off), rdx, (n + 8) * U * sdx)
    close(M.grouped_matmul_wgrad(dy, x, off), rdw, (rows + 8) * U * sdw)


def test_a_groups_infinities_stay_in_the_group():
    sizes, n, k = [7, 9, 20, 5], 64, 96
    gen = torch.Generator(device=DEV)
    gen.manual_seed(4)
    off = offsets_of(sizes)
    x, dy = (torch.randn(sum(sizes), c, device=DEV, generator=gen).bfloat16() for c in (k, n))
    w = torch.randn(4, n, k, device=DEV, generator=gen).bfloat16()
    clean = [M.grouped_matmul(x, w, off), M.grouped_matmul_dgrad(dy, w, off), M.grouped_matmul_wgrad(dy, x, off)]
    x2, dy2, w2 = x.clone(), dy.clone(), w.clone()
    x2[7:16], dy2[7:16], w2[1] = float("nan"), float("inf"), float("-inf")
    y, dx, dw = M.grouped_matmul(x2, w2, off), M.grouped_matmul_dgrad(dy2, w2, off), M.grouped_matmul_wgrad(dy2, x2, off)
    keep = torch.ones(sum(sizes), dtype=torch.bool, device=DEV)
    keep[7:16] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert torch.equal(dw[[0, 2, 3]], clean[2][[0, 2, 3]])
    assert not bool(torch.isfinite(y[7:16]).any())


def test_grouped_matmul_writes_only_its_result():
    sizes, n, k = [33, 0, 130], 72, 64
    off = offsets_of(sizes)
    rows = sum(sizes) + 4
    x, w, dy = (torch.ones(*s, device=DEV, dtype=torch.bfloat16) for s in ((rows, k), (3, n, k), (rows, n)))
    for call, shape in ((lambda o: M.grouped_matmul(x, w, off, out=o), (rows, n)),
                        (lambda o: M.grouped_matmul_dgrad(dy, w, off, out=o), (rows, k)),
                        (lambda o: M.grouped_matmul_wgrad(dy, x, off, out=o), (3, n, k))):
        count = torch.Size(shape).numel()
        raw = torch.full((count + 8192,), 7.0, device=DEV, dtype=torch.bfloat16)
        call(raw[4096:4096 + count].view(shape))
        assert bool((raw[:4096] == 7).all()) and bool((raw[4096 + count:] == 7).all())
        assert not bool((raw[4096:4096 + count] == 7).any())


def test_grouped_gradients_are_exact_differences():
    """The operator is linear in x and in w: with small whole numbers every sum is exact, and the change
    of <dy, y> along a direction is the gradient times it, to the last bit."""
    sizes, n, k = [5, 0, 40, 3], 24, 40
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    off = offsets_of(sizes)
    whole = lambda *s: torch.randint(-1, 2, s, device=DEV, generator=gen).bfloat16()
    x, w, dy, ex, ew = whole(48, k), whole(4, n, k), whole(48, n), whole(48, k), whole(4, n, k)
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(M.grouped_matmul(x, w, off), (x, w), dy)
    with torch.no_grad():
        at = lambda a, b: (M.grouped_matmul(a, b, off).double() * dy.double()).sum()
        assert float(at(x + ex, w) - at(x, w)) == float((dx.double() * ex.double()).sum())
        assert float(at(x, w + ew) - at(x, w)) == float((dw.double() * ew.double()).sum())


def test_gradients_through_strided_and_partial_use():
    off = offsets_of([3, 6])
    x = torch.randn(9, 32, device=DEV).bfloat16().requires_grad_()
    w = torch.randn(2, 16, 32, device=DEV).bfloat16()
    y = M.grouped_matmul(x, w, off)                       # only x asks for a gradient
    (g,) = torch.autograd.grad(y.sum(), x)                # an expanded gradient, all strides zero
    assert torch.equal(g, M.grouped_matmul_dgrad(torch.ones(9, 16, device=DEV, dtype=torch.bfloat16), w, off))
    w.requires_grad_()
    (h,) = torch.autograd.grad(M.grouped_matmul(x.detach(), w, off)[:, 1::2].sum(), w)
    ones = torch.zeros(9, 16, device=DEV, dtype=torch.bfloat16)
    ones[:, 1::2] = 1
    assert torch.equal(h, M.grouped_matmul_wgrad(ones, x.detach(), off))


def test_second_derivatives_are_refused():
    off = offsets_of([4])
    x = torch.randn(4, 16, device=DEV).bfloat16().requires_grad_()
    w = torch.randn(1, 8, 16, device=DEV).bfloat16().requires_grad_()
    dy = torch.ones(4, 8, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    (dx,) = torch.autograd.grad(M.grouped_matmul(x, w, off), x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.float().sum(), dy)


# ----------------------------------------------------------------------------- e4m3 products
def block_inputs(m, n, k, quant, seed, spread=1.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    x = (torch.randn(m, k, device=DEV, generator=gen) * torch.exp(spread * torch.randn(m, k // 128, device=DEV, generator=gen)).repeat_interleave(128, 1)).bfloat16()
    a, sa = api.quantise_rows(x, quant)
    w = torch.randn(n, k, device=DEV, generator=gen).to(torch.float8_e4m3fn)
    sw = torch.exp2(torch.randint(-6, 5, ((n + 127) // 128, k // 128), device=DEV, generator=gen).float())
    if quant == "block128":
        sw = sw * (1 + torch.rand(sw.shape, device=DEV, generator=gen))
    return a, sa, w, sw


def scale_values(sa, quant, blocks):
    return sa.view(torch.float32).double() if quant == "block128" else torch.exp2(sa[:, :blocks].double() - 127)


def block_reference(a, sa, w, sw, quant):
    blocks = a.shape[1] // 128
    av = a.view(torch.float8_e4m3fn).double() * scale_values(sa, quant, blocks).repeat_interleave(128, 1)
    wv = w.view(torch.float8_e4m3fn).double() * sw.double().repeat_interleave(128, 1).repeat_interleave(128, 0)[:w.shape[0]]
    return av @ wv.T, av.abs() @ wv.abs().T


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("nk", [(1, 128), (7, 256), (128, 384), (130, 640), (576, 1024), (1001, 2048)])
def test_matmul_block128(m, nk, quant):
    n, k = nk
    a, sa, w, sw = block_inputs(m, n, k, quant, seed=m * 7 + n)
    out = M.matmul_block128(a, sa, w, sw, quant)
    ref, mag = block_reference(a, sa, w, sw, quant)
    close(out, ref, (k + 8) * U * mag)
    assert M.operator_status(DEV) == 0


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("mnk", [(1024, 2048, 512), (2049, 300, 1408), (640, 4096, 7168)])
def test_matmul_block128_large(mnk, quant):
    m, n, k = mnk
    a, sa, w, sw = block_inputs(m, n, k, quant, seed=n)
    out = M.matmul_block128(a.view(torch.float8_e4m3fn), sa, w.view(torch.uint8), sw, quant)
    ref, mag = block_reference(a, sa, w, sw, quant)
    close(out, ref, (k + 8) * U * mag)


def test_matmul_block128_takes_scales_as_floats_and_views():
    a, sa, w, sw = block_inputs(9, 200, 640, "block128", seed=1)
    want = M.matmul_block128(a, sa, w, sw)
    assert torch.equal(M.matmul_block128(a, sa.view(torch.float32), w, sw), want)
    # rows taken from the middle of larger tensors: the scales are then aligned to 4 bytes only
    big_a, big_s = torch.cat([a, a]), torch.cat([sa, sa])
    assert torch.equal(M.matmul_block128(big_a[5:14], big_s[5:14], w, sw), torch.cat([want, want])[5:14])


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("m", [3, 200])
def test_matmul_block128_special_values(m, quant):
    """NaN bytes reach exactly the results that use them; all-zero rows give zeros; nothing is written outside."""
    n, k = 150, 384
    a, sa, w, sw = block_inputs(m, n, k, quant, seed=8)
    a[1] = 0
    a[2, 200] = 0x7F
    w.view(torch.uint8)[149, 5] = 0xFF
    raw = torch.full((m * n + 8192,), 7.0, device=DEV, dtype=torch.bfloat16)
    out = M.matmul_block128(a, sa, w, sw, quant, out=raw[4096:4096 + m * n].view(m, n))
    nan = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    nan[2], nan[:, 149] = True, True
    assert torch.equal(torch.isnan(out), nan)
    assert bool((out[1, :149] == 0).all())
    assert bool((raw[:4096] == 7).all()) and bool((raw[4096 + m * n:] == 7).all())


@pytest.mark.parametrize("m", [2, 40, 300])
def test_power_of_two_scales_at_their_limits(m):
    """The smallest scale, the largest finite one and NaN; weight scales count by their exponent."""
    n, k = 136, 256
    a, sa, w, sw = block_inputs(m, n, k, "block128_ue8m0", seed=12)
    sa[0, 0], sa[1, 1] = 0, 255
    sw.fill_(1.0)
    out = M.matmul_block128(a, sa, w, sw, "block128_ue8m0")
    assert bool(torch.isnan(out[1]).all()) and not bool(torch.isnan(out[0]).any())
    keep = [i for i in range(m) if i != 1]
    ref, mag = block_reference(a[keep], sa[keep], w, sw, "block128_ue8m0")
    close(out[keep], ref, (k + 8) * U * mag + 2.0 ** -110)
    assert torch.equal(M.matmul_block128(a[keep], sa[keep], w, sw * 1.75, "block128_ue8m0"), out[keep])


def test_every_kernel_of_the_product_is_reached():
    """Rows from one to many: the tiles of 16, 32 and 128 rows with and without a split of K, and the
    128 x 256 tiles, each against 64 bits (the choice goes by m, n and k)."""
    for quant in ("block128", "block128_ue8m0"):
        for m, n, k in ((1, 128, 128), (16, 384, 4096), (17, 2304, 4096), (40, 4096, 2048), (100, 7744, 1024), (130, 640, 1920), (70, 18432, 256), (520, 2048, 640)):
            a, sa, w, sw = block_inputs(m, n, k, quant, seed=m)
            ref, mag = block_reference(a, sa, w, sw, quant)
            close(M.matmul_block128(a, sa, w, sw, quant), ref, (k + 8) * U * mag)
    assert M.operator_status() == 0


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("mnk", [(5, 63, 128), (5, 63, 640), (5, 63, 1024), (5, 63, 2048), (250, 4999, 384), (639, 200, 1408), (640, 63, 4096),
                                 (300, 63, 7168), (100, 18431, 640), (130, 2303, 5632), (130, 1100, 7168), (639, 200, 5632),
                                 (1030, 7743, 128), (333, 18431, 128), (2040, 2300, 3968)])
def test_every_form_of_the_choice(mnk, quant):
    """Sizes for 16, 32 and 128 rows to a tile, each with K whole and shared by 2, 4 and 8 CTAs, and for
    128 x 256 tiles of one CTA, by the estimates that choose among them."""
    m, n, k = mnk
    a, sa, w, sw = block_inputs(m, n, k, quant, seed=m + n)
    ref, mag = block_reference(a, sa, w, sw, quant)
    close(M.matmul_block128(a, sa, w, sw, quant), ref, (k + 8) * U * mag)
    assert M.operator_status() == 0


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("mnk", [(600, 7700, 7296), (7960, 3000, 2432), (2304, 18432, 1280)])
def test_tiles_of_a_pair_of_ctas(mnk, quant):
    """Sizes at which two CTAs share tiles of 256 x 256: a second half without rows, widths that are no
    multiple of 8, odd numbers of K blocks, several bands of rows."""
    m, n, k = mnk
    a, sa, w, sw = block_inputs(m, n, k, quant, seed=m + n)
    ref, mag = block_reference(a, sa, w, sw, quant)
    close(M.matmul_block128(a, sa, w, sw, quant), ref, (k + 8) * U * mag)
    assert M.operator_status() == 0


# ----------------------------------------------------------------------------- the gated activation
def silu_reference(gu, weight, dy):
    g, u = gu.double().chunk(2, 1)
    w = torch.ones(gu.shape[0], 1, dtype=torch.float64, device=gu.device) if weight is None else weight.double()[:, None]
    d = dy.double()
    s = torch.sigmoid(g)
    slack = (12 + 1.173 * g.abs()) * U
    y = w * g * s * u
    dg, du = w * d * u * s * (1 + g * (1 - s)), w * d * g * s
    terms = d * g * s * u
    width = g.shape[1]
    dw = terms.sum(1), ((width + 8) * U + slack.max(1).values) * terms.abs().sum(1)
    return (y, slack * y.abs()), (torch.cat([dg, du], 1), torch.cat([2 * slack * (w * d * u * s).abs() * (1 + g.abs()), slack * du.abs()], 1)), dw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 24), (257, 512), (5, 520), (33, 2048), (2, 14336), (1000, 104)])
def test_silu_mul_and_gradients(rows, width, weighted, dtype):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(rows + width)
    gu = (torch.randn(rows, 2 * width, device=DEV, generator=gen) * 2).to(dtype)
    dy = torch.randn(rows, width, device=DEV, generator=gen).to(dtype)
    weight = torch.rand(rows, device=DEV, generator=gen) - 0.25 if weighted else None
    if weighted:
        weight[0] = 0.0
    (ry, sy), (rg, sg), (rw, sw) = silu_reference(gu, weight, dy)
    close(M.silu_mul(gu, weight), ry, sy)
    leaves = [gu.requires_grad_()] + ([weight.requires_grad_()] if weighted else [])
    grads = torch.autograd.grad(M.silu_mul(gu, weight), leaves, dy)
    close(grads[0], rg, sg)
    if weighted:
        close(grads[1], rw, sw)


def test_silu_mul_far_values():
    """Gates of any size, infinities and NaN: the formula's values, not overflow's."""
    g = torch.tensor([0.0, -0.0, 30.0, -30.0, 87.0, -87.0, -100.0, 3e4, -3e4, float("inf")], device=DEV)
    gu = torch.zeros(2, 32, device=DEV, dtype=torch.bfloat16)
    gu[0, :10], gu[0, 16:] = g.bfloat16(), 2.0
    gu[1, 3], gu[1, 16:] = float("nan"), 1.0
    y = M.silu_mul(gu)
    ref = torch.nn.functional.silu(gu[0, :16].double()) * 2
    finite = torch.isfinite(ref)
    slack = (12 + 1.173 * gu[0, :16].double().abs()) * U * ref.abs()
    close(y[0][finite], ref[finite], slack[finite] + 2.0 ** -120)
    assert bool(torch.isinf(y[0, 9]))
    assert bool(torch.isnan(y[1, 3])) and int(torch.isnan(y[1]).sum()) == 1


def test_silu_gradient_against_differences():
    """The operator's gradient against central differences of the definition in 64 bits (step 1e-4: the
    truncation is below 1e-8 of the sum of magnitudes, far inside the rounding of the gradient)."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(2)
    gu = torch.randn(6, 64, device=DEV, generator=gen).half()
    weight = torch.rand(6, device=DEV, generator=gen)
    dy = torch.randn(6, 32, device=DEV, generator=gen).half()
    dgu, dweight = M.silu_mul_backward(gu, dy, weight)

    def loss(a, b):
        g, u = a.chunk(2, 1)
        return (b[:, None] * torch.nn.functional.silu(g) * u * dy.double()).sum()
    h = 1e-4
    for _ in range(8):
        ea = torch.randn(6, 64, device=DEV, generator=gen).double()
        eb = torch.randn(6, device=DEV, generator=gen).double()
        want = (loss(gu.double() + h * ea, weight.double() + h * eb) - loss(gu.double() - h * ea, weight.double() - h * eb)) / (2 * h)
        got = (dgu.double() * ea).sum() + (dweight.double() * eb).sum()
        size = (dgu.double() * ea).abs().sum() + (dweight.double() * eb).abs().sum()
        assert abs(float(got - want)) <= float(size) * (half_step(torch.float16) + 1e-5)


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 128), (5, 384), (300, 1152), (16, 14336)])
def test_silu_mul_quantise_is_quantise_of_silu_mul(rows, width, weighted, quant):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(rows)
    gu = torch.randn(rows, 2 * width, device=DEV, generator=gen).bfloat16()
    gu[rows // 2] = 0                                     # a row whose groups are all zero
    weight = torch.rand(rows, device=DEV, generator=gen) if weighted else None
    q, s = M.silu_mul_quantise(gu, quant, weight)
    q2, s2 = api.quantise_rows(M.silu_mul(gu, weight), quant)
    used = width // 128 * (4 if quant == "block128" else 1)   # the bytes that pad a row's scales are nobody's
    assert torch.equal(q, q2) and torch.equal(s[:, :used], s2[:, :used])


# ----------------------------------------------------------------------------- streams, graphs, repeatability
def _everything():
    """One call of each operator on fixed inputs: (call, inputs that may change between replays)."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(11)
    sizes = [40, 0, 300, 7, 1]
    off = offsets_of(sizes)
    x = torch.randn(350, 256, device=DEV, generator=gen).bfloat16()
    w = torch.randn(5, 320, 256, device=DEV, generator=gen).bfloat16()
    dy = torch.randn(350, 320, device=DEV, generator=gen).bfloat16()
    rw = torch.rand(350, device=DEV, generator=gen)
    few = offsets_of([1, 0, 2, 0, 1])
    blocks = {q: block_inputs(m, 392, 512, q, seed=6) for q, m in (("block128", 200), ("block128_ue8m0", 200))}
    small = {q: tuple(t[:2].contiguous() if i < 2 else t for i, t in enumerate(v)) for q, v in blocks.items()}

    def call(stream=None):
        out = [M.grouped_matmul(x, w, off, stream=stream), M.grouped_matmul_dgrad(dy, w, off, stream=stream),
               M.grouped_matmul_wgrad(dy, x, off, stream=stream), M.grouped_matmul(x[:4], w, few, stream=stream),
               M.grouped_matmul_dgrad(dy[:4], w, few, stream=stream),
               M.silu_mul(dy, rw, stream=stream), *M.silu_mul_backward(dy, dy[:, :160].contiguous(), rw, stream=stream)]
        for q in blocks:
            out += [M.matmul_block128(*blocks[q], quant=q, stream=stream), M.matmul_block128(*small[q], quant=q, stream=stream)]
        return out
    return call, (x, w, dy, rw)


def test_repeated_calls_give_the_same_bits():
    call, _ = _everything()
    first = [t.clone() for t in call()]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))


def test_calls_on_other_streams():
    call, _ = _everything()
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(3)]
    got = [call(s) for s in streams]                      # the same calls at once on three streams
    for s in streams:
        s.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(want, g))
    with torch.cuda.stream(streams[0]):
        g = call()
    streams[0].synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, g))


def test_two_captured_graphs_replayed_together():
    call, inputs = _everything()
    call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for t in inputs:
        t.mul_(0.5)                                       # replays see the new values
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_a_captured_training_step():
    off = offsets_of([10, 0, 23])
    x = torch.randn(33, 64, device=DEV).bfloat16().requires_grad_()
    w1 = torch.randn(3, 96, 64, device=DEV).bfloat16().requires_grad_()
    dy = torch.randn(33, 48, device=DEV).bfloat16()

    def step():
        return torch.autograd.grad(M.silu_mul(M.grouped_matmul(x, w1, off)), (x, w1), dy)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    with torch.no_grad():
        x.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_results_given_by_the_caller():
    off = offsets_of([3, 30])
    x, w = torch.randn(33, 64, device=DEV).bfloat16(), torch.randn(2, 48, 64, device=DEV).bfloat16()
    dy = torch.randn(33, 48, device=DEV).bfloat16()
    gu, rw = torch.randn(9, 512, device=DEV).half(), torch.rand(9, device=DEV)
    q = block_inputs(5, 70, 256, "block128", seed=2)
    for call in (lambda **o: M.grouped_matmul(x, w, off, **o), lambda **o: M.grouped_matmul_dgrad(dy, w, off, **o),
                 lambda **o: M.grouped_matmul_wgrad(dy, x, off, **o), lambda **o: M.silu_mul(gu, rw, **o), lambda **o: M.matmul_block128(*q, **o)):
        want = call()
        out = torch.empty_like(want)
        assert call(out=out) is out and torch.equal(out, want)
    qs, ss = M.silu_mul_quantise(gu, "block128", rw)
    q2, s2 = torch.empty_like(qs), torch.empty_like(ss)
    M.silu_mul_quantise(gu, "block128", rw, q=q2, scales=s2)
    assert torch.equal(qs, q2) and torch.equal(ss, s2)


def test_calls_from_a_thread_that_has_made_none():
    """The first CUDA work of a thread: nothing has made the context current there yet."""
    import threading
    call, _ = _everything()
    want, got = call(), []
    torch.cuda.synchronize()
    t = threading.Thread(target=lambda: got.extend(call()))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_threads_at_once():
    import threading
    call, _ = _everything()
    want = call()
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        s = torch.cuda.Stream(DEV)
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = call()
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))


def test_the_wrappers_refuse_what_does_not_fit():
    off = offsets_of([2, 2])
    x = torch.randn(4, 64, device=DEV).bfloat16()
    w = torch.randn(2, 32, 64, device=DEV).bfloat16()
    q = torch.zeros(4, 128, dtype=torch.uint8, device=DEV)
    s, sw = torch.ones(4, 1, device=DEV), torch.ones(1, 1, device=DEV)
    wide = torch.randn(4, 128, device=DEV).bfloat16()
    for call in (lambda: M.grouped_matmul(x.half(), w, off), lambda: M.grouped_matmul(x.float(), w.float(), off),
                 lambda: M.grouped_matmul(x[:, :60], w[:, :, :60], off), lambda: M.grouped_matmul(wide[:, ::2], w, off),
                 lambda: M.grouped_matmul(x[:, :60].contiguous(), w[:, :, :60].contiguous(), off),
                 lambda: M.grouped_matmul(x, w, off.long()), lambda: M.grouped_matmul(x, w, off[:2]),
                 lambda: M.grouped_matmul(x, w, off.cpu()), lambda: M.grouped_matmul(x, w[0], off),
                 lambda: M.grouped_matmul(x.requires_grad_(), w, off, out=torch.empty(4, 32, device=DEV, dtype=torch.bfloat16)),
                 lambda: M.grouped_matmul_wgrad(x.detach(), x.detach()[:3], off), lambda: M.grouped_matmul_dgrad(x.detach(), w, off),
                 lambda: M.matmul_block128(q, s[:3], q, sw), lambda: M.matmul_block128(q, s, q, sw.half()),
                 lambda: M.matmul_block128(q, s, q, sw, quant="block128_ue8m0"), lambda: M.matmul_block128(q[:, :100], s, q[:, :100], sw),
                 lambda: M.matmul_block128(q, s, q, sw, out=torch.empty(4, 4, device=DEV)),
                 lambda: M.silu_mul(wide.float()), lambda: M.silu_mul(wide[:, :24].contiguous()), lambda: M.silu_mul(wide, s),
                 lambda: M.silu_mul(wide, s[:, 0].double()), lambda: M.silu_mul_quantise(wide, "block128"),
                 lambda: M.silu_mul_backward(wide, wide)):
        with pytest.raises(M.FmoeError):
            call()


# ----------------------------------------------------------------------------- as they are used
def _route(T, E, K, gen):
    ids, weight = M.route(torch.randn(T, E, device=DEV, generator=gen), K)
    order = torch.argsort(ids.flatten(), stable=True)
    counts = torch.bincount(ids.flatten(), minlength=E)
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    return ids, weight, order, off


def test_an_expert_layer_trains_through_its_parts():
    """Routed rows, both products, the weighted activation and the sum per token: the result against the
    fused operator, all gradients against 64-bit autograd of the same layer.  In bf16 every stage rounds
    (2^-8 of its value); a handful of roundings along every path, independent from element to element,
    leave the whole within 2^-6 in the 2-norm."""
    T, H, I, E, K = 200, 256, 384, 8, 2
    gen = torch.Generator(device=DEV)
    gen.manual_seed(21)
    ids, weight, order, off = _route(T, E, K, gen)
    x = torch.randn(T, H, device=DEV, generator=gen).bfloat16()
    w1 = (torch.randn(E, 2 * I, H, device=DEV, generator=gen) * 0.05).bfloat16()
    w2 = (torch.randn(E, H, I, device=DEV, generator=gen) * 0.05).bfloat16()
    dy = torch.randn(T, H, device=DEV, generator=gen).bfloat16()
    token = order // K

    def layer(x, w1, w2, weight):
        gu = M.grouped_matmul(x[token], w1, off)
        rows = M.grouped_matmul(M.silu_mul(gu, weight.flatten()[order]), w2, off)
        return torch.zeros(T, H, device=DEV).index_add(0, token, rows.float()).bfloat16()
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2, weight)]
    y = layer(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)

    fused = M.fused_moe(M.FusedMoeTraits(), M.FusedMoeArgs(a=x, g=w1, d=w2, topk_ids=ids, topk_weight=weight))
    rel = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())
    assert rel(y.detach(), fused) <= 2.0 ** -6

    exact = [t.detach().double().requires_grad_() for t in leaves]
    xe, w1e, w2e, we = exact
    flat = ids.flatten()[order].long()
    gu = torch.einsum("rh,rih->ri", xe[token], w1e[flat])
    act = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:] * we.flatten()[order][:, None]
    ye = torch.zeros(T, H, device=DEV, dtype=torch.float64).index_add(0, token, torch.einsum("ri,rhi->rh", act, w2e[flat]))
    for got, want in zip(grads, torch.autograd.grad(ye, exact, dy.double())):
        assert rel(got, want) <= 2.0 ** -6
    assert M.operator_status(DEV) == 0


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("T", [1, 130])
def test_a_dense_layer_serves_in_e4m3(T, quant):
    """quantise -> product -> gated activation as e4m3 -> product: every stage against 64 bits on its own
    inputs, so each has its own bound."""
    H, I = 512, 640
    gen = torch.Generator(device=DEV)
    gen.manual_seed(T)
    _, _, w1, s1 = block_inputs(1, 2 * I, H, quant, seed=31)
    _, _, w2, s2 = block_inputs(1, H, I, quant, seed=32)
    x = torch.randn(T, H, device=DEV, generator=gen).bfloat16()
    a, sa = M.quantise_rows(x, quant)
    gu = M.matmul_block128(a, sa, w1, s1 / 64, quant)
    ref, mag = block_reference(a, sa, w1, s1 / 64, quant)
    close(gu, ref, (H + 8) * U * mag)
    q, sq = M.silu_mul_quantise(gu, quant)
    out = M.matmul_block128(q, sq, w2, s2, quant)
    ref, mag = block_reference(q, sq, w2, s2, quant)
    close(out, ref, (I + 8) * U * mag)
    g, u = gu.double().chunk(2, 1)
    act = torch.nn.functional.silu(g) * u
    v = q.view(torch.float8_e4m3fn).double() * scale_values(sq, quant, I // 128).repeat_interleave(128, 1)
    # rounded to bf16, then to e4m3 (2^-4 of the value, or half of its smallest step, 2^-10, times the scale)
    step = scale_values(sq, quant, I // 128).repeat_interleave(128, 1) * 2.0 ** -10
    assert bool(((v - act).abs() <= (2.0 ** -4 + 2.0 ** -7) * act.abs() + step).all())


def test_torch_ops_have_the_same_results_and_gradients():
    import therock_b200.torch_op  # noqa: F401
    ns = torch.ops.therock_b200
    off = offsets_of([10, 0, 23])
    x = torch.randn(33, 64, device=DEV).bfloat16().requires_grad_()
    w = torch.randn(3, 96, 64, device=DEV).bfloat16().requires_grad_()
    rw = torch.rand(33, device=DEV).requires_grad_()
    dy = torch.randn(33, 48, device=DEV).bfloat16()
    a = ns.silu_mul(ns.grouped_matmul(x, w, off), rw)
    b = M.silu_mul(M.grouped_matmul(x, w, off), rw)
    assert torch.equal(a, b)
    assert all(torch.equal(g, h) for g, h in zip(torch.autograd.grad(a, (x, w, rw), dy), torch.autograd.grad(b, (x, w, rw), dy)))
    (g,) = torch.autograd.grad(ns.silu_mul(x), x, dy[:, :32])
    assert torch.equal(g, M.silu_mul_backward(x.detach(), dy[:, :32].contiguous())[0])
    q = block_inputs(5, 70, 256, "block128", seed=2)
    assert torch.equal(ns.matmul_block128(*q), M.matmul_block128(*q))


# ----------------------------------------------------------------------------- calls that are easy to get wrong
def _differentiable_calls():
    import therock_b200.torch_op  # noqa: F401
    ns = torch.ops.therock_b200
    off = offsets_of([10, 0, 23])
    x = torch.randn(33, 64, device=DEV).bfloat16()
    w = torch.randn(3, 96, 64, device=DEV).bfloat16()
    rw = torch.rand(33, device=DEV)
    return {"grouped": ((x, w), lambda x, w: M.grouped_matmul(x, w, off)), "silu": ((x, rw), M.silu_mul),
            "op_grouped": ((x, w), lambda x, w: ns.grouped_matmul(x, w, off)), "op_silu": ((x, rw), ns.silu_mul)}


@pytest.mark.parametrize("name", ["grouped", "silu", "op_grouped", "op_silu"])
def test_a_captured_backward_pass_beside_a_living_graph(name):
    """A leaf's node lives as long as any graph of it does, on the stream that graph was recorded on; the
    default stream cannot join a capture, so the pass is refused, and goes through once the graph is gone."""
    leaves, f = _differentiable_calls()[name]
    leaves = [t.requires_grad_() for t in leaves]

    def step():
        return torch.autograd.grad(f(*leaves), leaves, dy)
    living = f(*leaves)
    dy = torch.randn_like(living)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(g):
            step()
    want = torch.autograd.grad(living, leaves, dy)        # the eager graph is as good as before
    del living, g
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_captured_backward_pass_beside_a_graph_of_a_side_stream():
    leaves, f = _differentiable_calls()["grouped"]
    leaves = [t.requires_grad_() for t in leaves]
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        living = f(*leaves)
        dy = torch.randn_like(living)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = torch.autograd.grad(f(*leaves), leaves, dy)
    g.replay()
    torch.cuda.synchronize()
    want = torch.autograd.grad(living, leaves, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", ["grouped", "silu"])
def test_forward_mode_derivatives_are_refused(name):
    import torch.autograd.forward_ad as fwd
    (x, other), f = _differentiable_calls()[name]
    with fwd.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(fwd.make_dual(x, torch.ones_like(x)), other)


def test_results_share_no_memory_with_inputs():
    off = offsets_of([2, 2])
    x, w = torch.zeros(4, 64, device=DEV).bfloat16(), torch.zeros(2, 64, 64, device=DEV).bfloat16()
    q, s, sw = torch.zeros(4, 128, dtype=torch.uint8, device=DEV), torch.ones(4, 1, device=DEV), torch.ones(1, 1, device=DEV)
    gu = torch.zeros(4, 256, device=DEV).half()
    flat = gu.view(-1)
    for call in (lambda: M.grouped_matmul(x, w, off, out=x), lambda: M.grouped_matmul(x, w, off, out=w[1, 60:]),
                 lambda: M.grouped_matmul_dgrad(x, w, off, out=x), lambda: M.grouped_matmul_wgrad(w[0], w[1], off, out=w),
                 lambda: M.silu_mul(gu, out=flat[512:].view(4, 128)),
                 lambda: M.silu_mul_quantise(gu, "block128", q=flat[:256].view(torch.uint8).view(4, 128)),
                 lambda: M.silu_mul_quantise(gu, "block128", q=q, scales=q.view(-1)[496:].view(4, 4)),
                 lambda: M.matmul_block128(q, s, q, sw, out=q.view(-1)[:32].view(torch.bfloat16).view(4, 4))):
        with pytest.raises(M.FmoeError, match="share"):
            call()


def test_results_of_more_than_two_to_the_31_elements():
    """Row indices times widths that pass 32 bits: the first, the middle and the last rows."""
    rows, n = 270000, 8192
    at = torch.tensor([0, 1, 131071, 262143, 262144, 262145, rows - 2, rows - 1], device=DEV)
    torch.manual_seed(11)
    off = torch.tensor([0, 262145, rows - 1], dtype=torch.int32, device=DEV)     # and a last row of no group
    x = torch.randn(rows, 8, device=DEV).bfloat16()
    w = torch.randn(2, n, 8, device=DEV).bfloat16()
    y = M.grouped_matmul(x, w, off)
    xd, group = x[at].double(), (at >= 262145).long()
    ref = torch.einsum("rk,rnk->rn", xd, w.double()[group])
    mag = torch.einsum("rk,rnk->rn", xd.abs(), w.double().abs()[group])
    ref[-1], mag[-1] = 0, 0
    close(y[at], ref, (8 + 8) * U * mag)
    # y as the gradient: its sums over 8192 columns and over the rows
    dx = M.grouped_matmul_dgrad(y, w, off)
    yd = y[at].double()
    ref = torch.einsum("rn,rnk->rk", yd, w.double()[group])
    mag = torch.einsum("rn,rnk->rk", yd.abs(), w.double().abs()[group])
    close(dx[at], ref, (n + 8) * U * mag)
    dw = M.grouped_matmul_wgrad(y, x, off)
    lo, hi = 262145, rows - 1
    yg, xg = y[lo:hi].double(), x[lo:hi].double()
    close(dw[1], yg.T @ xg, (hi - lo + 8) * U * (yg.abs().T @ xg.abs()))
    del dw, dx, yg
    act = M.silu_mul(y)
    g, u = y[at].double().chunk(2, dim=1)
    slack = (12 + 1.173 * g.abs()) * U
    close(act[at], g * torch.sigmoid(g) * u, slack * (g * torch.sigmoid(g) * u).abs() + 2.0 ** -140)
    del y, act
    a, sa, b, sb = block_inputs(rows, n, 128, "block128", seed=4)
    out = M.matmul_block128(a, sa, b, sb)
    ref, mag = block_reference(a[at], sa[at], b, sb, "block128")
    close(out[at], ref, (128 + 8) * U * mag)


def test_weights_of_more_than_two_to_the_31_elements():
    groups, n, k = 520, 2048, 2056
    torch.manual_seed(12)
    w = torch.empty(groups, n, k, device=DEV, dtype=torch.bfloat16).normal_()
    sizes = [0] * groups
    sizes[0], sizes[511], sizes[519] = 3, 2, 20
    off = offsets_of(sizes)
    x, dy = torch.randn(25, k, device=DEV).bfloat16(), torch.randn(25, n, device=DEV).bfloat16()
    spans = [(0, 0, 3), (511, 3, 5), (519, 5, 25)]
    y, dx, dw = M.grouped_matmul(x, w, off), M.grouped_matmul_dgrad(dy, w, off), M.grouped_matmul_wgrad(dy, x, off)
    for g, lo, hi in spans:
        xd, dd, wd = x[lo:hi].double(), dy[lo:hi].double(), w[g].double()
        close(y[lo:hi], xd @ wd.T, (k + 8) * U * (xd.abs() @ wd.abs().T))
        close(dx[lo:hi], dd @ wd, (n + 8) * U * (dd.abs() @ wd.abs()))
        close(dw[g], dd.T @ xd, (hi - lo + 8) * U * (dd.abs().T @ xd.abs()))
    assert not bool(dw[1:511].any()) and not bool(dw[512:519].any())


def test_the_first_call_of_a_process_may_be_captured():
    """Set-up on a first call (attributes, occupancy) does not break a capture."""
    import subprocess
    import sys
    text = """
import torch, therock_b200 as M
d = "cuda:0"
torch.manual_seed(0)
off = torch.tensor([0, 5, 33], dtype=torch.int32, device=d)
x, w = torch.randn(33, 64, device=d).bfloat16(), torch.randn(2, 256, 64, device=d).bfloat16()
a, b = torch.randn(33, 256, device=d).to(torch.float8_e4m3fn), torch.randn(70, 256, device=d).to(torch.float8_e4m3fn)
sa, sb = torch.rand(33, 2, device=d), torch.rand(1, 2, device=d)
def calls():
    gu = M.grouped_matmul(x, w, off)
    y = M.silu_mul(gu)
    q, s = M.silu_mul_quantise(gu, "block128")
    dx, dw = M.grouped_matmul_dgrad(gu, w, off), M.grouped_matmul_wgrad(gu, x, off)
    return gu, y, q, s, dx, dw, M.matmul_block128(a, sa, b, sb)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = calls()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, calls()))
print("same")
"""
    r = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
