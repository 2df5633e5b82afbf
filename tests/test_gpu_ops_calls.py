"""Calls of the expert layer's parts beside the plain ones: results given by the caller inside a graph,
tracers, derivatives of other kinds, hooks on what a graph keeps."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import therock_b200 as M
from tests.test_gpu_ops import DEV, block_inputs, offsets_of

pytestmark = pytest.mark.gpu


def _calls_with_results():
    """name: (the call, its results' keyword names)"""
    off = offsets_of([3, 30])
    x, w = torch.randn(33, 64, device=DEV).bfloat16(), torch.randn(2, 48, 64, device=DEV).bfloat16()
    dy = torch.randn(33, 48, device=DEV).bfloat16()
    gu, rw = torch.randn(9, 512, device=DEV).half(), torch.rand(9, device=DEV)
    q = block_inputs(5, 70, 256, "block128", seed=2)
    return {"y": (lambda **o: M.grouped_matmul(x, w, off, **o), ("out",)), "dx": (lambda **o: M.grouped_matmul_dgrad(dy, w, off, **o), ("out",)),
            "dw": (lambda **o: M.grouped_matmul_wgrad(dy, x, off, **o), ("out",)), "silu": (lambda **o: M.silu_mul(gu, rw, **o), ("out",)),
            "block": (lambda **o: M.matmul_block128(*q, **o), ("out",)),
            "quantise": (lambda **o: M.silu_mul_quantise(gu, "block128", rw, **o), ("q", "scales"))}


@pytest.mark.parametrize("name", ["y", "dx", "dw", "silu", "block", "quantise"])
def test_a_result_over_a_tensor_that_a_graph_has_saved(name):
    """The graph's backward pass raises, as it does after any write in place, and does not use the new values."""
    call, names = _calls_with_results()[name]
    first = call()
    results = [torch.empty_like(t) for t in (first if isinstance(first, tuple) else (first,))]
    leaves = [torch.ones(t.shape, device=DEV, requires_grad=True) for t in results]
    with torch.no_grad():
        call(**dict(zip(names, results)))
    losses = [(leaf * t).sum() for leaf, t in zip(leaves, results)]       # each keeps its result for the leaf's gradient
    with torch.no_grad():
        call(**dict(zip(names, results)))
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("name", ["y", "dx", "dw", "silu", "block"])
def test_a_result_that_requires_a_gradient_is_refused(name):
    call, (key,) = _calls_with_results()[name]
    out = torch.empty_like(call()).requires_grad_()
    with pytest.raises(M.FmoeError, match="gradient"):
        call(**{key: out})
    with torch.no_grad():
        assert call(**{key: out}) is out


@pytest.mark.parametrize("recording", [True, False])
@pytest.mark.parametrize("second", [False, True])
@pytest.mark.parametrize("name", ["grouped", "silu"])
def test_a_tangent_is_not_dropped(name, second, recording):
    """Forward-mode derivatives are recorded under torch.no_grad too, so the call is refused there as well,
    with a result given by the caller or without."""
    off = offsets_of([10, 0, 23])
    x, w, rw = torch.randn(33, 64, device=DEV).bfloat16(), torch.randn(3, 32, 64, device=DEV).bfloat16(), torch.rand(33, device=DEV)
    f, inputs = (lambda a, b, **o: M.grouped_matmul(a, b, off, **o), [x, w]) if name == "grouped" else (M.silu_mul, [x, rw])
    out = f(*inputs)
    with fwd.dual_level(), torch.set_grad_enabled(recording):
        inputs[second] = fwd.make_dual(inputs[second], torch.ones_like(inputs[second]))
        for o in ({}, {"out": out}):
            with pytest.raises(M.FmoeError, match="forward-mode"):
                f(*inputs, **o)
        with fwd._set_fwd_grad_enabled(False):
            assert torch.equal(f(*inputs), out)


def _layer(name):
    import therock_b200.torch_op  # noqa: F401
    off = offsets_of([10, 0, 23])
    op = M.grouped_matmul if name == "M" else torch.ops.therock_b200.grouped_matmul
    x, w = (torch.randn(*s, device=DEV).bfloat16().requires_grad_() for s in ((33, 64), (3, 96, 64)))
    return x, w, lambda x, w: op(x, w, off), torch.randn(33, 96, device=DEV).bfloat16()


@pytest.mark.parametrize("name", ["M", "op"])
def test_a_captured_backward_pass_beside_a_living_graph_of_a_leaf_further_on(name):
    """The leaf whose node is on the default stream lies behind another operation."""
    x, w, f, dy = _layer(name)
    w.requires_grad_(False)
    living = x.exp()

    def step():
        return torch.autograd.grad(f(x.neg(), w), x, dy)[0]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(g):
            step()
    del living, g
    want = step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, got)


@pytest.mark.parametrize("name", ["M", "op"])
def test_a_captured_backward_pass_that_leaves_a_living_graphs_leaf_alone(name):
    """A gradient that the pass does not ask for stands in nobody's way."""
    x, w, f, dy = _layer(name)
    living = f(x.detach(), w)

    def step():
        return torch.autograd.grad(f(x, w), x, dy)[0]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(step(), got)
    (dw,) = torch.autograd.grad(living, w, dy)
    assert torch.equal(dw, M.grouped_matmul_wgrad(dy, x.detach(), offsets_of([10, 0, 23])))


def _saved_through(give_back):
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, give_back)


@pytest.mark.parametrize("which", ["grouped", "silu"])
def test_what_a_graph_kept_may_come_back_with_other_strides(which):
    x, w, f, dy = _layer("M")
    rw = torch.rand(33, device=DEV).requires_grad_()
    leaves, f, dy = ([x, w], f, dy) if which == "grouped" else ([x, rw], M.silu_mul, dy[:, :32].contiguous())
    want = torch.autograd.grad(f(*leaves), leaves, dy)

    def strided(t):
        return t if t.dim() < 2 else t.mT.contiguous().mT
    with _saved_through(strided):
        y = f(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))


@pytest.mark.parametrize("which", ["grouped", "silu"])
@pytest.mark.parametrize("index", [0, 1, 2])
@pytest.mark.parametrize("change", ["shorter", "wider type", "host", "flat"])
def test_what_a_graph_kept_is_checked_when_it_comes_back(change, index, which):
    """A hook that gives back something else ends the pass; nothing is read by the old sizes."""
    x, w, f, dy = _layer("M")
    rw = torch.rand(33, device=DEV).requires_grad_()
    leaves, f, dy = ([x, w], f, dy) if which == "grouped" else ([x, rw], M.silu_mul, dy[:, :32].contiguous())
    how = {"shorter": lambda t: t[:-1], "wider type": lambda t: t.double(), "host": lambda t: t.cpu(), "flat": lambda t: t[None]}[change]
    given = []

    def give_back(t):
        given.append(t)
        return how(t.detach()) if len(given) == index + 1 else t
    with _saved_through(give_back):
        y = f(*leaves)
    if which == "silu" and index == 2:
        torch.autograd.grad(y, leaves, dy)
        assert len(given) == 2
        return
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, dy)
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", ["y", "dx", "dw", "silu", "silu gradients", "block", "quantise"])
def test_a_tracer_does_not_record_an_empty_result(name):
    """make_fx and torch.jit.trace would see the allocation of the result only; the call is refused, with a
    result given by the caller too.  It is as good as ever under a mode that records nothing."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    if name == "silu gradients":
        gu, dy = torch.randn(9, 512, device=DEV).half(), torch.randn(9, 256, device=DEV).half()
        call, names = lambda: M.silu_mul_backward(gu, dy)[0], ()
    else:
        call, names = _calls_with_results()[name]
    want = call()
    x = torch.ones(3, device=DEV)
    given = [{}] + [dict(zip(names, want if isinstance(want, tuple) else (want,)))] * bool(names)
    for out in given:
        def program(x):
            r = call(**out)
            return (r[0] if isinstance(r, tuple) else r) + x[0]
        for trace in (lambda: make_fx(program)(x), lambda: make_fx(program, pre_dispatch=True)(x), lambda: torch.jit.trace(program, (x,), check_trace=False)):
            with pytest.raises(M.FmoeError, match="traced program"):
                trace()
        with FlopCounterMode(display=False):
            program(x)


TRANSFORMS = {"vmap": lambda f, x: torch.vmap(f)(x[None]), "functionalize": lambda f, x: torch.func.functionalize(f)(x),
              "grad": lambda f, x: torch.func.grad(lambda t: f(t).float().sum())(x), "jvp": lambda f, x: torch.func.jvp(f, (x,), (x,))}


@pytest.mark.parametrize("name,transform", [(n, t) for n in ("grouped", "silu", "quantise", "block") for t in TRANSFORMS
                                            if n != "block" or t in ("vmap", "functionalize")])     # bytes have no derivatives
def test_function_transforms_are_refused(name, transform):
    off, w = offsets_of([10, 0, 23]), torch.randn(3, 96, 256, device=DEV).bfloat16()
    a, sa, b, sb = block_inputs(33, 70, 256, "block128", seed=2)
    x = a.view(torch.float8_e4m3fn).bfloat16()
    f = {"grouped": lambda t: M.grouped_matmul(t, w, off), "silu": M.silu_mul, "quantise": lambda t: M.silu_mul_quantise(t, "block128")[0],
         "block": lambda t: M.matmul_block128(t, sa, b, sb)}[name]
    with pytest.raises(RuntimeError):
        TRANSFORMS[transform](f, a.view(torch.uint8) if name == "block" else x)


@pytest.mark.parametrize("name", ["grouped", "silu"])
def test_a_tracer_does_not_record_empty_gradients(name):
    """The backward pass of a call that was made before the trace began."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, f, dy = _layer("M")
    y = f(x, w) if name == "grouped" else M.silu_mul(x)
    dy = dy if name == "grouped" else dy[:, :32].contiguous()
    want = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
    with pytest.raises(RuntimeError, match="traced program"):
        make_fx(lambda dy: torch.autograd.grad(y, x, dy, retain_graph=True)[0])(dy)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)


def test_gradients_with_offsets_and_weights_from_the_middle_of_a_tensor():
    """Both need their types' alignment only, in the backward pass too."""
    x, w, _, dy = _layer("M")
    off = torch.cat([torch.full((1,), 7, dtype=torch.int32, device=DEV), offsets_of([10, 0, 23])])
    rw = torch.rand(34, device=DEV)
    for call, other in ((lambda o: torch.autograd.grad(M.grouped_matmul(x, w, o), (x, w), dy), off[1:]),
                        (lambda o: torch.autograd.grad(M.silu_mul(x, o.detach().requires_grad_()), x, dy[:, :32].contiguous()), rw[1:])):
        assert other.data_ptr() % 16
        assert all(torch.equal(a, b) for a, b in zip(call(other), call(other.clone())))


def test_traced_and_compiled_programs_hold_the_registered_operators():
    import therock_b200.torch_op  # noqa: F401
    from torch.fx.experimental.proxy_tensor import make_fx
    ns = torch.ops.therock_b200
    x, w, _, _ = _layer("M")
    off = offsets_of([10, 0, 23])
    q = block_inputs(33, 70, 256, "block128", seed=2)

    def layer(x, w, off, *q):
        return ns.silu_mul(ns.grouped_matmul(x, w, off)).float().square().sum() + ns.matmul_block128(*q).float().sum()
    rest = (off, *q)
    with torch.no_grad():
        for program in (make_fx(layer)(x, w, *rest), torch.jit.trace(layer, (x, w, *rest), check_trace=False),
                        make_fx(layer, tracing_mode="fake")(x, w, *rest)):
            assert torch.equal(program(-x, w, *rest), layer(-x, w, *rest))
    compiled = torch.compile(layer, backend="aot_eager", fullgraph=True, dynamic=True)
    want, got = torch.autograd.grad(layer(x, w, *rest), (x, w)), torch.autograd.grad(compiled(x, w, *rest), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", ["grouped_matmul", "grouped_matmul_dgrad", "grouped_matmul_wgrad", "matmul_block128", "silu_mul", "silu_mul_backward"])
def test_registered_operators_pass_opcheck(name):
    import therock_b200.torch_op  # noqa: F401
    x, w, _, dy = _layer("M")
    off, rw = offsets_of([10, 0, 23]), torch.rand(33, device=DEV).requires_grad_()
    a, sa, b, sb = block_inputs(33, 70, 256, "block128", seed=2)
    calls = {"grouped_matmul": [(x, w, off)], "grouped_matmul_dgrad": [(dy, w.detach(), off)], "grouped_matmul_wgrad": [(dy, x.detach(), off)],
             "matmul_block128": [(a, sa, b.view(torch.uint8), sb)], "silu_mul": [(x,), (x, rw)],
             "silu_mul_backward": [(x.detach(), dy[:, :32].contiguous()), (x.detach(), dy[:, :32].contiguous(), rw.detach())]}
    for args in calls[name]:
        assert set(torch.library.opcheck(getattr(torch.ops.therock_b200, name).default, args).values()) == {"SUCCESS"}


def test_the_first_calls_of_a_process_may_come_from_several_threads():
    """Set-up that a first call does (attributes of kernels, occupancy) is shared between threads."""
    import subprocess
    import sys
    text = """
import threading, torch, therock_b200 as M
d = "cuda:0"
torch.manual_seed(0)
off = torch.tensor([0, 5, 33], dtype=torch.int32, device=d)
x, w = torch.randn(33, 64, device=d).bfloat16(), torch.randn(2, 256, 64, device=d).bfloat16()
dy = torch.randn(33, 256, device=d).bfloat16()
a, b = torch.randn(2100, 1024, device=d).to(torch.float8_e4m3fn), torch.randn(2048, 1024, device=d).to(torch.float8_e4m3fn)
sa, sb = torch.rand(2100, 8, device=d), torch.rand(16, 8, device=d)
torch.cuda.synchronize()
def calls():
    return [M.grouped_matmul(x, w, off), M.grouped_matmul_dgrad(dy, w, off), M.grouped_matmul_wgrad(dy, x, off), M.silu_mul(dy),
            M.matmul_block128(a, sa, b, sb), M.matmul_block128(a[:3], sa[:3], b, sb)]
start, got = threading.Barrier(8), [None] * 8
def work(i):
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream(d)):
        got[i] = calls()
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
for t in threads: t.start()
for t in threads: t.join()
want = calls()
assert all(torch.equal(p, q) for g in got for p, q in zip(g, want))
print("same")
"""
    r = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


# ----------------------------------------------------------------------------- every kernel, and exact sums
FORMS = {("few_rows", rows, split) for rows in (16, 32, 128) for split in (1, 2, 4, 8)} | {("tiles", 128, 1), ("cta_pairs", 256, 1)}


def _whole(gen, limit, *shape):
    return torch.randint(-limit, limit + 1, shape, device=DEV, generator=gen)


def _exact_block(m, n, k, quant, seed):
    """Whole numbers up to 2 with scales of 1/2, 1 and 2: multiples of 1/4 below 2^17, so every 32-bit sum is
    exact in any order and the result is the reference rounded once."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    blocks, nb = k // 128, (n + 127) // 128
    a, w = _whole(gen, 2, m, k).float(), _whole(gen, 2, n, k).float()
    ea, ew = _whole(gen, 1, m, blocks), _whole(gen, 1, nb, blocks)
    sa = torch.exp2(ea.float()) if quant == "block128" else torch.nn.functional.pad((ea + 127).to(torch.uint8), (0, -blocks % 4), value=255)
    sw = torch.exp2(ew.float())
    out = M.matmul_block128(a.to(torch.float8_e4m3fn), sa.contiguous(), w.to(torch.float8_e4m3fn), sw, quant)
    ref = (a.double() * torch.exp2(ea.double()).repeat_interleave(128, 1)) @ (w.double() * sw.double().repeat_interleave(128, 1).repeat_interleave(128, 0)[:n]).T
    assert torch.equal(out, ref.bfloat16()), (m, n, k, float((out.double() - ref).abs().max()))


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
def test_every_form_of_the_product_is_run_and_exact(quant):
    """Each kernel, tile and split that the library may choose, found by asking it, at its smallest size and
    at one with odd sizes and many blocks of K."""
    found = {}
    for m in (1, 5, 16, 17, 33, 40, 65, 100, 130, 250, 300, 384, 520, 639, 1030, 2040, 4096, 7960):
        for n in (63, 128, 200, 1100, 2303, 4999, 7743, 9000, 18431):
            for k in (128, 384, 512, 1024, 1408, 2048, 2432, 3968, 5632, 7168, 7296):
                d = M.describe_matmul_block128(m, n, k, quant)
                assert d["cols_per_tile"] == (128 if d["kernel"] == "few_rows" else 256)
                if m * n * k <= 6e10:
                    found.setdefault((d["kernel"], d["rows_per_tile"], d["k_split"]), []).append((m * n * k, m, n, k))
    # whole K to a 128-row tile always takes longer than a 128 x 256 tile whose MMAs apply the scales
    assert set(found) == FORMS - ({("few_rows", 128, 1)} if quant == "block128_ue8m0" else set())
    for sizes in found.values():
        _, *smallest = min(sizes)
        _, *odd = max(s for s in sizes if s[0] <= max(4e9, min(sizes)[0]))
        for m, n, k in {tuple(smallest), tuple(odd)}:
            _exact_block(m, n, k, quant, seed=m + n + k)
    assert M.operator_status(DEV) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k", [([3, 0, 40], 136, 7168), ([300, 1], 7168, 72), ([2100, 4000], 264, 200)])
def test_long_sums_of_the_grouped_products_are_exact(sizes, n, k, dtype):
    """Whole numbers up to 2: every sum of a few thousand products is exact in 32 bits, so each result is the
    reference rounded once."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(n)
    rows, off = sum(sizes), offsets_of(sizes)
    x, w, dy = (_whole(gen, 2, *s).to(dtype) for s in ((rows, k), (len(sizes), n, k), (rows, n)))
    y, dx, dw = M.grouped_matmul(x, w, off), M.grouped_matmul_dgrad(dy, w, off), M.grouped_matmul_wgrad(dy, x, off)
    lo = 0
    for g, size in enumerate(sizes):
        at = slice(lo, lo + size)
        xg, dg, wg = x[at].double(), dy[at].double(), w[g].double()
        assert torch.equal(y[at], (xg @ wg.T).to(dtype)) and torch.equal(dx[at], (dg @ wg).to(dtype)) and torch.equal(dw[g], (dg.T @ xg).to(dtype))
        lo += size


# ----------------------------------------------------------------------------- the quantising form from float16
def _quantised(y, quant):
    """e4m3 bytes and scales of y's groups of 128 by the rule of quantise_rows: absmax / 448 (1 for zeros), or
    the smallest power of two that is no less; the reciprocal rounded once.  (A tensor divided by a number is
    a product with its reciprocal on the GPU; 64 bits round a quotient of 32-bit numbers as one division does.)"""
    v = y.float().view(y.shape[0], -1, 128)
    amax = v.abs().amax(2)
    s = torch.where(amax > 0, (amax.double() / 448).float(), torch.ones_like(amax))
    if quant == "block128_ue8m0":
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), torch.where(m == 0.5, e - 1, e))
    return (v * (1 / s.double()).float()[:, :, None]).view(y.shape).to(torch.float8_e4m3fn), s


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 128), (5, 384), (300, 1152), (16, 14336)])
def test_silu_mul_quantise_of_float16(rows, width, weighted, quant):
    """Rounded to float16 first, then quantised: bytes and scales of the rule applied to silu_mul's result."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(rows + width)
    gu = (torch.randn(rows, 2 * width, device=DEV, generator=gen) * 3).half()
    gu[rows // 2] = 0
    weight = torch.rand(rows, device=DEV, generator=gen) if weighted else None
    q, s = M.silu_mul_quantise(gu, quant, weight)
    want_q, want_s = _quantised(M.silu_mul(gu, weight), quant)
    groups = width // 128
    got_s = s.view(torch.float32) if quant == "block128" else torch.exp2(s[:, :groups].float() - 127)
    assert torch.equal(got_s, want_s) and torch.equal(q, want_q.view(torch.uint8))


@pytest.mark.parametrize("quant", ["block128", "block128_ue8m0"])
def test_a_group_that_overflows_float16_leaves_the_others_alone(quant):
    """Above 65504 float16 is infinite, and so is its group's f32 scale; a power-of-two scale stays at its largest."""
    gu = torch.ones(3, 768, device=DEV).half()
    want_q, want_s = M.silu_mul_quantise(gu, quant)
    gu[1, 130], gu[1, 384 + 130] = 300.0, 300.0
    assert bool(torch.isinf(M.silu_mul(gu)[1, 130]))
    q, s = M.silu_mul_quantise(gu, quant)
    rest = torch.ones_like(q, dtype=torch.bool)
    rest[1, 128:256] = False
    assert torch.equal(q[rest], want_q[rest])
    if quant == "block128":
        s, want_s = s.view(torch.float32), want_s.view(torch.float32)
    assert torch.equal(s[[0, 2], :3], want_s[[0, 2], :3]) and torch.equal(s[1, [0, 2]], want_s[1, [0, 2]])
    assert bool(torch.isinf(s[1, 1])) if quant == "block128" else int(s[1, 1]) == 254


# ----------------------------------------------------------------------------- ends of the ranges
def test_no_rows_at_all():
    """Empty results, zero gradients of the weights."""
    x, gu = (torch.empty(0, c, device=DEV, dtype=torch.bfloat16).requires_grad_() for c in (64, 96))
    w = torch.randn(3, 48, 64, device=DEV).bfloat16().requires_grad_()
    rw = torch.empty(0, device=DEV).requires_grad_()
    off = offsets_of([0, 0, 0])
    y = M.grouped_matmul(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 48) and dx.shape == (0, 64) and dw.shape == w.shape and not bool(dw.any())
    for weight in (None, rw):
        z = M.silu_mul(gu, weight)
        grads = torch.autograd.grad(z, [gu] + [weight] * (weight is not None), torch.empty_like(z))
        assert z.shape == (0, 48) and [g.shape for g in grads] == [gu.shape] + [rw.shape] * (weight is not None)
    q, s = M.silu_mul_quantise(torch.empty(0, 256, device=DEV).half(), "block128")
    assert q.shape == (0, 128) and s.shape == (0, 4)
    a, sa, b, sb = block_inputs(2, 70, 256, "block128", seed=1)
    assert M.matmul_block128(a[:0], sa[:0], b, sb).shape == (0, 70)
    assert M.operator_status(DEV) == 0


def test_the_most_groups():
    """1024 groups, most of them with a few rows, some with none, one with several pieces."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(9)
    sizes = torch.randint(0, 9, (1024,), device=DEV, generator=gen)
    sizes[0], sizes[511], sizes[1023] = 700, 0, 300
    off = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).int()
    rows, n, k = int(off[-1]), 72, 136
    x, w, dy = (_whole(gen, 2, *s).bfloat16() for s in ((rows, k), (1024, n, k), (rows, n)))
    group = torch.repeat_interleave(torch.arange(1024, device=DEV), sizes)
    y, dx, dw = M.grouped_matmul(x, w, off), M.grouped_matmul_dgrad(dy, w, off), M.grouped_matmul_wgrad(dy, x, off)
    xd, wd, dd = x.double(), w.double(), dy.double()
    assert torch.equal(y, torch.einsum("rk,rnk->rn", xd, wd[group]).bfloat16())
    assert torch.equal(dx, torch.einsum("rn,rnk->rk", dd, wd[group]).bfloat16())
    ref = torch.zeros(1024, n * k, device=DEV, dtype=torch.float64).index_add(0, group, (dd[:, :, None] * xd[:, None, :]).flatten(1))
    assert torch.equal(dw, ref.view(1024, n, k).bfloat16())


def test_an_activation_of_several_launches():
    """A launch covers 2^30 vectors of 8; rows behind that are another launch's, with the same results as alone."""
    rows, width = 8195, 1 << 20                                # 8192 rows are the first launch's
    gu = torch.empty(rows, 2 * width, device=DEV, dtype=torch.bfloat16).normal_()
    rw = torch.rand(rows, device=DEV)
    spans = [slice(0, 2), slice(8190, 8192), slice(8192, rows)]
    y = M.silu_mul(gu, rw)
    for at in spans:
        assert torch.equal(y[at], M.silu_mul(gu[at], rw[at].clone()))
    for weight in (rw, None):
        dgu, dw = M.silu_mul_backward(gu, y, weight)
        for at in spans:
            g, d = M.silu_mul_backward(gu[at], y[at], None if weight is None else weight[at].clone())
            assert torch.equal(dgu[at], g) and (weight is None or torch.equal(dw[at], d))
        del dgu, dw
    del y
    for quant in ("block128", "block128_ue8m0"):
        q, s = M.silu_mul_quantise(gu, quant, rw)
        for at in spans:
            p, t = M.silu_mul_quantise(gu[at], quant, rw[at].clone())
            assert torch.equal(q[at], p) and torch.equal(s[at], t)
        del q, s
