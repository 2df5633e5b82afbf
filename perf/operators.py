"""Timing cases of the operators an expert layer is built from when it is not one fused call.

  grouped_matmul     rows grouped by expert times that expert's weight, with both gradients (training; serving without them)
  matmul_block128    e4m3 activations and weights with one scale per 128 (dense layers beside the experts, serving)
  silu_mul           the gated activation between the two products, with its gradients, and with e4m3 rows as its result

A case names its operator in "op"; `run` computes it in plain 32-bit torch operations, or by the library's calls when `own` is set.
"""
import math

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # -- products grouped by expert
        # one token's two experts: the smallest call, a few megabytes of weights
        {"name": "grouped_token", "op": "grouped", "type": "bf16", "rows": 2, "groups": 8, "active": 2, "spare": 0, "n": 1024, "k": 512, "back": False},
        # 16 tokens in decode at two experts each, gate and up rows of an eight-expert layer: the weights are the work
        {"name": "grouped_decode", "op": "grouped", "type": "bf16", "rows": 32, "groups": 8, "active": 8, "spare": 0, "n": 28672, "k": 4096, "back": False},
        # a prompt of 4096 tokens through the same weights
        {"name": "grouped_prompt", "op": "grouped", "type": "bf16", "rows": 8192, "groups": 8, "active": 8, "spare": 0, "n": 28672, "k": 4096, "back": False},
        # a training step on one rank's 32 fine-grained experts, about 256 rows each, rows kept behind the last one
        {"name": "grouped_train_fine", "op": "grouped", "type": "bf16", "rows": 8192, "groups": 32, "active": 31, "spare": 256, "n": 4096, "k": 7168, "back": True},
        # a training step with odd group sizes and widths that fill no tile
        {"name": "grouped_train_odd", "op": "grouped", "type": "fp16", "rows": 1777, "groups": 12, "active": 9, "spare": 5, "n": 1416, "k": 1000, "back": True},
        # -- e4m3 products with a scale for each block of 128
        # one token through a projection
        {"name": "block_token", "op": "block", "quant": "block128", "rows": 1, "n": 4096, "k": 2048},
        # 16 tokens, the wide projection of a dense layer, power-of-two scales
        {"name": "block_decode", "op": "block", "quant": "block128_ue8m0", "rows": 16, "n": 18432, "k": 7168},
        # a small batch with an output width that ends inside a block
        {"name": "block_batch", "op": "block", "quant": "block128", "rows": 200, "n": 7168 + 576, "k": 2048},
        # prompts, both kinds of scale
        {"name": "block_prompt", "op": "block", "quant": "block128", "rows": 8192, "n": 4096, "k": 7168},
        {"name": "block_prompt_ue8m0", "op": "block", "quant": "block128_ue8m0", "rows": 8192, "n": 4096, "k": 7168},
        # -- the gated activation
        # a training step: rows weighted by their routing weight, all three gradients
        {"name": "silu_train", "op": "silu", "type": "bf16", "rows": 16384, "width": 2048, "weighted": True, "back": True, "quant": "none"},
        # 16 tokens at two experts each on the way to an e4m3 product
        {"name": "silu_decode_e4m3", "op": "silu", "type": "bf16", "rows": 32, "width": 14336, "weighted": False, "back": False, "quant": "block128_ue8m0"},
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["grouped", "grouped", "block", "block", "silu"])
    if op == "grouped":
        groups = _between(rng, 1, 64)
        active = rng.randint(max(1, groups // 2), groups)
        case = {"op": op, "type": rng.choice(["bf16", "bf16", "fp16"]), "rows": _between(rng, active, 8192), "groups": groups, "active": active,
                "spare": rng.choice([0, 0, 1, 77]), "n": 8 * _between(rng, 2, 1024), "k": 8 * _between(rng, 2, 1024), "back": rng.random() < 0.5}
        if case["rows"] >= 2048:  # room for the padded 32-bit copies of the plain form
            case["n"], case["k"] = min(case["n"], 4096), min(case["k"], 4096)
        while case["groups"] * case["n"] * case["k"] > 2 ** 29:  # a gigabyte of weights
            case["n"], case["k"] = max(8, case["n"] // 16 * 8), max(8, case["k"] // 16 * 8)
        return case
    if op == "block":
        return {"op": op, "quant": rng.choice(["block128", "block128_ue8m0"]), "rows": _between(rng, 1, 8192), "n": _between(rng, 16, 8192),
                "k": 128 * _between(rng, 1, 56)}
    quant = rng.choice(["none", "none", "block128", "block128_ue8m0"])
    width = 8 * _between(rng, 1, 1792) if quant == "none" else 128 * _between(rng, 1, 112)
    return {"op": op, "type": "bf16" if quant != "none" else rng.choice(["bf16", "fp16"]), "rows": _between(rng, 1, min(16384, 2 ** 25 // width)), "width": width,
            "weighted": rng.random() < 0.5, "back": quant == "none" and rng.random() < 0.6, "quant": quant}


def _type(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[case["type"]]


def _sizes(case, gen):
    """Rows of each group: every active group has one, the rest are shared out unevenly; which groups are active goes by the seed."""
    groups, active = case["groups"], case["active"]
    share = torch.exp(0.5 * torch.randn(active, generator=gen, dtype=torch.float64))
    edge = torch.cumsum(share, 0) / share.sum() * (case["rows"] - active)
    edge = torch.cat([torch.zeros(1, dtype=torch.float64), edge]).round().long()
    edge[-1] = case["rows"] - active
    sizes = torch.zeros(groups, dtype=torch.int64)
    sizes[torch.randperm(groups, generator=gen)[:active]] = 1 + edge[1:] - edge[:-1]
    return sizes


def _scale_of(amax, quant):
    """absmax / 448, or the smallest power of two that is no less."""
    s = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    if quant == "block128_ue8m0":
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), torch.where(m == 0.5, e - 1, e))
    return s


def _scale_rows(scale, quant):
    """Activation scales as the library keeps them: 32-bit numbers, or exponent bytes in rows of a multiple of four."""
    if quant == "block128":
        return scale.contiguous()
    byte = (torch.frexp(scale)[1] + 126).to(torch.uint8)
    return torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4)).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEVICE, generator=gen) * scale).to(dtype)

    if case["op"] == "grouped":
        host = torch.Generator()
        host.manual_seed(seed)
        sizes = _sizes(case, host)
        dtype, rows = _type(case), case["rows"] + case["spare"]
        # `longest` is what a plan on the host knows of the sizes; only the plain form needs it
        state = {"case": case, "longest": int(sizes.max()),
                 "offsets": torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(sizes, 0)]).to(torch.int32).to(DEVICE),
                 "x": normal(rows, case["k"], dtype=dtype), "w": torch.empty(case["groups"], case["n"], case["k"], dtype=dtype, device=DEVICE)}
        state["w"].normal_(0.0, 0.02, generator=gen)
        if case["back"]:
            state["dy"] = normal(rows, case["n"], dtype=dtype)
            state["x"].requires_grad_()
            state["w"].requires_grad_()
        return state
    if case["op"] == "block":
        quant, m, n, k = case["quant"], case["rows"], case["n"], case["k"]
        a = normal(m, k).view(m, k // 128, 128)
        sa = _scale_of(a.abs().amax(2), quant)
        nb = -(-n // 128)
        w = torch.nn.functional.pad(normal(n, k, scale=0.02), (0, 0, 0, nb * 128 - n)).view(nb, 128, k // 128, 128)
        sw = _scale_of(w.abs().amax(3).amax(1), quant)
        return {"case": case, "a": (a / sa[:, :, None]).view(m, k).to(torch.float8_e4m3fn), "a_scale": _scale_rows(sa, quant),
                "w": (w / sw[:, None, :, None]).view(nb * 128, k)[:n].to(torch.float8_e4m3fn).contiguous(), "w_scale": sw.contiguous()}
    dtype, rows, width = _type(case), case["rows"], case["width"]
    state = {"case": case, "gu": normal(rows, 2 * width, scale=1.5, dtype=dtype), "weight": None}
    if case["weighted"]:
        state["weight"] = torch.rand(rows, device=DEVICE, generator=gen)
    if case["back"]:
        state["dy"] = normal(rows, width, dtype=dtype)
        state["gu"].requires_grad_()
        if case["weighted"]:
            state["weight"].requires_grad_()
    return state


def _spread(rows, offsets, longest, *wide):
    """Where each row lies among its group's, and the given matrices as [groups, longest, columns] in 32 bits, zeros behind each group's rows."""
    at = torch.arange(rows, device=offsets.device)
    live = at < offsets[-1]
    group = torch.where(live, torch.searchsorted(offsets[1:].contiguous(), at.int(), right=True), 0)
    place = torch.where(live, at - offsets[group], longest)  # rows of no group go behind the others
    padded = [torch.zeros(offsets.numel() - 1, longest + 1, m.shape[1], device=m.device).index_put((group, place), m.float())[:, :longest] for m in wide]
    return live, group, place.clamp(max=longest - 1), padded


def _grouped(s):
    x, w, offsets = s["x"].detach(), s["w"].detach(), s["offsets"]
    if not s["case"]["back"]:
        live, group, place, (xp,) = _spread(x.shape[0], offsets, s["longest"], x)
        y = torch.bmm(xp, w.float().transpose(1, 2))[group, place]
        return torch.where(live[:, None], y, 0).to(x.dtype)
    live, group, place, (xp, dp) = _spread(x.shape[0], offsets, s["longest"], x, s["dy"])
    wf = w.float()
    y = torch.bmm(xp, wf.transpose(1, 2))[group, place]
    dx = torch.bmm(dp, wf)[group, place]
    dw = torch.bmm(dp.transpose(1, 2), xp)
    return {"y": torch.where(live[:, None], y, 0).to(x.dtype), "dx": torch.where(live[:, None], dx, 0).to(x.dtype), "dw": dw.to(w.dtype)}


def _block(s):
    a, w, k = s["a"].float(), s["w"].float(), s["case"]["k"]
    sa = s["a_scale"] if s["case"]["quant"] == "block128" else torch.exp2(s["a_scale"][:, :k // 128].float() - 127)
    a = a * sa.repeat_interleave(128, 1)
    w = w * s["w_scale"].repeat_interleave(128, 1).repeat_interleave(128, 0)[:w.shape[0]]
    return (a @ w.t()).to(torch.bfloat16)


def _values(q, scale):
    """What e4m3 rows with a scale for each 128 stand for, in the type that they were made from."""
    return (q.float().view(q.shape[0], -1, 128) * scale[:, :, None]).view(q.shape).to(torch.bfloat16)


def _silu(s):
    gu, weight, width = s["gu"].detach().float(), s["weight"], s["case"]["width"]
    g, u = gu[:, :width], gu[:, width:]
    sig = 1 / (1 + torch.exp(-g))
    act = g * sig * u
    y = act if weight is None else act * weight.detach()[:, None]
    y = y.to(s["gu"].dtype)
    if s["case"]["quant"] != "none":
        v = y.float().view(y.shape[0], -1, 128)
        scale = _scale_of(v.abs().amax(2), s["case"]["quant"])
        return _values((v * (1 / scale)[:, :, None]).view(y.shape).to(torch.float8_e4m3fn), scale)
    if not s["case"]["back"]:
        return y
    dy = s["dy"].float()
    back = dy if weight is None else dy * weight.detach()[:, None]
    out = {"y": y, "dgu": torch.cat([back * u * sig * (1 + g * (1 - sig)), back * g * sig], 1).to(s["gu"].dtype)}
    if weight is not None:
        out["dweight"] = (dy * act).sum(1)
    return out


def _own(s):
    import therock_b200 as M
    case = s["case"]
    if case["op"] == "grouped":
        y = M.grouped_matmul(s["x"], s["w"], s["offsets"])
        if not case["back"]:
            return y
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if case["op"] == "block":
        return M.matmul_block128(s["a"], s["a_scale"], s["w"], s["w_scale"], quant=case["quant"])
    if case["quant"] != "none":
        q, scale = M.silu_mul_quantise(s["gu"], case["quant"], s["weight"])
        groups = case["width"] // 128
        scale = scale.view(torch.float32) if case["quant"] == "block128" else torch.exp2(scale[:, :groups].float() - 127)
        return _values(q.view(torch.float8_e4m3fn), scale)
    y = M.silu_mul(s["gu"], s["weight"])
    if not case["back"]:
        return y
    if s["weight"] is None:
        return {"y": y, "dgu": torch.autograd.grad(y, s["gu"], s["dy"])[0]}
    dgu, dweight = torch.autograd.grad(y, (s["gu"], s["weight"]), s["dy"])
    return {"y": y, "dgu": dgu, "dweight": dweight}


def run(state):
    if own:
        return _own(state)
    return {"grouped": _grouped, "block": _block, "silu": _silu}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "grouped":
        rows, n, k = case["rows"], case["n"], case["k"]
        moved = 2 * (rows * k + (rows + case["spare"]) * n + case["active"] * n * k)
        if case["back"]:  # dy and the groups' weights once more for dx, all of dw written; x is read for y and for dw
            moved += 2 * (rows * n + (rows + case["spare"]) * k + case["groups"] * n * k)
        return {"bytes": moved, "flops": 2 * rows * n * k * (3 if case["back"] else 1)}
    if case["op"] == "block":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 2 * m * n + m * (k // 128) * (4 if case["quant"] == "block128" else 1) + 4 * -(-n // 128) * (k // 128), "flops": 2 * m * n * k}
    cells = case["rows"] * case["width"]
    moved = 4 * cells + (cells if case["quant"] != "none" else 2 * cells)
    if case["back"]:
        moved += 6 * cells
    return {"bytes": moved + (8 if case["back"] else 4) * case["rows"] * case["weighted"], "flops": cells * (20 if case["back"] else 6)}


def exact(case, seed):
    if case["op"] == "silu" and case["quant"] != "none":
        return None  # what 8 bits hold goes by ties and borders, not by a formula in 64 bits
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "grouped":
            ends = s["offsets"].tolist()
            x = s["x"].double()
            y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=DEVICE)
            dx, dw = (torch.zeros_like(x), torch.zeros(s["w"].shape, dtype=torch.float64, device=DEVICE)) if case["back"] else (None, None)
            for g in range(case["groups"]):
                lo, hi = ends[g], ends[g + 1]
                if lo == hi:
                    continue
                wg = s["w"][g].double()
                y[lo:hi] = torch.einsum("mk,nk->mn", x[lo:hi], wg)
                if case["back"]:
                    dyg = s["dy"][lo:hi].double()
                    dx[lo:hi] = torch.einsum("mn,nk->mk", dyg, wg)
                    dw[g] = torch.einsum("mn,mk->nk", dyg, x[lo:hi])
            return {"y": y, "dx": dx, "dw": dw} if case["back"] else y
        if case["op"] == "block":
            col = torch.arange(case["k"], device=DEVICE) // 128
            row = torch.arange(case["n"], device=DEVICE) // 128
            sa = s["a_scale"].double() if case["quant"] == "block128" else torch.pow(2.0, s["a_scale"].double() - 127)
            return torch.einsum("mk,nk->mn", s["a"].double() * sa[:, col], s["w"].double() * s["w_scale"].double()[row][:, col])
        g, u = s["gu"].double().chunk(2, 1)
        weight = torch.ones(case["rows"], dtype=torch.float64, device=DEVICE) if s["weight"] is None else s["weight"].double()
        sig = torch.sigmoid(g)
        y = weight[:, None] * g * sig * u
        if not case["back"]:
            return y
        dy = s["dy"].double()
        dg = weight[:, None] * dy * u * (sig + g * sig * (1 - sig))
        out = {"y": y, "dgu": torch.cat([dg, weight[:, None] * dy * g * sig], 1)}
        if s["weight"] is not None:
            out["dweight"] = (dy * g * sig * u).sum(1)
        return out
