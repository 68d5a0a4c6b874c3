"""The training-step operators, measured: an AdamW step over many tensors (moments in 32 or in 8 bits), the norm of all
gradients with its clip factor, and the balance loss over the superpoints with its counts and gradients.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes the inputs on the GPU,
``run()`` is one pass -- in plain torch, or through the framework where ``own`` is set --, ``exact()`` the same in 64
bits from the definition, ``work()`` what a pass has to read, write and compute.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 256          # elements that share a scale when the moments are held in 8 bits
TOP = 448.0          # largest value of the 8-bit format (4 exponent bits, 3 mantissa bits)
LOW = 2.0 ** -9      # its smallest positive value
BETAS, EPS = (0.9, 0.999), 1e-8
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _framework():
    path = os.path.join(os.getcwd(), "fast-sp-gs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the smallest step: a narrow deformation network in one flat tensor, the radius and weight of 64 superpoints
        dict(name="step32 small net", op="step", sizes="59982,64,64", ptype="float32", gtype="float32", bits=32,
             master=False, clip=0.0),
        # a network of many layers, trained in 16 bits with a master copy, clipped: weights, biases, odd lengths
        dict(name="step32 layers bf16 master", op="step", sizes="ragged:120:1:180000", ptype="bfloat16",
             gtype="bfloat16", bits=32, master=True, clip=1.0),
        # all tensors of two million Gaussians (58 floats each)
        dict(name="step32 scene 2M", op="step", sizes="scene:2000000", ptype="float32", gtype="float32", bits=32,
             master=False, clip=0.0),
        # the shipped deformation network (8 x 256) and the kernel weights of 512 superpoints, small state
        dict(name="step8 motion net", op="step", sizes="523320,512,512", ptype="float32", gtype="float32", bits=8,
             master=False, clip=0.0),
        # all tensors of the 300 k scene, state in 8 bits
        dict(name="step8 scene 300k", op="step", sizes="scene:300000", ptype="float32", gtype="float32", bits=8,
             master=False, clip=0.0),
        # the two-million scene held in 16 bits with an 8-bit state, clipped: the smallest memory per Gaussian
        dict(name="step8 scene 2M bf16", op="step", sizes="scene:2000000", ptype="bfloat16", gtype="bfloat16", bits=8,
             master=False, clip=1.0),
        # gradient norm of a small network's layers
        dict(name="norm layers", op="norm", sizes="ragged:40:1:70000", gtype="float32", clip=1.0),
        # gradient norm of the two-million scene
        dict(name="norm scene 2M", op="norm", sizes="scene:2000000", gtype="float32", clip=0.5),
        # balance of the blend weights of the 300 k scene: three nearest of 512 superpoints
        dict(name="balance 300k x 3", op="balance", rows=300000, near=3, points=512, masked=0.0),
        # the stress scene: eight nearest of 4096, part of the Gaussians left out
        dict(name="balance 2M x 8", op="balance", rows=2000000, near=8, points=4096, masked=0.03),
        # a learned association table of the 300 k scene, value and gradient in one call
        dict(name="table 300k x 512", op="table", rows=300000, near=3, points=512, masked=0.0, gtype="float32",
             autograd=False),
        # a small one in 16 bits, odd width, through autograd
        dict(name="table 20k x 333 bf16", op="table", rows=20000, near=2, points=333, masked=0.05, gtype="bfloat16",
             autograd=True),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["step", "step", "step", "norm", "balance", "table"])
    if op in ("step", "norm"):
        total = log(1000, 30_000_000)
        kind = rng.choice(["scene", "ragged", "flat"])
        if kind == "scene":
            sizes = f"scene:{max(1, total // 58)}"
        elif kind == "ragged":
            count = rng.randint(2, 150)
            sizes = f"ragged:{count}:{log(1, 50)}:{max(100, min(400_000, 4 * total // count))}"
        else:
            sizes = f"{total},{log(1, 5000)}"
        gtype = rng.choice(["float32", "bfloat16", "float16"])
        clip = rng.choice([0.0, 0.1, 1.0])
        if op == "norm":
            return dict(op=op, sizes=sizes, gtype=gtype, clip=clip or 5.0)
        ptype = gtype if gtype != "float32" else rng.choice(["float32", "float32", "bfloat16"])
        return dict(op=op, sizes=sizes, ptype=ptype, gtype=gtype, bits=rng.choice([8, 32]),
                    master=ptype != "float32" and rng.random() < 0.5, clip=clip)
    near = rng.randint(1, 8)
    masked = rng.choice([0.0, 0.02, 0.3])
    if op == "balance":
        return dict(op=op, rows=log(100, 2_000_000), near=near, points=log(max(near, 8), 4096), masked=masked)
    points = log(max(near, 8), 4096)
    return dict(op=op, rows=max(1, min(log(100, 300_000), 120_000_000 // points)), near=near, points=points,
                masked=masked, gtype=rng.choice(["float32", "bfloat16", "float16"]), autograd=rng.random() < 0.4)


def _sizes(text):
    """The lengths of a case's tensors."""
    if text.startswith("scene:"):   # position, SH DC, SH rest, opacity, scale, rotation
        return [int(text[6:]) * k for k in (3, 3, 45, 1, 2, 4)]
    if text.startswith("ragged:"):
        count, low, high = (int(v) for v in text[7:].split(":"))
        r = random.Random(count * 1_000_003 + high)
        return [int(round(math.exp(r.uniform(math.log(low), math.log(high))))) for _ in range(count)]
    return [int(v) for v in text.split(",")]


def work(case):
    if case["op"] in ("step", "norm"):
        n = sum(_sizes(case["sizes"]))
        g = 4 if case["gtype"] == "float32" else 2
        if case["op"] == "norm":
            return {"bytes": n * g, "flops": 2 * n}
        p = 4 if case["ptype"] == "float32" else 2
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (g + state + (8 + p if case["master"] else 2 * p)), "flops": (18 if case["clip"] else 15) * n}
    n, k, m = case["rows"], case["near"], case["points"]
    if case["op"] == "balance":
        return {"bytes": n * k * 16 + (n if case["masked"] else 0) + 8 * m, "flops": 4 * n * k}
    size = 4 if case["gtype"] == "float32" else 2
    return {"bytes": 2 * n * m * size + 8 * n * k + (n if case["masked"] else 0) + 8 * m, "flops": 9 * n * m}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _normal(n, gen, spread):
    """Values whose size differs from element to element by factors of e^spread, as gradients do."""
    x = torch.randn(n, device="cuda", generator=gen)
    return x * torch.exp(torch.randn(n, device="cuda", generator=gen) * spread)


def _to8(x, positive):
    """Rows of BLOCK values -> (8-bit values, scale): value = 8-bit value * scale of its row."""
    top = x.abs().amax(dim=1, keepdim=True)
    scale = top / TOP
    y = torch.where(top > 0, x * (TOP / top), torch.zeros_like(x))
    y = torch.where(x > 0, y.clamp_min(LOW), y) if positive else y
    return y.to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    if case["op"] in ("step", "norm"):
        sizes = _sizes(case["sizes"])
        # the tensors lie in one buffer, each at the start of a block: what a flat parameter store looks like
        starts = [0]
        for n in sizes:
            starts.append(starts[-1] + -(-n // BLOCK) * BLOCK)
        rows = starts[-1] // BLOCK
        spans = list(zip(starts, sizes))
        inside = torch.zeros(starts[-1], dtype=torch.bool, device="cuda")
        for a, n in spans:
            inside[a:a + n] = True
        g = torch.where(inside, _normal(starts[-1], gen, 1.0) * 1e-3, 0.0)
        seen = torch.rand(rows, 1, device="cuda", generator=gen) > 0.1      # what no view saw has no gradient
        g = (g.view(rows, BLOCK) * seen).view(-1).to(TYPES[case["gtype"]])
        grads = [g[a:a + n] for a, n in spans]
        if case["op"] == "norm":
            return dict(case=case, flat=g, grads=grads)
        p = torch.where(inside, torch.randn(starts[-1], device="cuda", generator=gen) * 0.3, 0.0)
        m = torch.where(inside, _normal(starts[-1], gen, 1.0) * 4e-4, 0.0)
        v = torch.where(inside, (_normal(starts[-1], gen, 0.7) * 1e-3) ** 2 + 0.2 * m * m, 0.0)
        s = dict(case=case, p=p.to(TYPES[case["ptype"]]), g=g, spans=spans)
        if case["master"]:
            s["master"] = p
        if case["bits"] == 8:
            s["m"], s["m_scale"] = _to8(m.view(rows, BLOCK), False)
            s["s"], s["s_scale"] = _to8(v.sqrt().view(rows, BLOCK), True)
            for k in ("m", "s"):
                s[k], s[k + "_scale"] = s[k].reshape(-1), s[k + "_scale"].reshape(-1)
        else:
            s["m"], s["v"] = m, v
        s["step"] = torch.full((len(sizes),), 40.0, device="cuda")
        # every other tensor decays: weights do, biases and positions do not
        half = len(sizes) - len(sizes) // 2
        decays = [i % 2 == 0 for i in range(len(sizes))]
        s["groups"] = ((2e-3, 0.01), (5e-4, 0.0))
        pick = torch.zeros(rows, 1, device="cuda")
        for (a, n), d in zip(spans, decays):
            pick[a // BLOCK:-(-(a + n) // BLOCK)] = 0.0 if d else 1.0
        s["lr"] = torch.where(pick > 0, 5e-4, 2e-3)
        s["keep"] = torch.where(pick > 0, 1.0, 1.0 - 2e-3 * 0.01)
        s["half"], s["decays"] = half, decays
        if own:
            s["optimizer"], s["params"], s["grads"] = _optimizer(s)
        return s
    n, k, m = case["rows"], case["near"], case["points"]
    # some superpoints are near many Gaussians, some near few; the K of a Gaussian are distinct
    popular = torch.exp(torch.randn(m, device="cuda", generator=gen) * 0.7).cumsum(0)
    first = torch.searchsorted(popular, torch.rand(n, device="cuda", generator=gen) * popular[-1]).clamp_(max=m - 1)
    idx = (first[:, None] + torch.arange(k, device="cuda") * max(1, m // (2 * k))) % m
    mask = torch.rand(n, device="cuda", generator=gen) >= case["masked"] if case["masked"] else None
    s = dict(case=case, idx=idx.contiguous(), mask=mask)
    if case["op"] == "balance":
        s["w"] = torch.softmax(torch.randn(n, k, device="cuda", generator=gen), dim=1)
    else:
        z = torch.randn(n, m, device="cuda", generator=gen) * 1.5
        s["z"] = z.scatter_add_(1, idx, torch.full((n, k), 2.0, device="cuda")).to(TYPES[case["gtype"]])
    return s


def _optimizer(s):
    """The framework's optimiser over the tensors of a step case, with its state where the case's buffers are."""
    _framework()
    from fsgs.optim import AdamW
    case = s["case"]
    params = [torch.nn.Parameter(s["p"][a:a + n]) for a, n in s["spans"]]
    grads = [s["g"][a:a + n] for a, n in s["spans"]]
    for p in params:
        p.grad_dtype = s["g"].dtype
    groups = [dict(params=[p for p, d in zip(params, s["decays"]) if d == first], lr=lr, weight_decay=wd)
              for first, (lr, wd) in zip((True, False), s["groups"])]
    opt = AdamW([g for g in groups if g["params"]], betas=BETAS, eps=EPS, state_bits=case["bits"],
                master_weights=case["master"], max_grad_norm=case["clip"] or None)
    for i, (p, (a, n)) in enumerate(zip(params, s["spans"])):
        st = dict(step=s["step"][i], exp_avg=s["m"][a:a + n])
        if case["bits"] == 8:
            rows = slice(a // BLOCK, -(-(a + n) // BLOCK))
            st.update(exp_avg_scale=s["m_scale"][rows], exp_avg_sq_root=s["s"][a:a + n],
                      exp_avg_sq_root_scale=s["s_scale"][rows])
        else:
            st["exp_avg_sq"] = s["v"][a:a + n]
        if case["master"]:
            st["master"] = s["master"][a:a + n]
        opt.state[p] = st
    return opt, params, grads


# ---- one pass --------------------------------------------------------------------------------------------------------

def _step_outputs(s, norm):
    names = ["p", "m", "step"] + (["m_scale", "s", "s_scale"] if s["case"]["bits"] == 8 else ["v"])
    out = {k: s[k] for k in names + (["master"] if s["case"]["master"] else [])}
    return dict(out, norm=norm) if norm is not None else out


def _plain_norm(g, most):
    norm = g.float().square().sum(dtype=torch.float64).sqrt().float()
    return norm, (most / (norm + 1e-6)).clamp(max=1.0)


def _plain_step(s):
    case = s["case"]
    b1, b2 = BETAS
    rows = lambda t: t.view(-1, BLOCK)  # noqa: E731
    norm = None
    g = rows(s["g"]).float()
    if case["clip"]:
        norm, factor = _plain_norm(s["g"], case["clip"])
        g = g * factor
    s["step"] += 1
    t = s["step"][0].double()
    c1, c2 = (1 - b1 ** t).float(), (1 - b2 ** t).sqrt().float()
    if case["bits"] == 8:
        m = rows(s["m"]).float() * s["m_scale"][:, None]
        v = (rows(s["s"]).float() * s["s_scale"][:, None]).square()
    else:
        m, v = rows(s["m"]), rows(s["v"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    root = v.sqrt()
    p = rows(s["master"] if case["master"] else s["p"]).float()
    p = p * s["keep"] - (s["lr"] / c1) * (m / (root / c2 + EPS))
    if case["master"]:
        rows(s["master"]).copy_(p)
    rows(s["p"]).copy_(p)
    if case["bits"] == 8:
        for k, x, positive in (("m", m, False), ("s", root, True)):
            code, scale = _to8(x, positive)
            rows(s[k]).copy_(code)
            s[k + "_scale"].copy_(scale[:, 0])
    else:
        rows(s["m"]).copy_(m)
        rows(s["v"]).copy_(v)
    return _step_outputs(s, norm)


def _plain_balance(s):
    case, idx, m = s["case"], s["idx"], s["case"]["points"]
    valid = torch.ones_like(idx[:, 0], dtype=torch.bool) if s["mask"] is None else s["mask"]
    n = valid.sum()
    pairs = valid[:, None].expand_as(idx)
    # every pair of a row that counts, in a bin of its own; the others in one bin more
    counts = torch.bincount(torch.where(pairs, idx, m).reshape(-1), minlength=m + 1)[:m]
    total = counts.sum()
    if case["op"] == "balance":
        share = (m * counts.double() / (total * n)).float()
        grad = torch.where(pairs, share[idx], 0.0)
        return dict(loss=(grad * s["w"]).sum(dtype=torch.float64).float(), grad=grad, counts=counts)
    # a constant taken off all shares changes no gradient: with the mean taken off, no two near values are subtracted
    share = ((m * counts.double() - total) / (total * n)).float()
    z = s["z"].float()
    e = torch.exp(z - z.amax(dim=1, keepdim=True))
    p = e / e.sum(dim=1, keepdim=True)
    inner = (p * share).sum(dim=1, keepdim=True)
    grad = torch.where(valid[:, None], p * (share - inner), 0.0).to(s["z"].dtype)
    loss = 1.0 + torch.where(valid, inner[:, 0], 0.0).sum(dtype=torch.float64)
    return dict(loss=loss.float(), grad=grad, counts=counts)


def _own(s):
    case = s["case"]
    _framework()
    if case["op"] == "step":
        for p, g in zip(s["params"], s["grads"]):
            p.grad = g
        s["optimizer"].step()
        return _step_outputs(s, s["optimizer"].grad_norm if case["clip"] else None)
    if case["op"] == "norm":
        from fsgs.optim import grad_norm
        norm, factor = grad_norm(s["grads"], max_norm=case["clip"])
        return dict(norm=norm, factor=factor)
    from fsgs import loss
    if case["op"] == "balance":
        value, grad, counts = loss.balance_value_and_grad(s["w"], s["idx"], case["points"], mask=s["mask"])
    elif case["autograd"]:
        z = s["z"].detach().requires_grad_()
        value, counts = loss.table_balance_loss(z, s["idx"], mask=s["mask"])
        grad, = torch.autograd.grad(value, z)
        value = value.detach()
    else:
        value, grad, counts = loss.table_balance_value_and_grad(s["z"], s["idx"], mask=s["mask"])
    return dict(loss=value, grad=grad, counts=counts)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "step":
        return _plain_step(state)
    if op == "norm":
        norm, factor = _plain_norm(state["flat"], state["case"]["clip"])
        return dict(norm=norm, factor=factor)
    return _plain_balance(state)


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------

def _nearest8(y):
    """Nearest value with 4 exponent and 3 mantissa bits, ties to even, of float64 numbers of at most TOP."""
    _, e = torch.frexp(y)
    spacing = torch.ldexp(torch.ones_like(y), e.clamp_min(-5) - 4)
    return torch.round(y / spacing) * spacing


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("step", "norm"):
        g = (s["flat"] if case["op"] == "norm" else s["g"]).double()
        length = (g * g).sum().sqrt()
        factor = min(1.0, case["clip"] / (float(length) + 1e-6)) if case["clip"] else 1.0
        if case["op"] == "norm":
            return dict(norm=length, factor=torch.tensor(factor, dtype=torch.float64))
        g *= factor
        m0, v0 = s["m"].double(), (s["s"] if case["bits"] == 8 else s["v"]).double()
        if case["bits"] == 8:
            m0 *= s["m_scale"].double().repeat_interleave(BLOCK)
            v0 = (v0 * s["s_scale"].double().repeat_interleave(BLOCK)) ** 2
        m1 = BETAS[0] * m0 + (1 - BETAS[0]) * g
        v1 = BETAS[1] * v0 + (1 - BETAS[1]) * g * g
        del m0, v0, g
        t = 41
        update = (m1 / (1 - BETAS[0] ** t)) / (torch.sqrt(v1 / (1 - BETAS[1] ** t)) + EPS)
        p1 = (s["master"] if case["master"] else s["p"]).double()
        for (a, n), d in zip(s["spans"], s["decays"]):
            lr, wd = s["groups"][0 if d else 1]
            p1[a:a + n] -= lr * wd * p1[a:a + n] + lr * update[a:a + n]
        del update
        out = dict(p=p1, m=m1, step=torch.full((len(s["spans"]),), float(t), dtype=torch.float64))
        if case["master"]:
            out["master"] = p1
        if case["bits"] == 8:
            for k, x in (("m", m1), ("s", v1.sqrt())):
                largest = x.view(-1, BLOCK).abs().max(dim=1).values
                scale = (largest / TOP).float().double()     # held in 32 bits
                y = x / scale.repeat_interleave(BLOCK).clamp_min(1e-300)
                y = torch.where((x > 0) & (y < LOW), torch.full_like(y, LOW), y) if k == "s" else y
                out[k], out[k + "_scale"] = _nearest8(y.clamp(-TOP, TOP)), scale
        else:
            out["v"] = v1
        return dict(out, norm=length) if case["clip"] else out
    n, m = case["rows"], case["points"]
    rows = torch.arange(n, device="cuda") if s["mask"] is None else s["mask"].nonzero()[:, 0]
    used = s["idx"][rows].reshape(-1)
    counts = torch.zeros(m, dtype=torch.int64, device="cuda").index_add_(0, used, torch.ones_like(used))
    f = counts.double() / used.numel()
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    if case["op"] == "balance":
        mean = torch.zeros(m, dtype=torch.float64, device="cuda").index_add_(0, used, s["w"][rows].double().reshape(-1))
        grad = torch.zeros(n, case["near"], dtype=torch.float64, device="cuda")
        grad[rows] = m * f[s["idx"][rows]] / rows.numel()
        loss += m * (f * mean).sum() / rows.numel()
    else:
        grad = torch.zeros(n, m, dtype=torch.float64, device="cuda")
        for part in rows.split(50_000):
            p = torch.softmax(s["z"][part].double(), dim=1)
            inner = p @ f
            grad[part] = m / rows.numel() * p * (f - inner[:, None])
            loss += m * inner.sum() / rows.numel()
    return dict(loss=loss, grad=grad, counts=counts)
