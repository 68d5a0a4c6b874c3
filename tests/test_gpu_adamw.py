"""The AdamW step and the gradient norm against the formulas evaluated in float64, one step at a time from the state
that the step before left.

Tolerances, e = 2^-24 (half a unit of float32).  With g' = c g (c: the clip factor, 6 e off: the norm 3, its inverse and
product 3) and M = |b1 m| + |(1 - b1) g'|: the first moment is 12 e M off (8-bit states add a product: e), the second 20 e
relative, so its root 11 e, the denominator 15 e; the quotient is the device's approximate one (2 units: 4 e), the factor
lr / (1 - b1^t) and its product 2 e.  The update U = lr / (1 - b1^t) M / (sqrt(v) / sqrt(1 - b2^t) + eps) is thus at
most 34 e U off and the parameter, with its own product, sum and rounded constant, 4 e |p| more; 40 e U + 4 e |p| is
asked for, and half a unit of the parameter's type on top where that has 16 bits.  A moment in 8 bits is off by half a
step of its format, 2^-4 relative or 2^-10 of its scale where the format is denormal; sqrt(v) by a whole smallest step,
2^-9 of its scale, since it never rounds to zero."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
B = 256


def _make(sizes, ptype, gtype, seed=0, offset=0, spread=2.0):
    """Parameters and gradients as slices of longer buffers, `offset` elements from an aligned start."""
    gen = torch.Generator().manual_seed(seed)
    params, grads = [], []
    for n in sizes:
        x = torch.randn(n + 16, generator=gen) * 0.5
        g = torch.randn(n + 16, generator=gen) * torch.exp(spread * torch.randn(n + 16, generator=gen)) * 1e-3
        g[torch.rand(n + 16, generator=gen) < 0.1] = 0
        p = torch.nn.Parameter(x.to(ptype).cuda()[offset:offset + n])
        p.grad_dtype = gtype
        params.append(p)
        grads.append(g.to(gtype).cuda()[offset:offset + n])
    return params, grads


def _values(opt, p):
    """(m, sqrt(v), scale of m, scale of sqrt(v)) of a parameter in float64; scales per element, 0 where 32 bits."""
    st = opt.state[p]
    if opt.state_bits == 32:
        z = torch.zeros_like(st["exp_avg"], dtype=torch.float64)
        return st["exp_avg"].double(), st["exp_avg_sq"].double().sqrt(), z, z
    ms, ss = (st[k].double().repeat_interleave(B)[:p.numel()] for k in ("exp_avg_scale", "exp_avg_sq_root_scale"))
    return st["exp_avg"].double() * ms, st["exp_avg_sq_root"].double() * ss, ms, ss


def _snapshot(opt, params):
    out = []
    for p in params:
        m, s, _, _ = _values(opt, p) if opt.state.get(p) else (torch.zeros_like(p, dtype=torch.float64),) * 4
        master = opt.state[p].get("master") if opt.state.get(p) else None
        out.append(((p if master is None else master).detach().double().clone(), m.clone(), s.clone(),
                    float(opt.state[p]["step"]) if opt.state.get(p) else 0.0))
    return out


def _check_step(opt, before, params, grads, factor=1.0):
    group_of = {id(p): g for g in opt.param_groups for p in g["params"]}
    for (p0, m0, s0, t0), p, g in zip(before, params, grads):
        grp = group_of[id(p)]
        (b1, b2), lr, wd, eps = grp["betas"], grp["lr"], grp["weight_decay"], grp["eps"]
        g = g.double() * factor
        m1 = b1 * m0 + (1 - b1) * g
        v1 = b2 * s0 ** 2 + (1 - b2) * g ** 2
        t = t0 + 1
        rate, den = lr / (1 - b1 ** t), v1.sqrt() / math.sqrt(1 - b2 ** t) + eps
        want = p0 * (1 - lr * wd) - rate * m1 / den
        size = (b1 * m0).abs() + ((1 - b1) * g).abs()
        tol = 40 * E * rate * size / den + 4 * E * p0.abs() + 1e-40
        st = opt.state[p]
        assert float(st["step"]) == t
        half = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[p.dtype]
        if "master" in st:
            assert bool(((st["master"].double() - want).abs() <= tol).all())
            assert torch.equal(st["master"].to(p.dtype), p.detach())
        smallest = 2.0 ** -25 if p.dtype == torch.float16 else 0.0     # half a step of fp16's denormals
        assert bool(((p.detach().double() - want).abs() <= tol + half * (want.abs() + tol) + smallest).all())
        m, s, ms, ss = _values(opt, p)
        mt = 13 * E * size + 1e-40
        stol = 11 * E * v1.sqrt() + 1e-40
        if opt.state_bits == 8:
            mt = mt + torch.maximum(2.0 ** -4 * m1.abs(), 2.0 ** -10 * ms) * (1 + 8 * E)
            stol = stol + torch.maximum(2.0 ** -4 * v1.sqrt(), 2.0 ** -9 * ss) * (1 + 8 * E)
            assert bool((s[v1 > 1e-60] > 0).all()), "a positive second moment was rounded to zero"
            for name, x in (("exp_avg_scale", m1), ("exp_avg_sq_root_scale", v1.sqrt())):
                top = torch.nn.functional.pad(x.abs(), (0, -x.numel() % B)).view(-1, B).amax(dim=1)
                room = torch.nn.functional.pad(size if name == "exp_avg_scale" else x, (0, -x.numel() % B)).view(-1, B).amax(dim=1)
                assert bool(((st[name].double() * 448 - top).abs() <= 16 * E * room + 1e-30).all()), name
        assert bool(((m - m1).abs() <= mt).all()) and bool(((s - v1.sqrt()).abs() <= stol).all())


SIZES = (1, 7, 255, 256, 257, 1000, 2047, 2048, 2049, 9001)
KINDS = [(torch.float32, torch.float32, 32, False), (torch.float32, torch.float32, 8, False),
         (torch.bfloat16, torch.bfloat16, 32, False), (torch.bfloat16, torch.float32, 32, True),
         (torch.bfloat16, torch.bfloat16, 8, True), (torch.bfloat16, torch.float32, 8, False),
         (torch.float16, torch.float16, 32, True), (torch.float16, torch.float32, 32, False),
         (torch.float16, torch.float16, 8, False), (torch.float16, torch.float32, 8, True)]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("ptype,gtype,bits,master", KINDS)
def test_step_vs_formula(ptype, gtype, bits, master, offset):
    from fsgs.optim import AdamW
    params, _ = _make(SIZES, ptype, gtype, offset=offset)
    opt = AdamW([dict(params=params[:4], weight_decay=0.1), dict(params=params[4:], lr=3e-4, betas=(0.8, 0.99))],
                lr=1e-2, weight_decay=0.0, state_bits=bits, master_weights=master)
    for k in range(3):
        _, grads = _make(SIZES, ptype, gtype, seed=k + 1, offset=offset)
        for p, g in zip(params, grads):
            p.grad = g
        before = _snapshot(opt, params)
        opt.step()
        _check_step(opt, before, params, grads)


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_clipped_by_their_norm(bits):
    """More tensors than one launch takes, of two types, with and without clipping taking hold."""
    from fsgs.optim import AdamW
    sizes = [(k * 37) % 700 + 1 for k in range(600)]
    a, _ = _make(sizes[:300], torch.float32, torch.float32)
    b, _ = _make(sizes[300:], torch.bfloat16, torch.bfloat16)
    params = a + b
    opt = AdamW(params, lr=1e-3, state_bits=bits, max_grad_norm=0.5, master_weights=True)
    for k, amount in enumerate((1.0, 1e-3)):
        ga, gb = _make(sizes[:300], torch.float32, torch.float32, seed=5 + k)[1], _make(sizes[300:], torch.bfloat16, torch.bfloat16, seed=7 + k)[1]
        grads = [g * amount for g in ga + gb]
        for p, g in zip(params, grads):
            p.grad = g
        before = _snapshot(opt, params)
        opt.step()
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
        assert abs(float(opt.grad_norm) - norm) <= 4 * E * norm
        factor = min(1.0, 0.5 / (norm + 1e-6))
        assert (factor < 1.0) == (k == 0)
        _check_step(opt, before, params, grads, factor)


def test_follows_torchs_adamw():
    """Twenty steps beside torch's AdamW in float64: float32 rounding only."""
    from fsgs.optim import AdamW
    params, _ = _make((300, 5000), torch.float32, torch.float32)
    twins = [torch.nn.Parameter(p.detach().double()) for p in params]
    opt, ref = AdamW(params, lr=1e-3, weight_decay=0.05), torch.optim.AdamW(twins, lr=1e-3, weight_decay=0.05)
    for k in range(20):
        for p, q, g in zip(params, twins, _make((300, 5000), torch.float32, torch.float32, seed=k)[1]):
            p.grad, q.grad = g, g.double()
        opt.step()
        ref.step()
    for p, q in zip(params, twins):
        # a step is below lr / (1 - b1) sqrt(1 - b2^t) / ... < 10 lr, each off by 40 e of that, and 4 e |p|
        assert float((p.double() - q).abs().max()) <= 20 * (40 * E * 10 * 1e-3 + 4 * E * float(q.abs().max()))


@pytest.mark.parametrize("bits", [8, 32])
def test_dropped_steps_change_nothing(bits):
    from fsgs.optim import AdamW
    params, grads = _make((700, 3), torch.float32, torch.float32)
    for p, g in zip(params, grads):
        p.grad = g
    opt = AdamW(params, state_bits=bits)
    one = torch.ones(1, device="cuda")
    opt.step(gate=one, grad_scale=one)

    def frozen():
        return [t.clone().view(torch.uint8) for p in params for t in [p.detach().reshape(-1)] +
                [v.reshape(-1) for v in opt.state[p].values()]]

    before = frozen()
    nan, inf = float("nan"), float("inf")
    for gate, scale in ((0.0, None), (-1.0, None), (nan, None), (-inf, None), (None, 0.0), (None, nan), (None, inf),
                        (None, -1.0), (1.0, nan), (0.0, 1.0)):
        opt.step(gate=None if gate is None else one * gate, grad_scale=None if scale is None else one * scale)
        assert all(torch.equal(x, y) for x, y in zip(before, frozen())), (gate, scale)
    clipped = AdamW(params, state_bits=bits, max_grad_norm=1.0)
    clipped.step()
    clipped.load_state_dict(opt.state_dict())
    state, opt = opt, clipped
    before = frozen()
    for bad in (nan, inf, -inf):
        params[1].grad = torch.tensor([0.0, bad, 1.0], device="cuda")
        opt.step()
        assert not math.isfinite(float(opt.grad_norm))
        assert all(torch.equal(x, y) for x, y in zip(before, frozen())), bad
    params[1].grad = grads[1]
    opt.step()
    assert float(opt.state[params[0]]["step"]) == 2.0 and math.isfinite(float(opt.grad_norm))


def test_a_bad_gradient_spoils_its_element_or_its_block():
    from fsgs.optim import AdamW
    for bits in (32, 8):
        params, grads = _make((1000,), torch.float32, torch.float32)
        grads[0][300] = float("nan")
        params[0].grad = grads[0]
        opt = AdamW(params, state_bits=bits)
        opt.step()
        assert torch.isnan(params[0]).nonzero().flatten().tolist() == [300]
        bad = torch.isnan(_values(opt, params[0])[0]).nonzero().flatten().tolist()
        assert bad == ([300] if bits == 32 else list(range(256, 512)))


def test_eight_bit_moments_at_the_ends_of_the_range():
    """Blocks of zeros, of denormals, with one huge or one tiny element among others; the largest element of a block
    keeps its value to float32 rounding (its 8-bit value is 448 exactly)."""
    from fsgs.optim import AdamW
    g = torch.zeros(6 * B)
    g[B:2 * B] = 1e-40
    g[2 * B] = 1e18
    g[2 * B + 1:3 * B] = 1e-3
    g[3 * B:4 * B] = 1.0
    g[3 * B + 5] = 1e-12
    g[4 * B:5 * B] = -2.0 ** -60
    p = torch.nn.Parameter(torch.zeros(6 * B, device="cuda"))
    p.grad = g.cuda()
    opt = AdamW([p], lr=1.0, weight_decay=0.0, state_bits=8, eps=1e-8)
    opt.step()
    m, s, ms, ss = (t.cpu() for t in _values(opt, p))
    assert bool(torch.isfinite(p).all()) and bool(torch.isfinite(m).all()) and bool(torch.isfinite(s).all())
    for lo, hi in ((0, 2 * B), (5 * B, 6 * B)):
        assert not bool(m[lo:hi].any()) and not bool(s[lo:hi].any())
    for i in (2 * B, 3 * B, 4 * B):
        assert abs(float(m[i]) - 0.1 * float(g[i])) <= 8 * E * 0.1 * abs(float(g[i]))
        assert abs(float(s[i]) - math.sqrt(1e-3) * abs(float(g[i]))) <= 16 * E * math.sqrt(1e-3) * abs(float(g[i]))
    assert float(s[3 * B + 5]) == 2.0 ** -9 * float(ss[3 * B + 5]) > 0 and float(m[3 * B + 5]) == 0.0
    # no eps: where both moments of an element are zero the update is 0 / 0 of the formula, elsewhere finite
    assert bool((p.detach().cpu()[3 * B:4 * B] < 0).all())


def test_a_captured_step_counts_its_replays():
    from fsgs.optim import AdamW
    for bits, clip in ((32, None), (8, 0.3)):
        sizes = (5000, 17)
        a, grads = _make(sizes, torch.float32, torch.float32)
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        fixed = [torch.zeros_like(g) for g in grads]
        oa, ob = (AdamW(x, lr=1e-2, state_bits=bits, max_grad_norm=clip) for x in (a, b))
        for p, g in zip(a, fixed):
            p.grad = g
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="captured|capture"):
            with torch.cuda.graph(graph):
                oa.step()
        oa.init_state()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            oa.step()
        for k in range(4):
            now = _make(sizes, torch.float32, torch.float32, seed=20 + k)[1]
            for f, g, q in zip(fixed, now, b):
                f.copy_(g)
                q.grad = g
            graph.replay()
            ob.step()
            for p, q in zip(a, b):
                assert torch.equal(p, q) and float(oa.state[p]["step"]) == k + 1
                for name, t in ob.state[q].items():
                    assert torch.equal(oa.state[p][name].float(), t.float()), name


def test_on_another_stream_and_with_changing_tensors():
    """A side stream; gradients that come and go, are strided, or have new memory each step; a learning rate, a
    parameter's storage and a state tensor that are replaced between steps."""
    from fsgs.optim import AdamW
    params, _ = _make((64, 513, 12), torch.float32, torch.float32)
    opt = AdamW(params, lr=1e-2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for k in range(6):
            grads = _make((64, 513, 12), torch.float32, torch.float32, seed=40 + k)[1]
            use = [0, 2] if k == 1 else [0, 1, 2]
            grads[1] = torch.stack([grads[1], grads[1]], dim=1)[:, 1]       # stride 2
            for i, (p, g) in enumerate(zip(params, grads)):
                p.grad = None
                if i in use:
                    p.grad = g
            if k == 2:
                opt.param_groups[0]["lr"] = 5e-3
            if k == 3:
                params[0].data = params[0].data.clone()
            if k == 4:
                opt.state[params[2]]["exp_avg"] = opt.state[params[2]]["exp_avg"].clone()
            if k == 5:
                opt.param_groups[0]["betas"] = (0.7, 0.95)
            sel = [params[i] for i in use]
            before = _snapshot(opt, sel)
            opt.step()
            _check_step(opt, before, sel, [grads[i] for i in use])
        assert float(opt.state[params[1]]["step"]) == 5 and float(opt.state[params[0]]["step"]) == 6
    torch.cuda.current_stream().wait_stream(stream)


def test_refusals_on_the_device():
    from fsgs.optim import AdamW, grad_norm
    p = torch.nn.Parameter(torch.zeros(4, 6, device="cuda").t())
    p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="contiguous"):
        AdamW([p]).step()
    q = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    q.grad = torch.ones(8, device="cuda")
    opt = AdamW([q], max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="grad_scale"):
        opt.step(grad_scale=torch.ones(1, device="cuda"))
    for bad in (torch.ones(1), torch.ones(2, device="cuda"), torch.ones(1, device="cuda", dtype=torch.float64)):
        with pytest.raises(RuntimeError, match="gate"):
            opt.step(gate=bad)
    opt.step()
    opt.state[q]["exp_avg"] = torch.zeros(7, device="cuda")
    with pytest.raises(RuntimeError, match="exp_avg"):
        opt.step()
    del opt.state[q]["exp_avg"]
    with pytest.raises(RuntimeError, match="exp_avg"):
        opt.step()
    r = torch.nn.Parameter(torch.zeros(8))
    r.grad = torch.ones(8)
    with pytest.raises(RuntimeError, match="one device"):
        AdamW([torch.nn.Parameter(q.detach()), q, r]).step()
    with pytest.raises(RuntimeError):
        grad_norm([torch.ones(3, device="cuda"), torch.ones(3, device="cuda", dtype=torch.float64)])
    with pytest.raises(RuntimeError):
        grad_norm([torch.ones(3, device="cuda")], max_norm=0.0)


def test_empty_tensors():
    from fsgs.optim import AdamW, grad_norm
    params, grads = _make((0, 5, 0, 300, 0), torch.float32, torch.float32)
    for p, g in zip(params, grads):
        p.grad = g
    opt = AdamW(params, state_bits=8, max_grad_norm=100.0)
    before = _snapshot(opt, params)
    opt.step()
    _check_step(opt, before, params, grads)
    norm, factor = grad_norm([torch.zeros(0, device="cuda")], max_norm=1.0)
    assert float(norm) == 0.0 and float(factor) == 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_vs_double(dtype):
    """Eight squares are added in float32 (their sum 8 e off at most), the rest in double: 4 e relative on the norm, 1 e
    for its own rounding; the factor 3 roundings more."""
    from fsgs.optim import grad_norm
    gen = torch.Generator().manual_seed(1)
    sizes = [1, 3, 8191, 8192, 8193, 100_001] + [k % 50 for k in range(500)]
    ts = [(torch.randn(n + 3, generator=gen) * 10.0 ** (k % 5 - 3)).to(dtype).cuda()[k % 3:k % 3 + n] for k, n in enumerate(sizes)]
    ts.append(torch.randn(40, 30, generator=gen).to(dtype).cuda().t())
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    norm, factor = grad_norm(ts, max_norm=0.25)
    assert abs(float(norm) - want) <= 5 * E * want
    assert abs(float(factor) - 0.25 / (want + 1e-6)) <= 9 * E * float(factor)
    again, _ = grad_norm(ts, max_norm=0.25)
    assert torch.equal(norm, again)
    assert float(grad_norm(ts)[1]) == 1.0


def test_norm_at_the_ends_of_the_range():
    from fsgs.optim import grad_norm
    big = torch.full((100_000,), 1e17, device="cuda")
    norm, factor = grad_norm([big], max_norm=1.0)
    assert abs(float(norm) / (1e17 * math.sqrt(1e5)) - 1) < 1e-6 and 0 < float(factor) < 1e-19
    for bad in (float("inf"), float("nan")):
        t = torch.ones(50_000, device="cuda")
        t[31_234] = bad
        norm, factor = grad_norm([t, torch.ones(3, device="cuda")], max_norm=1.0)
        assert not math.isfinite(float(norm)) and float(factor) == 0.0
    mixed = [torch.ones(9, device="cuda"), torch.ones(7, device="cuda", dtype=torch.bfloat16),
             torch.ones(9, device="cuda", dtype=torch.float16)]
    assert float(grad_norm(mixed)[0]) == 5.0


def test_the_plan_follows_the_optimiser():
    """Between steps: states replaced or cleared, a group added, a parameter put in another's place, hooks, a scheduler,
    a state dictionary loaded: each following step is the formula's."""
    from fsgs.optim import AdamW
    params, _ = _make((400, 30, 2100), torch.float32, torch.float32)
    opt = AdamW(params[:2], lr=1e-2)
    seen = []
    opt.register_step_pre_hook(lambda o, args, kwargs: seen.append("pre"))
    opt.register_step_post_hook(lambda o, args, kwargs: seen.append("post"))
    sched = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)

    def one(sel, seed):
        for p, g in zip(params, _make((400, 30, 2100), torch.float32, torch.float32, seed=seed)[1]):
            p.grad = g
        before = _snapshot(opt, sel)
        opt.step()
        _check_step(opt, before, sel, [p.grad for p in sel])

    one(params[:2], 1)
    assert seen == ["pre", "post"]
    sched.step()
    assert opt.param_groups[0]["lr"] == 5e-3
    one(params[:2], 2)
    opt.state[params[0]] = {k: v.clone() for k, v in opt.state[params[0]].items()}
    one(params[:2], 3)
    del opt.state[params[1]]
    one(params[:2], 4)
    assert float(opt.state[params[1]]["step"]) == 1 and float(opt.state[params[0]]["step"]) == 4
    opt.add_param_group(dict(params=[params[2]], lr=1e-3, weight_decay=0.3))
    one(params, 5)
    opt.load_state_dict(opt.state_dict())
    one(params, 6)
    other = torch.nn.Parameter(torch.randn(30, device="cuda"))
    opt.state[other] = opt.state.pop(params[1])
    opt.param_groups[0]["params"][1] = params[1] = other
    one(params, 7)
    assert float(opt.state[other]["step"]) == 4
    params[2].data = params[2].data[:1000]          # same address, another length
    opt.state[params[2]] = {k: v if k == "step" else v[:1000].clone() for k, v in opt.state[params[2]].items()}
    g = torch.randn(1000, device="cuda")
    params[2].grad = None
    params[0].grad = None
    params[2].grad = g
    before = _snapshot(opt, [params[1], params[2]])
    opt.step()
    _check_step(opt, before, [params[1], params[2]], [params[1].grad, g])
    with torch.autograd.profiler.profile():
        one_grad = [p.grad for p in params[1:]]
        before = _snapshot(opt, params[1:])
        opt.step()
    _check_step(opt, before, params[1:], one_grad)


@pytest.mark.parametrize("bits", [8, 32])
def test_moments_are_the_formula_operation_by_operation(bits):
    """The moments bit for bit as float32 operations one after another give them, roots, scales and 8-bit values too: a
    moment beside a border between two 8-bit values falls on the formula's side."""
    from fsgs.optim import AdamW
    n = 64 * B
    gen = torch.Generator().manual_seed(11)
    spread = lambda: (torch.randn(n, generator=gen) * torch.exp(torch.randn(n, generator=gen))).cuda()  # noqa: E731
    p = torch.nn.Parameter(spread())
    opt = AdamW([p], state_bits=bits)
    opt.init_state()
    st = opt.state[p]
    rows = lambda t: t.view(-1, B)  # noqa: E731

    def pack(x, positive):
        top = x.abs().amax(dim=1, keepdim=True)
        y = x * (448.0 / top)
        y = torch.where(x > 0, y.clamp_min(2.0 ** -9), y) if positive else y
        return y.to(torch.float8_e4m3fn), top

    m, s = rows(spread() * 1e-3), rows(spread().abs() * 1e-3)
    if bits == 8:
        for x, name, positive in ((m, "exp_avg", False), (s, "exp_avg_sq_root", True)):
            code, top = pack(x, positive)
            st[name].copy_(code.view(-1))
            st[name + "_scale"].copy_(top[:, 0] / 448.0)
        m, s = (rows(st[k].float()) * st[k + "_scale"][:, None] for k in ("exp_avg", "exp_avg_sq_root"))
        v = s * s
    else:
        v = s * s
        st["exp_avg"].copy_(m.reshape(-1))
        st["exp_avg_sq"].copy_(v.reshape(-1))
    p.grad = spread() * 1e-3
    g = rows(p.grad)
    m, v = m * 0.9 + g * (1 - 0.9), v * 0.999 + g * g * (1 - 0.999)
    opt.step()
    if bits == 32:
        assert torch.equal(rows(st["exp_avg"]), m) and torch.equal(rows(st["exp_avg_sq"]), v)
        return
    for x, name, positive in ((m, "exp_avg", False), (v.sqrt(), "exp_avg_sq_root", True)):
        code, top = pack(x, positive)
        assert torch.equal(rows(st[name]).float(), code.float()), name
        assert bool(((st[name + "_scale"] - top[:, 0] / 448.0).abs() <= 2 * E * top[:, 0] / 448.0).all()), name


def test_a_gradient_whose_square_overflows():
    """|g| = 1e21: the second moment is infinite, the element's update zero (m / infinity) in 32 and in 8 bits; with 8 bits
    its block's moments are spoiled, its neighbours' parameters of this step are not."""
    from fsgs.optim import AdamW
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(600, device="cuda"))
        g = torch.full((600,), 1e-2, device="cuda")
        g[300] = 1e21
        p.grad = g
        AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits).step()
        assert float(p[300]) == 1.0
        others = torch.cat([p.detach()[:300], p.detach()[301:]])
        # first step: m / (1 - b1) = g, sqrt(v / (1 - b2)) = |g|
        assert float((others - (1.0 - 1e-3 / (1 + 1e-8 / 1e-2))).abs().max()) <= 44 * E


def test_two_graphs_of_one_optimiser():
    """Two captured steps of the same optimiser, each with gradients of its own, replayed in turn beside eager steps: they
    share its state, counts and workspaces."""
    from fsgs.optim import AdamW
    a, _ = _make((3000, 40), torch.float32, torch.float32)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    oa, ob = (AdamW(x, lr=1e-2, state_bits=8, max_grad_norm=0.2) for x in (a, b))
    oa.init_state()
    sets = [_make((3000, 40), torch.float32, torch.float32, seed=s)[1] for s in (31, 32, 33)]
    graphs = []
    for grads in sets[:2]:
        for p, g in zip(a, grads):
            p.grad = g
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            oa.step()
        graphs.append(graph)
    for k in (0, 1, 2, 1, 0, 2, 0):
        for p, q, g in zip(a, b, sets[k]):
            p.grad, q.grad = g, g
        if k < 2:
            graphs[k].replay()
        else:
            oa.step()
        ob.step()
        assert torch.equal(oa.grad_norm, ob.grad_norm)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            assert all(torch.equal(oa.state[p][n].float(), t.float()) for n, t in ob.state[q].items())


def test_tensors_beyond_32_bits_of_elements():
    """2^31 + 777 bf16 elements with 8-bit moments, clipped: the ends against the formula, the norm against a double sum."""
    from fsgs.optim import AdamW
    n = 2 ** 31 + 777
    p = torch.nn.Parameter(torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda"))
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[:5000] = 1.0
    g[-5000:] = -2.0
    g[n // 2] = 4.0
    p.grad = g
    opt = AdamW([p], lr=0.25, weight_decay=0.0, state_bits=8, max_grad_norm=1e9)
    opt.step()
    assert abs(float(opt.grad_norm) - math.sqrt(5000 + 20000 + 16)) <= 5 * E * 160
    # the first step is lr sign(g): m / (1 - b1) = g, sqrt(v / (1 - b2)) = |g|; bf16 at 0.25 and 0.75 rounds to 2^-8 of them
    assert float((p[:5000].float() - 0.25).abs().max()) <= 0.25 * 2.0 ** -8
    assert float((p[-5000:].float() - 0.75).abs().max()) <= 0.75 * 2.0 ** -8
    assert float((p[n // 2].float() - 0.25).abs()) <= 0.25 * 2.0 ** -8
    assert bool((p[5000:10_000] == 0.5).all()) and bool((p[-10_000:-5000] == 0.5).all())
    st = opt.state[p]
    assert st["exp_avg_scale"].numel() == (n + B - 1) // B and float(st["exp_avg_scale"][-1]) > 0


def test_parameters_that_share_memory_are_refused():
    from fsgs.optim import AdamW
    base = torch.zeros(1000, device="cuda")
    for a, b in ((base, base), (base[:500], base[499:]), (base[100:101], base)):
        params = [torch.nn.Parameter(a), torch.nn.Parameter(b)]
        for p in params:
            p.grad = torch.ones_like(p)
        with pytest.raises(RuntimeError, match="share memory"):
            AdamW(params).step()
    assert not bool(base.any())
    params = [torch.nn.Parameter(x) for x in (base[500:], base[:500], base[500:500])]   # neighbours, and an empty one inside
    for p in params:
        p.grad = torch.ones_like(p)
    AdamW(params, lr=0.5, weight_decay=0.0).step()
    # the first step is lr g / (|g| + eps), 40 E U off
    assert float((base + 0.5 / (1 + 1e-8)).abs().max()) <= 40 * E * 0.5


def test_numbers_on_the_device_are_refused():
    from fsgs.optim import AdamW
    p = [torch.nn.Parameter(torch.zeros(8, device="cuda"))]
    for kw in (dict(lr=torch.tensor(1e-3, device="cuda")), dict(weight_decay=torch.tensor(0.1, device="cuda"))):
        with pytest.raises(RuntimeError, match="numbers on the host"):
            AdamW(p, **kw)


def test_states_that_changed_where_they_lie_are_refused():
    """A state tensor cut, of another type, transposed or replaced at the same address since the last step, and another form
    of the state asked for: refused before anything is launched; put back, the next step is the formula's."""
    from fsgs.optim import AdamW
    for bits, dtype, master in ((32, torch.float32, False), (8, torch.bfloat16, True)):
        params, grads = _make((600, 24), dtype, torch.float32)
        for p, g in zip(params, grads):
            p.grad = g
        opt = AdamW(params, state_bits=bits, master_weights=master)
        opt.step()
        st = opt.state[params[1]]

        def refused(what):
            frozen = [t.clone() for p in params for t in [p.detach()] + list(opt.state[p].values())]
            with pytest.raises(RuntimeError, match=what):
                opt.step()
            after = [t for p in params for t in [p.detach()] + list(opt.state[p].values())]
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(frozen, after))

        for name in [n for n in st if n != "step"]:
            whole = st[name]
            there = whole.data_ptr()
            changed = [whole.view(torch.int8).view(-1)[:whole.numel()], whole.view(-1)[:whole.numel() // 2]]
            if whole.numel() == 24:
                changed.append(whole.view(6, 4).t())
            for other in changed:
                assert other.data_ptr() == there or other.numel() == 0
                st[name] = other
                refused(name)
                st[name] = whole
            whole.data, kept = whole.data.view(-1)[:0], whole.data        # the same tensor, cut in place
            refused(name)
            whole.data = kept
        # given back and replaced by a shorter one, for which the allocator may hand out the same address
        name = "exp_avg"
        kept = st[name].clone()
        del whole, changed, other, st[name]
        st[name] = torch.zeros(7, dtype=kept.dtype, device="cuda")
        refused(name)
        st[name] = kept
        opt.state_bits = 40 - bits
        refused("state")
        opt.state_bits = bits
        if dtype != torch.float32:
            del st["master"]
            opt.master_weights = False
            opt.step()                                                   # a state that has what is asked for
            opt.master_weights = True
            refused("master")
            st["master"] = params[1].detach().float()
        before = _snapshot(opt, params)
        opt.step()
        _check_step(opt, before, params, grads)


def test_a_step_marks_what_it_writes():
    """A graph that has saved a parameter before a step raises in its backward pass, as after torch's optimisers; every
    state that a step writes counts as modified, gradients do not, and tensors without a version are left alone."""
    from fsgs.loss import table_balance_loss
    from fsgs.optim import AdamW
    for bits, dtype, master in ((32, torch.float32, False), (8, torch.bfloat16, True)):
        z = torch.nn.Parameter(torch.randn(60, 40, device="cuda").to(dtype))
        z.grad = torch.ones_like(z)
        opt = AdamW([z], state_bits=bits, master_weights=master)
        opt.step()
        table, _ = table_balance_loss(z, torch.zeros(60, 2, dtype=torch.int64, device="cuda"))
        square = (z * z).sum()
        held = [z] + list(opt.state[z].values())
        before, grad = [t._version for t in held], z.grad._version
        opt.step()
        assert all(t._version > v for t, v in zip(held, before)) and z.grad._version == grad
        for loss in (table, square):
            with pytest.raises(RuntimeError, match="modified"):
                loss.backward()
        with torch.inference_mode():
            p = torch.zeros(5, device="cuda")
            p.grad = torch.ones(5, device="cuda")
            AdamW([p], lr=0.5, weight_decay=0.0, state_bits=bits).step()
        assert float((p + 0.5 / (1 + 1e-8)).abs().max()) <= 40 * E * 0.5     # the first step is lr g / (|g| + eps)


def test_loaded_numbers_on_the_device_are_read():
    """A state of torch's AdamW with its learning rate on the device: read once, when it is loaded; a step can be captured."""
    from fsgs.optim import AdamW
    params, grads = _make((300,), torch.float32, torch.float32)
    params[0].grad = grads[0]
    ref = torch.optim.AdamW(params, lr=torch.tensor(2.0 ** -7, device="cuda"), capturable=True)
    ref.step()
    opt = AdamW(params)
    opt.load_state_dict(ref.state_dict())
    assert type(opt.param_groups[0]["lr"]) is float and opt.param_groups[0]["lr"] == 2.0 ** -7
    assert torch.is_tensor(ref.param_groups[0]["lr"])
    before = _snapshot(opt, params)
    opt.step()
    _check_step(opt, before, params, grads)


def test_numbers_put_on_the_device_between_steps_are_refused():
    from fsgs.optim import AdamW
    params, grads = _make((300,), torch.float32, torch.float32)
    params[0].grad = grads[0]
    opt = AdamW(params, lr=1e-2)
    group = opt.param_groups[0]
    opt.step()
    for key, bad, good in (("lr", torch.tensor(0.1, device="cuda"), 1e-3), ("weight_decay", torch.tensor(0.1, device="cuda"), 0.0),
                           ("eps", torch.tensor(0.1, device="cuda"), torch.tensor(1e-6)),
                           ("betas", (torch.tensor(0.5, device="cuda"), 0.9), (0, 0.9))):
        group[key] = bad
        with pytest.raises(RuntimeError, match="numbers on the host"):
            opt.step()
        group[key] = good
    group["eps"] = float(group["eps"])
    before = _snapshot(opt, params)
    group["eps"] = torch.tensor(group["eps"], dtype=torch.float64)         # a tensor on the host is read at each step
    opt.step()
    group["eps"] = float(group["eps"])
    _check_step(opt, before, params, grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_over_the_whole_range_of_the_type(dtype):
    """Gradients whose squares leave the range of float32 on either side, alone, in all tensors, and beside zeros and beside
    others: 4 e relative on the norm and 1 e for its own rounding, half a denormal where it is one.  The factor: 4 e more,
    or half a denormal, or (above 2^126) the inverse's half denormal of 2^-150 times the limit."""
    from fsgs.optim import grad_norm
    gen = torch.Generator().manual_seed(4)
    lo, hi = (2.0 ** -24, 6e4) if dtype == torch.float16 else (1e-45, 3e38) if dtype == torch.float32 else (1e-40, 3e38)
    sizes = (1, 7, 300, 8192, 50_001)
    for amount in (lo, 1e-38, 1e-30, 1e-23, 1e-20, 1e-18, 1e-16, 1.0, 1e15, 6e18, 1e19, 1e25, 1e36, hi):
        if not lo <= amount <= hi:
            continue
        for others in (None, 0.0, 1e-25, 1e-12):
            ts = []
            for k, n in enumerate(sizes):
                x = (torch.rand(n + 1, generator=gen) + 0.5).double() * amount
                if others is not None:
                    x = torch.where(torch.rand(n + 1, generator=gen) < 1e-3, x, others)
                ts.append(x.clamp(max=float(torch.finfo(dtype).max)).to(dtype).cuda()[k % 2:n + k % 2])
            want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
            norm, factor = (float(t) for t in grad_norm(ts, max_norm=0.25))
            if want > 3.4e38:
                assert norm == math.inf and factor == 0.0
                continue
            assert abs(norm - want) <= 5 * E * want + 2.0 ** -150, (amount, others, norm, want)
            limit = min(1.0, 0.25 / (want + 1e-6))
            assert abs(factor - limit) <= 9 * E * limit + 2.0 ** -150 * 1.25, (amount, others, factor, limit)
            assert float(grad_norm([t for t in ts] * 2, max_norm=0.25)[0]) > norm or want == 0.0
    assert float(grad_norm([torch.zeros(70_000, dtype=dtype, device="cuda"), -torch.zeros(9, dtype=dtype, device="cuda")])[0]) == 0.0
    for bad in (math.inf, -math.inf, math.nan):
        t = torch.full((9000,), 1e-30 if dtype != torch.float16 else 1e-7, dtype=dtype, device="cuda")
        t[7777] = bad
        norm, factor = grad_norm([t], max_norm=1.0)
        assert not math.isfinite(float(norm)) and float(factor) == 0.0


def test_an_optimiser_let_go_of_while_its_step_runs():
    """Made on one stream, stepped on another that is busy, dropped: the memory that it brought along is not handed out again
    before that step is done."""
    import gc
    from fsgs.optim import AdamW
    params, grads = _make((700,), torch.float32, torch.float32)
    params[0].grad = grads[0]
    opt = AdamW(params, max_grad_norm=1.0)
    opt.step()
    torch.cuda.synchronize()
    own = [opt._work[1], *opt._norm]
    places, sizes = {t.untyped_storage().data_ptr() for t in own}, [t.untyped_storage().nbytes() for t in own]
    state = dict(opt.state)                        # the parameters' states are the caller's here
    stream = torch.cuda.Stream()
    busy, done = torch.cuda.Event(), torch.cuda.Event()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(1_000_000_000)           # half a second
        busy.record()
        opt.step()
        done.record()
    del own, opt
    gc.collect()
    handed_out = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(30)]
    waiting = not busy.query()
    assert waiting and not places & {t.data_ptr() for t in handed_out}
    done.synchronize()
    assert float(state[params[0]]["step"]) == 2


def test_eight_bit_second_moments_over_many_steps():
    """Constant gradients per element beside a twin with 32 bits, the block's largest element holding its own.  A value
    (8 + k) 2^j of the format has half a step of h = 1 / (2 (8 + k)) above it (1 / (2 k) where it is k smallest steps), so
    s = sqrt(v) rises as long as sqrt(b2 + (1 - b2) (g / s)^2) >= 1 + h and rests at
    g / s < sqrt(((1 + h)^2 - b2) / (1 - b2)); it never falls, as sqrt(b2) = 0.9995 is within half a step of 1; and when the
    largest element grows, all grow with it (a step takes 0.8 % of their share at most, less than 1/32).  Float32 adds 2e-5."""
    from fsgs.optim import AdamW
    b2, lr = 0.999, 1e-3
    first = torch.tensor([0.9 * 2.0 ** -(i % 17) * (1 - (i // 17) / 40) for i in range(B)], device="cuda")
    first[0] = 1.0
    params = [torch.nn.Parameter(torch.zeros(B, device="cuda")) for _ in range(2)]
    eight, whole = opts = [AdamW([p], lr=lr, betas=(0.9, b2), weight_decay=0.0, eps=1e-12, state_bits=bits)
                           for p, bits in zip(params, (8, 32))]

    def run(g, steps):
        before = [p.detach().clone() for p in params]
        for _ in range(steps):
            before = [p.detach().clone() for p in params]
            for p, o in zip(params, opts):
                p.grad = g
                o.step()
        st = eight.state[params[0]]
        held = (st["exp_avg_sq_root"].double() * st["exp_avg_sq_root_scale"].double())
        return (held, whole.state[params[1]]["exp_avg_sq"].double().sqrt(), st["exp_avg_sq_root"].double(),
                [(b - p.detach()).double() for b, p in zip(before, params)])

    def half_step(code):
        low = 2.0 ** -6                                    # the smallest normal value; steps of 2^-9 below it
        _, e = torch.frexp(code)
        return torch.where(code >= low, torch.ldexp(torch.ones_like(code), e - 5), 2.0 ** -10) / code

    held, true, codes, _ = run(first, 50)
    fine = codes >= 2.0 ** -6
    assert bool(fine.any()) and bool((~fine).any())
    off = (held / true - 1).abs()
    assert float(off[fine].max()) <= 1 / 16 + 1e-3 and float(off.max()) <= 1.0 + 1e-3
    # gradients that vanish: the bytes stay, where 32 bits go down to 0.999^1500
    gone = first.clone()
    gone[1:] = 0
    held, true, now, _ = run(gone, 3000)
    assert torch.equal(now, codes) and float((held / true)[1:].min()) > 3
    # gradients that grow thirty times
    grown = (first * 30).clamp(max=0.9)
    grown[0] = 1.0
    held, true, codes, moved = run(grown, 400)
    bound = (((1 + half_step(codes)) ** 2 - b2) / (1 - b2)).sqrt()
    assert float(bound.max()) < 35.4 and float(bound[codes >= 2.0 ** -6].max()) < 11.41
    ratio = grown.double() / held
    assert bool((ratio <= bound * (1 + 1e-3)).all()) and float(ratio.max()) > 4
    # the step: m = g, held as a value of the format, 1/16 off, and bias corrections that have gone to 1 (0.999^3450 = 0.03)
    assert bool((moved[0] <= lr * bound * (1 + 1 / 16) * 1.03).all()) and float(moved[1][1:].max()) < lr * 2
    # the largest grows four times: the others' bytes stay and their values go with it
    loud = grown.clone()
    loud[0] = 4.0
    after, true, now, _ = run(loud, 3000)
    assert torch.equal(now, codes)
    share = after / held
    assert float(share.min()) > 3.8 and float(share.max()) < 4.1


def test_a_state_given_to_two_parameters_is_refused():
    from fsgs.optim import AdamW
    params, grads = _make((40, 40, 9), torch.float32, torch.float32)
    for p, g in zip(params, grads):
        p.grad = g
    opt = AdamW(params)
    opt.step()
    kept = opt.state[params[1]]
    frozen = [t.clone() for p in params for t in [p.detach()] + list(opt.state[p].values())]
    for shared in (opt.state[params[0]], dict(kept, step=opt.state[params[2]]["step"])):
        opt.state[params[1]] = shared
        with pytest.raises(RuntimeError, match="share a state"):
            opt.step()
    opt.state[params[1]] = kept
    assert all(torch.equal(a, b) for a, b in zip(frozen, [t for p in params for t in [p.detach()] + list(opt.state[p].values())]))
    before = _snapshot(opt, params)
    opt.step()
    _check_step(opt, before, params, grads)


def test_roots_are_rounded_correctly():
    """The root of the second moment for a quarter of a million mantissas, read back through the scale of a block in which it
    is the largest: the float32 nearest to the root of fl(g^2) / 2, times the float32 nearest to 1/448."""
    from fsgs.optim import AdamW
    n, gen = 2 ** 18, torch.Generator("cuda").manual_seed(6)
    g = torch.full((n, B), 2.0 ** -20, device="cuda")              # nothing in a lane leaves the range of the fast root
    g[:, 8] = 1.0 + torch.randint(0, 2 ** 23, (n,), device="cuda", generator=gen).float() * 2.0 ** -23
    p = torch.nn.Parameter(torch.zeros(n * B, device="cuda"))
    p.grad = g.view(-1)
    opt = AdamW([p], betas=(0.0, 0.5), state_bits=8)
    opt.step()
    root = ((g[:, 8] * g[:, 8]).double() / 2).sqrt().float()
    assert torch.equal(opt.state[p]["exp_avg_sq_root_scale"], root * torch.tensor(1 / 448, dtype=torch.float32, device="cuda"))
