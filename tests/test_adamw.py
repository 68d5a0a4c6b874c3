"""AdamW on the CPU: what it refuses, and what its state dictionary keeps."""
import copy

import pytest
import torch

from fsgs.optim import AdamW, grad_norm


def _with_state(opt):
    """State as a step would have left it, filled with values that survive no cast unnoticed."""
    for k, p in enumerate(p for g in opt.param_groups for p in g["params"]):
        st = opt._state_of(p)
        for name, t in st.items():
            if t.dtype == torch.float8_e4m3fn:
                t.copy_((torch.arange(t.numel()).reshape(t.shape) % 13 - 6.0).to(torch.float8_e4m3fn))
            else:
                t.copy_(torch.linspace(1.00001, 2.00001, t.numel()).reshape(t.shape) * (k + 1))
    return opt


def _params(dtype=torch.float32):
    return [torch.nn.Parameter(torch.randn(n, dtype=torch.float32).to(dtype)) for n in (5, 300)]


@pytest.mark.parametrize("kw", [dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)),
                                dict(eps=-1e-8), dict(weight_decay=-0.1), dict(max_grad_norm=0.0), dict(max_grad_norm=-1.0)])
def test_refused_settings(kw):
    with pytest.raises(RuntimeError):
        AdamW(_params(), **kw)


def test_refused_parameters():
    with pytest.raises(RuntimeError):
        AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    p = _params()
    p[0].grad = torch.ones(5)
    for opt in (AdamW(p), AdamW(p, state_bits=8, max_grad_norm=1.0)):
        with pytest.raises(RuntimeError):
            opt.step()                         # no CPU path
        with pytest.raises(RuntimeError):
            opt.init_state()
    AdamW(_params()).step()                    # nothing has a gradient: nothing to do
    for bad in ([], [torch.zeros(3)]):
        with pytest.raises(RuntimeError):
            grad_norm(bad)


@pytest.mark.parametrize("bits,dtype,master", [(32, torch.float32, False), (8, torch.float32, False),
                                               (32, torch.bfloat16, True), (8, torch.float16, True), (8, torch.bfloat16, False)])
def test_state_dict_keeps_types_and_bits(bits, dtype, master, tmp_path):
    a = _with_state(AdamW(_params(dtype), lr=3e-4, state_bits=bits, master_weights=master))
    torch.save(a.state_dict(), tmp_path / "s.pt")
    sd = torch.load(tmp_path / "s.pt")
    b = AdamW(_params(dtype), state_bits=bits, master_weights=master)
    for _ in range(2):                         # into an optimiser without state, and into one with it
        before = {p: dict(st) for p, st in b.state.items()}
        b.load_state_dict(sd)
        assert b.param_groups[0]["lr"] == 3e-4
        for p, q in zip(a.param_groups[0]["params"], b.param_groups[0]["params"]):
            assert set(a.state[p]) == set(b.state[q]) == set(a._names(p))
            for name, t in a.state[p].items():
                u = b.state[q][name]
                assert u.dtype == t.dtype and u.shape == t.shape and torch.equal(u.float(), t.float()), name
                assert q not in before or before[q][name] is u, "state tensors that are there are written, not replaced"


def test_state_dicts_that_do_not_fit_are_refused():
    sd32 = _with_state(AdamW(_params())).state_dict()
    sd8 = _with_state(AdamW(_params(), state_bits=8)).state_dict()
    for opt, sd in ((AdamW(_params(), state_bits=8), sd32), (AdamW(_params()), sd8),
                    (AdamW(_params(torch.bfloat16), master_weights=True), sd32),
                    (AdamW(_params()[:1]), sd32), (AdamW(_params()[::-1]), sd32)):
        with pytest.raises(RuntimeError):
            opt.load_state_dict(sd)
        assert len(opt.state) == 0


def test_state_of_torchs_adamw_loads():
    p = _params()
    ref = torch.optim.AdamW(p, lr=1e-2)
    for q in p:
        q.grad = torch.randn_like(q)
    ref.step()
    opt = AdamW(p, lr=1.0)
    opt.load_state_dict(ref.state_dict())
    for q in p:
        assert float(opt.state[q]["step"]) == 1.0
        assert torch.equal(opt.state[q]["exp_avg"], ref.state[q]["exp_avg"])
        assert torch.equal(opt.state[q]["exp_avg_sq"], ref.state[q]["exp_avg_sq"])


def test_copies_keep_their_settings():
    a = _with_state(AdamW(_params(torch.bfloat16), state_bits=8, master_weights=True, max_grad_norm=2.0))
    b = copy.deepcopy(a)
    assert (b.state_bits, b.master_weights, b.max_grad_norm) == (8, True, 2.0) and b.grad_norm is None
    assert {len(s) for s in b.state.values()} == {6}


def test_loading_a_state_that_has_none_starts_again_in_place():
    """What a fresh optimiser saves has no state: a loaded one starts again as new, in the tensors that it had (a captured
    step may be using them)."""
    a = _with_state(AdamW(_params(torch.bfloat16), state_bits=8, master_weights=True))
    held = {p: dict(st) for p, st in a.state.items()}
    a.load_state_dict(AdamW(_params(torch.bfloat16), state_bits=8, master_weights=True).state_dict())
    for p, before in held.items():
        st = a.state[p]
        assert all(st[n] is t for n, t in before.items()) and torch.equal(st["master"], p.detach().float())
        assert all(not bool(st[n].float().any()) for n in st if n != "master")


@pytest.mark.parametrize("of", [lambda p: torch.optim.AdamW(p, amsgrad=True), lambda p: torch.optim.AdamW(p, maximize=True),
                                lambda p: torch.optim.Adam(p, weight_decay=0.1)])
def test_state_dicts_of_another_rule_are_refused(of):
    opt = AdamW(_params())
    with pytest.raises(RuntimeError, match="amsgrad"):
        opt.load_state_dict(of(_params()).state_dict())
    opt.load_state_dict(torch.optim.Adam(_params()).state_dict())    # without weight decay the two are one


def test_a_schedule_follows_the_steps():
    opt = AdamW(_params(), lr=1.0)
    schedule = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    for _ in range(2):
        opt.step()                             # nothing has a gradient
        schedule.step()
    assert opt.param_groups[0]["lr"] == 0.25 and schedule.get_last_lr() == [0.25]
    AdamW(_params(), lr=torch.tensor(0.5))     # on the host: read at each step


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=float("nan")),
                                 dict(params=[torch.zeros(3, dtype=torch.float64)])])
def test_a_refused_group_is_not_kept(bad):
    opt = AdamW(_params(), lr=1e-3)
    with pytest.raises(RuntimeError):
        opt.add_param_group(dict(dict(params=[torch.zeros(3)]), **bad))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[torch.zeros(3)], lr=0.5))
    assert [g["lr"] for g in opt.param_groups] == [1e-3, 0.5]


def test_a_group_with_settings_of_another_kind_is_not_kept():
    opt = AdamW(_params(), lr=1e-3)
    for bad in (dict(betas=0.9), dict(lr="fast"), dict(eps=None)):
        with pytest.raises((TypeError, ValueError)):
            opt.add_param_group(dict(params=[torch.zeros(3)], **bad))
    assert len(opt.param_groups) == 1


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=float("nan")), dict(weight_decay=-0.5)])
def test_loaded_settings_are_checked(bad):
    """What the constructor refuses is refused in a state dictionary too, before anything has changed."""
    opt = _with_state(AdamW(_params(), lr=1e-3))
    held = {p: {n: t.clone() for n, t in st.items()} for p, st in opt.state.items()}
    sd = _with_state(AdamW(_params(), lr=0.25)).state_dict()
    sd["param_groups"][0].update(bad)
    with pytest.raises(RuntimeError):
        opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] == 1e-3 and opt.param_groups[0]["betas"] == (0.9, 0.999)
    assert all(torch.equal(opt.state[p][n], t) for p, st in held.items() for n, t in st.items())


def test_hooks_of_loading():
    """A pre-hook sees the whole state dictionary and may return another one, a post-hook sees the loaded state; afterwards
    the optimiser has the hooks that it had."""
    src = _with_state(AdamW(_params(), lr=0.25))
    opt, seen = AdamW(_params(), lr=1.0), []

    def before(o, sd):
        seen.append(len(sd["state"]))
        sd["state"] = {k: dict(v, step=torch.tensor(7.0)) for k, v in sd["state"].items()}
        sd["param_groups"] = [dict(g, lr=0.5) for g in sd["param_groups"]]
        return sd

    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(lambda o: seen.append([float(o.state[p]["step"]) for p in o.param_groups[0]["params"]]))
    for n in (1, 2):
        given = src.state_dict()
        opt.load_state_dict(given)
        assert seen == [2, [7.0, 7.0]] * n and opt.param_groups[0]["lr"] == 0.5
        assert given["param_groups"][0]["lr"] == 0.25
        for p, q in zip(src.param_groups[0]["params"], opt.param_groups[0]["params"]):
            assert torch.equal(src.state[p]["exp_avg"], opt.state[q]["exp_avg"])

    def refuse(o, sd):
        return dict(sd, state={k: {n: t for n, t in v.items() if n != "exp_avg"} for k, v in sd["state"].items()})

    handle = opt.register_load_state_dict_pre_hook(refuse)
    with pytest.raises(RuntimeError, match="exp_avg"):
        opt.load_state_dict(src.state_dict())
    handle.remove()
    opt.load_state_dict(src.state_dict())
    assert seen == [2, [7.0, 7.0]] * 2 + [2] + [2, [7.0, 7.0]]


@pytest.mark.parametrize("bad", [lambda: 0.0, 1.0, [1.0], "open"])
def test_a_gate_that_is_no_tensor_is_refused(bad):
    """A closure too: the step of this optimiser takes a gate in the first place."""
    opt = AdamW(_params())
    for call in (lambda: opt.step(bad), lambda: opt.step(gate=bad), lambda: opt.step(grad_scale=bad)):
        with pytest.raises(RuntimeError, match="one-element float32 tensors"):
            call()
