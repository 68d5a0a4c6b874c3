"""What the balance losses refuse (no GPU), and the layout of the argument structures of the training-step operators."""
import re
import os

import pytest
import torch

from conftest import ROOT


def test_refusals_without_a_device():
    from fsgs.loss import balance_loss, balance_value_and_grad, table_balance_loss, table_balance_value_and_grad
    w, idx = torch.ones(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    for call in (lambda: balance_loss(w, idx, 3), lambda: balance_value_and_grad(w, idx, 3),
                 lambda: table_balance_loss(w, idx), lambda: table_balance_value_and_grad(w, idx)):
        with pytest.raises(RuntimeError):
            call()


def test_entry_points_check_their_arguments():
    """The C side refuses before anything is launched (no device is needed to see it)."""
    from fsgs._lib import lib
    L = lib()
    need = L.fsgs_balance_workspace_bytes
    pairs_ws, table_ws = need(4, 2, 3, 0), need(4, 2, 3, 1)
    assert pairs_ws % 16 == 0 and need(10, 3, 70_000, 0) - need(0, 3, 70_000, 0) == 128 and need(0, 1, 1, 1) > 0
    for bad in ((-1, 2, 3, 0), (4, 0, 3, 0), (4, 2, 0, 0), (4, 2, 3, 2), (1 << 36, 2, 3, 0), (1 << 26, 2, 2048, 1)):
        assert need(*bad) == 0, bad
    ok = dict(N=4, K=2, M=3, idx=4096, mask=0, form=0, counts=4096, ws=4096, n=pairs_ws)

    def count(**kw):
        a = dict(ok, **kw)
        return L.fsgs_balance_count(a["N"], a["K"], a["M"], a["idx"], a["mask"], a["form"], a["counts"], a["ws"], a["n"], None)

    for bad in (dict(N=-1), dict(K=0), dict(M=0), dict(idx=0), dict(counts=0), dict(form=2)):
        assert count(**bad) == -1, bad
    assert count(ws=0) == -3 and count(ws=4100) == -3 and count(n=pairs_ws - 1) == -3 and count(N=1 << 40) == -5

    def pairs(N=4, K=2, M=3, w=4096, c=4096, ws=4096, n=pairs_ws, loss=4096, g=0):
        return L.fsgs_balance_pairs(N, K, M, w, c, ws, n, 1.0, None, loss, g, 0, None)

    assert pairs(w=0) == -1 and pairs(c=0) == -1 and pairs(N=-1) == -1 and pairs(ws=0) == -3 and pairs(n=8) == -3 and pairs(N=1 << 40) == -5
    assert pairs(loss=0) == 0                                      # nothing asked for

    def table(N=4, M=3, type=0, t=4096, rs=3, c=4096, ws=4096, n=table_ws, loss=4096, g=0, gs=3):
        return L.fsgs_balance_table(N, M, type, t, rs, None, c, ws, n, 1.0, None, loss, g, gs, None)

    for bad in (dict(N=-1), dict(M=0), dict(type=3), dict(t=0), dict(rs=2), dict(c=0), dict(g=4096, gs=2)):
        assert table(**bad) == -1, bad
    assert table(ws=0) == -3 and table(n=5) == -3 and table(loss=0) == 0 and table(N=1 << 40) == -5


def test_step_entry_points_check_their_arguments():
    from fsgs import _lib
    L = _lib.lib()
    def step(n=1, p=0, g=0, bits=32, b1=0.9, b2=0.999, eps=1e-8, ws=4096, size=None, **kw):
        t = (_lib.AdamWTensor * 1)()
        for k in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step"):
            setattr(t[0], k, 4096)
        t[0].numel = 8
        for k, v in kw.items():
            setattr(t[0], k, v)
        import ctypes
        return L.fsgs_adamw_multi(n, ctypes.addressof(t), p, g, bits, b1, b2, eps, None, None, ws,
                                  L.fsgs_adamw_workspace_bytes() if size is None else size, None)
    for bad in (dict(n=-1), dict(p=3), dict(g=-1), dict(bits=16), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
                dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(step=None), dict(numel=-1),
                dict(bits=8, exp_avg_scale=None), dict(bits=8, exp_avg_sq_scale=None)):
        assert step(**bad) == -1, bad
    for bad in (dict(p=0, g=1), dict(p=1, g=2), dict(p=2, g=1), dict(p=0, master=4096)):
        assert step(**bad) == -2, bad
    assert step(numel=1 << 50) == -5 and step(n=0) == 0 and step(ws=None) == step(ws=4100) == step(size=15) == -3
    n = L.fsgs_grad_norm_workspace_bytes()
    one = (_lib.NormTensor * 1)()
    import ctypes
    def norm(count=1, most=1.0, ws=4096, size=n, out=4096, **kw):
        one[0].data, one[0].numel, one[0].type = 4096, 8, 0
        for k, v in kw.items():
            setattr(one[0], k, v)
        return L.fsgs_grad_norm(count, ctypes.addressof(one), most, ws, size, out, None)
    for bad in (dict(count=-1), dict(most=0.0), dict(most=float("nan")), dict(out=None), dict(data=None), dict(numel=-1), dict(type=3)):
        assert norm(**bad) == -1, bad
    assert norm(ws=None) == -3 and norm(ws=4100) == -3 and norm(size=n - 1) == -3


def test_argument_structures_follow_the_header():
    from fsgs import _lib
    header = open(os.path.join(ROOT, "include", "fsgs.h")).read()
    for cname, cls in (("fsgs_adamw_tensor", _lib.AdamWTensor), ("fsgs_norm_tensor", _lib.NormTensor)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), header, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = [d.split()[-1].lstrip("*") for d in body.split(";") if d.strip()]
        assert names == [f[0] for f in cls._fields_], cname
