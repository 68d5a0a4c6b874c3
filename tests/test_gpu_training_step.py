"""The training-step operators together, as ``DynamicScene.train_views`` runs them: balance loss on the kernel weights, its
gradient through the kernel weights into the exchange bucket, the norm of the dense gradients and the AdamW step with
8-bit moments, beside the masked Adam of the Gaussians."""
import math

import pytest
import torch

import motion_oracle as mo
from test_gpu_adamw import E, _check_step, _snapshot

pytestmark = pytest.mark.gpu

W, H, P, M, K = 96, 64, 3000, 48, 3


def _scene(**kw):
    from fsgs import workloads as wl
    from fsgs.motion import MotionNet
    from fsgs.scene import DynamicScene
    surf = wl.surfels(P, seed=5, log_scale_mean=-3.2)
    centres = wl.superpoints(surf["means"], M=M, seed=1)["centres"]
    gen = torch.Generator().manual_seed(2)
    net = MotionNet(M, width=64, local_frame=True, seed=4)
    with torch.no_grad():
        net.views()["heads.weight"].copy_(torch.randn(net.views()["heads.weight"].shape, generator=gen) * 0.02)
    weights = (torch.full((M,), -1.2) + 0.2 * torch.randn(M, generator=gen), torch.randn(M, generator=gen) * 0.5)
    cams = [{k: v.cuda() for k, v in wl.camera(W, H, eye=e).items()} for e in ((0.0, 0.0, 4.0), (1.0, 0.5, 3.5))]
    return DynamicScene(surf, centres, K=K, device="cuda", motion_net=net, kernel_weights=weights, **kw), cams


def _balance64(scene):
    """Loss, counts and gradients of raw radius and raw weight in float64."""
    rr, rw = (p.detach().cpu().double().requires_grad_() for p in (scene.sp_radius, scene.sp_weight))
    idx = scene.knn_idx.cpu()
    w = mo.kernel_weights(scene.knn_d2.cpu().double(), idx, rr, rw)
    counts = torch.bincount(idx.reshape(-1), minlength=M)
    loss = M * (w * (counts.double() / (P * K))[idx]).sum() / P
    loss.backward()
    return float(loss), counts, rr.grad, rw.grad


def test_balance_alone_reaches_the_kernel_weights():
    """Views without an image gradient: what is left in the bucket is the balance term.  The kernels of the weights and of
    their adjoint are held to 1e-4 relative elsewhere; the same here."""
    scene, cams = _scene(balance=0.7)
    want, counts, g_r, g_w = _balance64(scene)
    zero = torch.zeros(3, H, W, device="cuda")
    kept = {}
    scene.dense_optimizer.step_gated = lambda gate: kept.update(r=scene.sp_radius.grad.clone(), w=scene.sp_weight.grad.clone())
    for views in ([dict(cam=cams[0], t=torch.tensor([0.3]).cuda(), g_images=zero)], []):
        scene.train_views(views, (W, H))
        assert torch.equal(scene.superpoint_counts.cpu(), counts)
        assert abs(float(scene.balance_loss) - 0.7 * want) <= 1e-5
        for got, ref in ((kept["r"], g_r), (kept["w"], g_w)):
            assert float((got.cpu().double() - 0.7 * ref).norm()) <= 1e-4 * float(0.7 * ref.norm())


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_together(bits):
    scene, cams = _scene(balance=0.05, lr_deform=1e-3, adamw=dict(state_bits=bits, weight_decay=0.02, max_grad_norm=0.05, eps=1e-8))
    opt = scene.dense_optimizer
    gen = torch.Generator().manual_seed(3)
    for k in range(3):
        views = [dict(cam=c, t=torch.tensor([0.2 + 0.1 * k]).cuda(), g_images=torch.randn(3, H, W, generator=gen).cuda() * 1e-3)
                 for c in cams]
        before = _snapshot(opt, scene.dense_params)
        scene.train_views(views, (W, H))
        grads = [scene.bucket.view_of(p).clone() for p in scene.dense_params]
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
        assert abs(float(opt.grad_norm) - norm) <= 4 * E * norm and norm > 0.05
        _check_step(opt, before, [p for p in scene.dense_params], [g.reshape(p.shape) for g, p in zip(grads, scene.dense_params)],
                    0.05 / (norm + 1e-6))
    scene.check()
    assert scene.sp_radius.grad is None and float(opt.state[scene.sp_radius]["step"]) == 3
    assert int(scene.superpoint_counts.sum()) == P * K
    # the optimiser goes on after the Gaussians have changed, and through its state dictionary
    scene.prune(torch.arange(P, device="cuda") % 5 == 0)
    saved = opt.state_dict()
    opt.load_state_dict(saved)
    scene.train_views([dict(cam=cams[0], t=torch.tensor([0.5]).cuda(), g_images=torch.zeros(3, H, W, device="cuda"))], (W, H))
    assert float(opt.state[scene.sp_radius]["step"]) == 4 and int(scene.superpoint_counts.sum()) == scene.num_points * K


def test_an_overflowed_view_drops_the_dense_step_too():
    """The gate that drops the Gaussians' step (tests of the mask) reaches AdamW: closed, nothing of it changes."""
    scene, _ = _scene(adamw=dict(state_bits=8), balance=0.1)
    scene.train_views([], (W, H))
    opt = scene.dense_optimizer
    before = [t.clone() for p in scene.dense_params for t in [p.detach()] + list(opt.state[p].values())]
    for p, v in zip(scene.dense_params, (scene.bucket.view_of(p) for p in scene.dense_params)):
        p.grad = v
    opt.step_gated(torch.full((1,), -math.inf, device="cuda") + 1.0)
    after = [t for p in scene.dense_params for t in [p.detach()] + list(opt.state[p].values())]
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(before, after))


def test_balance_needs_kernel_weights():
    from fsgs import workloads as wl
    from fsgs.scene import DynamicScene
    surf = wl.surfels(100, seed=5, log_scale_mean=-3.2)
    with pytest.raises(ValueError):
        DynamicScene(surf, wl.superpoints(surf["means"], M=8, seed=1)["centres"], K=2, device="cuda", balance=1.0)


def test_hooks_and_schedules_of_the_dense_optimiser():
    """What a user hangs on the scene's AdamW runs with its steps: step hooks, and a schedule that counts them."""
    import warnings
    scene, _ = _scene(adamw=dict(lr=1e-3))
    opt, seen = scene.dense_optimizer, []
    opt.register_step_pre_hook(lambda o, args, kwargs: seen.append("pre"))
    opt.register_step_post_hook(lambda o, args, kwargs: seen.append("post"))
    schedule = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    with warnings.catch_warnings():
        warnings.simplefilter("error")             # a schedule stepped before its optimiser warns
        for k in range(2):
            scene.train_views([], (W, H))
            schedule.step()
            assert seen == ["pre", "post"] * (k + 1) and opt.param_groups[0]["lr"] == 1e-3 * 0.5 ** (k + 1)
    assert float(opt.state[scene.sp_radius]["step"]) == 2
