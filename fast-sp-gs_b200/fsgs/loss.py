"""Losses of the training step: the image loss, and the balance of the Gaussians over the superpoints.

Image loss, fused: ``lambda_l1 * mean|image - target| + lambda_ssim * (1 - mean SSIM)``
(the reference's rgb + ssim terms: exps/d_nerf.yaml:64-65, losses/image_loss.py, losses/ssim.py:69-99) in one forward
kernel (map, derivative maps, both sums) and one backward kernel that writes dL/dimage in the [3,H,W] layout the
compositing backward reads."""
import torch

from . import ops
from ._lib import check, host, lib

C1, C2 = 0.01 ** 2, 0.03 ** 2


class _L1SSIM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, image, target, lambda_l1, lambda_ssim):
        ops._need(image.is_cuda and image.dtype == torch.float32 and image.shape == target.shape and image.dim() == 3,
                  "l1_ssim_loss: image and target must be float32 CUDA tensors [C,H,W] of equal shape")
        image, target = image.contiguous(), target.contiguous()
        C, H, W = image.shape
        maps = torch.empty(4, C, H, W, device=image.device, dtype=torch.float32)
        sums = torch.zeros(2, device=image.device, dtype=torch.float32)
        p = ops._ptr
        check(lib().fsgs_ssim_forward(1, C, H, W, C1, C2, p(image), p(target), p(maps[0]), p(maps[1]), p(maps[2]),
                                      p(maps[3]), p(sums), ops._stream()), "fsgs_ssim_forward")
        n = float(C * H * W)
        ctx.save_for_backward(image, target, maps)
        ctx.weights = (lambda_l1 / n, lambda_ssim / n)
        return lambda_l1 * (sums[1] / n) + lambda_ssim * (1.0 - sums[0] / n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss):
        image, target, maps = ctx.saved_tensors
        C, H, W = image.shape
        w_l1, w_ssim = ctx.weights
        g = float(g_loss) if g_loss.device.type == "cpu" else None
        out = torch.empty_like(image)
        p = ops._ptr
        if g is None:
            # upstream scale lives on the device: keep it there (no synchronisation), scale afterwards
            check(lib().fsgs_ssim_backward(1, C, H, W, C1, C2, p(image), p(target), None, -w_ssim, w_l1, p(maps[1]),
                                           p(maps[2]), p(maps[3]), p(out), ops._stream()), "fsgs_ssim_backward")
            out = out * g_loss
        else:
            check(lib().fsgs_ssim_backward(1, C, H, W, C1, C2, p(image), p(target), None, -w_ssim * g, w_l1 * g,
                                           p(maps[1]), p(maps[2]), p(maps[3]), p(out), ops._stream()),
                  "fsgs_ssim_backward")
        return out, None, None, None


def l1_ssim_loss(image, target, lambda_l1=0.8, lambda_ssim=0.2):
    """Scalar loss (device tensor) of a rendered ``image`` [C,H,W] against ``target``; differentiable in ``image``."""
    return _L1SSIM.apply(image, target, float(lambda_l1), float(lambda_ssim))


def l1_ssim_value_and_grad(image, target, lambda_l1=0.8, lambda_ssim=0.2):
    """(loss, dL/dimage) without autograd: two kernel launches.  ``dL/dimage`` is ready to be handed to
    ``torch.autograd.backward(images, grad)`` or to the compositing backward directly."""
    image, target = image.detach().contiguous(), target.contiguous()
    C, H, W = image.shape
    maps = torch.empty(4, C, H, W, device=image.device, dtype=torch.float32)
    sums = torch.zeros(2, device=image.device, dtype=torch.float32)
    grad = torch.empty_like(image)
    n = float(C * H * W)
    p = ops._ptr
    check(lib().fsgs_ssim_forward(1, C, H, W, C1, C2, p(image), p(target), p(maps[0]), p(maps[1]), p(maps[2]),
                                  p(maps[3]), p(sums), ops._stream()), "fsgs_ssim_forward")
    check(lib().fsgs_ssim_backward(1, C, H, W, C1, C2, p(image), p(target), None, -lambda_ssim / n, lambda_l1 / n,
                                   p(maps[1]), p(maps[2]), p(maps[3]), p(grad), ops._stream()),
          "fsgs_ssim_backward")
    return lambda_l1 * (sums[1] / n) + lambda_ssim * (1.0 - sums[0] / n), grad


# ---- balance over the superpoints ------------------------------------------------------------------------------------

def balance_loss(weights, idx, M, mask=None):
    """``(loss, counts)``: how evenly the Gaussians use the ``M`` superpoints.  ``weights`` [N,K] float32 are the blend
    weights of each Gaussian's superpoints ``idx`` [N,K] int64 (``lbs_weights``, ``motion.kernel_weights``); ``counts``
    [M] int64 is the number of pairs that name each superpoint, and

        ``loss = M * sum_m (counts_m / sum(counts)) * (1 / n) * sum of the weights of the pairs that name m``

    is 1 when every superpoint has its share.  Differentiable in ``weights`` (the counts carry no gradient).  ``mask``
    (bool [N]): the Gaussians that count, ``n`` of them; an index outside 0 .. M-1 is a pair that does not count.  No
    Gaussian or no pair that counts: loss 0.  No synchronisation; the same inputs give the same bits.

    Forward and backward can be captured into a CUDA graph.  While an earlier graph of ``weights``, made on a stream outside
    the capture, is still alive (a loss that somebody holds), the captured backward pass raises: its gradient could not be
    handed over.  ``balance_value_and_grad`` has no such limit."""
    return host().balance_pairs(weights, idx, int(M), mask, 1.0, None, True)


def balance_value_and_grad(weights, idx, M, mask=None, weight=1.0, grad=None):
    """``(weight * loss, weight * dloss/dweights, counts)`` of ``balance_loss`` without autograd.  ``grad`` (float32 [N,K],
    contiguous): the gradient is added to it instead of written to a new tensor."""
    return host().balance_pairs(weights, idx, int(M), mask, float(weight), grad, False)


def table_balance_loss(table, idx, mask=None):
    """``(loss, counts)`` for a ``table`` [N,M] (float32, bfloat16 or float16 logits) of how each Gaussian is spread over all
    ``M`` superpoints, and the superpoints ``idx`` [N,K] int64 that it is bound to:

        ``loss = M * sum_m (counts_m / sum(counts)) * mean over the Gaussians of softmax(table)_m``

    ``balance_loss`` with the probabilities of all superpoints in the place of the K blend weights, differentiable in
    ``table`` (gradient in its type).  It acts on the softmax over the whole row, so it also falls where probability goes to
    the M - K superpoints that a Gaussian is not bound to.  For the ``"table"`` weighting of ``lbs_weights``, a softmax over
    the K gathered entries, the balance of what is blended is ``balance_loss(lbs_weights(d2, idx, "table", table=table),
    idx, M)``, which reaches those entries alone.  A row of nothing but -infinity adds nothing.  ``mask``, indices outside 0 .. M-1
    and ``counts`` as in ``balance_loss``; a captured backward pass too.  The gradient of a table
    of N rows is of the order of a probability times M / N: below 6e-8 a float16 table loses it, so scale the loss."""
    return host().balance_table(table, idx, mask, 1.0, True)


def table_balance_value_and_grad(table, idx, mask=None, weight=1.0):
    """``(weight * loss, weight * dloss/dtable, counts)`` of ``table_balance_loss`` without autograd: one pass that reads
    the table once and writes the gradient once."""
    return host().balance_table(table, idx, mask, float(weight), False)
