"""Losses of the training step: the image loss, and the balance of the Gaussians over the superpoints.

Image loss, fused: ``lambda_l1 * mean|image - target| + lambda_ssim * (1 - mean SSIM)``
(the reference's rgb + ssim terms: exps/d_nerf.yaml:64-65, losses/image_loss.py, losses/ssim.py:69-99) in one forward
kernel (map, derivative maps, both sums) and one backward kernel that writes dL/dimage in the [3,H,W] layout the
compositing backward reads."""
import torch

from . import ops
from ._lib import lib, check

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

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # FSGS_F32, FSGS_BF16, FSGS_F16


def _balance_check(what, rows, idx, M, mask):
    ops._need(rows.is_cuda and rows.dim() == 2, f"{what}: a two-dimensional CUDA tensor is expected")
    ops._need(idx.dim() == 2 and idx.dtype == torch.int64 and idx.shape[0] == rows.shape[0] and idx.shape[1] > 0 and
              idx.device == rows.device, f"{what}: idx must be int64 [N,K] on the same device")
    ops._need(0 < int(M) < 2 ** 31, f"{what}: the number of superpoints must be positive")
    ops._need(mask is None or (mask.dtype in (torch.bool, torch.uint8) and tuple(mask.shape) == (rows.shape[0],) and
                               mask.device == rows.device), f"{what}: mask must be bool [N] on the same device")


_PAIRS, _TABLE = 0, 1   # FSGS_BALANCE_PAIRS, FSGS_BALANCE_TABLE


def _balance_count(idx, M, mask, form):
    """(counts with T and n behind them, workspace for the other two calls), see fsgs_balance_count."""
    N, K = idx.shape
    idx, mask = idx.contiguous(), None if mask is None else mask.contiguous()
    size = int(lib().fsgs_balance_workspace_bytes(N, K, M, form))
    ops._need(size > 0, "balance: more than 2^36 pairs or table entries")
    counts = torch.empty(M + 2, dtype=torch.int64, device=idx.device)
    ws = torch.empty(size, dtype=torch.uint8, device=idx.device)
    p = ops._ptr
    check(lib().fsgs_balance_count(N, K, M, p(idx), p(mask), form, p(counts), p(ws), size, ops._stream()),
          "fsgs_balance_count")
    return counts, ws


def _pairs(N, K, M, weights, ws, scale, upstream, loss, grad, accumulate):
    p = ops._ptr
    check(lib().fsgs_balance_pairs(N, K, M, p(weights), p(ws), ws.numel(), scale, p(upstream), p(loss), p(grad),
                                   int(accumulate), ops._stream()), "fsgs_balance_pairs")


def _table(table, mask, ws, scale, upstream, loss, grad):
    p, (N, M) = ops._ptr, table.shape
    check(lib().fsgs_balance_table(N, M, _TYPES[table.dtype], p(table), table.stride(0) if N > 1 else M, p(mask), p(ws),
                                   ws.numel(), scale, p(upstream), p(loss), p(grad), M, ops._stream()), "fsgs_balance_table")


def _check_weights(weights, idx, M, mask):
    _balance_check("balance_loss", weights, idx, M, mask)
    ops._need(weights.dtype == torch.float32 and weights.shape == idx.shape, "balance_loss: weights must be float32 [N,K]")


def _check_table(table, idx, mask):
    _balance_check("table_balance_loss", table, idx, table.shape[-1] if table.dim() == 2 else 0, mask)
    ops._need(table.dtype in _TYPES, "table_balance_loss: float32, bfloat16 or float16 table")


def _rows_of(table):
    """The table itself where its rows are runs of memory that do not overlap, else a copy."""
    one = table.stride(1) == 1 or table.shape[1] == 1
    return table if one and (table.stride(0) >= table.shape[1]) else table.contiguous()


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weights, idx, M, mask):
        weights = weights.contiguous()
        with ops._on_device(weights.device):
            counts, ws = _balance_count(idx, M, mask, _PAIRS)
            loss = torch.empty((), device=weights.device)
            _pairs(*idx.shape, M, weights, ws, 1.0, None, loss, None, False)
        ctx.save_for_backward(ws)
        ctx.size = (*idx.shape, M)
        out = counts[:M]
        ctx.mark_non_differentiable(out)
        return loss, out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _):
        ws, = ctx.saved_tensors
        N, K, M = ctx.size
        grad = torch.empty(N, K, device=ws.device)
        with ops._on_device(ws.device):
            _pairs(N, K, M, None, ws, 1.0, g_loss, None, grad, False)
        return grad, None, None, None


def balance_loss(weights, idx, M, mask=None):
    """``(loss, counts)``: how evenly the Gaussians use the ``M`` superpoints.  ``weights`` [N,K] float32 are the blend
    weights of each Gaussian's superpoints ``idx`` [N,K] int64 (``lbs_weights``, ``motion.kernel_weights``); ``counts``
    [M] int64 is the number of pairs that name each superpoint, and

        ``loss = M * sum_m (counts_m / sum(counts)) * (1 / n) * sum of the weights of the pairs that name m``

    is 1 when every superpoint has its share.  Differentiable in ``weights`` (the counts carry no gradient).  ``mask``
    (bool [N]): the Gaussians that count, ``n`` of them; an index outside 0 .. M-1 is a pair that does not count.  No
    Gaussian or no pair that counts: loss 0.  No synchronisation; the same inputs give the same bits."""
    _check_weights(weights, idx, M, mask)
    return _BalanceLoss.apply(weights, idx, int(M), mask)


def balance_value_and_grad(weights, idx, M, mask=None, weight=1.0, grad=None):
    """``(weight * loss, weight * dloss/dweights, counts)`` of ``balance_loss`` without autograd.  ``grad`` (float32 [N,K],
    contiguous): the gradient is added to it instead of written to a new tensor."""
    _check_weights(weights, idx, M, mask)
    ops._need(grad is None or (grad.shape == weights.shape and grad.dtype == torch.float32 and grad.is_contiguous() and
                               grad.device == weights.device), "balance_value_and_grad: grad must be contiguous float32 [N,K]")
    weights = weights.detach().contiguous()
    with ops._on_device(weights.device):
        counts, ws = _balance_count(idx, int(M), mask, _PAIRS)
        loss = torch.empty((), device=weights.device)
        out = torch.empty_like(weights) if grad is None else grad
        _pairs(*idx.shape, int(M), weights, ws, float(weight), None, loss, out, grad is not None)
    return loss, out, counts[:M]


class _TableBalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, idx, mask):
        table, mask = _rows_of(table), None if mask is None else mask.contiguous()
        with ops._on_device(table.device):
            counts, ws = _balance_count(idx, table.shape[1], mask, _TABLE)
            loss = torch.empty((), device=table.device)
            _table(table, mask, ws, 1.0, None, loss, None)
        ctx.save_for_backward(table, mask, ws)
        out = counts[:table.shape[1]]
        ctx.mark_non_differentiable(out)
        return loss, out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _):
        table, mask, ws = ctx.saved_tensors
        grad = torch.empty(table.shape, dtype=table.dtype, device=table.device)
        with ops._on_device(table.device):
            _table(table, mask, ws, 1.0, g_loss, None, grad)
        return grad, None, None


def table_balance_loss(table, idx, mask=None):
    """``(loss, counts)`` for a learned association ``table`` [N,M] (float32, bfloat16 or float16 logits; the ``"table"``
    weighting of ``lbs_weights``) and the superpoints ``idx`` [N,K] int64 that each Gaussian is bound to:

        ``loss = M * sum_m (counts_m / sum(counts)) * mean over the Gaussians of softmax(table)_m``

    ``balance_loss`` with the probabilities of all superpoints in the place of the K blend weights; the gradient of the
    table (in its type) is formed in the same pass over it that forms the softmax.  A row of nothing but -infinity adds
    nothing.  ``mask``, indices outside 0 .. M-1 and ``counts`` as in ``balance_loss``."""
    _check_table(table, idx, mask)
    return _TableBalanceLoss.apply(table, idx, mask)


def table_balance_value_and_grad(table, idx, mask=None, weight=1.0):
    """``(weight * loss, weight * dloss/dtable, counts)`` of ``table_balance_loss`` without autograd: one pass that reads
    the table once and writes the gradient once."""
    _check_table(table, idx, mask)
    table, mask = _rows_of(table.detach()), None if mask is None else mask.contiguous()
    with ops._on_device(table.device):
        counts, ws = _balance_count(idx, table.shape[1], mask, _TABLE)
        loss = torch.empty((), device=table.device)
        grad = torch.empty(table.shape, dtype=table.dtype, device=table.device)
        _table(table, mask, ws, float(weight), None, loss, grad)
    return loss, grad, counts[:table.shape[1]]
