"""utils/loss.py counterpart: `sdf_bce_loss` (:44-62), HIP-backed (clid_loss_fwd_bwd), and the class head's softmax cross
entropy without its logits (clid_ce_fwd / clid_ce_bwd)."""
from __future__ import annotations

import torch

from . import _lib, linear


class _BceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, label, sigma, weight, weighted):
        lib = _lib.load()
        pred_c = _lib.require_cuda(pred.detach().contiguous(), "pred", torch.float32)
        label_c = _lib.require_cuda(label.detach().contiguous(), "label", torch.float32)
        w_c = _lib.require_cuda(weight.detach().contiguous(), "weight", torch.float32) if weighted else None
        out = torch.zeros(4, device=pred.device, dtype=torch.float32)
        d_pred = torch.empty_like(pred_c)
        _lib.check(
            lib.clid_loss_fwd_bwd(_lib.ptr(pred_c), _lib.ptr(label_c), _lib.ptr(w_c), pred_c.numel(), float(sigma),
                                  int(bool(weighted)), None, 0, 0.0, _lib.ptr(out), _lib.ptr(d_pred), None,
                                  _lib.stream()),
            "clid_loss_fwd_bwd",
        )
        ctx.save_for_backward(d_pred)
        return out[1]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (d_pred,) = ctx.saved_tensors
        return g * d_pred, None, None, None, None


def sdf_bce_loss(pred, label, sigma, weight, weighted=False, bce_reduction="mean"):
    """BCE-with-logits between pred/sigma and sigmoid(label/sigma) (utils/loss.py:44-62)."""
    if bce_reduction != "mean":
        raise NotImplementedError("sdf_bce_loss: only bce_reduction='mean' is used by the mapping loop")
    return _BceLoss.apply(pred, label, sigma, weight, weighted)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index, reduction):
        n, k = weight.shape
        (x2, ldx), (w, ldw) = linear.rows_of(x, k), linear.rows_of(weight, k)
        b = None if bias is None else bias.contiguous()
        t = target.to(torch.int64).contiguous()
        rows, dev = x2.shape[0], x.device
        loss = torch.empty(target.shape if reduction == 0 else (), dtype=torch.float32, device=dev)
        args = linear.CeArgs(x2.data_ptr(), w.data_ptr(), _lib.ptr(b), t.data_ptr(), None, loss.data_ptr(), None, None, None, None, ldx, ldw,
                             rows, ignore_index, k, n, linear.DTYPES[x.dtype], reduction)
        need = linear.load().clid_ce_saved(args)
        if need < 0:
            _lib.check(int(need), "clid_ce_saved")
        saved = torch.empty(need, dtype=torch.uint8, device=dev)
        args.saved = saved.data_ptr()
        if rows or reduction:
            linear.call("clid_ce_fwd", "clid_ce_workspace", args, dev)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        ctx.save_for_backward(x, weight, t, saved, bias)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, weight, t, saved, bias = ctx.saved_tensors
        n, k = weight.shape
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dtype, dev = x.dtype, x.device
        dx = torch.empty(x.shape, dtype=dtype, device=dev) if need_x else None
        dw = torch.empty((n, k), dtype=dtype, device=dev) if need_w else None
        db = torch.empty(n, dtype=dtype, device=dev) if need_b else None
        (x2, ldx), (w, ldw) = linear.rows_of(x, k), linear.rows_of(weight, k)
        rows = x2.shape[0]
        if rows == 0:
            for v in (dw, db):
                if v is not None:
                    v.zero_()
        else:
            b = None if bias is None else bias.contiguous()
            g = g.to(torch.float32).contiguous()
            linear.call("clid_ce_bwd", "clid_ce_bwd_workspace",
                        linear.CeArgs(x2.data_ptr(), w.data_ptr(), _lib.ptr(b), t.data_ptr(), saved.data_ptr(), None, g.data_ptr(), _lib.ptr(dx),
                                      _lib.ptr(dw), _lib.ptr(db), ldx, ldw, rows, ctx.ignore_index, k, n, linear.DTYPES[dtype],
                                      ctx.reduction), dev)
        return dx, dw, db, None, None, None


def linear_cross_entropy(x, weight, bias, target, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of the logits x weight^T + bias against `target`, with its gradients, never storing the logits: they
    are made a piece of the classes at a time, in the forward pass for their running maximum and sum, in the backward pass again.

    x [..., k], weight [n, k], bias [n] or None of one type (float32, bfloat16, float16) on one GPU; target [...] int64 or int32
    class numbers.  The loss is fp32: a value, or [...] with reduction="none".  Rows with target == ignore_index count for nothing,
    whatever they hold; "mean" divides by the rows that count and is 0 where there are none.  Any other target outside [0, n)
    makes its row's loss and the gradients that it reaches NaN.  Differentiates once, backward only."""
    if reduction not in linear.REDUCTIONS:
        raise NotImplementedError(f"linear_cross_entropy: reduction must be mean, sum or none, got {reduction!r}")
    linear.check_operands("linear_cross_entropy", x, weight, bias)
    if not isinstance(target, torch.Tensor) or target.dtype not in (torch.int64, torch.int32) or target.device != x.device:
        raise RuntimeError(f"linear_cross_entropy: target must be int64 or int32 on {x.device}")
    if target.shape != x.shape[:-1]:
        raise RuntimeError(f"linear_cross_entropy: target must have shape {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    ignore_index = int(ignore_index)
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise RuntimeError(f"linear_cross_entropy: ignore_index must be an int64, got {ignore_index}")
    return _LinearCrossEntropy.apply(x, weight, bias, target, ignore_index, linear.REDUCTIONS[reduction])
