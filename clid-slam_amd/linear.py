"""Dense operators at any width, on the hand-written kernels of include/clid_dense.h (csrc/dense/): the layer of a decoder
(model/decoder.py:58-76) and the class of each row (utils/mesher.py:118-131).  The class head's loss is in `loss.py`.

`Decoder` uses them for every shape but the geometry decoder's 11 -> 64 -> 1, which has its own fused kernels.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_vp, _i32, _i64 = C.c_void_p, C.c_int32, C.c_int64

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "leaky_relu": 2, "gelu": 3, "silu": 4}
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class LinearArgs(C.Structure):
    _fields_ = [("x", _vp), ("w", _vp), ("bias", _vp), ("residual", _vp), ("y", _vp), ("z_out", _vp),
                ("ldx", _i64), ("ldw", _i64), ("ldr", _i64), ("rows", _i64),
                ("k", _i32), ("n", _i32), ("dtype", _i32), ("act", _i32), ("ws", _vp), ("ws_bytes", _i64)]


class LinearBwdArgs(C.Structure):
    _fields_ = [("x", _vp), ("w", _vp), ("dy", _vp), ("z", _vp), ("dx", _vp), ("dw", _vp), ("db", _vp),
                ("ldx", _i64), ("ldw", _i64), ("lddy", _i64), ("rows", _i64),
                ("k", _i32), ("n", _i32), ("dtype", _i32), ("act", _i32), ("ws", _vp), ("ws_bytes", _i64)]


class CeArgs(C.Structure):
    _fields_ = [("x", _vp), ("w", _vp), ("bias", _vp), ("target", _vp), ("order", _vp), ("stat", _vp), ("total", _vp), ("loss_out", _vp),
                ("g", _vp), ("dx", _vp), ("dw", _vp), ("db", _vp),
                ("ldx", _i64), ("ldw", _i64), ("rows", _i64), ("ignore_index", _i64),
                ("k", _i32), ("n", _i32), ("dtype", _i32), ("reduction", _i32), ("ws", _vp), ("ws_bytes", _i64)]


class LabelArgs(C.Structure):
    _fields_ = [("x", _vp), ("w", _vp), ("bias", _vp), ("label", _vp), ("log_prob", _vp),
                ("ldx", _i64), ("ldw", _i64), ("rows", _i64),
                ("k", _i32), ("n", _i32), ("dtype", _i32), ("reserved", _i32), ("ws", _vp), ("ws_bytes", _i64)]


_SIGS = {
    "clid_linear_workspace": (_i64, [C.POINTER(LinearArgs)]),
    "clid_linear_fwd": (C.c_int, [C.POINTER(LinearArgs), _vp]),
    "clid_linear_bwd_workspace": (_i64, [C.POINTER(LinearBwdArgs)]),
    "clid_linear_bwd": (C.c_int, [C.POINTER(LinearBwdArgs), _vp]),
    "clid_ce_workspace": (_i64, [C.POINTER(CeArgs)]),
    "clid_ce_fwd": (C.c_int, [C.POINTER(CeArgs), _vp]),
    "clid_ce_bwd_workspace": (_i64, [C.POINTER(CeArgs)]),
    "clid_ce_bwd": (C.c_int, [C.POINTER(CeArgs), _vp]),
    "clid_label_workspace": (_i64, [C.POINTER(LabelArgs)]),
    "clid_label_fwd": (C.c_int, [C.POINTER(LabelArgs), _vp]),
}
EXPORTS = tuple(_SIGS)
_bound = None


def load():
    """The shared library with the dense entry points' signatures set (once)."""
    global _bound
    if _bound is None:
        lib = _lib.load()
        for name, (res, args) in _SIGS.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _bound = lib
    return _bound


def call(entry: str, workspace: str, args, device) -> None:
    """One entry point on torch's current stream of `device`, with its workspace from torch's allocator: a buffer of this call
    alone, which the allocator gives back in stream order (and keeps for a graph that is being captured)."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return call(entry, workspace, args, device)
    lib = load()
    need = getattr(lib, workspace)(C.byref(args))
    if need < 0:
        _lib.check(int(need), workspace)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    args.ws, args.ws_bytes = _lib.ptr(ws), need
    _lib.check(getattr(lib, entry)(C.byref(args), _lib.stream()), entry)


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """`t` as [rows, width] with contiguous columns: a view wherever its strides allow, else a copy."""
    t = t.detach().reshape(-1, width)
    if t.shape[0] > 1 and t.stride(0) < width or width > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def ld_of(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def check_operands(what: str, x, weight, bias=None, residual=None) -> None:
    """x [..., k], weight [n, k], bias [n], residual [..., n]: on one GPU, of one of the three types."""
    for name, t in (("x", x), ("weight", weight)):
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{what}: {name} must be a tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{what}: x must live on the GPU (got {x.device}); the HIP path has no CPU fallback")
    if x.dtype not in DTYPES:
        raise RuntimeError(f"{what}: x must be float32, bfloat16 or float16, got {x.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise RuntimeError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)} must be [..., k] and [n, k] with n, k >= 1")
    n = weight.shape[0]
    for name, t, shape in (("weight", weight, weight.shape), ("bias", bias, (n,)), ("residual", residual, (*x.shape[:-1], n))):
        if t is None:
            continue
        if t.shape != shape:
            raise RuntimeError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
        if t.dtype != x.dtype or t.device != x.device:
            raise RuntimeError(f"{what}: {name} must be {x.dtype} on {x.device} like x, got {t.dtype} on {t.device}")


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _forward(x, weight, bias, act, residual, keep_z):
    n, k = weight.shape
    x2, w = rows_of(x, k), rows_of(weight, k)
    b = None if bias is None else bias.detach().contiguous()
    r = None if residual is None else rows_of(residual, n)
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    z = torch.empty((x2.shape[0], n), dtype=x.dtype, device=x.device) if keep_z else None
    if x2.shape[0]:
        args = LinearArgs(_lib.ptr(x2), _lib.ptr(w), _lib.ptr(b), _lib.ptr(r), _lib.ptr(y), _lib.ptr(z), ld_of(x2), ld_of(w),
                          ld_of(r) if r is not None else n, x2.shape[0], k, n, DTYPES[x.dtype], act)
        call("clid_linear_fwd", "clid_linear_workspace", args, x.device)
    return y, z


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        # what the backward pass reads of z: nothing without an activation; its sign, which y has too where nothing was added
        # (float16 excepted: a z under 2^-25 would be 0 in y)
        sign_of_y = act in (ACTIVATIONS["relu"], ACTIVATIONS["leaky_relu"]) and residual is None and x.dtype != torch.float16
        y, z = _forward(x, weight, bias, act, residual, act != 0 and not sign_of_y)
        ctx.act = act
        ctx.save_for_backward(x, weight, y if sign_of_y else z)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        n, k = weight.shape
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty((n, k), dtype=x.dtype, device=x.device) if need_w else None
        db = torch.empty(n, dtype=x.dtype, device=x.device) if need_b else None
        x2, w, dy2 = rows_of(x, k), rows_of(weight, k), rows_of(dy, n)
        if x2.shape[0] == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif need_x or need_w or need_b:
            args = LinearBwdArgs(_lib.ptr(x2), _lib.ptr(w), _lib.ptr(dy2), _lib.ptr(z), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db),
                                 ld_of(x2), ld_of(w), ld_of(dy2), x2.shape[0], k, n, DTYPES[x.dtype], ctx.act)
            call("clid_linear_bwd", "clid_linear_bwd_workspace", args, x.device)
        return dx, dw, db, (dy if need_r else None), None


def linear_act(x, weight, bias=None, activation: str = "none", residual=None):
    """y = activation(x weight^T + bias) + residual in one pass over x and weight, with its gradients.

    x [..., k], weight [n, k] (torch.nn.Linear's layout), bias [n], residual [..., n] and y all of one type (float32, bfloat16,
    float16) on one GPU; rows may be a view of a wider buffer.  `activation`: none, relu, leaky_relu (slope 0.01), gelu (erf),
    silu.  Sums are fp32; y is rounded once, after the residual.  Runs on torch's current stream, captures into a graph,
    differentiates once."""
    if activation not in ACTIVATIONS:
        raise NotImplementedError(f"linear_act: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    check_operands("linear_act", x, weight, bias, residual)
    if wants_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, ACTIVATIONS[activation])
    return _forward(x, weight, bias, ACTIVATIONS[activation], residual, False)[0]


@torch.no_grad()
def linear_label(x, weight, bias=None):
    """(label, log_prob) of z = x weight^T + bias without storing z: label [...] int64 = the lowest class with the largest z (a
    NaN counts as largest, as in torch.argmax), log_prob [...] float32 = log softmax(z) at it.  Operands as in `linear_act`; not
    differentiable (the class head's training loss is `loss.linear_cross_entropy`)."""
    check_operands("linear_label", x, weight, bias)
    n, k = weight.shape
    x2, w = rows_of(x, k), rows_of(weight, k)
    b = None if bias is None else bias.detach().contiguous()
    label = torch.empty(x.shape[:-1], dtype=torch.int64, device=x.device)
    log_prob = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if x2.shape[0]:
        args = LabelArgs(_lib.ptr(x2), _lib.ptr(w), _lib.ptr(b), _lib.ptr(label), _lib.ptr(log_prob), ld_of(x2), ld_of(w),
                         x2.shape[0], k, n, DTYPES[x.dtype], 0)
        call("clid_label_fwd", "clid_label_workspace", args, x.device)
    return label, log_prob
