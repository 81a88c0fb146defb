"""Dense operators at any width, on the hand-written kernels of include/clid_dense.h (csrc/dense/): the layer of a decoder
(model/decoder.py:58-76) and the class of each row (utils/mesher.py:118-131).  The class head's loss is in `loss.py`.

`Decoder` uses them for every shape but the geometry decoder's 11 -> 64 -> 1, which has its own fused kernels.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad

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
                ("k", _i32), ("n", _i32), ("dtype", _i32), ("act", _i32), ("z_is_y", _i32), ("reserved", _i32), ("ws", _vp), ("ws_bytes", _i64)]


class CeArgs(C.Structure):
    _fields_ = [("x", _vp), ("w", _vp), ("bias", _vp), ("target", _vp), ("saved", _vp), ("loss_out", _vp),
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
    "clid_ce_saved": (_i64, [C.POINTER(CeArgs)]),
    "clid_ce_workspace": (_i64, [C.POINTER(CeArgs)]),
    "clid_ce_fwd": (C.c_int, [C.POINTER(CeArgs), _vp]),
    "clid_ce_bwd_workspace": (_i64, [C.POINTER(CeArgs)]),
    "clid_ce_bwd": (C.c_int, [C.POINTER(CeArgs), _vp]),
    "clid_label_workspace": (_i64, [C.POINTER(LabelArgs)]),
    "clid_label_fwd": (C.c_int, [C.POINTER(LabelArgs), _vp]),
}
EXPORTS = tuple(_SIGS)
_functions = {}


def load():
    """The shared library with the dense entry points' signatures set (once)."""
    lib = _lib.load()
    if not _functions:
        bound = {}
        for name, (res, args) in _SIGS.items():
            bound[name] = fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _functions.update(bound)
    return lib


# (The small shapes are over in 10 us on the GPU, so what Python does around a call is kept to what is needed: no tensor is made only to read its
# pointer, and one buffer holds what a call leaves for its backward pass.)
def call(entry: str, workspace: str, args, device) -> None:
    """One entry point on torch's current stream of `device`, with its workspace from torch's allocator: a buffer of this call
    alone, which the allocator gives back in stream order (and keeps for a graph that is being captured)."""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return call(entry, workspace, args, device)
    fn, ref = _functions or load() and _functions, C.byref(args)
    need = fn[workspace](ref)
    if need:
        if need < 0:
            _lib.check(int(need), workspace)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        args.ws, args.ws_bytes = ws.data_ptr(), need
    rc = fn[entry](ref, _lib.stream())
    if rc:
        _lib.check(rc, entry)


def rows_of(t: torch.Tensor, width: int):
    """(`t` as rows of `width` contiguous columns, elements between rows): t itself or a view wherever its strides allow, else a
    copy.  Called without gradients (inside autograd functions, under no_grad)."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    rows, (ld, step) = t.shape[0], t.stride()
    if width > 1 and step != 1 or rows > 1 and ld < width:
        t = t.contiguous()
        ld = width
    return t, (ld if rows > 1 else width)


def check_operands(what: str, x, weight, bias=None, residual=None) -> None:
    """x [..., k], weight [n, k], bias [n], residual [..., n]: on one GPU, of one of the three types."""
    for name, t in (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)):
        if not isinstance(t, torch.Tensor) and (t is not None or name in ("x", "weight")):
            raise RuntimeError(f"{what}: {name} must be a tensor")
    if torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise RuntimeError(f"{what}: make_fx records the tensors that a call makes but not the kernels that fill them")
    if not x.is_cuda:
        raise RuntimeError(f"{what}: x must live on the GPU (got {x.device}); the HIP path has no CPU fallback")
    dtype, shape, wshape = x.dtype, x.shape, weight.shape
    if dtype not in DTYPES:
        raise RuntimeError(f"{what}: x must be float32, bfloat16 or float16, got {dtype}")
    if len(wshape) != 2 or len(shape) < 1 or shape[-1] != wshape[1] or 0 in wshape:
        raise RuntimeError(f"{what}: x {tuple(shape)} and weight {tuple(wshape)} must be [..., k] and [n, k] with n, k >= 1")
    if max(wshape) >= 1 << 20:  # (also before a ctypes structure keeps the low 32 bits of it)
        raise RuntimeError(f"{what}: bad argument: weight {tuple(wshape)} must have n, k < 2^20")
    _like(what, "weight", weight, wshape, dtype, x.device)
    if bias is not None:
        _like(what, "bias", bias, wshape[:1], dtype, x.device)
    if residual is not None:
        _like(what, "residual", residual, (*shape[:-1], wshape[0]), dtype, x.device)


def _like(what, name, t, shape, dtype, device):
    if t.shape != shape:
        raise RuntimeError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        raise RuntimeError(f"{what}: {name} must be {dtype} on {device} like x, got {t.dtype} on {t.device}")


def through_function(*tensors) -> bool:
    """Whether a call goes through its autograd Function rather than straight to the launch: gradients are wanted; or an operand
    carries a forward-mode tangent, which the Function refuses (a launch of its own would return a derivative of zero without a word);
    or torch.jit.trace is recording, which keeps a Function as a node and of a launch nothing."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return torch._C._is_tracing()


def _forward(x, weight, bias, act, residual, keep_z):
    n, k = weight.shape
    (x2, ldx), (w, ldw) = rows_of(x, k), rows_of(weight, k)
    r, ldr = (None, n) if residual is None else rows_of(residual, n)
    b = None if bias is None else bias.contiguous()
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    z = torch.empty(y.shape, dtype=torch.float32 if x.dtype == torch.float32 else torch.float16, device=x.device) if keep_z else None
    rows = x2.shape[0]
    if rows:
        call("clid_linear_fwd", "clid_linear_workspace",
             LinearArgs(x2.data_ptr(), w.data_ptr(), _lib.ptr(b), _lib.ptr(r), y.data_ptr(), _lib.ptr(z), ldx, ldw, ldr, rows, k, n,
                        DTYPES[x.dtype], act), x.device)
    return y, z


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        # what the backward pass reads of z: nothing without an activation; its sign, which y has too where nothing was added
        # (float16 excepted: a z under 2^-25 would be 0 in y)
        sign_of_y = act in (ACTIVATIONS["relu"], ACTIVATIONS["leaky_relu"]) and residual is None and x.dtype != torch.float16
        y, z = _forward(x, weight, bias, act, residual, act != 0 and not sign_of_y)
        ctx.act, ctx.z_is_y = act, int(sign_of_y)
        ctx.save_for_backward(x, weight, y if sign_of_y else z)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        n, k = weight.shape
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dtype, device = x.dtype, x.device
        dx = torch.empty(x.shape, dtype=dtype, device=device) if need_x else None
        dw = torch.empty((n, k), dtype=dtype, device=device) if need_w else None
        db = torch.empty(n, dtype=dtype, device=device) if need_b else None
        (x2, ldx), (w, ldw), (dy2, lddy) = rows_of(x, k), rows_of(weight, k), rows_of(dy, n)
        rows = x2.shape[0]
        if rows == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif need_x or need_w or need_b:
            call("clid_linear_bwd", "clid_linear_bwd_workspace",
                 LinearBwdArgs(x2.data_ptr(), w.data_ptr(), dy2.data_ptr(), _lib.ptr(z), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), ldx, ldw,
                               lddy, rows, k, n, DTYPES[dtype], ctx.act, ctx.z_is_y), device)
        return dx, dw, db, (dy if need_r else None), None


def linear_act(x, weight, bias=None, activation: str = "none", residual=None):
    """y = activation(x weight^T + bias) + residual in one pass over x and weight, with its gradients.

    x [..., k], weight [n, k] (torch.nn.Linear's layout), bias [n], residual [..., n] and y all of one type (float32, bfloat16,
    float16) on one GPU; rows may be a view of a wider buffer.  `activation`: none, relu, leaky_relu (slope 0.01), gelu (erf),
    silu.  Sums are fp32; y is rounded once, after the residual.  Runs on torch's current stream, captures into a graph,
    differentiates once, backward only (forward-mode tangents are refused)."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise NotImplementedError(f"linear_act: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    check_operands("linear_act", x, weight, bias, residual)
    if through_function(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, act)
    with torch.no_grad():
        return _forward(x, weight, bias, act, residual, False)[0]


def _label(x, weight, bias):
    n, k = weight.shape
    (x2, ldx), (w, ldw) = rows_of(x, k), rows_of(weight, k)
    b = None if bias is None else bias.contiguous()
    label = torch.empty(x.shape[:-1], dtype=torch.int64, device=x.device)
    log_prob = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rows = x2.shape[0]
    if rows:
        call("clid_label_fwd", "clid_label_workspace",
             LabelArgs(x2.data_ptr(), w.data_ptr(), _lib.ptr(b), label.data_ptr(), log_prob.data_ptr(), ldx, ldw, rows, k, n, DTYPES[x.dtype], 0),
             x.device)
    return label, log_prob


class _LinearLabel(torch.autograd.Function):  # for torch.jit.trace alone (through_function)
    @staticmethod
    def forward(ctx, x, weight, bias):
        label, log_prob = _label(x, weight, bias)
        ctx.mark_non_differentiable(label, log_prob)
        return label, log_prob


@torch.no_grad()
def linear_label(x, weight, bias=None):
    """(label, log_prob) of z = x weight^T + bias without storing z: label [...] int64 = the lowest class with the largest z (a
    NaN counts as largest, as in torch.argmax), log_prob [...] float32 = log softmax(z) at it.  Operands as in `linear_act`; not
    differentiable (the class head's training loss is `loss.linear_cross_entropy`)."""
    check_operands("linear_label", x, weight, bias)
    if torch._C._is_tracing():
        return _LinearLabel.apply(x, weight, bias)
    return _label(x, weight, bias)
