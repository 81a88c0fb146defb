"""The dense operators (linear_act, linear_cross_entropy, linear_label) against plain 64-bit forms (dense_ref.py), their refusals,
and a run of them together through Decoder and the mesher."""
import ctypes as C
import math
import os
import re
import subprocess

import pytest
import torch

import dense_ref as ref
from clid_slam_amd import Decoder, HotPathConfig, _lib
from clid_slam_amd import linear as L
from clid_slam_amd.linear import linear_act, linear_label
from clid_slam_amd.loss import linear_cross_entropy

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "clid_dense.h")
gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- CPU: the ABI and the refusals ----------------------------------------------------------------------------------------
def test_header_and_bindings_agree(tmp_path):
    names = sorted(set(re.findall(r"\b(clid_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S))))
    lib = L.load()
    assert sorted(L.EXPORTS) == names
    for n in names:
        assert hasattr(lib, n)
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(){printf("%%zu %%zu %%zu %%zu %%zu %%zu %%zu %%zu",'
                   "sizeof(clid_linear_args), offsetof(clid_linear_args, ws), sizeof(clid_linear_bwd_args), offsetof(clid_linear_bwd_args, ws),"
                   "sizeof(clid_ce_args), offsetof(clid_ce_args, ws), sizeof(clid_label_args), offsetof(clid_label_args, ws)); return 0;}\n" % HEADER)
    subprocess.check_call(["gcc", str(src), "-o", str(tmp_path / "sz")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "sz")]).split()]
    want = []
    for s in (L.LinearArgs, L.LinearBwdArgs, L.CeArgs, L.LabelArgs):
        want += [C.sizeof(s), s.ws.offset]
    assert got == want


def test_entry_points_refuse_bad_arguments():
    lib = L.load()
    for fn, make in (("clid_linear_fwd", L.LinearArgs), ("clid_linear_bwd", L.LinearBwdArgs), ("clid_ce_fwd", L.CeArgs),
                     ("clid_ce_bwd", L.CeArgs), ("clid_label_fwd", L.LabelArgs)):
        a = make(rows=4, k=0, n=4)
        assert getattr(lib, fn)(C.byref(a), None) == -1 and fn.encode() in lib.clid_last_error()
        a = make(rows=4, k=8, n=4, dtype=7)
        assert getattr(lib, fn)(C.byref(a), None) == -1
        a = make(rows=4, k=8, n=4)  # null pointers
        assert getattr(lib, fn)(C.byref(a), None) == -1
        a = make(rows=1 << 31, k=8, n=4)
        assert getattr(lib, fn)(C.byref(a), None) == -1
        assert getattr(lib, fn)(None, None) == -1
    # a workspace that is too small, or not aligned as the header asks (never launched: the addresses are no memory)
    a = L.CeArgs(x=4096, w=4096, target=4096, saved=4096, loss_out=4096, ldx=100, ldw=100, rows=4, k=100, n=100, reduction=1)
    need = lib.clid_ce_workspace(C.byref(a))
    assert need > 0 and need % 256 == 0
    for a.ws, a.ws_bytes in ((4096, need - 1), (4097, need), (None, need)):
        assert lib.clid_ce_fwd(C.byref(a), None) == -1 and b"workspace" in lib.clid_last_error()
    a.saved = 4097
    assert lib.clid_ce_fwd(C.byref(a), None) == -1
    for fn in ("clid_linear_workspace", "clid_linear_bwd_workspace", "clid_ce_workspace", "clid_ce_bwd_workspace", "clid_label_workspace"):
        assert getattr(lib, fn)(None) < 0


def test_no_cpu_fallback_and_bad_names():
    x, w = torch.zeros(4, 8), torch.zeros(5, 8)
    for f in (lambda: linear_act(x, w), lambda: linear_label(x, w), lambda: linear_cross_entropy(x, w, None, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="GPU"):
            f()
    with pytest.raises(NotImplementedError, match="activation"):
        linear_act(x, w, activation="tanh")
    with pytest.raises(NotImplementedError, match="reduction"):
        linear_cross_entropy(x, w, None, torch.zeros(4, dtype=torch.int64), reduction="max")
    with pytest.raises(RuntimeError, match="tensor"):
        linear_act(None, w)


# ---- GPU ---------------------------------------------------------------------------------------------------------------------
def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def strided(t, pad, offset):
    """the values of t as rows of a wider buffer that starts `offset` elements into its storage"""
    m, k = t.shape
    store = torch.full((m * (k + pad) + offset,), float("nan"), dtype=t.dtype, device=t.device)
    v = store[offset:].view(m, k + pad)[:, :k]
    v.copy_(t)
    return v


SHAPES = [(1, 1, 1), (1, 8, 5), (3, 11, 64), (17, 64, 21), (64, 64, 64), (1, 4100, 130), (5, 2051, 7), (65, 100, 130), (257, 333, 129),
          (1000, 64, 64), (2, 64, 5000), (300, 40, 700), (31, 72, 1), (513, 256, 264)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", list(L.ACTIVATIONS))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_act(shape, act, dtype):
    m, k, n = shape
    dt = TYPES[dtype]
    gen = generator(m * 1000003 + k * 1009 + n)
    exact = act in ("relu", "leaky_relu")  # small eighths: z is exact in fp32, so no z changes its side of the kink
    make = (lambda *s: torch.randint(-8, 9, s, generator=gen, device="cuda") / 8) if exact else (lambda *s: normal(gen, *s))
    bias, res = (m + n) % 3 != 0, (m + k) % 2 == 0
    x = strided(make(m, k).to(dt), (0, 1, 8)[(m + k + n) % 3], (0, 3)[k % 2]).requires_grad_()
    w = strided((make(n, k) * (1.0 if exact else k ** -0.5)).to(dt), (0, 5, 8)[n % 3], (0, 1)[n % 2]).requires_grad_()
    b = make(n).to(dt).requires_grad_() if bias else None
    r = normal(gen, m, n).to(dt).requires_grad_() if res else None
    dy = normal(gen, m, n).to(dt)
    y = linear_act(x, w, b, activation=act, residual=r)
    assert y.dtype == dt
    leaves = {"dx": x, "dw": w, "db": b, "dr": r}
    leaves = {q: t for q, t in leaves.items() if t is not None}
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    want = ref.linear(x, w, b, r, act, dy)
    for name, (v, tol) in want.items():
        if name == "y" or name in got:
            ref.close(y if name == "y" else got[name], v, tol, name)
    if res:
        assert torch.equal(got["dr"], dy)
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, activation=act, residual=r), y)  # the same bits without and with gradients
    again = torch.autograd.grad(linear_act(x, w, b, activation=act, residual=r), list(leaves.values()), dy)
    assert all(torch.equal(a, g) for a, g in zip(again, got.values()))  # and every time


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", list(L.REDUCTIONS))
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 8, 2), (5, 11, 21), (64, 64, 21), (130, 72, 64), (33, 100, 1000), (257, 130, 333), (7, 512, 4099),
                                   (600, 64, 513), (1, 300, 2000), (16, 200, 1500), (17, 129, 130), (32, 1031, 700)], ids=str)
@pytest.mark.parametrize("ignored", [0.0, 0.5, 1.0])
def test_cross_entropy(shape, reduction, dtype, ignored):
    m, k, n = shape
    dt = TYPES[dtype]
    gen = generator(m * 1000003 + k * 1009 + n + int(ignored * 4))
    w = strided((normal(gen, n, k) * k ** -0.5).to(dt), (0, 5, 8)[n % 3], (0, 1)[n % 2]).requires_grad_()
    target = torch.randint(0, n, (m,), generator=gen, device="cuda")
    x = normal(gen, m, k) + 8 * torch.rand(m, 1, generator=gen, device="cuda") * w.detach().float()[target]
    x = strided(x.to(dt), (0, 1, 8)[(m + k + n) % 3], (0, 3)[k % 2])
    lost = torch.rand(m, generator=gen, device="cuda") < ignored
    target = target.masked_fill(lost, -1)
    x[lost] = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dt, device="cuda")[torch.arange(int(lost.sum()), device="cuda") % 3][:, None]
    x.requires_grad_()
    b = normal(gen, n).to(dt).requires_grad_() if (m + n) % 2 else None
    g = normal(gen, m).abs() + 0.5 if reduction == "none" else torch.full((), 64.0, device="cuda")
    kind = torch.int32 if m % 2 else torch.int64
    loss = linear_cross_entropy(x, w, b, target.to(kind), ignore_index=-1, reduction=reduction)
    assert loss.dtype == torch.float32
    leaves = {q: t for q, t in {"dx": x, "dw": w, "db": b}.items() if t is not None}
    got = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()), g)))
    for name, (v, tol) in ref.cross_entropy(x, w, b, target, -1, reduction, g).items():
        if name == "loss" or name in got:
            ref.close(loss if name == "loss" else got[name], v, tol, name)
    assert not got["dx"][lost].any()
    again = linear_cross_entropy(x, w, b, target.to(kind), ignore_index=-1, reduction=reduction)
    assert torch.equal(again, loss)
    assert all(torch.equal(a, q) for a, q in zip(torch.autograd.grad(again, list(leaves.values()), g), got.values()))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 8, 2), (5, 11, 21), (4099, 64, 21), (130, 72, 64), (33, 100, 1000), (3, 512, 40001), (1, 300, 2000),
                                   (16, 256, 777), (70, 130, 600)], ids=str)
def test_label(shape, dtype):
    m, k, n = shape
    dt = TYPES[dtype]
    gen = generator(m + k + n)
    # eighths: logits are exact in fp32, ties are ties, and the lowest column wins them
    w = (torch.randint(-4, 5, (n, k), generator=gen, device="cuda") / 8).to(dt)
    x = (torch.randint(-4, 5, (m, k), generator=gen, device="cuda") / 8).to(dt)
    b = (torch.randint(-4, 5, (n,), generator=gen, device="cuda") / 8).to(dt) if m % 2 else None
    label, lp = linear_label(strided(x, m % 3, k % 2), strided(w, n % 3 * 4, n % 2), b)
    _, _, z, ez = ref.logits(x, w, b)
    best = z.amax(1, keepdim=True)
    want = torch.where(z == best, torch.arange(n, device="cuda"), n).amin(1)
    assert torch.equal(label, want)
    v = -torch.log1p(torch.where(torch.arange(n, device="cuda") == want[:, None], 0.0, torch.exp(z - best)).sum(1))
    ref.close(lp, v, (gamma_of(n) + 16 * ref.U + ref.U * (best - z).clamp(max=100).amax(1)) * v.abs() + 1e-37, "log_prob")


def gamma_of(n):
    return ref.gamma(n)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(4096, 264, 4100), (333, 8200, 260), (260, 72, 20011), (4099, 1000, 40)], ids=str)
def test_large_tiles_and_cuts(shape, dtype):
    """Sizes that take the larger tiles, and k cut into parts."""
    m, k, n = shape
    dt = TYPES[dtype]
    gen = generator(m + n)
    x, w, b = (normal(gen, m, k).to(dt).requires_grad_(), (normal(gen, n, k) * k ** -0.5).to(dt).requires_grad_(), normal(gen, n).to(dt).requires_grad_())
    r, dy, t = normal(gen, m, n).to(dt), normal(gen, m, n).to(dt), torch.randint(0, n, (m,), generator=gen, device="cuda")
    t[::3] = -100
    y = linear_act(x, w, b, activation="gelu", residual=r)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, [x, w, b], dy))) | {"y": y}
    for name, (v, tol) in ref.linear(x, w, b, r, "gelu", dy).items():
        ref.close(got[name], v, tol, name)
    g = torch.full((), 256.0, device="cuda")
    loss = linear_cross_entropy(x, w, b, t)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(loss, [x, w, b], g))) | {"loss": loss}
    for name, (v, tol) in ref.cross_entropy(x, w, b, t, -100, "mean", g).items():
        ref.close(got[name], v, tol, "cross entropy " + name)
    label, _ = linear_label(x, w, b)
    _, _, z, ez = ref.logits(x, w, b)
    top = z.topk(2, dim=1)
    clear = top.values[:, 0] - top.values[:, 1] > 2 * ez.amax(1)
    # (how many rows are clear says nothing about the kernel, only that the comparison is not empty: two largest of normal logits are
    # about 0.3 apart, and 2 ez reaches 0.06 at k = 8200)
    assert torch.equal(label[clear], top.indices[clear, 0]) and clear.float().mean() > 0.5


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,pad", [((150003, 64, 64), 0), ((150003, 11, 64), 0), ((140001, 64, 21), 1), ((200000, 40, 33), 8)], ids=str)
def test_many_rows_of_narrow_layers(shape, pad, dtype):
    """More than 65536 rows: a wave takes several turns of 32, by copies to LDS and (rows that are not whole aligned chunks) through registers."""
    m, k, n = shape
    dt, gen = TYPES[dtype], generator(m + k)
    x = strided(normal(gen, m, k).to(dt), pad, 0).requires_grad_()
    w, b = (normal(gen, n, k) * k ** -0.5).to(dt).requires_grad_(), normal(gen, n).to(dt).requires_grad_()
    dy = normal(gen, m, n).to(dt)
    y = linear_act(x, w, b, activation="gelu")
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, [x, w, b], dy))) | {"y": y}
    for name, (v, tol) in ref.linear(x, w, b, None, "gelu", dy).items():
        ref.close(got[name], v, tol, name)
    t = torch.randint(0, n, (m,), generator=gen, device="cuda")
    t[::3] = -100
    g = torch.full((), 4096.0, device="cuda")
    loss = linear_cross_entropy(x, w, b, t)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(loss, [x, w, b], g))) | {"loss": loss}
    for name, (v, tol) in ref.cross_entropy(x, w, b, t, -100, "mean", g).items():
        ref.close(got[name], v, tol, "cross entropy " + name)
    label, _ = linear_label(x, w, b)
    _, _, z, ez = ref.logits(x, w, b)
    top = z.topk(2, dim=1)
    clear = top.values[:, 0] - top.values[:, 1] > 2 * ez.amax(1)  # k <= 64: 2 ez is under 1e-3, and two largest of 21 and more are rarely that near
    assert torch.equal(label[clear], top.indices[clear, 0]) and clear.float().mean() > 0.9
    gx = torch.autograd.grad(linear_act(x, w.detach(), activation="silu"), x, dy)[0]  # dx alone
    ref.close(gx, *ref.linear(x, w, None, None, "silu", dy)["dx"], "dx alone")


@gpu
@pytest.mark.parametrize("dtype,m", [("bf16", 8192), ("f16", 7000), ("f32", 4096)])
def test_cross_entropy_in_several_pieces(dtype, m):
    """A backward pass whose dz takes more than one piece of the classes (512 MB of it)."""
    k, n, dt, gen = 24, 40003, TYPES[dtype], generator(17)
    x, w, b = (normal(gen, m, k).to(dt).requires_grad_(), (normal(gen, n, k) * k ** -0.5).to(dt).requires_grad_(), normal(gen, n).to(dt).requires_grad_())
    t = torch.randint(0, n, (m,), generator=gen, device="cuda")
    g = normal(gen, m).abs()
    loss = linear_cross_entropy(x, w, b, t, reduction="none")
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(loss, [x, w, b], g))) | {"loss": loss}
    for name, (v, tol) in ref.cross_entropy(x, w, b, t, -100, "none", g).items():
        ref.close(got[name], v, tol, name)


@gpu
@pytest.mark.parametrize("shape", [(5, 8, 9), (5, 100, 70), (200, 100, 70)], ids=str)
def test_infinities_stay_infinities(shape):
    """What a plain product gives: an infinity in x times a weight's sign, NaN where it meets a zero, nothing in the other rows."""
    m, k, n = shape
    for dt in TYPES.values():
        gen = generator(m)
        x, w = normal(gen, m, k).to(dt), normal(gen, n, k).to(dt)
        w[:, 3] = 1.0
        w[0, 3] = 0.0
        w[1, 3] = -0.5
        x[1, 3], x[2, 3], x[4, 3] = float("inf"), -float("inf"), float("nan")
        y = linear_act(x, w)
        want = x.double() @ w.double().t()
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
        odd = torch.isinf(want)
        assert torch.equal(y[odd].double(), want[odd])


@gpu
def test_calls_from_two_threads():
    import threading

    gen = generator(8)
    x, w, t = normal(gen, 700, 96), normal(gen, 130, 96), torch.randint(0, 130, (700,), generator=gen, device="cuda")
    want = [linear_act(x, w, activation="gelu"), linear_cross_entropy(x, w, None, t), *linear_label(x, w)]
    torch.cuda.synchronize()
    wrong = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = [linear_act(x, w, activation="gelu"), linear_cross_entropy(x, w, None, t), *linear_label(x, w)]
                s.synchronize()
                if not all(torch.equal(a, q) for a, q in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


@gpu
def test_label_of_odd_rows():
    nan, inf = float("nan"), float("inf")
    for n in (3, 70, 700):
        w = torch.zeros(n, 8, device="cuda")
        w[1, 0] = w[2, 0] = 1.0
        x = torch.zeros(4, 8, device="cuda")
        x[1, 0] = 5.0
        b = torch.full((n,), -inf, device="cuda")  # every class masked but one
        b[2] = 0.0
        label, lp = linear_label(x, w, b)
        assert label.tolist() == [2] * 4 and lp.tolist() == [0.0] * 4
        label, lp = linear_label(x, w, torch.full((n,), -inf, device="cuda"))  # none left: the first, no probability
        assert label.tolist() == [0] * 4 and torch.isnan(lp).all()
        low = torch.full((n,), torch.finfo(torch.float32).min, device="cuda")
        label, lp = linear_label(x[:1], w, low)
        assert label.tolist() == [0] and abs(lp.item() + torch.log(torch.tensor(float(n))).item()) < 1e-5
        b[:] = 0.0
        b[n - 1] = nan
        label, lp = linear_label(x, w, b)
        assert label.tolist() == [n - 1] * 4 and torch.isnan(lp).all()


@gpu
def test_cross_entropy_of_masked_classes_and_bad_targets():
    inf = float("inf")
    for n in (5, 300):
        gen = generator(n)
        x, w = normal(gen, 6, 16).requires_grad_(), normal(gen, n, 16).requires_grad_()
        b = torch.zeros(n, device="cuda")
        b[1:3] = -inf
        target = torch.tensor([0, 3, 1, 4, -100, 0], device="cuda")
        loss = linear_cross_entropy(x, w, b, target, reduction="none")
        assert loss[2] == inf and loss[4] == 0
        g = torch.tensor([1.0, 1.0, 0.0, 1.0, 1.0, 1.0], device="cuda")
        gx, gw = torch.autograd.grad(loss, [x, w], g)
        keep = torch.tensor([0, 1, 3, 5], device="cuda")
        want = ref.cross_entropy(x[keep], w, b, target[keep], -100, "sum", torch.ones((), device="cuda"))
        ref.close(gx[keep], *want["dx"], "dx")
        ref.close(gw, *want["dw"], "dw")
        bad = linear_cross_entropy(x, w, None, torch.tensor([0, n, -1, 2, 1 << 40, 1], device="cuda"), reduction="none")
        assert torch.isnan(bad).tolist() == [False, True, True, False, True, False]


@gpu
@pytest.mark.parametrize("m,k,n", [(40, 100, 72), (40, 100, 65), (40, 24, 70), (300, 96, 264), (20, 100, 72), (300, 16, 21)])
def test_a_target_behind_the_last_class_reaches_its_own_row_only(m, k, n):
    """Targets n .. n + 200 (in the last tile's empty columns, and behind them): NaN in their rows, nothing in the others'."""
    for dt in TYPES.values():
        gen = generator(n)
        x, w = normal(gen, m, k).to(dt).requires_grad_(), (normal(gen, n, k) * k ** -0.5).to(dt).requires_grad_()
        target = torch.randint(0, n, (m,), generator=gen, device="cuda")
        bad = torch.arange(m, device="cuda") % 3 == 2  # the last row of some sizes among them
        target[bad] = n + 7 * torch.arange(int(bad.sum()), device="cuda") % 200
        target[2], target[m - 1], bad[m - 1] = n, n + 1, True
        loss = linear_cross_entropy(x, w, None, target, reduction="none")
        gx = torch.autograd.grad(loss, x, torch.ones(m, device="cuda"))[0]
        good = ~bad
        want = ref.cross_entropy(x[good], w, None, target[good], -100, "sum", torch.ones((), device="cuda"))
        ref.close(gx[good], *want["dx"], "dx")
        assert torch.isnan(gx[bad]).all() and torch.equal(torch.isnan(loss), bad)


@gpu
def test_no_rows_and_leading_dimensions():
    for dt in TYPES.values():
        x = torch.zeros(0, 16, device="cuda", dtype=dt, requires_grad=True)
        w = torch.ones(5, 16, device="cuda", dtype=dt, requires_grad=True)
        b = torch.ones(5, device="cuda", dtype=dt, requires_grad=True)
        y = linear_act(x, w, b, activation="gelu")
        assert y.shape == (0, 5)
        gx, gw, gb = torch.autograd.grad(y.sum(), [x, w, b])
        assert gx.shape == (0, 16) and not gw.any() and not gb.any()
        t = torch.zeros(0, dtype=torch.int64, device="cuda")
        for red, shape in (("mean", ()), ("sum", ()), ("none", (0,))):
            loss = linear_cross_entropy(x, w, b, t, reduction=red)
            assert loss.shape == shape and not loss.any()
            gx, gw = torch.autograd.grad(loss.sum(), [x, w])
            assert not gw.any()
        label, lp = linear_label(x, w, b)
        assert label.shape == (0,) and lp.shape == (0,)
        gen = generator(1)
        x3, w3 = normal(gen, 2, 3, 16).to(dt), normal(gen, 7, 16).to(dt)
        assert torch.equal(linear_act(x3, w3), linear_act(x3.view(6, 16), w3).view(2, 3, 7))
        assert torch.equal(linear_act(x3[0, 0], w3), linear_act(x3[0], w3)[0])  # one vector
        assert linear_label(x3, w3)[0].shape == (2, 3)
        assert linear_cross_entropy(x3, w3, None, torch.ones(2, 3, dtype=torch.int64, device="cuda"), reduction="none").shape == (2, 3)
        e = x3[0, :1].expand(9, 16)  # one row, nine times
        assert torch.equal(linear_act(e, w3), linear_act(e.contiguous(), w3))
        wt = normal(gen, 16, 7).to(dt).t()  # a transposed weight
        assert torch.equal(linear_act(x3[0], wt), linear_act(x3[0], wt.contiguous()))


@gpu
def test_refusals_on_the_gpu():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(5, 8, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        linear_act(x.double(), w.double())
    with pytest.raises(RuntimeError, match="k"):
        linear_act(x, torch.zeros(5, 9, device="cuda"))
    with pytest.raises(RuntimeError, match="weight"):
        linear_act(x, w.half())
    with pytest.raises(RuntimeError, match="weight"):
        linear_act(x, w.cpu())
    with pytest.raises(RuntimeError, match="bias"):
        linear_act(x, w, torch.zeros(4, device="cuda"))
    with pytest.raises(RuntimeError, match="residual"):
        linear_act(x, w, residual=torch.zeros(4, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="target"):
        linear_cross_entropy(x, w, None, t.float())
    with pytest.raises(RuntimeError, match="target"):
        linear_cross_entropy(x, w, None, t[:3])
    with pytest.raises(RuntimeError, match="target"):
        linear_cross_entropy(x, w, None, t.cpu())
    y = linear_act(x.requires_grad_(), w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(y.sum(), x, create_graph=True)[0].sum(), x)


@gpu
def test_sizes_and_numbers_out_of_range_are_refused():
    x, w = torch.zeros(2, 1 << 20, device="cuda"), torch.zeros(3, 1 << 20, device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    for f in (lambda: linear_act(x, w), lambda: linear_label(x, w), lambda: linear_cross_entropy(x, w, None, t)):
        with pytest.raises(RuntimeError, match="bad argument"):
            f()
    for index in (1 << 63, -(1 << 63) - 1, (1 << 64) - 1):
        with pytest.raises(RuntimeError, match="ignore_index"):
            linear_cross_entropy(x[:, :8], w[:, :8], None, t, ignore_index=index)


@gpu
@pytest.mark.parametrize("op", ["linear", "cross_entropy"])
def test_gradients_against_differences(op):
    """The directional derivative against (f(+h) - f(-h)) / 2h in fp32: its truncation is h^2 / 6 times the third derivative along
    the direction, estimated by the same difference in 64 bits, its rounding the two values' tolerances over 2h."""
    gen = generator(11)
    m, k, n, h = 40, 24, 50, 2.0 ** -6
    x, w, b = normal(gen, m, k), normal(gen, n, k) * k ** -0.5, normal(gen, n)
    dy, t = normal(gen, m, n), torch.randint(0, n, (m,), generator=gen, device="cuda")

    def f(x, w, b):
        return (linear_act(x, w, b, activation="gelu") * dy).sum() if op == "linear" else linear_cross_entropy(x, w, b, t, reduction="sum")

    def f64(x, w, b):
        if op == "linear":
            return (ref.act(x @ w.t() + b, "gelu")[0] * dy.double()).sum()
        return -torch.log_softmax(x @ w.t() + b, 1)[torch.arange(m), t].sum()

    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    grads = torch.autograd.grad(f(*leaves), leaves)
    for i in range(3):
        d = normal(gen, *leaves[i].shape)
        d = d / d.norm()
        plus, minus = [list((x, w, b)) for _ in range(2)]
        plus[i], minus[i] = plus[i] + h * d, minus[i] - h * d
        with torch.no_grad():
            num = (f(*plus).double() - f(*minus).double()) / (2 * h)
            num64 = (f64(*[v.double() for v in plus]) - f64(*[v.double() for v in minus])) / (2 * h)
            if op == "linear":
                rounding = sum((ref.linear(*v, None, "gelu")["y"][1] * dy.double().abs()).sum() for v in (plus, minus))
                rounding = rounding + ref.gamma(m * n) * 2 * (ref.linear(*plus, None, "gelu")["y"][0] * dy.double()).abs().sum()
            else:
                rounding = sum(ref.cross_entropy(*v, t, -100, "sum")["loss"][1] for v in (plus, minus))
        exact = torch.autograd.functional.vjp(f64, tuple(v.double() for v in (x, w, b)))[1][i]
        want = (exact * d.double()).sum()
        got = (grads[i].double() * d.double()).sum()
        assert abs(num - got) <= rounding / (2 * h) + 1.01 * abs(num64 - want) + abs(got - want), (i, num, got)
        assert abs(got - want) <= 1e-4 * grads[i].double().norm()  # a unit direction: fp32 sums of m n terms are within gamma of it


@gpu
def test_other_streams_and_captured_graphs():
    gen = generator(5)
    for m, k, n, dt in ((40, 64, 21, torch.float32), (300, 256, 700, torch.bfloat16), (2, 512, 1000, torch.float16)):
        x, w, b = normal(gen, m, k).to(dt), (normal(gen, n, k) * k ** -0.5).to(dt), normal(gen, n).to(dt)
        dy, t = normal(gen, m, n).to(dt), torch.randint(0, n, (m,), generator=gen, device="cuda")

        def step(x, w, b):
            xg, wg, bg = (v.detach().requires_grad_() for v in (x, w, b))
            y = linear_act(xg, wg, bg, activation="silu")
            loss = linear_cross_entropy(xg, wg, bg, t)
            return [y.detach(), *torch.autograd.grad(y, [xg, wg, bg], dy), loss.detach(), *torch.autograd.grad(loss, [xg, wg, bg]), *linear_label(x, w, b)]

        want = step(x, w, b)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step(x, w, b)
        s.synchronize()
        assert all(torch.equal(a, q) for a, q in zip(got, want))
        # two graphs that share nothing but their inputs, replayed in turn between eager work, on new inputs each time
        graphs = []
        sx, sw, sb = x.clone(), w.clone(), b.clone()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(s):
                step(sx, sw, sb)
            s.synchronize()
            with torch.cuda.graph(g, stream=s):
                out = step(sx, sw, sb)
            graphs.append((g, out))
        for i in range(3):
            sx.copy_(normal(gen, m, k).to(dt))
            want = step(sx, sw, sb)
            for g, out in graphs:
                for v in out:
                    v.zero_()
            for g, out in graphs:
                g.replay()
            torch.cuda.synchronize()
            for g, out in graphs:
                assert all(torch.equal(a, q) for a, q in zip(out, want))


@gpu
def test_large_offsets():
    """Rows behind 2^32 bytes: the last rows of a tall x are right and the result's other rows are too."""
    m, k, n = (1 << 25) + 37, 72, 8  # x: 4.8 GB in bf16, y: 0.5 GB
    gen = generator(3)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 1, (1 << 24) + 5, 29826161, 29826162, m - 66, m - 2, m - 1], device="cuda")
    x[rows] = normal(gen, len(rows), k).to(torch.bfloat16)
    w = (normal(gen, n, k) * k ** -0.5).to(torch.bfloat16)
    y = linear_act(x, w)
    v, tol = ref.linear(x[rows], w, None, None, "none")["y"]
    ref.close(y[rows], v, tol, "y")
    y[rows] = 0
    assert not y.any()
    label, _ = linear_label(x, w)
    assert torch.equal(label[rows], (x[rows].double() @ w.double().t()).argmax(1))
    label[rows] = 0
    assert not label.any()


@gpu
def test_more_rows_than_threads_of_one_launch():
    """2^28 + 100 rows: a thread for every 16th of a row would be more than 2^32."""
    m, k, n = (1 << 28) + 100, 1, 65
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    w = (torch.arange(n, device="cuda") / 32)[:, None].to(torch.bfloat16)
    rows = torch.tensor([0, 1, 77, (1 << 25) + 3, (1 << 27) + 5, 1 << 28, m - 1], device="cuda")
    x[rows] = 1.0
    label, log_prob = linear_label(x, w)
    assert (label[rows] == n - 1).all()
    lp = torch.log_softmax(w.double()[:, 0], 0)[-1]
    assert (log_prob[rows].double() - lp).abs().max() <= (ref.gamma(n) + 16 * ref.U) * lp.abs()
    label[rows] = 0
    assert not label.any()  # all zeros: the lowest class
    log_prob[rows] = log_prob[2].item()
    assert (log_prob == log_prob[2]).all() and abs(log_prob[2].item() + math.log(n)) <= 32 * ref.U * math.log(n)
    del label, log_prob
    target = torch.zeros(m, dtype=torch.int64, device="cuda")
    loss = linear_cross_entropy(x, w, None, target, reduction="none")
    zero = math.log(n)
    assert (loss[rows].double() + torch.log_softmax(w.double()[:, 0], 0)[0]).abs().max() <= (ref.gamma(n) + 32 * ref.U) * 5
    loss[rows] = loss[2].item()
    assert (loss == loss[2]).all() and abs(loss[2].item() - zero) <= 32 * ref.U * zero


def head_config():
    cfg = HotPathConfig()
    cfg.device = "cuda"
    return cfg


@gpu
@pytest.mark.parametrize("hidden,level,classes,leaky", [(64, 1, 21, False), (64, 2, 21, True), (128, 3, 300, False)])
def test_semantic_head_trains_and_answers(hidden, level, classes, leaky):
    """A semantic decoder's step as a user takes it: sem_loss and its gradients through every layer, sem_label_prob, sem_label."""
    torch.manual_seed(7)
    cfg = head_config()
    cfg.mlp_leaky_relu = leaky
    dec = Decoder(cfg, hidden, level, classes)
    gen = generator(9)
    feat = normal(gen, 500, 11).requires_grad_()
    label = torch.randint(0, classes, (500,), generator=gen, device="cuda")
    label[::5] = -100
    loss = dec.sem_loss(feat, label)
    params = list(dec.parameters())
    got = torch.autograd.grad(loss, [feat, *params])
    f64 = feat.detach().double().requires_grad_()
    p64 = [p.detach().double().requires_grad_() for p in params]
    h, fn = f64, (torch.nn.functional.leaky_relu if leaky else torch.relu)
    for i in range(level):
        h = fn(h @ p64[2 * i].t() + p64[2 * i + 1])
    lp = torch.log_softmax(h @ p64[-2].t() + p64[-1], 1)
    keep = label != -100
    want_loss = -lp[keep, label[keep]].mean()
    want = torch.autograd.grad(want_loss, [f64, *p64])
    # fp32 through level + 1 layers of at most 300 terms: relative errors of at most (level + 2) gamma(300) of each norm, and the
    # hidden units within gamma of the kink (a share of gamma of them, each worth one of `hidden`)
    bound = 4 * (level + 2) * ref.gamma(300)
    assert abs(loss.item() - want_loss.item()) <= bound * want_loss.item()
    for a, q in zip(got, want):
        assert (a.double() - q).norm() <= bound * q.norm()
    prob = dec.sem_label_prob(feat)
    assert (prob.double() - lp).abs().max() <= bound * lp.abs().max()
    top = lp.detach().topk(2, dim=1).values
    clear = top[:, 0] - top[:, 1] > 2 * bound * lp.abs().max()
    assert torch.equal(dec.sem_label(feat)[clear], lp.argmax(1)[clear]) and clear.sum() > 400


@gpu
def test_decoder_of_any_shape_matches_the_fused_one():
    """sdf of an 11 -> 64 -> 1 decoder through the layers equals the fused kernels'; a two-layer one equals plain torch."""
    torch.manual_seed(3)
    cfg = head_config()
    dec = Decoder(cfg, 64, 1, 1)
    feat = normal(generator(2), 300, 11)
    fused = dec.sdf(feat)
    dec._native_shape = False
    layers = dec.sdf(feat)
    assert (fused - layers).abs().max() <= 2 * ref.gamma(64) * 8 * dec.sdf_scale
    deep = Decoder(cfg, 96, 2, 1)
    h = feat.double()
    for layer in deep.layers:
        h = torch.relu(h @ layer.weight.double().t() + layer.bias.double())
    want = (h @ deep.lout.weight.double().t() + deep.lout.bias.double()).squeeze(1) * deep.sdf_scale
    assert (deep.sdf(feat).double() - want).abs().max() <= ref.gamma(96) * 8 * deep.sdf_scale


@gpu
@pytest.mark.parametrize("weighted_first", [True, False])
def test_mesher_asks_the_semantic_head(weighted_first):
    import shim_io
    from clid_slam_amd.mesher import Mesher

    torch.manual_seed(5)
    cfg = shim_io.config(weighted_first=weighted_first)
    nm = shim_io.neural_points(cfg)
    sdf, sem = shim_io.decoder(cfg), Decoder(cfg, 64, 1, 21)
    gen = generator(4)
    x = nm.local_neural_points[:400] + 0.1 * normal(gen, min(400, len(nm.local_neural_points)), 3)
    x[::7] += 500.0  # far from the map: no neighbour
    mesher = Mesher(cfg, nm, {"sdf": sdf, "semantic": sem})
    s, label, _, mask = mesher.query_points(x, 150, query_sem=True, query_locally=True, mask_min_nn_count=1, out_torch=True)
    s0, none, _, _ = mesher.query_points(x, 150, query_locally=True, out_torch=True)
    assert none is None and torch.equal(s, s0) and label.dtype == torch.int64
    with torch.no_grad():
        feature, _, weight, nn, _ = nm.query_feature(x, training_mode=False, query_locally=True)
        lp = sem.sem_label_prob(feature)
        lp = lp if weighted_first else (lp * weight).sum(1)
    top = lp.topk(2, dim=1).values
    clear = (top[:, 0] - top[:, 1] > 1e-4) & (nn >= 1)
    assert clear.sum() > 100 and torch.equal(label[clear], lp.argmax(1)[clear]) and not label[nn < 1].any() and (nn < 1).any()
    with pytest.raises(RuntimeError, match="semantic"):
        Mesher(cfg, nm, {"sdf": sdf}).query_points(x, 150, query_sem=True)
