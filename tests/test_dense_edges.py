"""Calls of the dense operators at the edge of what they promise, and results that need more than the tests of whole layers ask for."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import dense_ref as ref
from clid_slam_amd import Decoder, HotPathConfig
from clid_slam_amd import linear as L
from clid_slam_amd.linear import linear_act, linear_label
from clid_slam_amd.loss import linear_cross_entropy
from test_dense_ops import generator, normal

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = float("inf")

# one size of each family of kernels: narrow, at most 32 rows, tiles
FAMILIES = [(5, 8, 9), (300, 16, 40), (1, 100, 70), (4, 72, 20), (32, 64, 700), (33, 64, 700), (300, 72, 66)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FAMILIES, ids=str)
def test_a_logit_of_plus_infinity_is_nan_in_its_row_at_every_size(shape, dtype):
    """log softmax of a row with an infinity is inf - inf: NaN, for every class; its label is the infinity, the other rows are untouched."""
    m, k, n = shape
    dt, gen = TYPES[dtype], generator(m + n)
    w = (normal(gen, n, k) * k ** -0.5).to(dt)
    w[:, 3] = -0.5
    w[7, 3] = 2.0
    x = normal(gen, m, k).to(dt)
    x[::2, 3] = INF  # class 7 gets +inf, the others -inf
    odd = torch.arange(m, device="cuda") % 2 == 0
    label, log_prob = linear_label(x, w)
    assert (label[odd] == 7).all() and torch.equal(torch.isnan(log_prob), odd)
    for target in (2, 7):
        t = torch.full((m,), target, device="cuda")
        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = linear_cross_entropy(xg, wg, None, t, reduction="none")
        assert torch.equal(torch.isnan(loss), odd)
        gx = torch.autograd.grad(loss, xg, torch.ones(m, device="cuda"))[0]
        assert torch.isnan(gx[odd]).all()
        if (~odd).any():
            want = ref.cross_entropy(x[~odd], w, None, t[~odd], -100, "none", torch.ones(m, device="cuda")[~odd])
            ref.close(loss[~odd], *want["loss"], "loss")
            ref.close(gx[~odd], *want["dx"], "dx")
    b = torch.zeros(n, dtype=dt, device="cuda")
    b[n - 1] = INF  # one class of every row
    x[::2, 3] = 0.0
    label, log_prob = linear_label(x, w, b)
    assert (label == n - 1).all() and torch.isnan(log_prob).all()
    assert torch.isnan(linear_cross_entropy(x, w, b, torch.zeros(m, dtype=torch.int64, device="cuda"), reduction="none")).all()


# ---- CPU: the launch replaced by a count ---------------------------------------------------------------------------------------
@pytest.fixture
def launches(monkeypatch):
    """The entry points that calls reach, with CPU operands."""
    seen = []

    class Lib:
        @staticmethod
        def clid_ce_saved(args):
            return 256

    checks = L.check_operands

    def check(what, x, weight, bias=None, residual=None):
        if not x.is_cuda:  # everything but the refusal of CPU tensors
            with monkeypatch.context() as m:
                m.setattr(torch.Tensor, "is_cuda", True)
                return checks(what, x, weight, bias, residual)
        return checks(what, x, weight, bias, residual)

    monkeypatch.setattr(L, "check_operands", check)
    monkeypatch.setattr(L, "load", Lib)
    monkeypatch.setattr(L, "call", lambda entry, workspace, args, device: seen.append(entry))
    return seen


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_derivatives_are_refused_and_never_lost(launches, which, grad_mode):
    ops = {"x": torch.randn(4, 8), "weight": torch.randn(5, 8), "bias": torch.randn(5), "residual": torch.randn(4, 5)}
    target = torch.zeros(4, dtype=torch.int64)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        assert linear_act(**ops).shape == (4, 5)  # no tangent anywhere: an ordinary call
        ops[which] = forward_ad.make_dual(ops[which], torch.ones_like(ops[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            linear_act(**ops, activation="relu")
        if which != "residual":
            with pytest.raises(NotImplementedError, match="jvp"):
                linear_cross_entropy(ops["x"], ops["weight"], ops["bias"], target)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")  # (that the trace keeps shapes is what traces do)
@pytest.mark.parametrize("op", ["linear", "label", "cross_entropy"])
def test_a_traced_call_launches_at_every_replay(launches, op):
    """torch.jit.trace records no launch that a tensor's bare pointer is handed to: it would give back memory that nothing has written."""
    w, target = torch.randn(5, 8), torch.zeros(4, dtype=torch.int64)

    def f(x):
        if op == "linear":
            return linear_act(x, w, activation="relu")
        return linear_label(x, w) if op == "label" else linear_cross_entropy(x, w, None, target)

    with torch.no_grad():
        traced = torch.jit.trace(f, (torch.randn(4, 8),), check_trace=False)
        for _ in range(3):
            before = len(launches)
            traced(torch.randn(4, 8))
            assert len(launches) == before + 1


@pytest.mark.parametrize("op", ["linear", "label", "cross_entropy"])
def test_make_fx_is_refused(launches, op):
    from torch.fx.experimental.proxy_tensor import make_fx

    w, target = torch.randn(5, 8), torch.zeros(4, dtype=torch.int64)
    f = {"linear": lambda x: linear_act(x, w), "label": lambda x: linear_label(x, w)[0], "cross_entropy": lambda x: linear_cross_entropy(x, w, None, target)}[op]
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(f)(torch.randn(4, 8))
    assert not launches


@gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_traced_decoder_answers_as_the_decoder_itself():
    cfg = HotPathConfig()
    cfg.device = "cuda"
    torch.manual_seed(2)
    dec = Decoder(cfg, 48, 2, 5).requires_grad_(False)
    gen = generator(3)
    x = [normal(gen, 200, 11) for _ in range(3)]
    mlp = torch.jit.trace(lambda v: dec.mlp(v), (x[0],))
    label = torch.jit.trace(lambda v: dec.sem_label(v), (x[0],))
    for v in x:
        assert torch.equal(mlp(v), dec.mlp(v)) and torch.equal(label(v), dec.sem_label(v))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(300, 72, 66), (2000, 40, 100), (20, 72, 66), (300, 64, 21), (20000, 24, 70)], ids=str)
def test_factors_of_rows_that_do_not_count_reach_nothing(shape, dtype):
    """reduction="none": whatever dL/dloss holds for an ignored row, the others' gradients have the same bits."""
    m, k, n = shape
    dt, gen = TYPES[dtype], generator(m + k)
    x, w, b = normal(gen, m, k).to(dt).requires_grad_(), (normal(gen, n, k) * k ** -0.5).to(dt).requires_grad_(), normal(gen, n).to(dt).requires_grad_()
    t = torch.randint(0, n, (m,), generator=gen, device="cuda")
    lost = torch.arange(m, device="cuda") % 3 == 1
    t[lost] = -100
    g = (normal(gen, m).abs() + 0.5).masked_fill(lost, 0.0)
    want = ref.cross_entropy(x, w, b, t, -100, "none", g)
    first = None
    for other in (0.0, 1e30, -3e38, 1e-30, INF, float("nan")):
        loss = linear_cross_entropy(x, w, b, t, reduction="none")
        got = torch.autograd.grad(loss, [x, w, b], torch.where(lost, other, g))
        for name, v in zip(("dx", "dw", "db"), got):
            ref.close(v, *want[name], f"{name}, {other}")
        first = first or got
        assert all(torch.equal(a, q) for a, q in zip(got, first))


@pytest.mark.parametrize("k,n", [(1 << 20, 3), ((1 << 32) + 8, 3), (8, (1 << 32) + 3), (1 << 31, 1)], ids=str)
def test_widths_are_refused_before_they_are_cut_to_32_bits(k, n):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(2, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
        t = torch.empty(2, dtype=torch.int64, device="cuda")
        for f in (lambda: linear_act(x, w), lambda: linear_label(x, w), lambda: linear_cross_entropy(x, w, None, t)):
            with pytest.raises(RuntimeError, match="bad argument"):
                f()


def test_how_a_width_would_be_cut():
    """ctypes takes the low 32 bits of a number without a word: what the check above is for."""
    assert L.LinearArgs(k=(1 << 32) + 8).k == 8


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(300, 72, 64), (40, 264, 66), (4096, 80, 96), (300, 8, 50), (20, 72, 64)], ids=str)
def test_confident_rows_keep_their_relative_accuracy(m, k, n, dtype):
    """log_prob and loss of rows whose other classes together are 2^-6 to 2^-1 of the largest: log1p of that sum, in which nothing
    of the largest one's 1 may be rounded away.

    z = -x[m, 0] for every class but the first, exact in every type, so the sum's terms are off by what exp makes of z log2(e) rounded
    twice (2 u |z|) and its own 2 u; the n of them add (n + 3) u at most, three times that where a sum that holds the 1 is used (down
    to 1/2 of it), log1p 8 u."""
    dt = TYPES[dtype]
    x = torch.zeros(m, k, device="cuda")
    others = torch.linspace(2.0 ** -6, 0.5, m, device="cuda", dtype=torch.float64) * 1.01
    x[:, 0] = -torch.log(others / (n - 1))
    x = x.to(dt)
    w = torch.zeros(n, k, dtype=dt, device="cuda")
    w[1:, 0] = -1.0
    z = x[:, 0].double()
    want = torch.log1p((n - 1) * torch.exp(-z))
    tol = (3 * (n + 3) + 2 * z + 16) * ref.U * want
    label, log_prob = linear_label(x, w)
    assert not label.any()
    ref.close(log_prob, -want, tol, "log_prob")
    loss = linear_cross_entropy(x, w, None, torch.zeros(m, dtype=torch.int64, device="cuda"), reduction="none")
    ref.close(loss, want, tol, "loss")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("m,k,n", [(40, 72, 66), (300, 100, 130), (2049, 64, 500), (4500, 24, 300), (140001, 16, 65), (70, 9, 20011)], ids=str)
def test_bias_gradient_sums_what_was_not_rounded_yet(m, k, n, reduction, dtype):
    """db is the sum of dz in fp32, before dz is rounded to the operands' type for the products: as far from 64 bits as a sum in fp32
    and one rounding of its result."""
    dt, gen = TYPES[dtype], generator(m + n)
    x, w, b = normal(gen, m, k).to(dt), (normal(gen, n, k) * k ** -0.5).to(dt), normal(gen, n).to(dt).requires_grad_()
    t = torch.randint(0, n, (m,), generator=gen, device="cuda")
    t[::5] = -100
    g = normal(gen, m).abs() if reduction == "none" else torch.full((), 512.0 if reduction == "mean" else 1.0, device="cuda")
    loss = linear_cross_entropy(x, w, b, t, reduction=reduction)
    got = torch.autograd.grad(loss, b, g)[0]
    v, tol = ref.cross_entropy(x.float(), w.float(), b.detach().float(), t, -100, reduction, g)["db"]
    ref.close(got, v, ref.rounded(v, tol, dt), "db")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(40, 16, 24), (5, 100, 70), (33, 100, 72), (300, 130, 70), (2000, 64, 64)], ids=str)
def test_what_a_dead_relu_unit_is_sent_reaches_nothing(shape, residual, dtype):
    """relu's backward pass selects: an overflowed dy (infinity, NaN) at a unit whose z <= 0 is 0 and not 0 times infinity."""
    m, k, n = shape
    dt, gen = TYPES[dtype], generator(m + k)
    make = lambda *s: torch.randint(-8, 9, s, generator=gen, device="cuda") / 8  # noqa: E731  (z exact: no z changes its side of the kink)
    x, w, b = make(m, k).to(dt).requires_grad_(), make(n, k).to(dt).requires_grad_(), make(n).to(dt).requires_grad_()
    r = normal(gen, m, n).to(dt) if residual else None
    dy = normal(gen, m, n).to(dt)
    want = ref.linear(x, w, b, r, "relu", dy)
    with torch.no_grad():
        dead = x.double() @ w.double().t() + b.double() <= 0
    assert dead.any()
    for sent in (INF, -INF, float("nan")):
        y = linear_act(x, w, b, activation="relu", residual=r)
        got = torch.autograd.grad(y, [x, w, b], dy.masked_fill(dead, sent))
        for name, v in zip(("dx", "dw", "db"), got):
            ref.close(v, *want[name], f"{name}, {sent}")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 8, 9), (6, 100, 70), (40, 100, 70)], ids=str)
def test_activations_of_odd_values_answer_as_torch_does(shape, dtype):
    """z of NaN, the infinities and zero: values and slopes are numbers, infinities and NaN where torch's own are (in float64)."""
    m, k, n = shape
    dt = TYPES[dtype]
    fs = {"relu": torch.relu, "leaky_relu": torch.nn.functional.leaky_relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}
    for name, f in fs.items():
        for value in (INF, -INF, float("nan"), 0.0, -0.0):
            x, w = torch.zeros(m, k, dtype=dt, device="cuda"), torch.zeros(n, k, dtype=dt, device="cuda")
            x[:, 0], w[:, 0] = value, 1.0
            b = torch.zeros(n, dtype=dt, device="cuda", requires_grad=True)
            y = linear_act(x, w, b, activation=name)
            db = torch.autograd.grad(y, b, torch.ones_like(y))[0]
            z = torch.full((1,), value, dtype=torch.float64, requires_grad=True)
            v = f(z)
            slope = torch.autograd.grad(v, z)[0].item()
            # (exact numbers all: 0, 1, 1/2; leaky_relu's 0.01 has one rounding to fp32 and one to the type)
            assert torch.allclose(y.double().cpu(), v.detach().expand(m, n), rtol=0, atol=0, equal_nan=True), (name, value)
            assert torch.allclose(db.double().cpu(), torch.full((n,), m * slope, dtype=torch.float64), rtol=2.0 ** -8, atol=0, equal_nan=True), (name, value, db[0], slope)


@gpu
def test_results_beyond_the_threads_of_one_launch():
    """2^30 + 300 rows of 257 classes: the tiles are more than 2^32 threads, so one launch after the other takes its share of the rows."""
    m, k, n = (1 << 30) + 300, 8, 257
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 140 << 30:
        pytest.skip("needs 140 GB of free memory")
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    gen = generator(1)
    w = (torch.arange(n, device="cuda") % 101 / 64)[:, None].repeat(1, k).to(torch.bfloat16)
    w[:, 1:] = normal(gen, n, k - 1).to(torch.bfloat16)
    rows = torch.cat([torch.arange(0, m, (1 << 24) + 77, device="cuda"), torch.tensor([m - 301, m - 300, m - 2, m - 1], device="cuda")])
    x[rows] = normal(gen, len(rows), k).to(torch.bfloat16)
    label, log_prob = linear_label(x, w)
    lp = torch.log_softmax(x[rows].double() @ w.double().t(), 1)
    top = lp.topk(2, dim=1)
    clear = top.values[:, 0] - top.values[:, 1] > 1e-4
    assert clear.sum() > 40 and torch.equal(label[rows][clear], top.indices[clear, 0])
    # z is off by gamma(8) sum |x w| < 100 gamma(8), the statistics by gamma(257)
    assert (log_prob[rows].double() - top.values[:, 0]).abs().max() <= 200 * ref.gamma(8) + ref.gamma(n) * 8
    label[rows] = 0
    assert not label.any()  # all zeros: the lowest class
    log_prob[rows] = log_prob[1].item()
    assert (log_prob == log_prob[1]).all()
    del x, label, log_prob, lp
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,k,n", [(40, 100, 65), (2048, 1024, 32000), (8192, 2048, 65536), (300000, 64, 72), (1 << 20, 64, 72), (1 << 22, 64, 300), (5000000, 8, 130000)])
def test_workspaces_are_as_large_as_the_header_says(rows, k, n, dtype):
    import ctypes as C

    lib = L.load()
    a = L.CeArgs(x=4096, w=4096, dx=4096, dw=4096, db=4096, ldx=k, ldw=k, rows=rows, k=k, n=n, dtype=dtype, reduction=1)
    value = 6 if dtype == 0 else 2
    k32, n32, slack = (k + 31) // 32 * 32, (n + 31) // 32 * 32, 4096
    copies = value * (rows + n) * k32
    forward = lib.clid_ce_workspace(C.byref(a))
    assert value * rows * k <= forward <= copies + rows * (8 * (-(-n // 32)) + 4) + rows + slack
    piece = max(512 << 20, value * 256 * rows)
    backward = lib.clid_ce_bwd_workspace(C.byref(a))
    dz = backward - copies - (4 * rows * k if piece < value * rows * n32 else 0)
    # dz itself, k cut into at most 64 parts of the results of dx or dw, 4 bytes a column and run of at least 32 rows for db
    parts = 64 * 4 * (k + 8) * max(rows, n32)
    assert dz <= piece * (1 + 4 / (32 * value)) * 1.01 + parts + slack
    assert backward >= value * rows * (k + min(n, 256))
    a = L.LabelArgs(x=4096, w=4096, ldx=k, ldw=k, rows=rows, k=k, n=n, dtype=dtype)
    assert lib.clid_label_workspace(C.byref(a)) <= copies + 12 * rows * (-(-n // 32)) + slack


def whole(gen, bits, *shape):
    """odd whole numbers of up to `bits` bits, either sign"""
    return (torch.randint(0, 1 << (bits - 1), shape, generator=gen, device="cuda") * 2 + 1) * (torch.randint(0, 2, shape, generator=gen, device="cuda") * 2 - 1).float()


def one_a_column(gen, values, rows):
    """[rows, len(values)]: values[c] at a row of its own choice in each column, zeros elsewhere; and those rows"""
    at = torch.randint(0, rows, (len(values),), generator=gen, device="cuda")
    out = torch.zeros(rows, len(values), device="cuda")
    out[at, torch.arange(len(values), device="cuda")] = values
    return out, at


# Tiles of 64, 128 and 256 with k whole and cut, for the layer's product (operands' rows along k) and both gradients' (one or both operands' rows
# across k), then the few-row and the narrow kernels
@gpu
@pytest.mark.parametrize("m,k,n", [(40, 72, 70), (4096, 264, 1024), (333, 8200, 260), (8000, 96, 4000), (4096, 1024, 1024), (2100, 2000, 130), (20, 100, 70), (300, 64, 48)], ids=str)
def test_fp32_products_keep_every_bit_of_their_operands(m, k, n):
    """One term a sum, whose product fits 24 bits: 12-bit numbers with 12-bit numbers, 24-bit ones with powers of two.  In three bf16
    parts of 8 bits each that takes hi hi, hi mid, mid hi, mid mid, and hi lo, lo hi."""
    gen = generator(m + k + n)

    def grads(x, w, dy):
        x, w = x.requires_grad_(), w.requires_grad_()
        return torch.autograd.grad(linear_act(x, w), [x, w], dy)

    def power(count):
        return 2.0 ** torch.randint(-8, 9, (count,), generator=gen, device="cuda")

    for of_x, of_w in ((12, 12), (24, 0), (0, 24)):  # bits; 0: powers of two
        value = lambda bits, *s: whole(gen, bits, *s) if bits else power(math.prod(s)).view(s)  # noqa: E731
        # y: x has one value a row, w is full; then the other way about
        xt, at = one_a_column(gen, value(of_x, m), k)
        w = value(of_w, n, k)
        assert torch.equal(linear_act(xt.t().contiguous(), w).double(), xt.sum(0).double()[:, None] * w.double()[:, at].t())
        wt, at = one_a_column(gen, value(of_w, n), k)
        x = value(of_x, m, k)
        assert torch.equal(linear_act(x, wt.t().contiguous()).double(), x.double()[:, at] * wt.sum(0).double())
        # dx: dy has one value a row, w is full; w has one value a column, dy is full
        dyt, at = one_a_column(gen, value(of_x, m), n)
        w = value(of_w, n, k)
        assert torch.equal(grads(torch.zeros(m, k, device="cuda"), w, dyt.t().contiguous())[0].double(), dyt.sum(0).double()[:, None] * w.double()[at])
        w, at = one_a_column(gen, value(of_w, k), n)
        dy = value(of_x, m, n)
        assert torch.equal(grads(torch.zeros(m, k, device="cuda"), w, dy)[0].double(), dy.double()[:, at] * w.sum(0).double())
        # dw: dy has one value a column, x is full; x has one value a column, dy is full
        dy, at = one_a_column(gen, value(of_w, n), m)
        x = value(of_x, m, k)
        assert torch.equal(grads(x, torch.zeros(n, k, device="cuda"), dy)[1].double(), dy.sum(0).double()[:, None] * x.double()[at])
        x, at = one_a_column(gen, value(of_x, k), m)
        dy = value(of_w, m, n)
        assert torch.equal(grads(x, torch.zeros(n, k, device="cuda"), dy)[1].double(), (dy.double()[at] * x.sum(0).double()[:, None]).t())


def test_operands_that_are_no_tensors_are_named(launches):
    x, w = torch.zeros(4, 8), torch.zeros(5, 8)
    for name, call in (("bias", lambda: linear_act(x, w, 0.5)), ("residual", lambda: linear_act(x, w, residual=1.0)), ("bias", lambda: linear_label(x, w, [0.0] * 5)),
                       ("bias", lambda: linear_cross_entropy(x, w, 0, torch.zeros(4, dtype=torch.int64))), ("weight", lambda: linear_act(x, None))):
        with pytest.raises(RuntimeError, match=f"{name} must be a tensor"):
            call()
    assert not launches


@gpu
@pytest.mark.parametrize("m,k,n,dtype,reduction", [(300, 72, 66, "bf16", "mean"), (20000, 24, 70, "f16", "none"), (300, 64, 21, "f32", "mean"), (20, 100, 70, "f32", "sum"),
                                                   (2049, 64, 500, "f32", "none")])
def test_a_captured_step_follows_its_targets(m, k, n, dtype, reduction):
    """How many rows count is read on the device: a replay on other targets (none, all, some ignored, factors with them) is the eager result."""
    dt, gen = TYPES[dtype], generator(m)
    x, w, b = normal(gen, m, k).to(dt), (normal(gen, n, k) * k ** -0.5).to(dt), normal(gen, n).to(dt)
    t, g = torch.randint(0, n, (m,), generator=gen, device="cuda"), normal(gen, m) if reduction == "none" else torch.full((), 8.0, device="cuda")

    def step():
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        loss = linear_cross_entropy(*leaves, t, reduction=reduction)
        return [loss.detach(), *torch.autograd.grad(loss, leaves, g)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    for share in (0.5, 1.0, 0.0, 0.9, 0.1):
        t.copy_(torch.randint(0, n, (m,), generator=gen, device="cuda"))
        t[torch.rand(m, generator=gen, device="cuda") < share] = -100
        if reduction == "none":
            g.copy_(normal(gen, m))
        want = step()
        for v in out:
            v.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, q) for a, q in zip(out, want)), share
        if share == 1.0:
            assert not any(v.any() for v in out)
