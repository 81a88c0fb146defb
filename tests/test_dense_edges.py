"""Calls of the dense operators at the edge of what they promise, and results that need more than the tests of whole layers ask for."""
import pytest
import torch

import dense_ref as ref
from clid_slam_amd.linear import linear_label
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
