"""linear_cross_entropy of float32 matrices whose rows, columns, probabilities and gradients lie many powers of two apart, and
gradients that are no numbers: what is large, or lost, in one row must not cost another its precision.

Bounds.  As in test_gpu_operators_loss.py, first order, but weighted by the probabilities: an entry of the vocabulary that nobody
expects does not add to a logarithm's error, however large its logit.  A float32 product is off by its own rounding and by at most as
much again, a value of dz by its rounding to 24 bits and by what lies below 2^-120."""
import numpy as np
import pytest
import torch

import operator_oracle as O
from test_gpu_operators_loss import make

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = O.U32
NOTHING = 2.0 ** -120


@pytest.fixture(scope="module")
def ops():
    from mccl_amd import kernels, operators
    kernels.hip_kernels_init(0)
    return operators


def oracle(h, w, t, g):
    """Losses, lse, dh, dw for the rows' gradients g, and a bound of each."""
    h, w, t = O.f64(h), O.f64(w), t.cpu().numpy()
    n, v, d = len(h), len(w), h.shape[1]
    rows = np.arange(n)
    z = h @ w.T
    ez = (2 * d + 2) * U * (np.abs(h) @ np.abs(w).T)
    top = z.max(1, keepdims=True)
    lse = np.log(np.exp(z - top).sum(1)) + top[:, 0]
    away = z - lse[:, None]
    p = np.exp(away)
    el = (p * (ez + 8 * U * np.abs(away))).sum(1) + 120 * U + 8 * U * np.abs(lse)
    valid = t != -100
    at = np.where(valid, t, 0)
    loss = np.where(valid, lse - z[rows, at], 0.0)
    eloss = np.where(valid, el + ez[rows, at] + U * np.abs(loss), 0.0)
    g = np.where(valid, g, 0.0)[:, None]
    dz = p.copy()
    dz[rows, at] -= 1
    edz = np.minimum(p * (ez + el[:, None] + 8 * U * (1 + np.abs(away))) + 5 * U * np.abs(dz), 2.0) + NOTHING
    edz, dz = edz * np.abs(g) + NOTHING * np.abs(g).max(), dz * g
    eh = edz @ np.abs(w) + (2 * v + 6) * U * (np.abs(dz) @ np.abs(w))
    ew = edz.T @ np.abs(h) + (2 * n + 6) * U * (np.abs(dz).T @ np.abs(h))
    return loss, lse, dz @ w, dz.T @ h, eloss, el, eh, ew


def check(ops, h, w, t, grad):
    loss, lse = ops.linear_cross_entropy_forward(h, w, t, reduction="none")
    dh, dw = ops.linear_cross_entropy_backward(grad, h, w, t, lse, reduction="none")
    wl, wlse, wh, ww, el, elw, eh, ew = oracle(h, w, t, O.f64(grad))
    O.close(lse, wlse, elw, "lse")
    O.close(loss, wl, el, "loss")
    O.close(dh, wh, eh, "dhidden")
    O.close(dw, ww, ew, "dweight")


def gradients(n, seed=5):
    return torch.randn(n, generator=torch.Generator().manual_seed(seed)).cuda()


# small tiles; large ones (257 tokens of 16385 entries are more than half a round of the device's units)
@pytest.mark.parametrize("shape", [(40, 300, 64), (257, 16385, 72)], ids=str)
@pytest.mark.parametrize("e", [34, 50, 100])
@pytest.mark.parametrize("where", ["hidden", "ignored", "weight", "column"])
def test_float32_matrices_of_rows_far_apart(ops, where, e, shape):
    h, w, t = make(*shape, F32, seed=21)
    t[7] = 3
    if where in ("hidden", "ignored"):
        h[7] *= 2.0 ** e
    if where == "ignored":
        t[7] = -100
    if where == "weight":
        w[11] *= 2.0 ** e
    if where == "column":       # large, and without a partner
        h[:, 5] = 2.0 ** e
        w[:, 5] = 0.0
    check(ops, h, w, t, gradients(len(h)))


def test_float32_matrices_with_a_large_row_each(ops):
    """Padding 2^100 times as large as the tokens, and an entry 2^100 times as large as the others: both matrices at the end of their range."""
    h, w, t = make(60, 300, 64, F32, seed=25)
    h[7] *= 2.0 ** 100
    w[11] *= 2.0 ** 100
    t[7] = -100
    grad = gradients(60)
    loss, lse = ops.linear_cross_entropy_forward(h, w, t, reduction="none")
    dh, dw = ops.linear_cross_entropy_backward(grad, h, w, t, lse, reduction="none")
    rest = torch.arange(60) != 7
    wl, wlse, wh, ww, el, elw, eh, ew = oracle(h[rest], w, t[rest], O.f64(grad)[rest.numpy()])
    O.close(lse[rest], wlse, elw, "lse")
    O.close(loss[rest], wl, el, "loss")
    O.close(dh[rest], wh, eh, "dhidden")
    O.close(dw, ww, ew, "dweight")
    assert float(loss[7]) == 0.0 and not dh[7].any()


@pytest.mark.parametrize("e", [30, 60])
def test_float32_gradients_of_entries_that_nobody_expects(ops, e):
    """Half of the vocabulary has probabilities around 2^-e; those rows of dweight are held to their own size."""
    h, w, t = make(60, 300, 64, F32, seed=22)
    t = (t.clamp(min=0) // 2) * 2
    h[:, 0], w[:, 0] = 1.0, 0.0
    w[1::2, 0] = -e * 0.6931472
    check(ops, h, w, t, gradients(60))


def test_float32_gradients_of_tokens_far_apart(ops):
    h, w, t = make(60, 300, 64, F32, seed=23)
    check(ops, h, w, t, gradients(60) * torch.logspace(-30, 3, 60, device="cuda"))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_a_gradient_that_is_no_number_stays_in_its_row(ops, dtype, value):
    h, w, t = make(300, 520, 64, dtype, seed=24)
    t[5], t[9] = 3, -100
    grad = gradients(300)
    grad[5] = 0.0
    lse = ops.linear_cross_entropy_forward(h, w, t)[1]
    clean, _ = ops.linear_cross_entropy_backward(grad, h, w, t, lse, reduction="none")
    for row in (5, 9):
        bad = grad.clone()
        bad[row] = value
        dh, dw = ops.linear_cross_entropy_backward(bad, h, w, t, lse, reduction="none")
        rest = torch.arange(300) != row
        assert torch.equal(dh[rest], clean[rest])
        if row == 5:
            assert not torch.isfinite(dh[5]).any() and not torch.isfinite(dw).any()
        else:                   # an ignored token's gradient reaches nobody
            assert not dh[9].any() and torch.isfinite(dw).all()
    only = torch.zeros(300, device="cuda")
    only[5] = value
    dh, _ = ops.linear_cross_entropy_backward(only, h, w, t, lse, reduction="none")
    assert not torch.isfinite(dh[5]).any() and not dh[torch.arange(300) != 5].any()
