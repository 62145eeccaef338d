"""Operators over matrices whose elements and bytes 32 bits do not count, and over more rows than one launch takes.

A row's result does not depend on where it lies: rows near the places where 32 bits run over are computed again from
a small matrix of those rows and have to have the same bits (tests of that shape hold the small matrix to the formulas in
64 bits).  Masks do depend on the row, and are held to the generator's."""
import numpy as np
import pytest
import torch

import operator_oracle as O
from test_gpu_operators_loss import DZ, LOST, SPLIT

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SEED = 0x0123456789ABCDEF
ROWS, COLS = 524400, 8200   # 4.3e9 elements
SOME = sorted({0, 1, 2 ** 30 // COLS, 2 ** 31 // COLS, 2 ** 31 // COLS + 1, 2 ** 32 // COLS - 1, 2 ** 32 // COLS, 2 ** 32 // COLS + 1, ROWS - 1})


@pytest.fixture(scope="module")
def ops():
    from mccl_amd import kernels, operators
    kernels.hip_kernels_init(0)
    yield operators
    torch.cuda.empty_cache()


def filled(*shape, dtype=BF16, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(generator=g)


def keep_rows(rows, cols, p, seed, offset):
    groups = (cols + 7) // 8
    c = np.zeros((len(rows), groups, 4), np.uint64)
    c[..., 0] = np.arange(groups)
    c[..., 1] = np.asarray(rows)[:, None]
    c[..., 2], c[..., 3] = offset & 0xFFFFFFFF, offset >> 32
    w = O.philox(c, (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([(w >> np.uint64(16 * h)) & np.uint64(0xFFFF) for h in (0, 1)], -1).reshape(len(rows), groups * 8)
    return bits[:, :cols] >= O.threshold(p)


def test_norms_of_more_than_four_giga_elements(ops):
    assert ROWS * COLS > 2 ** 32
    x, dy = filled(ROWS, COLS), filled(ROWS, COLS, seed=2)
    w, b = filled(COLS, seed=3), filled(COLS, seed=4)
    some = torch.tensor(SOME, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    for got, want in zip((y, mean, rstd), ops.layer_norm_forward(x[some], w, b)):
        assert torch.equal(got[some], want)
    del y
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    assert torch.equal(dx[some], ops.layer_norm_backward(dy[some], x[some], mean[some], rstd[some], w)[0])
    del dx
    # each sum has 524400 terms in 32 bits, at most (terms + 30) u of the sum of magnitudes off (its lanes' shares are shorter)
    ww, wb, mw, mb = (torch.zeros(COLS, dtype=torch.float64, device="cuda") for _ in range(4))
    for i in range(0, ROWS, 40000):
        d = dy[i:i + 40000].double()
        u = (x[i:i + 40000].double() - mean[i:i + 40000, None]) * rstd[i:i + 40000, None].double()
        wb += d.sum(0)
        mb += d.abs().sum(0)
        d *= u
        ww += d.sum(0)
        mw += d.abs().sum(0)
    bound = (ROWS + 30) * O.U32
    O.close(dw, O.f64(ww), bound * O.f64(mw), "dweight")
    O.close(db, O.f64(wb), bound * O.f64(mb), "dbias")


def test_dropout_of_more_than_four_giga_elements(ops):
    x = filled(ROWS, COLS)
    some = torch.tensor(SOME, device="cuda")
    kept = keep_rows(SOME, COLS, 0.25, SEED, 9)
    want = np.where(kept, O.f64(x[some]) * O.factor(0.25), 0.0)
    O.close(ops.dropout_forward(x, 0.25, SEED, 9)[some], want, 2 * O.U32 * np.abs(want), "dropout")
    res = filled(ROWS, COLS, seed=5)
    y, s, mean, rstd = ops.dropout_add_layer_norm_forward(x, res, None, None, 0.25, SEED, 9)
    t = want + O.f64(res[some])
    O.close(s[some], t, 2 * O.U32 * (np.abs(want) + np.abs(t)), "s")
    del y, res
    dx, dres, _, _ = ops.dropout_add_layer_norm_backward(x, None, s, mean, rstd, None, 0.25, SEED, 9, with_bias=False)
    assert torch.equal(dres[some], ops.layer_norm_backward(x[some], s[some], mean[some], rstd[some], None, with_bias=False)[0])
    assert torch.equal((dx[some] != 0).cpu() | torch.from_numpy(~kept) | (dres[some] == 0).cpu(), torch.ones(len(SOME), COLS, dtype=torch.bool))
    assert not dx[some].cpu()[torch.from_numpy(~kept)].any()


def test_more_rows_than_a_launch_takes(ops):
    rows, cols = (1 << 21) + 77, 24
    x, dy = filled(rows, cols, dtype=F32), filled(rows, cols, dtype=F32, seed=2)
    some = torch.tensor([0, (1 << 21) - 1, 1 << 21, rows - 1], device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x)
    for got, want in zip((y, mean, rstd), ops.layer_norm_forward(x[some])):
        assert torch.equal(got[some], want)
    d = (x.double() - x.double().mean(1, keepdim=True))
    assert float((y - d / (d.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()).abs().max()) < 200 * O.U32 * float(y.abs().max())
    dx, _, db = ops.layer_norm_backward(dy, x, mean, rstd)
    assert torch.equal(dx[some], ops.layer_norm_backward(dy[some], x[some], mean[some], rstd[some])[0])
    O.close(db, O.f64(dy.double().sum(0)), (rows + 30) * O.U32 * O.f64(dy.double().abs().sum(0)), "dbias")


def test_sums_of_more_columns_than_one_launch_takes(ops):
    """A grid holds 2^32 lanes, and the parameters' sums take 32 a column."""
    cols = (1 << 27) + 40
    x, dy = filled(1, cols), filled(1, cols, seed=2)
    w = torch.ones(cols, dtype=BF16, device="cuda")
    mean, rstd = torch.full((1,), 0.25, device="cuda"), torch.full((1,), 1.5, device="cuda")
    _, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    assert torch.equal(db, dy[0])                     # one row: its sum is itself
    u = (x[0].float() - 0.25) * 1.5
    assert torch.equal(dw, (dy[0].float() * u).bfloat16())


# what is short in one call goes in small tiles, what is long in large ones
@pytest.mark.parametrize("tokens", [5, 300])
@pytest.mark.parametrize("dtype,vocab,width", [(BF16, 530001, 4096), (F32, 270001, 4096)], ids=str)
def test_a_weight_of_more_than_four_giga_bytes(ops, dtype, vocab, width, tokens):
    assert vocab * width * (2 if dtype == BF16 else 4) > 2 ** 32
    w = filled(vocab, width, dtype=dtype).mul_(2 / width ** 0.5)
    h = filled(tokens, width, dtype=dtype, seed=2)
    t = torch.randint(0, vocab, (tokens,), generator=torch.Generator().manual_seed(3)).cuda()
    past = 2 ** 32 // (width * w.element_size())  # the first row behind 4 GiB
    t[0], t[1], t[2] = vocab - 1, past - 1, past
    assert int(t.max()) < vocab
    loss, lse = ops.linear_cross_entropy_forward(h, w, t, reduction="none")
    grad = torch.linspace(-1.0, 1.0, tokens, device="cuda")
    dh, dw = ops.linear_cross_entropy_backward(grad, h, w, t, lse, reduction="none")

    # the formula in 64 bits and the bounds of test_gpu_operators_loss.py, in parts of the vocabulary
    parts = [slice(i, min(i + 20000, vocab)) for i in range(0, vocab, 20000)]
    at = torch.arange(tokens, device="cuda")
    h, g = h.double(), grad.double()[:, None]
    logits = lambda m, part: torch.mm(m, part.t().contiguous())
    z = torch.cat([logits(h, w[i].double()) for i in parts], 1)
    ez = torch.cat([logits(h.abs(), w[i].double().abs()) for i in parts], 1) * (2 * width * O.U32 + SPLIT[dtype])
    l, top = torch.logsumexp(z, 1), z.max(1).values
    el = ez.max(1).values + 120 * O.U32 + 8 * O.U32 * l.abs() + 4 * O.U32 * (top - z.min(1).values)
    O.close(lse, O.f64(l), O.f64(el), "lse")
    want = l - z[at, t]
    O.close(loss, O.f64(want), O.f64(el + ez[at, t] + O.U32 * want.abs()), "loss")
    wh, eh = torch.zeros_like(h), torch.zeros_like(h)
    for i in parts:
        away = z[:, i] - l[:, None]
        p = torch.exp(away)
        dz = p.clone()
        here = (t >= i.start) & (t < i.stop)
        dz[at[here], t[here] - i.start] -= 1
        edz = p * (ez[:, i] + el[:, None] + 8 * O.U32 * (1 + away.abs())) + (DZ[dtype] + 4 * O.U32) * dz.abs() + LOST[dtype]
        edz, dz = edz * g.abs() + LOST[dtype] * float(g.abs().max()), dz * g
        part = w[i].double()
        wh += torch.mm(dz, part)
        eh += torch.mm(edz, part.abs()) + (2 * vocab * O.U32 + SPLIT[dtype] + 4 * O.U32) * torch.mm(dz.abs(), part.abs())
        some = torch.unique(torch.cat([t[here] - i.start, torch.tensor([0, i.stop - i.start - 1], device="cuda")]))
        ww = torch.mm(dz[:, some].t().contiguous(), h)
        ew = torch.mm(edz[:, some].t().contiguous(), h.abs()) + (2 * tokens * O.U32 + SPLIT[dtype] + 4 * O.U32) * torch.mm(dz[:, some].abs().t().contiguous(), h.abs())
        O.close(dw[i][some], O.f64(ww), O.f64(ew), f"dweight {i}")
    O.close(dh, O.f64(wh), O.f64(eh), "dhidden")
