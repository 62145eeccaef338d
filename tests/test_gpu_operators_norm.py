"""layer_norm, dropout and dropout_add_layer_norm against plain 64-bit forms (operator_oracle.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

import operator_oracle as O

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]
# rows of less than a packet up to rows that no block holds; whole and ragged packets
SHAPES = [(1, 1), (3, 7), (5, 8), (70, 64), (33, 65), (19, 200), (7, 513), (260, 768), (4, 1024), (5, 1537), (3, 2049), (6, 4100), (3, 8193),
          (2, 16384), (3, 16385), (2, 40003)]


@pytest.fixture(scope="module")
def ops():
    from mccl_amd import kernels, operators
    kernels.hip_kernels_init(0)
    return operators


def make(shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).cuda()


def check_forward(ops, x, w, b, eps=1e-5):
    y, mean, rstd = ops.layer_norm_forward(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and mean.shape == x.shape[:-1]
    wy, wm, wr, ey, em, er = O.norm(O.f64(x).reshape(-1, x.shape[-1]), O.f64(w), O.f64(b), eps)
    O.close(mean, wm, em, "mean")
    O.close(rstd, wr, er, "rstd")
    O.close(y, wy, ey, "y")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_layer_norm_forward(ops, shape, types):
    x = make(shape, types[0], 1, 2.0, 0.5)
    check_forward(ops, x, make(shape[1:], types[1], 2, 0.3, 1.0), make(shape[1:], types[1], 3))


@pytest.mark.parametrize("has_weight,has_bias", [(False, False), (True, False), (False, True)])
def test_layer_norm_forward_without_parameters(ops, has_weight, has_bias):
    x = make((9, 300), BF16, 4)
    check_forward(ops, x, make((300,), BF16, 5) if has_weight else None, make((300,), BF16, 6) if has_bias else None)


def test_layer_norm_of_rows_far_from_zero_and_of_equal_values(ops):
    """A mean a thousand times the spread, and no spread at all."""
    x = make((4, 1000), F32, 7, 1.0, 1000.0)
    x[2] = 3.25
    check_forward(ops, x, None, None)
    assert torch.equal(ops.layer_norm_forward(x)[0][2], torch.zeros(1000, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_of_strided_and_misaligned_rows(ops, dtype):
    wide = make((12, 1000), dtype, 8)
    for x in (wide[:, 3:771], wide[::2, 1:514], wide.view(3, 4, 1000)[:, :, 16:80], wide.t()[:50], wide[:0], wide[:1].expand(5, 1000)):
        y, mean, rstd = ops.layer_norm_forward(x)
        assert y.shape == x.shape
        if x.numel():
            wy, wm, wr, ey, _, _ = O.norm(O.f64(x).reshape(-1, x.shape[-1]), None, None, 1e-5)
            O.close(y, wy, ey, str(x.stride()))


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinities_and_nan_stay_in_their_row(ops, value):
    x = make((6, 700), BF16, 9)
    x[3, 411] = value
    y, mean, rstd = ops.layer_norm_forward(x)
    assert torch.isnan(y[3]).all()
    clean = [0, 1, 2, 4, 5]
    assert torch.isfinite(y[clean]).all()
    dy = make((6, 700), BF16, 10)
    dx, _, _ = ops.layer_norm_backward(dy, x, mean, rstd)
    assert torch.isfinite(dx[clean]).all() and torch.isnan(dx[3]).all()


def backward_case(shape, types, seed=20):
    x = make(shape, types[0], seed, 2.0, 0.5)
    w = make(shape[1:], types[1], seed + 1, 0.3, 1.0)
    dy = make(shape, types[0], seed + 2, 0.1)
    _, m, r, _, _, _ = O.norm(O.f64(x), None, None, 1e-5)
    return x, w, dy, torch.from_numpy(m).float().cuda(), torch.from_numpy(r).float().cuda()


@pytest.mark.parametrize("shape", SHAPES + [(3000, 24), (1500, 1030)], ids=str)
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_layer_norm_backward(ops, shape, types):
    x, w, dy, mean, rstd = backward_case(shape, types)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    assert dx.dtype == types[0] and dw.dtype == db.dtype == types[1]
    wx, ww, wb, ex, ew, eb = O.norm_backward(O.f64(dy), O.f64(x), O.f64(mean), O.f64(rstd), O.f64(w))
    O.close(dx, wx, ex, "dx")
    O.close(dw, ww, ew, "dweight")
    O.close(db, wb, eb, "dbias")
    for a, b in zip((dx, dw, db), ops.layer_norm_backward(dy, x, mean, rstd, w)):
        assert torch.equal(a, b), "another call gives another result"


@pytest.mark.parametrize("cols", [100, 20000])
def test_layer_norm_backward_without_parameters_and_strided(ops, cols):
    wide, dwide = make((8, cols + 24), F16, 30), make((8, cols + 9), F16, 31)
    x, dy = wide[:, 5:5 + cols], dwide[:, 2:2 + cols]
    _, m, r, _, _, _ = O.norm(O.f64(x), None, None, 1e-5)
    mean, rstd = torch.from_numpy(m).float().cuda(), torch.from_numpy(r).float().cuda()
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, None, with_bias=False)
    assert dw is None and db is None
    wx, _, _, ex, _, _ = O.norm_backward(O.f64(dy), O.f64(x), O.f64(mean), O.f64(rstd), None)
    O.close(dx, wx, ex, "dx")
    _, _, db = ops.layer_norm_backward(dy, x, mean, rstd, None)
    O.close(db, O.f64(dy).sum(0), 40 * O.U32 * np.abs(O.f64(dy)).sum(0), "dbias")


def test_layer_norm_backward_of_no_rows(ops):
    e = torch.empty(0, 40, dtype=BF16, device="cuda")
    s = torch.empty(0, device="cuda")
    dx, dw, db = ops.layer_norm_backward(e, e, s, s, torch.ones(40, dtype=BF16, device="cuda"))
    assert dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == db.shape == (40,)


def test_layer_norm_gradient_against_differences(ops):
    """Central differences of the kernel's own forward pass.  With step h the truncation is h^2 / 6 times the third
    derivative (below 100 here: rows of 12 values around 1, rstd below 4), the rounding 2^-23 sum|dy y| / h."""
    x, w, b, dy = make((3, 12), F32, 40), make((12,), F32, 41, 0.3, 1.0), make((12,), F32, 42), make((3, 12), F32, 43)
    leaf = [t.clone().requires_grad_() for t in (x, w, b)]
    ops.layer_norm(*leaf).backward(dy)
    h = 2.0 ** -7
    value = lambda *a: float((ops.layer_norm_forward(*a)[0].double() * dy.double()).sum())
    tol = h * h / 6 * 100 + 36 * 2.0 ** -22 / h
    for k, t in enumerate((x, w, b)):
        for i in range(t.numel()):
            up, down = [a.clone() for a in (x, w, b)], [a.clone() for a in (x, w, b)]
            up[k].view(-1)[i] += h
            down[k].view(-1)[i] -= h
            assert abs((value(*up) - value(*down)) / (2 * h) - float(leaf[k].grad.view(-1)[i])) < tol


# ---- dropout ------------------------------------------------------------------------

SEED = 0x0123456789ABCDEF


@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (70, 64), (33, 65), (513, 24), (5, 4100), (2, 70001)], ids=str)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("p", [0.1, 0.5, 1e-7, 1 - 1e-7])
def test_dropout(ops, shape, dtype, p):
    x, res = make(shape, dtype, 50), make(shape, dtype, 51)
    offset = (3 << 48) | 17
    want = O.dropped(O.f64(x), p, SEED, offset)
    O.close(ops.dropout_forward(x, p, SEED, offset), want, 2 * O.U32 * np.abs(want), "dropout")
    both = ops.dropout_forward(x, p, SEED, offset, residual=res)
    O.close(both, want + O.f64(res), 2 * O.U32 * np.abs(want) + O.U32 * np.abs(want + O.f64(res)), "with residual")
    assert torch.equal(ops.dropout_backward(x, p, SEED, offset), ops.dropout_forward(x, p, SEED, offset))


def test_dropout_of_all_and_of_nothing(ops):
    x, res = make((9, 33), BF16, 52), make((9, 33), BF16, 53)
    assert torch.equal(ops.dropout_forward(x, 0.0, 1), x)
    assert not ops.dropout_forward(x, 1.0, 1).any()
    assert torch.equal(ops.dropout_forward(x, 1.0, 1, residual=res), res)
    assert ops.dropout_forward(x[:0], 0.3, 1).shape == (0, 33)


def test_a_dropped_element_is_zero_whatever_it_held(ops):
    x = torch.full((40, 100), float("nan"), device="cuda")
    kept = torch.from_numpy(O.keep(40, 100, 0.4, 5, 6)).cuda()
    y = ops.dropout_forward(x, 0.4, 5, 6)
    assert torch.isnan(y[kept]).all() and not y[~kept].any()
    x.fill_(float("inf"))
    y = ops.dropout_backward(x, 0.4, 5, 6)
    assert torch.isinf(y[kept]).all() and not y[~kept].any()


def test_masks_depend_on_seed_offset_row_and_column_alone(ops):
    ones = torch.ones(64, 200, device="cuda")
    first = ops.dropout_forward(ones, 0.5, 9, 9)
    assert torch.equal(first, ops.dropout_forward(torch.ones(64, 200, dtype=F32, device="cuda"), 0.5, 9, 9))
    assert torch.equal(first[:10], ops.dropout_forward(ones[:10], 0.5, 9, 9))
    assert torch.equal(first[:, :77], ops.dropout_forward(ones[:, :77], 0.5, 9, 9))
    assert torch.equal(first.bfloat16(), ops.dropout_forward(ones.bfloat16(), 0.5, 9, 9))
    masks = ops.MaskStream(9, rank=1)
    others = [ops.dropout_forward(ones, 0.5, 10, 9), ops.dropout_forward(ones, 0.5, 9, 10)] + [ops.dropout_forward(ones, 0.5, *masks.next()) for _ in range(2)]
    for o in others:                       # 12800 fair draws: a share of 0.5 +- 6 standard deviations agrees
        assert abs(float((o == first).float().mean()) - 0.5) < 6 * 0.5 / 12800 ** 0.5


def test_mask_stream_continues_from_its_state(ops):
    a = ops.MaskStream(7, rank=3)
    a.next()
    b = ops.MaskStream(0)
    b.load_state_dict(a.state_dict())
    assert a.next() == b.next() and a.next() != ops.MaskStream(7, rank=2).next()


# ---- both in one pass -------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1, 1), (5, 8), (33, 65), (19, 200), (7, 513), (260, 768), (5, 1537), (6, 4100), (2, 16384), (3, 16385)], ids=str)
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_dropout_add_layer_norm(ops, shape, types, p):
    x, res = make(shape, types[0], 60), make(shape, types[0], 61, 2.0)
    w, b = make(shape[1:], types[1], 62, 0.3, 1.0), make(shape[1:], types[1], 63)
    y, s, mean, rstd = ops.dropout_add_layer_norm_forward(x, res, w, b, p, SEED, 4, 1e-5)
    t = O.f64(res) + O.dropped(O.f64(x), p, SEED, 4)
    et = 2 * O.U32 * (np.abs(O.f64(x)) * max(1.0, O.factor(p)) + np.abs(t))
    O.close(s, t, et, "s")
    wy, wm, wr, ey, em, er = O.norm(t, O.f64(w), O.f64(b), 1e-5)
    # what the sum is off by in 32 bits goes through the norm: at most that, its mean and its share of the spread
    more = et.mean(1)
    O.close(mean, wm, em + more, "mean")
    O.close(rstd, wr, er + wr * wr * 2 * et.max(1), "rstd")
    O.close(y, wy, ey + np.abs(O.f64(w)) * wr[:, None] * (et + more[:, None] + np.abs(t - wm[:, None]) * (wr * 2 * et.max(1))[:, None]), "y")

    dy, ds = make(shape, types[0], 64, 0.1), make(shape, types[0], 65, 0.1)
    for extra in (ds, None):
        dx, dres, dw, db = ops.dropout_add_layer_norm_backward(dy, extra, s, mean, rstd, w, p, SEED, 4)
        wx, ww, wb, ex, ew, eb = O.norm_backward(O.f64(dy), O.f64(s), O.f64(mean), O.f64(rstd), O.f64(w))
        total = wx + (0 if extra is None else O.f64(extra))
        ex = ex + O.U32 * np.abs(total)
        O.close(dres, total, ex, "dresidual")
        kept = 1.0 if p == 0.0 else O.keep(*shape, p, SEED, 4) * O.factor(p)
        O.close(dx, total * kept, ex * kept + 2 * O.U32 * np.abs(total) * kept, "dx")
        O.close(dw, ww, ew, "dweight")
        O.close(db, wb, eb, "dbias")


def test_differentiable_forms(ops):
    """The three functions in a row against the same graph in torch, 64 bits, with the masks as constants."""
    x, res, w, b = (make(s, F32, 70 + i) for i, s in enumerate([(17, 96), (17, 96), (96,), (96,)]))
    dy, dz = make((17, 96), F32, 75), make((17, 96), F32, 76)
    leaf = [t.clone().requires_grad_() for t in (x, res, w, b)]
    masks = ops.MaskStream(3)
    y, s = ops.dropout_add_layer_norm(leaf[0], leaf[1], leaf[2], leaf[3], 0.2, masks)
    z = ops.dropout(ops.layer_norm(y, leaf[2], leaf[3]), 0.4, masks, residual=s)
    torch.autograd.backward([y, z], [dy, dz])
    wide = [t.double().requires_grad_() for t in (x, res, w, b)]
    k = [torch.from_numpy(O.keep(17, 96, p, 3, i) * O.factor(p)).cuda() for i, p in enumerate((0.2, 0.4))]
    s2 = wide[1] + wide[0] * k[0]
    ln = lambda t: torch.nn.functional.layer_norm(t, (96,), wide[2], wide[3])
    y2 = ln(s2)
    z2 = s2 + ln(y2) * k[1]
    torch.autograd.backward([y2, z2], [dy.double(), dz.double()])
    for got, want in zip([y, z] + [t.grad for t in leaf], [y2, z2] + [t.grad for t in wide]):
        # a chain of 2 norms in fp32: some hundred roundings of numbers up to the largest
        assert float((got.double() - want).detach().abs().max()) < 500 * O.U32 * float(want.detach().abs().max())


def test_a_sum_that_nobody_differentiates(ops):
    x, res = (make((5, 64), F32, i).requires_grad_() for i in (80, 81))
    y, s = ops.dropout_add_layer_norm(x, res)
    s.sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x)) and torch.equal(res.grad, torch.ones_like(x))


def test_other_streams_and_recordings(ops):
    x, res, w, b = (make(s, BF16, 90 + i) for i, s in enumerate([(300, 520), (300, 520), (520,), (520,)]))
    dy = make((300, 520), BF16, 95)

    def step():
        y, s, mean, rstd = ops.dropout_add_layer_norm_forward(x, res, w, b, 0.1, 5, 6)
        return (y, s) + ops.dropout_add_layer_norm_backward(dy, y, s, mean, rstd, w, 0.1, 5, 6)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        for a, c in zip(got, want):
            assert torch.equal(a, c)
        eager = step()
        torch.cuda.synchronize()
        for a, c in zip(eager, want):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_a_float32_bias_without_a_weight_has_a_float32_gradient(ops, dtype):
    """Its sum over the rows is not rounded to the rows' type on the way."""
    x, dy, b = make((300, 200), dtype, 100), make((300, 200), dtype, 101), make((200,), F32, 102)
    _, mean, rstd = ops.layer_norm_forward(x, None, b)
    want, bound = O.f64(dy).sum(0), 330 * O.U32 * np.abs(O.f64(dy)).sum(0)
    for mine, theirs in ((x, dy), (x[:, 1:], dy[:, 1:])):      # (adjacent rows, and rows that lie apart)
        last = slice(200 - mine.shape[1], 200)
        leaf = b[last].clone().requires_grad_()
        ops.layer_norm(mine, None, leaf).backward(theirs)
        O.close(leaf.grad, want[last], bound[last], "layer_norm")
        leaf = b[last].clone().requires_grad_()
        ops.dropout_add_layer_norm(mine, mine, None, leaf)[0].backward(theirs)
        O.close(leaf.grad, want[last], bound[last], "seam")
    db = ops.layer_norm_backward(dy, x, mean, rstd, bias_dtype=F32)[2]
    O.close(db, want, bound, "dbias")
    assert ops.layer_norm_backward(dy, x, mean, rstd)[2].dtype == dtype
    from mccl_amd import MCCLError
    for weight, bad in ((None, torch.float64), (None, F16 if dtype == BF16 else BF16), (x[0], F32), (b, dtype)):
        with pytest.raises(MCCLError, match=r"^\[MCCL\] bias"):
            ops.layer_norm_backward(dy, x, mean, rstd, weight, bias_dtype=bad)


def test_what_is_frozen_costs_nothing(ops):
    """A backward pass writes what somebody asks for: without the parameters' gradients it is one launch."""
    from mccl_amd import kernels
    q = kernels.hip_kernels_init(0)
    x, res, w, b, dy = (make(s, BF16, 120 + i) for i, s in enumerate([(300, 200), (300, 200), (200,), (200,), (300, 200)]))

    def gradients(call, *wanted):
        leaves = [t.clone().requires_grad_(want) for t, want in zip((x, res, w, b), wanted)]
        y = call(*leaves)
        n = q.launch_count()
        y.backward(dy)
        return [t.grad for t in leaves], q.launch_count() - n

    norm = lambda x, res, w, b: ops.layer_norm(x, w, b)
    seam = lambda x, res, w, b: ops.dropout_add_layer_norm(x, res, w, b, 0.3, ops.MaskStream(5))[0]
    for call in (norm, seam):
        every, launches = gradients(call, True, call is seam, True, True)
        assert launches == 2
        for wanted in ((True, False, False, False), (False, False, True, False), (False, False, False, True), (True, False, False, True)) + (
                ((False, True, False, False), (True, True, False, False)) if call is seam else ()):
            got, launches = gradients(call, *wanted)
            assert launches == (2 if wanted[2] or wanted[3] else 1), wanted
            for a, e, want in zip(got, every, wanted):
                assert torch.equal(a, e) if want else a is None


def test_a_seam_without_a_residual(ops):
    x, w, b, dy = (make(s, F32, 125 + i) for i, s in enumerate([(20, 96), (96,), (96,), (20, 96)]))
    zero = torch.zeros_like(x)
    got = []
    for res in (None, zero):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y, s = ops.dropout_add_layer_norm(leaves[0], res, leaves[1], leaves[2], 0.2, ops.MaskStream(4))
        torch.autograd.backward([y, s], [dy, dy])
        got.append([y, s] + [t.grad for t in leaves])
    for a, c in zip(*got):
        assert torch.equal(a, c)


def test_launches_are_counted(ops):
    from mccl_amd import kernels
    q = kernels.hip_kernels_init(0)
    n = q.launch_count()
    ops.dropout_forward(torch.ones(4, 4, device="cuda"), 0.5, 1)
    assert q.launch_count() == n + 1


def test_refusals(ops):
    from mccl_amd import MCCLError, _lib as L, kernels
    x = torch.ones(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    s = torch.ones(4, device="cuda")
    for call in (lambda: ops.layer_norm_forward(x.cpu()),
                 lambda: ops.layer_norm_forward(x.double()),
                 lambda: ops.layer_norm_forward(x, w[:7]),
                 lambda: ops.layer_norm_forward(x, w.bfloat16()),
                 lambda: ops.layer_norm_forward(x.bfloat16(), w, w.bfloat16()),
                 lambda: ops.layer_norm_forward(x, w.cpu()),
                 lambda: ops.layer_norm_forward(torch.ones((), device="cuda")),
                 lambda: ops.layer_norm_forward(torch.ones(3, 0, device="cuda")),
                 lambda: ops.layer_norm_forward(x, eps=-1.0),
                 lambda: ops.layer_norm_forward(x, eps=float("nan")),
                 lambda: ops.layer_norm_backward(x[:3], x, s, s),
                 lambda: ops.layer_norm_backward(x.half(), x, s, s),
                 lambda: ops.layer_norm_backward(x, x, s[:3], s),
                 lambda: ops.layer_norm_backward(x, x, s, s.double()),
                 lambda: ops.dropout_forward(x, 1.5, 1),
                 lambda: ops.dropout_forward(x, float("nan"), 1),
                 lambda: ops.dropout_forward(x, 0.5, 1, residual=x.half()),
                 lambda: ops.dropout_forward(x, 0.5, 1, residual=x[:2]),
                 lambda: ops.dropout_add_layer_norm(x, x, p=0.5),
                 lambda: ops.MaskStream(1, rank=-1)):
        with pytest.raises(MCCLError, match=r"^\[MCCL\] "):
            call()
    # the C entries themselves
    q = kernels.hip_kernels_init(0)
    lib = L.lib()

    def forward(**kw):
        a = L.Norm(L.F32, L.F32, 4, 8, 1e-5, 0.0, 0, 0, None, None, s.data_ptr(), s.data_ptr(), x.data_ptr(), None, torch.empty_like(x).data_ptr())
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.mcclx_layer_norm_forward(q.handle, None, C.byref(a))

    assert forward() == L.OK
    assert forward(dtype=7) == L.ERR_UNSUPPORTED
    assert forward(param_dtype=L.BF16) == L.ERR_UNSUPPORTED
    for bad in (dict(x=None), dict(y=None), dict(mean=None), dict(x=x.data_ptr() + 1), dict(x_stride=7), dict(rows=1 << 33), dict(cols=1 << 31),
                dict(cols=0), dict(p=-0.5), dict(eps=-1.0), dict(rows=1 << 20)):
        assert forward(**bad) == L.ERR_INVALID, bad
    a = L.Norm(L.F32, L.F32, 4, 8)
    a.s = a.dy = x.data_ptr()
    a.mean = a.rstd = s.data_ptr()
    assert lib.mcclx_layer_norm_backward(q.handle, None, C.byref(a)) == L.ERR_INVALID and "workspace" in L.last_error()
    assert lib.mcclx_layer_norm_forward(q.handle, None, None) == L.ERR_INVALID
    torch.cuda.synchronize()


def test_rows_further_apart_than_addresses_reach(ops):
    """(rows - 1) * stride in bytes is a multiple of 2^64: no range check sees anything of it."""
    from mccl_amd import _lib as L, kernels
    q, lib = kernels.hip_kernels_init(0), L.lib()
    rows = (1 << 24) + 1
    x, s = torch.ones(1, 8, device="cuda"), torch.ones(rows, device="cuda")
    work = torch.empty(int(lib.mcclx_layer_norm_workspace_bytes(q.handle, rows, 8)), dtype=torch.uint8, device="cuda")
    a = L.Norm(L.F32, L.F32, rows, 8)
    a.s, a.dy, a.mean, a.rstd = x.data_ptr(), x.data_ptr(), s.data_ptr(), s.data_ptr()
    a.s_stride = a.dy_stride = 1 << 40
    a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
    assert lib.mcclx_layer_norm_backward(q.handle, None, C.byref(a)) == L.ERR_INVALID and "elements apart" in L.last_error()


def test_a_workspace_that_ends_early(ops):
    """16 MB are needed and claimed, 512 bytes are there (in an allocation of at most 2 MB, torch's unit for small tensors)."""
    from mccl_amd import _lib as L, kernels
    q, lib = kernels.hip_kernels_init(0), L.lib()
    x, s = torch.ones(4096, 8192, dtype=BF16, device="cuda"), torch.ones(4096, device="cuda")
    w, small = torch.ones(8192, dtype=BF16, device="cuda"), torch.empty(512, dtype=torch.uint8, device="cuda")
    need = lib.mcclx_layer_norm_workspace_bytes(q.handle, 4096, 8192)
    assert need > 2 << 20
    a = L.Norm(L.BF16, L.BF16, 4096, 8192)
    a.s, a.dy, a.mean, a.rstd, a.weight, a.dweight = x.data_ptr(), x.data_ptr(), s.data_ptr(), s.data_ptr(), w.data_ptr(), w.data_ptr()
    a.workspace, a.workspace_bytes = small.data_ptr(), need
    assert lib.mcclx_layer_norm_backward(q.handle, None, C.byref(a)) == L.ERR_INVALID and "workspace" in L.last_error()
