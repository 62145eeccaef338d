"""Every layout that a row's length picks in the norm kernels: both edges of each and a length that is no number of packets, and enough
rows that a block of a backward pass takes several turns."""
import pytest
import torch

import operator_oracle as O
import test_gpu_operators_norm as N

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F32), (BF16, BF16)]
# lanes x packets of eight: 64, 128, 256, 512, 1024, 1536, 2048, 24 * 128, 4096, 6144, 8192 and 16384 columns are the ends of one layout each
COLS = [63, 64, 65, 100, 128, 129, 250, 256, 257, 400, 512, 513, 1000, 1025, 1111, 1535, 1536, 2001, 2048, 2600, 3071, 3073, 3500, 4095, 4096, 4097, 5001,
        6143, 6144, 6145, 7001, 8191, 8192, 9000, 16383]
# a device of 256 units holds this many rows of the layout at a time, and as many again, and some
TURNS = [(70001, 24), (33001, 100), (17001, 200), (9001, 400), (4500, 1000), (2700, 1111), (2300, 2001), (1100, 3071), (1100, 4001), (1100, 6101), (600, 8001)]


@pytest.fixture(scope="module")
def ops():
    from mccl_amd import kernels, operators
    kernels.hip_kernels_init(0)
    return operators


def backward(ops, shape, types):
    x, w, dy, mean, rstd = N.backward_case(shape, types)
    wx, ww, wb, ex, ew, eb = O.norm_backward(O.f64(dy), O.f64(x), O.f64(mean), O.f64(rstd), O.f64(w))
    first = ops.layer_norm_backward(dy, x, mean, rstd, w)
    for got, want, bound, what in zip(first, (wx, ww, wb), (ex, ew, eb), ("dx", "dweight", "dbias")):
        O.close(got, want, bound, what)
    for a, b in zip(first, ops.layer_norm_backward(dy, x, mean, rstd, w)):
        assert torch.equal(a, b), "another call gives another result"


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("cols", COLS)
def test_layouts(ops, cols, types):
    for rows in (1, 11):
        N.check_forward(ops, N.make((rows, cols), types[0], 110, 2.0, 0.5), N.make((cols,), types[1], 111, 0.3, 1.0), N.make((cols,), types[1], 112))
        backward(ops, (rows, cols), types)
    N.test_dropout_add_layer_norm(ops, (11, cols), types, 0.3)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", TURNS, ids=str)
def test_turns(ops, shape, types):
    backward(ops, shape, types)
    N.test_dropout_add_layer_norm(ops, shape, types, 0.3)
