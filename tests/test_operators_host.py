"""The training operators without a GPU: the tests' own generator against published outputs, the layouts
of the C ABI, calls without a context."""
import ctypes as C

import numpy as np
import pytest

import operator_oracle as O


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, want):
    """The known-answer vectors that the generator's authors publish for philox4x32, 10 rounds."""
    got = O.philox(np.array(counter, np.uint64), key)
    assert tuple(int(v) for v in got) == want


def test_masks_keep_the_share_they_should():
    kept = O.keep(256, 1000, 0.1, 12345, 6)
    assert abs(kept.mean() - 0.9) < 6 * (0.09 / kept.size) ** 0.5
    assert O.threshold(0.1) == 6554 and O.threshold(1e-9) == 1 and O.threshold(1 - 1e-9) == 65535


def test_layout_matches_the_header():
    from mccl_amd import _lib as L
    assert C.sizeof(L.Norm) == 8 + 6 * 8 + 14 * 8 + 5 * 8 + 2 * 8
    assert C.sizeof(L.Loss) == 8 + 3 * 8 + 13 * 8


def test_calls_without_a_context():
    from mccl_amd import _lib as L
    lib = L.lib()
    assert lib.mcclx_layer_norm_forward(None, None, C.byref(L.Norm())) == L.ERR_STATE
    assert lib.mcclx_layer_norm_backward(None, None, C.byref(L.Norm())) == L.ERR_STATE
    assert lib.mcclx_dropout(None, None, 0, 1, 1, None, 1, None, 1, None, 0.5, 0, 0) == L.ERR_STATE
    assert lib.mcclx_layer_norm_workspace_bytes(None, 4, 4) == 0
    assert lib.mcclx_linear_cross_entropy_forward(None, None, C.byref(L.Loss())) == L.ERR_STATE
    assert lib.mcclx_linear_cross_entropy_backward(None, None, C.byref(L.Loss())) == L.ERR_STATE
    assert lib.mcclx_linear_cross_entropy_workspace_bytes(None, C.byref(L.Loss()), 0) == 0


def test_no_fallback_without_a_queue(monkeypatch):
    import torch
    from mccl_amd import MCCLError, kernels, operators
    monkeypatch.setattr(kernels, "_default", None)
    with pytest.raises(MCCLError, match="not called"):
        operators.layer_norm_forward(torch.ones(2, 2))


def test_ranks_that_resume_from_one_state_keep_masks_of_their_own():
    """The usual checkpoint: rank 0 saves, every rank loads."""
    from mccl_amd import operators
    saved = operators.MaskStream(7, rank=0)
    saved.next()
    state = saved.state_dict()
    following = saved.next()
    drawn = []
    for rank in range(4):
        stream = operators.MaskStream(99, rank=rank)
        stream.load_state_dict(state)
        assert (stream.seed, stream.rank, stream.count) == (7, rank, 1)
        drawn.append(stream.next())
    assert drawn[0] == following and len(set(drawn)) == 4
    alone = operators.MaskStream(0)                   # one that names no rank takes the state's
    alone.load_state_dict(operators.MaskStream(7, rank=3).state_dict())
    assert alone.next() == operators.MaskStream(7, rank=3).next()


def test_the_tests_check_every_pointer_whatever_the_environment_says():
    """Some refusals that they ask for are told by a range check alone."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    out = subprocess.run([sys.executable, "-c", "import conftest, os; print(os.environ['MCCLX_VALIDATE'])"], cwd=here, text=True, capture_output=True,
                         env={**os.environ, "MCCLX_VALIDATE": "0"}, check=True).stdout
    assert out.strip() == "1"
