"""CPU checks of the mixture-of-experts and 8-bit checkpoint entry points: shapes,
types, formats and NULL pointers are refused on the host before any device call, empty
calls succeed, workspaces are sized, and the Python wrappers check what they are given.
Also the plain implementations that the GPU tests compare with."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R

BAD = M.MI_ERR_INVALID_ARG
P = 256  # a non-NULL stand-in address: refused calls never use it


def _all(f, good, changes):
    for at, value in changes:
        a = list(good)
        a[at] = value
        assert f(*a, None) == BAD, (at, value)
        assert f.__name__ in M.last_error() if hasattr(f, "__name__") else True


def test_gate_refusals():
    fwd = [P, P, P, 4, 8, 2, 1, M.TYPE_F32]
    _all(M.lib.mi_moe_gate_forward, fwd,
         [(3, -1), (4, 0), (4, 1025), (5, 0), (5, 9), (5, 17), (7, 3), (7, -1), (0, None),
          (1, None), (2, None), (3, 2 ** 30 + 1)])
    bwd = [P, P, P, P, P, 4, 8, 2, 0, M.TYPE_F32]
    _all(M.lib.mi_moe_gate_backward, bwd,
         [(5, -1), (6, 0), (6, 1025), (7, 0), (7, 9), (9, 3), (0, None), (1, None), (2, None),
          (3, None), (4, None)])
    assert M.lib.mi_moe_gate_forward(None, None, None, 0, 8, 2, 1, 0, None) == M.MI_OK
    assert M.lib.mi_moe_gate_backward(None, None, None, None, None, 0, 8, 2, 0, 0, None) == M.MI_OK


def test_sort_refusals():
    _all(M.lib.mi_moe_sort, [P, P, P, P, 10, 8],
         [(4, -1), (5, 0), (5, 1025), (0, None), (1, None), (3, None)])
    assert M.lib.mi_moe_sort_workspace(0, 8) == 0
    assert M.lib.mi_moe_sort_workspace(4096, 8) == 0       # one workgroup needs none
    assert M.lib.mi_moe_sort_workspace(2 ** 31 - 1, 1024) <= 256 + 256 * 1024 * 4


@pytest.mark.parametrize("name,pointers,null", [
    ("mi_moe_dispatch_forward", 3, [0, 1, 2]), ("mi_moe_dispatch_backward", 3, [0, 1, 2]),
    ("mi_moe_combine_forward", 4, [0, 1, 2, 3]), ("mi_moe_combine_backward", 6, [0, 1, 2, 3, 4, 5])])
def test_row_refusals(name, pointers, null):
    f = getattr(M.lib, name)
    n = pointers
    _all(f, [P] * n + [4, 2, 8, 16, M.TYPE_BF16],
         [(n, -1), (n + 1, 0), (n + 1, 17), (n + 2, -1), (n + 3, 0), (n + 3, 2 ** 22 + 1),
          (n + 4, 3), (n, 2 ** 30 + 1)] + [(i, None) for i in null])
    assert f(*([None] * n), 0, 2, 8, 16, 0, None) == M.MI_OK


def test_checkpoint_refusals():
    for f in (M.lib.mi_float_to_ckpt8, M.lib.mi_ckpt8_to_float):
        _all(f, [P, P, P, 4, 8, 0, 0],
             [(3, -1), (3, 2 ** 30 + 1), (4, 0), (4, 2 ** 24 + 1), (5, 2), (5, -1), (6, 3),
              (0, None), (1, None), (2, None)])
        assert f(None, None, None, 0, 8, 0, 0, None) == M.MI_OK
    _all(M.lib.mi_bias_gelu_forward_ckpt8, [P, P, P, P, P, P, 4, 8, 2, 0, 0],
         [(6, -1), (7, 0), (8, 0), (8, 1025), (9, 2), (10, 3), (0, None), (1, None), (2, None),
          (3, None), (4, None), (5, None)])
    assert "need offsets" not in M.last_error()
    _all(M.lib.mi_gelu_backward_with_bias_backward_ckpt8, [P] * 8 + [4, 8, 2, 0, 0],
         [(8, -1), (9, 0), (10, 0), (10, 1025), (11, 2), (12, 3), (0, None), (1, None), (2, None),
          (3, None), (4, None), (5, None), (7, None)])
    none = [None] * 8
    assert M.lib.mi_gelu_backward_with_bias_backward_ckpt8(*none, 0, 8, 1, 0, 0, None) == M.MI_OK
    assert M.lib.mi_bias_gelu_forward_ckpt8(*none[:6], 0, 8, 1, 0, 0, None) == M.MI_OK
    assert M.lib.mi_gelu_backward_ckpt8_workspace(0, 8, 1) == 0
    need = M.lib.mi_gelu_backward_ckpt8_workspace(16384, 6400, 32)
    assert (32 + 1) * 6400 * 4 < need < 16384 * 6400 // 4  # a small part of the tensors
    # the largest shapes do not overflow: at most 1024 + 1023 partial rows
    # the largest shapes do not overflow: at most 1024 + 1023 partial rows, and none where
    # one band has all rows (few rows, or so many columns that they fill the chip)
    for rows, cols, groups in ((16, 4096, 1), (2 ** 30, 2 ** 24, 1024)):
        assert M.lib.mi_gelu_backward_ckpt8_workspace(rows, cols, groups) == 0
    for rows, cols, groups in ((2 ** 30, 8192, 1024), (2 ** 30, 1, 1), (2 ** 30, 512, 1)):
        need = M.lib.mi_gelu_backward_ckpt8_workspace(rows, cols, groups)
        assert 256 + cols * 4 <= need <= 256 + (1024 + groups - 1) * cols * 4, (rows, cols)


def test_wrappers_check_their_tensors():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="GPU"):
        M.moe_gate_forward(x, None, None, 4, 8, 2)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        M.moe_gate_forward(x.double(), None, None, 4, 8, 2)
    with pytest.raises(ValueError, match="need their type"):
        M.moe_gate_forward(P, P, P, 4, 8, 2)
    with pytest.raises(ValueError, match="given as type"):
        M.moe_dispatch_forward(x, P, P, 4, 2, 8, 8, type=M.TYPE_BF16)
    with pytest.raises(M.MIError) as e:  # addresses pass; the library refuses the rest
        M.moe_gate_forward(P, P, P, 4, 8, 9, type=M.TYPE_F32, stream=0)
    assert e.value.code == BAD
    with pytest.raises(M.MIError):
        M.bias_gelu_forward_ckpt8(P, P, None, P, P, P, 4, 8, 2, type=M.TYPE_F32, stream=0)
    assert M.ckpt8_scales(3, 33) == 6


def test_plain_checkpoint_is_the_format():
    """The plain form's codes are the nearest ones, for a scale that holds the block."""
    r = np.random.default_rng(0)
    x = r.standard_normal((50, 70)) * np.exp2(r.integers(-30, 30, (50, 1)))
    for fmt in ("int8", "e4m3"):
        q, s = R.to_ckpt8(x, fmt)
        v = R.from_ckpt8(q, s, fmt)
        step = np.repeat(np.exp2(s.astype(float) - 127), 32, 1)[:, :70]  # 2^e
        if fmt == "int8":
            cut = x >= 127.5 / 64 * step
            assert (np.abs(v - x)[~cut] <= step[~cut] / 128).all()
            assert (np.abs(v - x)[cut] <= step[cut] / 64).all()
        else:
            cut = np.abs(x) > 448 / 256 * step
            bound = np.maximum(np.abs(x) * 2.0 ** -4, step * 2.0 ** -8 * 2.0 ** -10)
            assert (np.abs(v - x)[~cut] <= bound[~cut]).all()
            assert (np.abs(v - x)[cut] <= 64 / 256 * step[cut]).all()
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, R.E4M3, equal_nan=True)


def test_plain_router_is_the_sort():
    l = np.array([[1, 3, 3, -np.inf, np.nan], [-np.inf] * 5, [0, -0.0, 0, -0.0, -1]])
    ids, w, _ = R.gate(l, 3, True)
    assert ids.tolist() == [[4, 1, 2], [-1, -1, -1], [0, 1, 2]]
    assert np.isnan(w[0]).all() and not w[1].any() and np.allclose(w[2], 1 / 3)
