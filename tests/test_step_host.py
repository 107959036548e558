"""CPU checks of the RMS norm, balance loss and many-tensor entry points: shapes, types,
formats and NULL pointers are refused on the host before any device call, empty calls
succeed, workspaces are sized, and the Python wrappers check what they are given."""
import ctypes

import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
import step_ref as S

BAD = M.MI_ERR_INVALID_ARG
P = 256  # a non-NULL stand-in address: refused calls never use it
NAN, INF = float("nan"), float("inf")


def _all(f, good, changes):
    for at, value in changes:
        a = list(good)
        a[at] = value
        assert f(*a, None) == BAD, (f.__name__, at, value)
        assert f.__name__ in M.last_error()


def test_rmsnorm_refusals():
    L = M.lib
    shape = [(-1, 0), (0, 1), (2 ** 24 + 1, 1), (-3, 1)]  # (value, place behind the pointers)
    for name, ptrs, null in (("mi_rmsnorm_forward", 4, [0, 1, 2]),
                             ("mi_residual_rmsnorm_forward", 6, [0, 1, 2, 3, 4])):
        good = [P] * ptrs + [4, 8, 1e-5, M.TYPE_BF16]
        _all(getattr(L, name), good, [(ptrs + p, v) for v, p in shape] + [(i, None) for i in null] +
             [(ptrs + 2, v) for v in (-1e-6, NAN, INF)] + [(ptrs + 3, v) for v in (3, -1)])
        assert getattr(L, name)(*([None] * ptrs), 0, 8, 1e-5, 0, None) == M.MI_OK
    for name, ptrs, null in (("mi_rmsnorm_forward_row8", 6, [0, 1, 2, 3]),
                             ("mi_residual_rmsnorm_forward_row8", 8, [0, 1, 2, 3, 4, 5])):
        good = [P] * ptrs + [4, 8, 1e-5, 0, M.ROW8_E4M3, M.TYPE_F16]
        _all(getattr(L, name), good, [(ptrs + p, v) for v, p in shape] + [(i, None) for i in null] +
             [(ptrs + 2, NAN), (ptrs + 3, 32), (ptrs + 3, -128), (ptrs + 4, 2), (ptrs + 4, -1),
              (ptrs + 5, 3)])
        assert getattr(L, name)(*([None] * ptrs), 0, 8, 1e-5, 128, 0, 0, None) == M.MI_OK
    for name in ("mi_rmsnorm_backward", "mi_rmsnorm_backward_residual"):
        good = [P] * 6 + [4, 8, M.TYPE_F32]
        _all(getattr(L, name), good, [(6 + p, v) for v, p in shape] + [(i, None) for i in range(6)] +
             [(8, 3)])
        assert getattr(L, name)(*([None] * 6), 0, 8, 0, None) == M.MI_OK


def test_rmsnorm_workspace():
    f = M.lib.mi_rmsnorm_backward_workspace
    assert f(0, 8, 0) == f(8, 0, 0) == f(8, 8, 3) == 0
    for rows, cols, type_ in ((1, 1, 0), (8192, 1600, 2), (2 ** 31 - 1, 2 ** 24, 0),
                              (2 ** 31 - 1, 64, 1), (300, 20000, 0)):
        assert cols * 4 < f(rows, cols, type_) <= 256 + min(rows, 512) * cols * 4, (rows, cols)


def test_balance_refusals():
    fwd = [P] * 6 + [4, 8, 2, 0.01, M.TYPE_F32]
    _all(M.lib.mi_moe_balance_forward, fwd,
         [(6, -1), (7, 0), (7, 1025), (8, 0), (8, 9), (8, 17), (10, 3), (6, 2 ** 30 + 1)] +
         [(i, None) for i in (0, 1, 3, 4, 5)])
    bwd = [P] * 5 + [4, 8, 2, 0.01, 1, M.TYPE_F32]
    _all(M.lib.mi_moe_balance_backward, bwd,
         [(5, -1), (6, 0), (6, 1025), (7, 0), (7, 9), (10, 3), (0, None), (2, None), (4, None)])
    assert M.lib.mi_moe_balance_backward(*([None] * 5), 0, 8, 2, 0.01, 1, 0, None) == M.MI_OK
    # no tokens: the results are still written, so their buffers are needed
    assert M.lib.mi_moe_balance_forward(None, None, None, P, P, None, 0, 8, 2, 0.01, 0, None) == BAD
    f = M.lib.mi_moe_balance_workspace
    assert f(0, 8) == f(16, 8) == f(16, 0) == 0  # one workgroup needs none
    assert f(2 ** 31 - 1, 1024) <= 256 + 512 * (2 * 1024 + 1) * 4


def _lists(n):
    return ((ctypes.c_void_p * n)(*[P] * n), (ctypes.c_void_p * n)(*[P] * n),
            (ctypes.c_longlong * n)(*[4] * n), (ctypes.c_int * n)(*[M.TYPE_F32] * n))


def test_tensor_list_refusals():
    t, o, s, y = _lists(3)
    f, a = M.lib.mi_tensors_clip, ctypes.addressof
    _all(f, [a(t), a(o), a(s), a(y), 3, 1.0, P, P],
         [(0, None), (2, None), (4, -1), (5, -1.0), (5, NAN), (6, None), (7, None)])
    _all(M.lib.mi_tensors_scale, [a(t), a(o), a(s), a(y), 3, P], [(0, None), (2, None), (5, None)])
    _all(M.lib.mi_tensors_norm_sq_acc, [a(t), a(s), a(y), 3, P], [(0, None), (1, None), (4, None)])

    def refused(what):
        assert f(a(t), a(o), a(s), a(y), 3, 1.0, P, P, None) == BAD
        assert "tensor 1" in M.last_error() and what in M.last_error()
    s[1] = -1
    refused("size")
    s[1] = 2 ** 62
    refused("size")
    s[1], y[1] = 4, 7
    refused("type")
    y[1], t[1] = 0, None
    refused("NULL")
    t[1], o[1] = P, None
    refused("NULL")
    # more elements together than a grid has units for
    t, o, s, y = _lists(3)
    s[0] = s[1] = s[2] = 2 ** 42
    assert f(a(t), a(o), a(s), a(y), 3, 1.0, P, P, None) == BAD and "elements" in M.last_error()
    # nothing to do
    t, o, s, y = _lists(2)
    s[0] = s[1] = 0
    t[0] = None
    assert M.lib.mi_tensors_norm_sq_acc(a(t), a(s), a(y), 2, P, None) == M.MI_OK
    assert M.lib.mi_tensors_scale(a(t), a(o), a(s), None, 2, P, None) == M.MI_OK
    assert M.lib.mi_tensors_scale(None, None, None, None, 0, P, None) == M.MI_OK
    # a kernel's partial sums, and where there are more, a description of each tensor
    assert M.lib.mi_tensors_workspace(0) <= M.lib.mi_tensors_workspace(96) < 10_000
    assert M.lib.mi_tensors_workspace(10 ** 6) < 200 * 10 ** 6
    assert M.lib.mi_tensors_workspace(-1) == 0


def test_workspace_of_a_list_without_tensors():
    """Clipping it still writes the norm, through the partial sums' place of one launch: 2048."""
    assert M.lib.mi_tensors_workspace(0) == M.lib.mi_tensors_workspace(1) == 256 + 2048 * 4


def test_wrappers_check_their_tensors():
    x = torch.zeros(4, 8)
    for f in (lambda: M.rmsnorm_forward(x, x, x, None, 4, 8),
              lambda: M.rmsnorm_backward(x, x, x, x, x, x, 4, 8),
              lambda: M.moe_balance_forward(x, None, None, None, None, None, 4, 8, 2, 0.01),
              lambda: M.TensorList([x])):
        with pytest.raises(ValueError, match="GPU"):
            f()
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        M.rmsnorm_forward(x.double(), P, P, P, 4, 8)
    with pytest.raises(ValueError, match="need their type"):
        M.residual_rmsnorm_forward_row8(P, P, P, P, P, P, None, None, 4, 8)
    with pytest.raises(ValueError, match="outs"):
        M.TensorList([], [x])
    with pytest.raises(M.MIError) as e:  # addresses pass; the library refuses the rest
        M.rmsnorm_forward_row8(P, P, P, P, None, None, 4, 8, block=64, type=M.TYPE_F32, stream=0)
    assert e.value.code == BAD and "block=64" in str(e.value)
    assert M.row8_scales(3, 129) == 3 and M.row8_scales(3, 129, M.ROW8_BLOCK) == 6
    empty = M.TensorList([])
    M.tensors_scale(empty, P, stream=0)  # an empty list is a successful no-op


def _apart(tensors, outs=None):
    """Whether a list of host tensors would be taken where it is written (no kernel runs)."""
    x = M.TensorList([])
    x.tensors, x.out_tensors, x._outs = tensors, outs, None if outs is None else x._data
    try:
        x._written()
        return True
    except ValueError as e:
        assert "overlap" in str(e)
        return False


def test_lists_that_are_written_must_not_overlap():
    x, y = torch.zeros(100), torch.zeros(100)
    assert _apart([]) and _apart([x, y]) and _apart([x[50:], x[:50], x[50:50]])
    assert not _apart([x, x]) and not _apart([x[:51], y, x[50:]]) and not _apart([x, x[3:4]])
    assert not _apart([x.half(), y, y[99:].view(torch.float16)])
    # the tensors may overlap each other where they are only read
    assert _apart([x, x], [y[:50], y[50:]]) and _apart([x[:51], x[50:]], [y[1:], y[:1]])
    assert not _apart([x, y], [y[:50], torch.zeros(5)]) and not _apart([x, x], [y, y[10:20]])
    assert not _apart([x[10:20]], [x]) and not _apart([x], [x[99:]]) and not _apart([x], [x])
    assert _apart([x[10:20]], [x[20:30]]) and _apart([x[10:20], y], [x[20:30], x[:10]])


def test_plain_codes_are_the_nearest():
    r = np.random.default_rng(0)
    y = r.standard_normal((20, 300)) * np.exp2(r.integers(-20, 20, (20, 1)))
    for largest, table in ((127.0, np.arange(-127, 128)), (448.0, np.unique(R.E4M3[:127]))):
        for block in (0, 128):
            s, v = S.scales_of(y, block, largest)
            assert s.shape == (20, 3 if block else 1) and np.abs(v).max() <= largest * (1 + 1e-15)
            near = np.abs(np.abs(v)[..., None] - np.abs(table)[None, None]).min(-1)
            fmt = "int8" if largest == 127 else "e4m3"
            assert (near <= S.code_bound(v, fmt)).all()
