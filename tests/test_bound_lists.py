"""CPU checks of lists of tensors in calls: what a bound call will read stays alive with it, and
what is written overlaps nothing else of the call.  The tensors are stand-ins; the library's
functions are not called, or replaced."""
import gc
import weakref

import pytest
import torch

import cme213_amd as M

P = 256  # a non-NULL stand-in address, which nothing reads


class Stand:
    """A tensor on the GPU, as far as a list looks at it."""
    is_cuda = True

    def __init__(self, address, n, dtype=torch.float32, device=0):
        self.address, self.n, self.dtype, self.device_number = address, n, dtype, device

    def numel(self):
        return self.n

    def element_size(self):
        return torch.empty(0, dtype=self.dtype).element_size()

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device_number

    def data_ptr(self):
        return self.address


@pytest.fixture(autouse=True)
def device_0(monkeypatch):
    monkeypatch.setattr(M, "_current_device", lambda: 0)


def _bind(name, args):
    if name == "mi_tensors_norm_sq_acc":
        return M.bind(name, args[0], *args[2:], P)
    if name == "mi_tensors_scale":
        return M.bind(name, *args, P)
    return M.bind(name, *args, 1.0, P, P)


CALLS = ["mi_tensors_norm_sq_acc", "mi_tensors_scale", "mi_tensors_clip"]


@pytest.mark.parametrize("with_outs", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_a_bound_call_keeps_its_list(name, with_outs):
    tensors = [Stand(0x10000 * (i + 1), 100) for i in range(50)]
    outs = [Stand(0x10000 * (i + 101), 100) for i in range(50)] if with_outs else None
    x = M.TensorList(tensors, outs)
    held = [weakref.ref(t) for t in [x] + tensors + (outs or [])]
    bound = _bind(name, x.args())
    del x, tensors, outs
    gc.collect()
    assert all(r() is not None for r in held)
    del bound
    gc.collect()
    assert all(r() is None for r in held)


def test_the_arguments_alone_keep_the_list():
    """As of a call of the library itself, whose arguments are all that is left of the list."""
    args = M.TensorList([Stand(0x10000, 7)]).args()
    gc.collect()
    assert args[4] == 1 and args[1] is None
    keeper = args[0].tensors
    ref = weakref.ref(keeper)
    del keeper, args
    gc.collect()
    assert ref() is None


@pytest.mark.parametrize("name", CALLS)
def test_a_bound_call_makes_the_lists_checks(name, monkeypatch):
    """What is written overlaps nothing else of the list, when the call is bound; the current
    device is the tensors', when it is made."""
    def args(tensors, outs=None):
        return M.TensorList([Stand(*t) for t in tensors],
                            outs and [Stand(*t) for t in outs]).args()
    writes = name != "mi_tensors_norm_sq_acc"
    apart = args([(0x1000, 64), (0x1100, 10)])
    for bad in (args([(0x1000, 65), (0x1100, 10)]), args([(0x1000, 4), (0x1000, 4)]),
                args([(0x1000, 4)], [(0x1000, 4)]), args([(0x1000, 4)] * 2, [(0x2000, 4), (0x2008, 4)])):
        if writes:
            with pytest.raises(ValueError, match="overlap"):
                _bind(name, bad)
        else:
            _bind(name, bad)
    _bind(name, apart)
    _bind(name, args([(0x1000, 4), (0x1000, 4)], [(0x2000, 4), (0x2010, 4)]))
    if writes:  # a list with outs, bound without them: its tensors are what is written
        both = args([(0x1000, 4), (0x1008, 4)], [(0x2000, 4), (0x2010, 4)])
        _bind(name, both)
        with pytest.raises(ValueError, match="overlap"):
            _bind(name, (both[0], None) + both[2:])
    calls = []
    monkeypatch.setattr(M.lib, name, lambda *a: calls.append(a) or M.MI_OK)
    monkeypatch.setattr(M, "_current_stream", lambda: None)
    bound = _bind(name, apart)
    elsewhere = _bind(name, args([(0x1000, 4, torch.float32, 1)]))
    bound()
    with pytest.raises(ValueError, match="current device"):
        elsewhere()
    monkeypatch.setattr(M, "_current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        bound()
    assert len(calls) == 1
    elsewhere()
    assert len(calls) == 2


def _calls(x):
    """The calls that write a list's tensors, as functions of where their scalars are."""
    return [lambda a: M.tensors_scale(x, a, stream=0), lambda a: M.tensors_clip(x, 1.0, a, P, stream=0),
            lambda a: M.tensors_clip(x, 1.0, P, a, stream=0),
            lambda a: M.bind("mi_tensors_scale", *x.args(), a, stream=0)(),
            lambda a: M.bind("mi_tensors_clip", *x.args(), 1.0, a, P, stream=0)(),
            lambda a: M.bind("mi_tensors_clip", *x.args(), 1.0, P, a, stream=0)()]


@pytest.mark.parametrize("with_outs", [False, True])
def test_scalars_lie_outside_the_list(monkeypatch, with_outs):
    """A scale, norm or clip scale among the elements would be written while others read it."""
    made = []
    for name in CALLS:
        monkeypatch.setattr(M.lib, name, lambda *a: made.append(a) or M.MI_OK)
    outs = [Stand(0x8000, 4), Stand(0x9000, 100)] if with_outs else None
    x = M.TensorList([Stand(0x1000, 4, torch.float16), Stand(0x2000, 100)], outs)
    inside = [0x1000, 0x1004, 0xffe, 0x2000, 0x218c, 0x218e] + [0x8000, 0x918c] * with_outs
    outside = [0xffc, 0x1008, 0x1ffc, 0x2190] + ([0x7ffc, 0x9190] if with_outs else [0x8000])
    for call in _calls(x):
        for a in inside:
            n = len(made)
            with pytest.raises(ValueError, match="scalar"):
                call(a)
            assert len(made) == n
        for a in outside + outside:
            n = len(made)
            call(a)
            assert len(made) == n + 1
