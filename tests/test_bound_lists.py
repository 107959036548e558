"""CPU checks of lists of tensors in bound calls: what a bound call will read stays alive with it.
The tensors are stand-ins, and no bound call is made."""
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
