"""Several operands checked at once, and tensors handed to C entry points as their memory."""
import pytest
import torch

from herbert_rs_amd.errors import BackendError
from herbert_rs_amd.kernels import lib, ops


def test_operands_off_the_gpu_or_no_tensors_are_refused_by_name():
    all_fit = lib.host().all_fit
    assert all_fit() == -1 and all_fit(torch.zeros(3), None, None) == -1 and all_fit(None, None, None) == -1
    with pytest.raises(TypeError, match="are needed"):
        all_fit(torch.zeros(3), None)
    for wrong in (torch.zeros(2), None, 7):
        with pytest.raises(BackendError, match="first must be a tensor on the GPU"):
            ops._check_all("kernel", ("first", "second"), wrong, torch.float32, (2,), torch.zeros(2), None, None)


@pytest.mark.gpu
def test_operands_are_checked_together():
    a, b = torch.zeros(3, 4, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    assert lib.host().all_fit(a, torch.float32, (3, None), b, torch.int32, None) == a.get_device()
    ops._check_all("kernel", ("a", "b"), a, torch.float32, (3, 4), b, None, (5,))
    for bad, text in (((a, torch.float32, (3, 5), b, None, (5,)), "a must have shape"), ((a, None, (3, 4), b, torch.float32, (5,)), "b must be torch.float32"),
                      ((a.t(), None, None, b, None, None), "a must be contiguous"), ((a, None, None, b.cpu(), None, None), "b must be a tensor on the GPU")):
        with pytest.raises(BackendError, match=text):
            ops._check_all("kernel", ("a", "b"), *bad)


@pytest.mark.gpu
def test_an_entry_point_takes_a_tensor_for_its_memory():
    x = torch.ones(1000, device="cuda")
    lib.call("elementwise", "hb_scale", x, 2.0, x.numel(), ops._stream())
    lib.call("elementwise", "hb_scale", x.data_ptr(), 3.0, x.numel(), ops._stream())
    assert (x == 6).all()
    with pytest.raises(TypeError, match="no memory"):
        lib.call("elementwise", "hb_scale", x.to_sparse(), 2.0, x.numel(), ops._stream())
