"""What the log probabilities of given tokens refuse (no GPU needed)."""
import pytest
import torch

from herbert_rs_amd.errors import BackendError
from herbert_rs_amd.kernels import lib, ops


@pytest.mark.parametrize("R, V, top, text", [(0, 5, 0, "bad sizes"), (1, 0, 0, "bad sizes"), (1, 5, 6, "bad sizes"), (1, 500, 65, "bad sizes"),
                                             (1, 5, -1, "bad sizes"), (1 << 30, 1 << 20, 0, "too many rows"), (1, 4097, 0, "room"), (1, 5, 2, "no room for 2")])
def test_calls_that_the_entry_refuses(R, V, top, text):
    with pytest.raises(BackendError, match=text):
        lib.call("logprobs", "hb_token_logprobs", None, R, V, None, None, None, None, None, top, None, None, None)


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(BackendError, match="on the GPU"):
        ops.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(2))
