"""The bounded waits of the bf16, tf32 and fp8 tensor-core kernels' finishing warps."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_warp_takes_one_way_out_of_a_wait():
    """Lanes that see different outcomes agree that the wait failed, as they do once any role has given up."""
    from lightcompress_b200 import _lib as L
    answers = torch.full((3,), 7, dtype=torch.int32, device='cuda')
    L.launch(0, 'lc_selftest_warp_wait', answers.data_ptr())
    torch.cuda.synchronize()
    assert answers.tolist() == [0, 0, -1]
    assert float((torch.ones(8, device='cuda') * 2).sum()) == 16.0
    assert L.lib.lc_selftest_warp_wait(None, None) == L.LC_ERR_ARG
