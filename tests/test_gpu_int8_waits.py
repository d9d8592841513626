"""The bounded waits of the int8 products: nothing here makes a product wait; a kernel of its own does."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_warp_takes_one_way_out_of_a_wait():
    """Lanes that see different outcomes agree that the wait failed; the context stays usable."""
    from lightcompress_b200 import _lib as L
    status = torch.zeros(2, dtype=torch.int32, device='cuda')
    answers = torch.full((3,), 7, dtype=torch.int32, device='cuda')
    L.launch(0, 'lc_selftest_int8_wait', status.data_ptr(), answers.data_ptr())
    torch.cuda.synchronize()
    assert answers.tolist() == [0, -1, 0]
    assert int(status[0]) == L.LC_ERR_TIMEOUT
    assert float((torch.ones(8, device='cuda') * 2).sum()) == 16.0


def test_wait_selftest_refusals():
    from lightcompress_b200 import _lib as L
    assert L.lib.lc_selftest_int8_wait(None, None, None) == L.LC_ERR_ARG


def test_a_wait_that_runs_out_in_any_thread_is_reported():
    """The thread that reports has found what it waited for; another one's wait has run out."""
    from lightcompress_b200 import _lib as L
    status = torch.zeros(2, dtype=torch.int32, device='cuda')
    answers = torch.zeros(3, dtype=torch.int32, device='cuda')
    L.launch(0, 'lc_selftest_int8_wait', status.data_ptr(), answers.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [L.LC_ERR_TIMEOUT] * 2
