"""The status word of a device's products, made by the code that makes it: torch's device functions are replaced, the word
lies on the CPU."""
import pytest
import torch


@pytest.fixture
def words(monkeypatch):
    """(the module, words handed to the compiled front)"""
    from lightcompress_b200 import int8_linear as il
    handed = []

    class Stream:
        def synchronize(self):
            pass

    class Front:
        def set_status(self, dev, at):
            handed.append((dev, at))
    monkeypatch.setattr(il, '_status', {})
    monkeypatch.setattr(il, '_calls', Front())
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda d=None: Stream())
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda d=None: None)
    return il, handed


def _expire(il):
    from lightcompress_b200 import _lib as L
    with torch.inference_mode(il._status[0].is_inference()):
        il._status[0].fill_(L.LC_ERR_TIMEOUT)


@pytest.mark.parametrize('mode', [torch.inference_mode, torch.no_grad, torch.enable_grad])
def test_an_expired_wait_is_reported_once_whatever_mode_the_word_was_made_in(words, mode):
    from lightcompress_b200 import _lib as L
    il, handed = words
    with mode():
        at = il._status_of(torch.zeros(1), 0)
        assert il._status_of(torch.zeros(1), 0) == at != 0
    assert handed == [(0, at)]
    il.check_status(0)
    for check_mode in (torch.enable_grad, torch.inference_mode):
        _expire(il)
        with check_mode():
            with pytest.raises(L.LcError, match='timed out'):
                il.check_status(0)
            il.check_status(0)                        # and cleared


def test_no_word_is_made_inside_a_capture_or_without_a_device(words, monkeypatch):
    il, handed = words
    assert il._status_of(torch.zeros(1), -1) == 0
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    assert il._status_of(torch.zeros(1), 0) == 0 and not handed


def test_threads_that_come_first_together_share_one_word(words, monkeypatch):
    """Kernels launched by one thread may not keep the address of a word that another thread's replaces."""
    import threading
    il, handed = words
    together = threading.Barrier(4)

    class Slow:
        def synchronize(self):
            threading.Event().wait(0.2)               # lets the other threads run, as torch's does
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda d=None: Slow())
    got = []

    def first():
        together.wait()
        got.append(il._status_of(torch.zeros(1), 0))
    threads = [threading.Thread(target=first) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and set(got) == {il._status[0].data_ptr()} and handed == [(0, got[0])]
