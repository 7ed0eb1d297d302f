"""The products' status word on the host: one word a device whatever threads
ask first, and no report lost between a check and the work after it."""

import threading
import time

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def quant(monkeypatch):
    """The module with an empty table and a device that needs no CUDA."""
    from rns8_b200 import quant

    class Stream:
        def synchronize(self):
            pass

    monkeypatch.setattr(quant, "_status", {})
    monkeypatch.setattr(quant.torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(quant.torch.cuda, "current_stream", lambda device: Stream())
    return quant


def test_one_word_for_threads_that_ask_at_once(quant, monkeypatch):
    zeros, made = torch.zeros, []

    def slow_zeros(*size, dtype, device):
        word = zeros(*size, dtype=dtype)
        made.append(word)
        time.sleep(0.05)  # an allocation releases the interpreter's lock
        return word

    monkeypatch.setattr(quant.torch, "zeros", slow_zeros)
    start, got = threading.Barrier(4), [None] * 4

    def ask(i):
        start.wait()
        got[i] = quant.device_status(3)

    threads = [threading.Thread(target=ask, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and all(w is made[0] for w in got)


def test_check_clears_the_word_before_it_returns(quant, monkeypatch):
    """The word is cleared on the GPU, in the order of one stream; a product on
    another stream may report as soon as the check is over."""
    did = []

    class Word:
        def item(self):
            did.append("read")
            return 0x100

        def zero_(self):
            did.append("clear")

    monkeypatch.setitem(quant._status, 0, Word())
    monkeypatch.setattr(quant.torch.cuda, "synchronize", lambda device: did.append("synchronize"))
    with pytest.raises(RuntimeError, match="0x100"):
        quant.check_status(0)
    assert did == ["synchronize", "read", "clear", "synchronize"]
