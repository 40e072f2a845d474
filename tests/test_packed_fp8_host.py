"""CPU: when fp8.PackedFp8 packs a weight again, and in which order, on stand-ins of the packing and of the device's calls."""
import pytest
import torch

from flash_diffusion_amd import fp8, ops


class _Packed:
    """what the stand-in packing returns: a copy of the weight's values"""

    def __init__(self, w, into):
        self.N, self.K = w.shape
        self.codes, self.codes_t, self.was = torch.zeros(1), None, w.clone()
        self.into = into


@pytest.fixture
def calls(monkeypatch):
    """the calls that a PackedFp8 makes, in order"""
    seen = []

    class Stream:
        def synchronize(self):
            seen.append("stream done")

    stream = Stream()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: seen.append("device done"))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    monkeypatch.setattr(ops, "pack_weight_fp8", lambda w, transposed=False, into=None: (seen.append("pack"), _Packed(w, into))[1])
    return seen


def _holds(p, w):
    got = p(w)
    return torch.equal(got.was, w.detach()) and p(w) is got


def test_a_transposed_data_is_another_weight(calls):
    w = torch.nn.Parameter(torch.randn(6, 6))
    p = fp8.PackedFp8()
    assert _holds(p, w)
    w.data = w.data.t()                       # the same version, address, type and shape
    assert _holds(p, w)


def test_data_at_the_address_of_data_that_was_freed_is_another_weight(calls):
    memory = bytearray(4 * 36)                # what an allocator hands out a second time

    def fresh(value):
        t = torch.frombuffer(memory, dtype=torch.float32).view(6, 6)
        t.numpy()[:] = value                  # (before the parameter holds it, and not counted as a write to it)
        return t

    w = torch.nn.Parameter(torch.zeros(6, 6))
    w.data = fresh(1.0)
    p = fp8.PackedFp8()
    assert _holds(p, w)
    address = w.data_ptr()
    for value in (2.0, 3.0):
        w.data = torch.zeros(0)
        w.data = fresh(value)
        assert w.data_ptr() == address and _holds(p, w)


def test_an_unchanged_weight_is_packed_once_and_a_written_one_again(calls):
    w = torch.nn.Parameter(torch.randn(5, 7), requires_grad=False)
    p = fp8.PackedFp8()
    for _ in range(3):
        assert _holds(p, w)
    assert calls.count("pack") == 1
    w.mul_(2.0)
    assert _holds(p, w) and calls.count("pack") == 2
    other = torch.nn.Parameter(w.data, requires_grad=False)          # the same memory behind another parameter
    assert _holds(p, other) and calls.count("pack") == 3


def test_packing_has_ended_when_the_call_returns(calls):
    """what reads the codes next need not ask again: a captured graph replayed on another stream waits for nothing of this one"""
    w = torch.nn.Parameter(torch.randn(5, 7), requires_grad=False)
    p = fp8.PackedFp8()
    first = p(w)
    assert calls == ["pack", "stream done"] and first.into is None
    p(w)
    assert calls == ["pack", "stream done"]
    w.mul_(2.0)
    second = p(w)
    assert calls[2:] == ["device done", "pack", "stream done"] and second.into is first     # (readers before, and behind)


def test_two_threads_pack_a_weight_once(calls, monkeypatch):
    import threading
    import time
    plain = ops.pack_weight_fp8
    monkeypatch.setattr(ops, "pack_weight_fp8", lambda *a: (time.sleep(0.05), plain(*a))[1])       # (the other thread comes in)
    w, p = torch.nn.Parameter(torch.randn(5, 7), requires_grad=False), fp8.PackedFp8()
    for turn in (1, 2):
        gate, got = threading.Barrier(2), []

        def work():
            gate.wait()
            got.append(p(w))

        threads = [threading.Thread(target=work) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert calls.count("pack") == turn and got[0] is got[1] and torch.equal(got[0].was, w)
        w.mul_(2.0)
