"""The order of `KdaVerify.accept` between torch's current stream, where its inputs are made and its answers are read, and the stream that it launches on: against a
fake of torch's streams.  No GPU."""
import contextlib
import importlib
import types

import pytest

torch = pytest.importorskip("torch")


class Streams:
    """torch.cuda's streams: which one is the current one, which are being captured, and what was asked of them in order."""

    def __init__(self):
        self.log, self.captured, fake = [], set(), self

        class Stream:
            def __init__(self, address):
                self.cuda_stream = address

            def wait_stream(self, other):
                fake.log.append(("wait", self.cuda_stream, other.cuda_stream))
                # (an event of a stream outside a capture cannot be waited for inside it; the other way round the waiting stream joins)
                assert not (self.cuda_stream in fake.captured and other.cuda_stream not in fake.captured)
                if other.cuda_stream in fake.captured:
                    fake.captured.add(self.cuda_stream)

            def synchronize(self):
                raise AssertionError("the host waits")

        self.ExternalStream = self.Stream = Stream
        self.at = Stream(1)

    def current_stream(self):
        return self.at

    def is_current_stream_capturing(self):
        return self.at.cuda_stream in self.captured

    @contextlib.contextmanager
    def stream(self, s):
        before, self.at = self.at, s
        yield
        self.at = before

    def synchronize(self):
        raise AssertionError("the host waits")


@pytest.fixture()
def round_of(pkg, monkeypatch):
    kernel, marks, verify = (importlib.import_module("glm53f-afd_b200." + n) for n in ("kernel", "marks", "verify"))
    monkeypatch.setattr(kernel, "DEVICE", "cpu")

    def make(pool_stream=None):
        cuda = Streams()
        monkeypatch.setattr(kernel, "_torch", lambda: torch)
        pool = marks.KvPool(marks.KvConfig(marks.KvLayout.new(1, 0), 2, 2))
        vf = verify.KdaVerify(pool, [None], 8, 2)
        vf.verify([(pool.slot(), 2), (pool.slot(), 4)])
        pool.stream = kernel.Stream(None if pool_stream is None else cuda.Stream(pool_stream))
        monkeypatch.setattr(kernel, "_torch", lambda: types.SimpleNamespace(cuda=cuda, int32=torch.int32))
        monkeypatch.setattr(verify.spec, "accept_batch", lambda *a, **kw: cuda.log.append(("launch", cuda.at.cuda_stream)))
        one = torch.zeros(2, dtype=torch.int32)
        return cuda, lambda **kw: vf.accept(torch.zeros(6, dtype=torch.int32), torch.zeros(6, 9), torch.zeros(6), one, one, **kw)

    return make


BOTH = [("wait", 7, 1), ("launch", 7), ("wait", 1, 7)]  # behind the inputs, and the answers behind it


def test_on_the_current_stream_nothing_waits(round_of):
    cuda, accept = round_of()
    accept()
    assert cuda.log == [("launch", 1)]
    cuda, accept = round_of(1)
    accept()
    assert cuda.log == [("launch", 1)]


def test_on_the_pools_own_stream(round_of):
    cuda, accept = round_of(7)
    accept()
    assert cuda.log == BOTH and cuda.at.cuda_stream == 1


def test_on_a_given_stream(round_of):
    cuda, accept = round_of()
    accept(stream=importlib.import_module("glm53f-afd_b200.kernel").Stream(cuda.Stream(7)))
    assert cuda.log == BOTH


def test_captured(round_of):
    cuda, accept = round_of(7)
    cuda.captured = {1}  # the launch's stream joins the capture and hands it back
    accept()
    assert cuda.log == BOTH and cuda.captured == {1, 7}
    cuda, accept = round_of(7)
    cuda.captured = {7}  # a capture that the current stream has no part in: the order is the captured one
    accept()
    assert cuda.log == [("launch", 7)] and cuda.captured == {7}
