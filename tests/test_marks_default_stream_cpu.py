"""A pool on the legacy default stream, whose address is 0, while torch's current stream is another: its copies come after the current stream's work, on the stream
that was given (torch makes a new one of that address).  Against the fake of torch's streams.  No GPU."""
import importlib
import types

import pytest

from test_verify_accept_default_stream_cpu import WithDefault

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("address", [0, 1, 7])
@pytest.mark.parametrize("torchs_own", [True, False])
def test_copies_follow_the_current_stream(pkg, monkeypatch, address, torchs_own):
    kernel, marks = (importlib.import_module("glm53f-afd_b200." + n) for n in ("kernel", "marks"))
    monkeypatch.setattr(kernel, "DEVICE", "cpu")
    pool = marks.KvPool(marks.KvConfig(marks.KvLayout.new(1, 0), 2, 2))
    cuda = WithDefault()
    monkeypatch.setattr(kernel, "_torch", lambda: types.SimpleNamespace(cuda=cuda))
    pool.stream = kernel.Stream(cuda.Stream(address) if torchs_own else type("Other", (), {"cuda_stream": address})())
    pool._after_current()
    assert cuda.log == ([] if address == 1 else [("wait", address, 1)])
