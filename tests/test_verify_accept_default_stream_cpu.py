"""`KdaVerify.accept` on the legacy default stream, whose address is 0, while torch's current stream is another: torch makes a new stream of that address.  Against the
fake of torch's streams.  No GPU."""
import importlib

import pytest

from test_verify_accept_streams_cpu import Streams, round_of  # noqa: F401  (the fixture)

pytest.importorskip("torch")


class WithDefault(Streams):
    def __init__(self):
        super().__init__()

        class External(self.Stream):
            def __init__(self, address):
                super().__init__(address or 99)

        self.ExternalStream = External

    def default_stream(self):
        return self.Stream(0)


@pytest.mark.parametrize("torchs_own", [True, False])
@pytest.mark.parametrize("address", [0, 7])
def test_the_stream_that_was_given(round_of, monkeypatch, address, torchs_own):  # noqa: F811
    monkeypatch.setattr(importlib.import_module("test_verify_accept_streams_cpu"), "Streams", WithDefault)
    cuda, accept = round_of()
    given = cuda.Stream(address) if torchs_own else type("Other", (), {"cuda_stream": address})()
    accept(stream=importlib.import_module("glm53f-afd_b200.kernel").Stream(given))
    assert cuda.log == [("wait", address, 1), ("launch", address), ("wait", 1, address)]
