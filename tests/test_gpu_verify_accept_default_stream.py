"""A round judged on the legacy default stream, given by name, while torch's current stream is another one that is still about to write the inputs."""
import importlib

import pytest

from test_gpu_accept import rule

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_inputs_and_answers_are_waited_for():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    K, marks, verify = (importlib.import_module("glm53f-afd_b200." + n) for n in ("kernel", "marks", "verify"))
    default = torch.cuda.default_stream()
    assert K.torch_stream(K.Stream(default)).cuda_stream == default.cuda_stream
    assert K.torch_stream(K.Stream(type("Other", (), {"cuda_stream": default.cuda_stream})())).cuda_stream == default.cuda_stream
    windows, vocab = [4, 3], 501
    gen = torch.Generator().manual_seed(9)
    rows = sum(windows)
    target, u, greedy = torch.randn(rows, vocab, generator=gen), torch.rand(rows, generator=gen), torch.zeros(2)
    tokens = target.argmax(-1).int().roll(1)
    tokens[2] = (int(tokens[2]) + 1) % vocab
    want = rule(windows, tokens, target, u, False, None, greedy)
    pool = marks.KvPool(marks.KvConfig(marks.KvLayout.new(1, 0), 2, 2), K.Stream(default))
    vf = verify.KdaVerify(pool, [None], 8, 4)
    made = [t.cuda() for t in (tokens, target, u, greedy)]
    given = [torch.zeros_like(t) for t in made]
    keep, nxt = (torch.full((2,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    vf.verify([(pool.slot(), n) for n in windows])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(20_000_000)  # about 10 ms
        for a, b in zip(given, made):
            a.copy_(b)
        vf.accept(*given[:3], keep, nxt, temperature=given[3])
        kept, after = keep.clone().tolist(), nxt.clone().tolist()
    assert (kept, after) == want and want[0] == [2, 3]
