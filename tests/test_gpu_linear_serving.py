"""A decoder layer with linear attention as it is served: fused projections, prefill, windows of drafted tokens, their verification and the
commit of what is kept.  And the same verification in a round of the KDA layers."""
import importlib

import pytest

from test_gpu_accept import rule

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HIDDEN, HEADS, QK, VOCAB, PER = 256, 4, 2, 1000, 128 * 128


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return {n: importlib.import_module("glm53f-afd_b200." + n) for n in ("kernel", "marks", "verify", "core", "linear", "spec", "proj")}


class Layer:
    """h = x + W_o y with y the linear attention of W_qkv x + b; logits = W_v silu(h W_u)."""

    def __init__(self, m, dtype, seed):
        self.m, gen = m, torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)
        mat = lambda n, k: m["proj"].Bf16Mat.dense((rn(n, k) * k ** -0.5).bfloat16())
        width = (2 * QK + HEADS) * 128
        self.qkv, self.o, self.up, self.head = mat(width, HIDDEN), mat(HIDDEN, HEADS * 128), mat(512, HIDDEN), mat(VOCAB, 512)
        self.bias = rn(width) * 0.1
        self.dtype = dtype

    def buffers(self, rows):
        z = lambda n, t=torch.bfloat16: torch.zeros(rows, n, dtype=t, device="cuda")
        return {"qkv": z((2 * QK + HEADS) * 128), "y": z(HEADS * 128), "h": z(HIDDEN), "up": z(512), "logits": z(VOCAB, torch.float32)}

    def parts(self, b):
        at, out = 0, []
        for n in (QK, QK, HEADS):
            out.append(b["qkv"][:, at:at + n * 128])
            at += n * 128
        return out

    def project_in(self, x, b):
        rows = x.shape[0]
        self.m["proj"].fused(x, HIDDEN, 0, self.qkv, rows, b["qkv"], b["qkv"].shape[1], 0, bias=self.bias)

    def project_out(self, x, b):
        p, rows = self.m["proj"], x.shape[0]
        p.fused(b["y"], HEADS * 128, 0, self.o, rows, b["h"], HIDDEN, 0, residual=x)
        p.fused(b["h"], HIDDEN, 0, self.up, rows, b["up"], 512, 0, activation="silu")
        p.bf16(b["up"], 512, 0, self.head, rows, b["logits"], VOCAB, 0, out_f32=True)


def cu_of(lens):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_windows_acceptance_commit(mods, dtype):
    lin, spec = mods["linear"], mods["spec"]
    layer = Layer(mods, dtype, 5)
    gen = torch.Generator(device="cuda").manual_seed(6)
    rn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)
    prompts, windows = [70, 200, 3], [4, 8, 1]
    slots = torch.tensor([2, 0, 3], device="cuda") * (HEADS * PER)
    state = torch.zeros(4, HEADS, 128, 128, dtype=dtype, device="cuda")

    # the prompts
    rows = sum(prompts)
    x, g = rn(rows, HIDDEN).bfloat16(), -torch.rand(rows, HEADS, device="cuda", generator=gen) * 0.1
    b = layer.buffers(rows)
    layer.project_in(x, b)
    ws = torch.empty(max(16, lin.prefill_workspace_bytes(HEADS, len(prompts), max(prompts))), dtype=torch.uint8, device="cuda")
    lin.prefill_varlen(HEADS, rows, cu_of(prompts), max(prompts), *layer.parts(b), g, state, slots, qk_heads=QK, out=b["y"], workspace=ws)
    layer.project_out(x, b)
    assert (state[1] == 0).all() and (state[2] != 0).any()
    after_prompts = state.clone()

    # a round: verify, judge, commit, captured as a server would
    rows, cu = sum(windows), cu_of(windows)
    x, g = rn(rows, HIDDEN).bfloat16(), -torch.rand(rows, HEADS, device="cuda", generator=gen) * 0.1
    b, u = layer.buffers(rows), torch.rand(rows, device="cuda", generator=gen) * 0.999
    tokens, heat = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.tensor([0.0, 0.2, 1.0], device="cuda")
    keep, nxt = torch.full((3,), -7, dtype=torch.int32, device="cuda"), torch.full((3,), -7, dtype=torch.int32, device="cuda")

    def one_round():
        layer.project_in(x, b)
        lin.decode_batch(HEADS, rows, cu, *layer.parts(b), g, state, slots, qk_heads=QK, state_out=None, out=b["y"])
        layer.project_out(x, b)
        spec.accept_batch(cu, tokens, b["logits"], u, keep, nxt, temperature=heat)
        lin.decode_batch(HEADS, rows, cu, *layer.parts(b), g, state, slots, qk_heads=QK, keep=keep)

    one_round()
    best = b["logits"].argmax(-1).int()
    tokens[1:] = best[:-1]  # what the target itself would choose
    tokens[3] = (best[2] + 1) % VOCAB  # but the last of the first window
    state.copy_(after_prompts)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        one_round()
    side.synchronize()
    eager = [t.clone() for t in (state, b["h"], keep, nxt)]
    graph = torch.cuda.CUDAGraph()
    state.copy_(after_prompts)
    with torch.cuda.graph(graph):
        one_round()
    for _ in range(2):
        state.copy_(after_prompts)
        keep.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got, want) for got, want in zip((state, b["h"], keep, nxt), eager))
    assert mods["core"].device_status() == 0
    want_keep, want_next = rule(windows, tokens, b["logits"], u, False, None, heat)
    assert keep.tolist() == want_keep and nxt.tolist() == want_next
    assert keep.tolist()[0] == 3 and keep.tolist()[2] == 1

    # the kept rows one token at a time: the same bits of states and rows
    serial, first = after_prompts.clone(), 0
    for i, n in enumerate(windows):
        for t in range(first, first + int(keep[i])):
            bt = layer.buffers(1)
            layer.project_in(x[t:t + 1], bt)
            lin.decode_batch(HEADS, 1, cu_of([1]), *layer.parts(bt), g[t:t + 1], serial, slots[i:i + 1], qk_heads=QK, out=bt["y"])
            layer.project_out(x[t:t + 1], bt)
            assert torch.equal(bt["h"], b["h"][t:t + 1])
        first += n
    assert torch.equal(serial, state)


def test_a_round_of_the_kda_layers_is_judged(mods):
    K, marks, verify = mods["kernel"], mods["marks"], mods["verify"]
    gen = torch.Generator(device="cuda").manual_seed(4)
    rn = lambda n, s=1.0, d=torch.bfloat16: (torch.randn(n, device="cuda", generator=gen) * s).to(d)
    buf = lambda t: K.DeviceBuffer(t.view(torch.uint8))
    h, windows = marks.KDA_HEADS, [5, 2]
    c, width, rows = K.channels(h), h * 128, sum(windows)
    w = K.Weights(h, buf(rn(c * 4, 0.5)), buf(rn(h, 0.5, torch.float32)), buf(rn(width, 1.0, torch.float32)), buf(1 + rn(128, 0.1)), 1e-5, -5.0)
    projected, gates = rn(rows * verify.KDA_P_COLS), rn(rows * width)
    target, u = torch.randn(rows, 777, device="cuda", generator=gen), torch.rand(rows, device="cuda", generator=gen) * 0.999
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    tokens[1:] = target.argmax(-1)[:-1].int()
    tokens[3] += 1 if int(tokens[3]) < 776 else -1
    greedy = torch.zeros(2, device="cuda")
    want = rule(windows, tokens, target, u, False, None, greedy)
    states = []
    for stream in (None, K.Stream(torch.cuda.Stream())):
        pool = marks.KvPool(marks.KvConfig(marks.KvLayout.new(1, 0), 2, 2))
        slots = [pool.slot(), pool.slot()]
        vf = verify.KdaVerify(pool, [w], 8, 4)
        vf.verify(list(zip(slots, windows)))
        vf.v.p.upload_at(0, projected.cpu().view(torch.int16).numpy().view("uint16"))
        out = K.RowView.dense(K.DeviceBuffer.zeroed(rows * width * 2), width)
        rv = K.RowView.dense(buf(gates), width)
        torch.cuda.synchronize()
        vf.layer(0, rv, rv, out, stream)
        keep, nxt = (torch.full((2,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        vf.accept(tokens, target, u, keep, nxt, temperature=greedy, stream=stream)
        if stream is not None:
            stream.synchronize()
        assert (keep.tolist(), nxt.tolist()) == want and want[0] == [3, 2]
        vf.commit(slots, keep.tolist(), stream)
        torch.cuda.synchronize()
        assert [s.tokens() for s in slots] == [3, 2]
        states.append(pool.state.t.clone())
    assert mods["core"].device_status() == 0 and torch.equal(*states)
