"""The gated linear recurrence on the GPU against 64 bits: rows one by one, packed sequences, gradients."""
import importlib

import pytest

torch = pytest.importorskip("torch")
import gated_oracle as ref  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def gated():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.gated")


def cu_of(lens, first=0):
    return torch.tensor([first, *(first + torch.tensor(lens).cumsum(0)).tolist()], dtype=torch.int32, device="cuda")


class Case:
    """Inputs of `lens` packed sequences; `pad` columns lie between rows, `apart` elements between the states."""

    def __init__(self, channels, lens, gate="decay", input="plain", g=F32, x=BF, pad=0, apart=0, seed=1):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
        self.channels, self.lens, self.rows, self.kinds = channels, lens, sum(lens), {"gate": gate, "input": input}
        wide = lambda t: torch.cat([t, t.new_full((t.shape[0], pad), 7.0)], 1)[:, :channels] if pad else t
        reach = torch.exp2(8 * torch.rand(channels, device="cuda", generator=gen))
        n = max(self.rows, 1)
        self.g = wide((-torch.rand(n, channels, device="cuda", generator=gen) * 2 / reach if gate == "decay" else torch.log(reach) + rn(n, channels)).to(g))
        self.x, self.dout = wide(rn(n, channels).to(x)), wide(rn(n, channels).to(x))
        batch = len(lens)
        self.state, self.dstate = rn(batch, channels), rn(batch, channels)
        self.cu = cu_of(lens)
        self.step = channels + apart
        self.off = torch.arange(batch, dtype=torch.int64, device="cuda").flip(0) * self.step  # the last request's state first

    def arena(self, states):
        t = torch.full((len(self.lens) * self.step,), 9.0, device="cuda")
        for i, o in enumerate(self.off.tolist()):
            t[o:o + self.channels] = states[i]
        return t

    def states(self, arena):
        return torch.stack([arena[o:o + self.channels] for o in self.off.tolist()])

    def like(self, t):
        return torch.full(t.shape, 5.0, dtype=t.dtype, device="cuda")

    def workspace(self, m):
        return torch.full((m.workspace_bytes(self.channels, len(self.lens), self.rows),), 255, dtype=torch.uint8, device="cuda")

    def prefill(self, m, workspace=None, saves=None, **kw):
        out, state = self.like(self.x), self.arena(self.state)
        m.prefill_varlen(self.channels, self.rows, self.cu, max(self.lens, default=0), self.g, self.x, state, self.off, out=out, saves=saves, workspace=workspace,
                         **self.kinds, **kw)
        return out[:self.rows], state

    def saves(self, m):
        return torch.full((m.saves_rows(len(self.lens), self.rows), self.channels), 3.0, device="cuda")

    def backward(self, m, saves, workspace=None, dstate=True):
        dg, dx, ds = self.like(self.g), self.like(self.x), self.arena(torch.zeros_like(self.state))
        m.backward_varlen(self.channels, self.rows, self.cu, max(self.lens, default=0), self.g, self.x, saves, self.off, self.dout, dg, dx,
                          dstate=self.arena(self.dstate) if dstate else None, dstate_in=ds, workspace=workspace, **self.kinds)
        return dg[:self.rows], dx[:self.rows], ds


SHAPES = [(1, [1]), (64, [128]), (65, [127, 0, 129]), (2, [0]), (200, [300, 65, 1, 0]), (63, [700]), (130, [5, 64, 63, 256, 257]), (1024, [100])]


@pytest.mark.parametrize("channels,lens", SHAPES, ids=lambda v: str(v).replace(" ", ""))
@pytest.mark.parametrize("gate,input", [("decay", "plain"), ("decay", "complement"), ("sigmoid", "plain"), ("sigmoid", "complement")])
@pytest.mark.parametrize("g,x,pad", [(F32, BF, 0), (BF, BF, 3), (BF, F32, 2), (F32, F32, 1)], ids=["f32-bf16", "bf16-bf16-odd", "bf16-f32-even", "f32-f32-odd"])
def test_sequences_and_gradients(gated, channels, lens, gate, input, g, x, pad):
    c = Case(channels, lens, gate, input, g, x, pad, apart=3)
    n = c.rows
    h, hb, end, endb = ref.forward(lens, c.g[:n], c.x[:n], c.state, gate, input)
    results = []
    for ws in (None, c.workspace(gated)):
        saves = c.saves(gated)
        out, state = c.prefill(gated, ws, saves)
        ref.close(out, h, hb, "out")
        ref.close(c.states(state), end, endb, "state")
        assert (state.view(len(lens), -1)[:, channels:] == 9).all()
        grads = c.backward(gated, saves, ws)
        for got, want, name in zip((*grads[:2], c.states(grads[2])), ref.backward(lens, c.g[:n], c.x[:n], c.state, c.dout[:n], c.dstate, gate, input), ("dg", "dx", "ds")):
            ref.close(got, *want, name)
        results.append((out, state, *grads))
    for a, b in zip(*results):  # the workspace changes no bit
        assert torch.equal(a, b)
    assert importlib.import_module("glm53f-afd_b200.core").device_status() == 0


@pytest.mark.parametrize("gate,input", [("decay", "plain"), ("sigmoid", "complement")])
def test_long_sequences_in_parts(gated, gate, input):
    """Many tiles a sequence, more than a look reaches; the same bits alone, beside others and a second time."""
    lens = [5000, 1, 9000, 4097]
    c = Case(192, lens, gate, input, F32, F32, seed=3)
    saves = c.saves(gated)
    out, state = c.prefill(gated, c.workspace(gated), saves)
    grads = c.backward(gated, saves, c.workspace(gated))
    h, hb, end, endb = ref.forward(lens, c.g, c.x, c.state, gate, input)
    ref.close(out, h, hb)
    ref.close(c.states(state), end, endb)
    for got, want in zip((*grads[:2], c.states(grads[2])), ref.backward(lens, c.g, c.x, c.state, c.dout, c.dstate, gate, input)):
        ref.close(got, *want)
    again = c.prefill(gated, c.workspace(gated), saves)
    assert torch.equal(again[0], out) and torch.equal(again[1], state)
    first = 0
    for i, n in enumerate(lens):
        alone, s = torch.empty_like(c.x[:n]), c.state[i].clone()
        gated.prefill_varlen(192, n, cu_of([n]), n, c.g[first:first + n], c.x[first:first + n], s, torch.zeros(1, dtype=torch.int64, device="cuda"), out=alone, **c.kinds)
        assert torch.equal(alone, out[first:first + n]) and torch.equal(s, c.states(state)[i])
        first += n


def test_gradients_against_differences(gated):
    """sum(w out) + sum(v end) moves by the gradients along a direction; in f32 types, by central differences of the 64-bit recurrence."""
    for gate, input in (("decay", "plain"), ("decay", "complement"), ("sigmoid", "plain"), ("sigmoid", "complement")):
        lens = [130, 70]
        c = Case(40, lens, gate, input, F32, F32, seed=4)
        saves = c.saves(gated)
        c.prefill(gated, None, saves)
        dg, dx, ds = c.backward(gated, saves)
        gen = torch.Generator(device="cuda").manual_seed(9)
        move = [torch.randn(t.shape, device="cuda", generator=gen, dtype=torch.float64) for t in (c.g, c.x, c.state)]

        def loss(eps):
            h, _, end, _ = ref.forward(lens, c.g.double() + eps * move[0], c.x.double() + eps * move[1], c.state.double() + eps * move[2], gate, input)
            return (h * c.dout.double()).sum() + (end * c.dstate.double()).sum()

        eps = 1e-5
        want = float((loss(eps) - loss(-eps)) / (2 * eps))
        parts = [(a.double() * b) for a, b in zip((dg, dx, c.states(ds)), move)]
        got = float(sum(p.sum() for p in parts))
        # Third derivatives times eps^2, and the f32 gradients' roundings: 200 steps at most, so 2000 u of the absolute sum.
        assert abs(got - want) <= 2000 * ref.U * float(sum(p.abs().sum() for p in parts)) + 1e-5 * abs(want)


def test_no_gradient_of_the_end_states(gated):
    c = Case(66, [130, 3], "sigmoid", "complement", BF, BF)
    saves = c.saves(gated)
    c.prefill(gated, None, saves)
    dg, dx, ds = c.backward(gated, saves, dstate=False)
    for got, want in zip((dg, dx, c.states(ds)), ref.backward(c.lens, c.g, c.x, c.state, c.dout, None, "sigmoid", "complement")):
        ref.close(got, *want)
    a, b = torch.empty_like(dg), torch.empty_like(dx)
    both = c.arena(c.dstate)
    gated.backward_varlen(66, c.rows, c.cu, 130, c.g, c.x, saves, c.off, c.dout, a, b, dstate=both, dstate_in=both, workspace=c.workspace(gated), **c.kinds)  # in place
    assert torch.equal(both, c.backward(gated, saves)[2])
    gated.backward_varlen(66, c.rows, c.cu, 130, c.g, c.x, saves, c.off, c.dout, a, b, workspace=c.workspace(gated), **c.kinds)
    assert torch.equal(a, dg) and torch.equal(b, dx)


@pytest.mark.parametrize("channels,lens", [(1, [1]), (64, [1] * 48), (257, [1, 8, 0, 3]), (4096, [17])], ids=lambda v: str(v).replace(" ", "")[:20])
@pytest.mark.parametrize("gate,input,g,x,pad", [("decay", "plain", F32, BF, 0), ("sigmoid", "complement", BF, BF, 1), ("decay", "complement", BF, F32, 2), ("sigmoid", "plain", F32, F32, 0)])
def test_row_by_row(gated, channels, lens, gate, input, g, x, pad):
    c = Case(channels, lens, gate, input, g, x, pad, apart=1)
    h, hb, end, endb = ref.forward(lens, c.g[:c.rows], c.x[:c.rows], c.state, gate, input)
    arena, out = c.arena(c.state), c.like(c.x)
    args = (channels, c.rows, c.cu, c.g, c.x)
    before = arena.clone()
    gated.decode_batch(*args, arena, c.off, out=out, state_out=None, **c.kinds)  # a verify
    assert torch.equal(arena, before)
    ref.close(out[:c.rows], h, hb)
    keep = torch.tensor([(3 * i + 1) % (n + 2) for i, n in enumerate(lens)], dtype=torch.int32, device="cuda")  # (some beyond the window)
    gated.decode_batch(*args, arena, c.off, keep=keep, **c.kinds)  # a commit
    serial = before.clone()
    for t in range(max(lens)):  # single rows
        live = [i for i, n in enumerate(lens) if t < min(n, int(keep[i]))]
        for i in live:
            row = sum(lens[:i]) + t
            one = torch.empty_like(c.x[:1])
            gated.decode_batch(channels, 1, cu_of([1]), c.g[row:row + 1], c.x[row:row + 1], serial, c.off[i:i + 1], out=one, **c.kinds)
            assert torch.equal(one[0], out[row])
    assert torch.equal(serial, arena)
    arena = c.arena(c.state)
    other = torch.zeros_like(arena)
    gated.decode_batch(*args, arena, c.off, state_out=other, **c.kinds)
    ref.close(c.states(other), end, endb)


def test_gates_at_their_ends(gated):
    """A decay of -inf and a sigmoid at its ends forget or keep exactly; what a row holds reaches no row before it and no other channel."""
    n, ch = 200, 64
    c = Case(ch, [n], "decay", "complement", F32, F32)
    c.g[50] = -float("inf")
    c.g[120, 3] = 0.0
    out, _ = c.prefill(gated, c.workspace(gated))
    h, hb, *_ = ref.forward([n], c.g, c.x, c.state, "decay", "complement")
    assert torch.equal(out[50], c.x[50]) and h[120, 3] == h[119, 3]
    # (Row 120 begins a thread's eight rows: its state comes from the composition of the rows before it, row 119's from the rows one by one.  Each is within
    # its bound of the same value, so they are within the two bounds' sum of one another.)
    assert (out[120, 3].double() - out[119, 3].double()).abs() <= hb[119, 3] + hb[120, 3]
    for gate in ("decay", "sigmoid"):
        c = Case(ch, [n], gate, "plain", F32, F32)
        clean, _ = c.prefill(gated, c.workspace(gated))
        c.x[130, 5], c.g[131, 7] = float("nan"), float("nan")
        out, state = c.prefill(gated, c.workspace(gated))
        assert out[130:, 5].isnan().all() and out[131:, 7].isnan().all() and torch.equal(out[:130], clean[:130])
        rest = [i for i in range(ch) if i not in (5, 7)]
        assert torch.equal(out[:, rest], clean[:, rest])
    c = Case(ch, [n], "sigmoid", "complement", F32, F32)
    c.g[10], c.g[20] = float("inf"), -float("inf")
    out, _ = c.prefill(gated, None)
    assert torch.equal(out[10], out[9]) and torch.equal(out[20], c.x[20])
    c = Case(ch, [n], "sigmoid", "complement", F32, F32)
    c.g[::3], c.g[1::3] = 100.0, -100.0  # (e^-100 is a subnormal number's)
    out, _ = c.prefill(gated, None)
    h, hb, *_ = ref.forward([n], c.g, c.x, c.state, "sigmoid", "complement")
    assert ((out.double() - h).abs() <= hb + ref.half_step(h, F32) + 1e-37).all()


def test_rows_of_no_request(gated):
    """Rows before the first and behind the last request are left as they are, whatever they hold."""
    c = Case(70, [150, 40], "sigmoid", "complement", BF, BF)
    for t in (c.g, c.x, c.dout):
        t[:10], t[140:] = float("nan"), float("nan")
    cu, off = cu_of([100, 0, 30], 10), torch.arange(3, dtype=torch.int64, device="cuda") * 70
    state = torch.randn(3, 70, device="cuda")
    start = state.clone()
    out, dg, dx = (torch.full((190, 70), 5.0, dtype=BF, device="cuda") for _ in range(3))
    saves = torch.empty(gated.saves_rows(3, 190), 70, device="cuda")
    ws = c.workspace(gated)
    kw = dict(gate="sigmoid", input="complement", workspace=torch.empty(gated.workspace_bytes(70, 3, 190), dtype=torch.uint8, device="cuda"))
    gated.prefill_varlen(70, 190, cu, 100, c.g, c.x, state, off, out=out, saves=saves, **kw)
    gated.backward_varlen(70, 190, cu, 100, c.g, c.x, saves, off, c.dout, dg, dx, **kw)
    for t in (out, dg, dx):
        assert (t[:10] == 5).all() and (t[140:] == 5).all() and not t[10:140].isnan().any()
    h, hb, end, endb = ref.forward([100, 0, 30], c.g[10:140], c.x[10:140], start, "sigmoid", "complement")
    ref.close(out[10:140], h, hb)
    ref.close(state, end, endb)


def test_many_requests(gated):
    """More requests than a look among them takes in one step."""
    gen = torch.Generator().manual_seed(2)
    lens = (torch.randint(0, 40, (1500,), generator=gen) ** 2 // 40).tolist()
    lens[700] = 300
    c = Case(6, lens, "decay", "plain", F32, F32)
    out, state = c.prefill(gated, c.workspace(gated))
    apart, s = c.prefill(gated, None)
    assert torch.equal(out, apart) and torch.equal(state, s)
    first = sum(lens[:700])
    h, hb, *_ = ref.forward([300], c.g[first:first + 300], c.x[first:first + 300], c.state[700:701], "decay", "plain")
    ref.close(out[first:first + 300], h, hb)


def test_streams_and_graphs(gated):
    """Two graphs with workspaces of their own replayed at once, and calls on two streams."""
    cases = [Case(320, [3000, 40], "sigmoid", "complement", BF, BF, seed=s) for s in (1, 2)]
    want = [c.prefill(gated, c.workspace(gated)) for c in cases]
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        out, state, ws = torch.zeros_like(c.x), c.arena(c.state), c.workspace(gated)
        start = state.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            state.copy_(start)
            gated.prefill_varlen(c.channels, c.rows, c.cu, 3000, c.g, c.x, state, c.off, out=out, workspace=ws, **c.kinds)
        graphs.append((g, out, state, ws, start))
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for s, (g, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (g, out, state, *_), (w_out, w_state) in zip(graphs, want):
        assert torch.equal(out, w_out) and torch.equal(state, w_state)
