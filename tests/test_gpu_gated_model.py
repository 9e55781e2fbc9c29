"""A small decoder of one gated recurrent layer with 4-bit projections, served and trained: prompts, drafted tokens verified, judged, reported and committed, the same as a captured
round, and the gradients of a run from the log probabilities back to the gates."""
import importlib

import pytest

torch = pytest.importorskip("torch")
import gated_oracle as oracle

pytestmark = pytest.mark.gpu
BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
U = 2.0 ** -24


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return {n: importlib.import_module("glm53f-afd_b200." + n) for n in ("gated", "spec", "proj")}


class Decoder:
    """tokens -> embedding -> [gate | input] -> recurrence -> output projection -> logits."""

    WIDTH, CHANNELS, VOCAB, KINDS = 256, 192, 500, {"gate": "sigmoid", "input": "complement"}

    def __init__(self, mods):
        self.m = mods
        gen = torch.Generator(device="cuda").manual_seed(5)
        rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
        self.embedding = rn(self.VOCAB, self.WIDTH).bfloat16()
        pack = lambda n, k, group, zeros: mods["proj"].Int4Mat.quantise(rn(n, k) * 2 * k ** -0.5, group=group, zeros=zeros)
        self.into, self.outof, self.head = pack(2 * self.CHANNELS, self.WIDTH, 64, False), pack(self.WIDTH, self.CHANNELS, 32, True), pack(self.VOCAB, self.WIDTH, 128, False)

    def inputs(self, tokens):
        rows, c = len(tokens), self.CHANNELS
        e = self.embedding[tokens.long()]
        gx = torch.empty(rows, 2 * c, dtype=BF, device="cuda")
        self.m["proj"].int4(e, self.WIDTH, self.into, rows, gx, 2 * c)
        return gx[:, :c], gx[:, c:]

    def logits(self, h):
        rows = len(h)
        y, out = torch.empty(rows, self.WIDTH, dtype=BF, device="cuda"), torch.empty(rows, self.VOCAB, device="cuda")
        self.m["proj"].int4(h, self.CHANNELS, self.outof, rows, y, self.WIDTH)
        self.m["proj"].int4(y, self.WIDTH, self.head, rows, out, self.VOCAB, out_f32=True)
        return out

    def prefill(self, tokens, lens, state, off):
        gated, rows = self.m["gated"], len(tokens)
        g, x = self.inputs(tokens)
        h = torch.empty(rows, self.CHANNELS, dtype=BF, device="cuda")
        workspace = torch.empty(gated.workspace_bytes(self.CHANNELS, len(lens), rows), dtype=torch.uint8, device="cuda")
        cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=I32, device="cuda")
        gated.prefill_varlen(self.CHANNELS, rows, cu, max(lens), g, x, state, off, out=h, workspace=workspace, **self.KINDS)
        return g, x, h

    def step(self, tokens, cu, state, off):
        g, x = self.inputs(tokens)
        h = torch.empty(len(tokens), self.CHANNELS, dtype=BF, device="cuda")
        self.m["gated"].decode_batch(self.CHANNELS, len(tokens), cu, g, x, state, off, out=h, **self.KINDS)
        return self.logits(h)

    def round(self, tokens, cu, state, off, keep, next, logprob):
        """Verify, judge (greedy), report and commit the kept rows."""
        rows, batch = len(tokens), len(keep)
        g, x = self.inputs(tokens)
        h = torch.empty(rows, self.CHANNELS, dtype=BF, device="cuda")
        self.m["gated"].decode_batch(self.CHANNELS, rows, cu, g, x, state, off, state_out=None, out=h, **self.KINDS)
        logits = self.logits(h)
        self.m["spec"].accept_batch(cu, tokens, logits, torch.full((rows,), 0.5, device="cuda"), keep, next, temperature=torch.zeros(batch, device="cuda"))
        judged = torch.cat([tokens[1:], tokens.new_full((1,), -1)])  # what each row's distribution is asked for: the token behind it
        self.m["spec"].logprobs(logits, judged, logprob, entropy=None)
        self.m["gated"].decode_batch(self.CHANNELS, rows, cu, g, x, state, off, keep=keep, out=None, **self.KINDS)
        return logits, judged


def test_prompts_drafts_and_a_captured_round(mods):
    d = Decoder(mods)
    gen = torch.Generator(device="cuda").manual_seed(6)
    lens = [37, 150]
    prompt = torch.randint(0, d.VOCAB, (sum(lens),), generator=gen, device="cuda", dtype=I32)
    off = torch.tensor([d.CHANNELS, 0], device="cuda")
    state = torch.zeros(2, d.CHANNELS, device="cuda")
    g, x, h = d.prefill(prompt, lens, state, off)
    want, bound, ends, ends_bound = oracle.forward(lens, g, x, torch.zeros(2, d.CHANNELS, device="cuda"), **d.KINDS)
    oracle.close(h, want, bound)
    oracle.close(state.flip(0), ends, ends_bound)

    # Token by token, greedy: what the rounds have to arrive at.
    first = d.logits(h[torch.tensor([lens[0] - 1, sum(lens) - 1], device="cuda")]).argmax(1).to(I32)
    single, cu1 = state.clone(), torch.tensor([0, 1, 2], dtype=I32, device="cuda")
    tokens, states, rows = [first], [], []
    for _ in range(3):
        rows.append(d.step(tokens[-1], cu1, single, off))
        states.append(single.clone())
        tokens.append(rows[-1].argmax(1).to(I32))

    # A round of windows of three: all drafts right, and the second wrong.
    wrong = (tokens[2][1] + 1) % d.VOCAB
    window = torch.stack([tokens[0][0], tokens[1][0], tokens[2][0], tokens[0][1], tokens[1][1], wrong])
    cu = torch.tensor([0, 3, 6], dtype=I32, device="cuda")
    keep, next, logprob = torch.zeros(2, dtype=I32, device="cuda"), torch.zeros(2, dtype=I32, device="cuda"), torch.zeros(6, device="cuda")
    start = state.clone()
    logits, judged = d.round(window, cu, state, off, keep, next, logprob)
    assert keep.tolist() == [3, 2] and next.tolist() == [int(tokens[3][0]), int(tokens[2][1])]
    for row, (request, t) in {0: (0, 0), 1: (0, 1), 2: (0, 2), 3: (1, 0), 4: (1, 1)}.items():
        assert torch.equal(logits[row], rows[t][request]), row  # up to eight rows' products do not depend on the others
    assert torch.equal(state[1], states[2][1]) and torch.equal(state[0], states[1][0])
    exact = torch.log_softmax(logits.double(), 1)
    for row in range(5):
        lp = exact[row, int(judged[row])]
        # the sum to u (vocab / 512 + 300), what stands before it to 4 u of itself, and as much for the largest logit
        assert abs(float(logprob[row] - lp)) <= U * (d.VOCAB / 512 + 300 + 8 * (abs(float(lp)) + float(logits[row].abs().max())))
    assert float(logprob[5]) == 0.0

    # The same round captured, from the same states.
    again, keep2, next2, lp2 = start.clone(), torch.zeros_like(keep), torch.zeros_like(next), torch.zeros_like(logprob)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        d.round(window, cu, again, off, keep2, next2, lp2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            d.round(window, cu, again, off, keep2, next2, lp2)
        for _ in range(2):
            again.copy_(start), keep2.zero_(), next2.zero_(), lp2.zero_()
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, state) and torch.equal(keep2, keep) and torch.equal(next2, next) and torch.equal(lp2, logprob)


@pytest.mark.parametrize("gate,input", [("decay", "plain"), ("sigmoid", "complement")])
def test_gradients_of_a_run(mods, gate, input):
    """The loss sum w_t log p(token_t) + v_t H_t of a recurrence's outputs through a head in 64 bits; every other step is the framework's, in f32.

    Bounds: those of each step, carried through the next ones.  A logit off by at most d moves each p by a factor within e^(2 d), and with it the entropy by 2 d (1 + H)."""
    gated, spec = mods["gated"], mods["spec"]
    lens, channels, vocab = [30, 1, 90], 24, 60
    rows = sum(lens)
    gen = torch.Generator(device="cuda").manual_seed(7)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    g = -torch.rand(rows, channels, generator=gen, device="cuda") if gate == "decay" else rn(rows, channels)
    x, state, head, w, v = rn(rows, channels), rn(len(lens), channels), rn(channels, vocab).double() * channels ** -0.5, rn(rows), rn(rows)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=I32)
    cu = torch.tensor([0, 30, 31, 121], dtype=I32, device="cuda")
    off = torch.arange(len(lens), device="cuda") * channels
    kinds = dict(gate=gate, input=input)

    h, end, saves = torch.empty_like(x), state.clone(), torch.empty(gated.saves_rows(len(lens), rows), channels, device="cuda")
    workspace = torch.empty(gated.workspace_bytes(channels, len(lens), rows), dtype=torch.uint8, device="cuda")
    gated.prefill_varlen(channels, rows, cu, max(lens), g, x, end, off, out=h, saves=saves, workspace=workspace, **kinds)
    logits = (h.double() @ head).float()
    logprob, entropy, lse = (torch.empty(rows, device="cuda") for _ in range(3))
    spec.logprobs(logits, tokens, logprob, entropy=entropy, lse=lse)
    dlogits = torch.empty_like(logits)
    spec.logprobs_backward(logits, tokens, lse, w, dlogits, entropy=entropy, dentropy=v)
    dh = (dlogits.double() @ head.T).float()
    dg, dx, ds = torch.empty_like(g), torch.empty_like(x), torch.empty_like(state)
    gated.backward_varlen(channels, rows, cu, max(lens), g, x, saves, off, dh, dg, dx, dstate_in=ds, workspace=workspace, **kinds)

    # In 64 bits, differentiated by the tape.
    g64, x64, s64 = (t.double().requires_grad_() for t in (g, x, state))
    hs, at = [], 0
    for b, n in enumerate(lens):
        a, c, _ = oracle.gates(g64[at:at + n], gate, input)
        last = s64[b]
        for t in range(n):
            last = a[t] * last + c[t] * x64[at + t]
            hs.append(last)
        at += n
    logp = torch.log_softmax(torch.stack(hs) @ head, 1)
    H = -(logp.exp() * logp).sum(1)
    ((w.double() * logp.gather(1, tokens.long()[:, None])[:, 0]).sum() + (v.double() * H).sum()).backward()

    with torch.no_grad():
        _, hb, _, _ = oracle.forward(lens, g, x, state, gate, input)
        hb = hb + U * torch.stack(hs).abs()  # h is rounded once
        lb = hb @ head.abs() + U * (torch.stack(hs) @ head).abs()
        d = lb.amax(1, keepdim=True)
        p, size, l, n, Hc = logp.exp(), logp.abs(), w.double().abs()[:, None], v.double().abs()[:, None], H[:, None]
        s = U * (vocab / 512 + 300)
        rel = s + U * (8 * size + 20 + 4 * (torch.stack(hs) @ head).abs().amax(1, keepdim=True))
        db = p * (l + n * (size + Hc)) * (rel + 2.2 * d) + n * p * (4 * s * (1 + Hc) + 16 * U * (size + Hc) + 2.2 * d * (2 + Hc))
        db.scatter_add_(1, tokens.long()[:, None], 8 * U * l)
        want_dl = (torch.nn.functional.one_hot(tokens.long(), vocab) - p) * w.double()[:, None] - v.double()[:, None] * p * (logp + Hc)
        dy = want_dl @ head.T
        yb = (db + U * want_dl.abs()) @ head.T.abs() + U * dy.abs()
        (vg, bg), (vx, bx), (vs, bs) = oracle.backward(lens, g, x, state, dy, None, gate, input)
        # What dh's own error does behind the bounds of the backward pass.
        at, eg, ex, es = 0, [], [], []
        before_all = torch.stack(hs)
        for b, m in enumerate(lens):
            a, c, slope = oracle.gates(g[at:at + m], gate, input)
            e, E = torch.zeros(channels, dtype=F64, device="cuda"), []
            for t in reversed(range(m)):
                e = yb[at + t] + (a[t + 1] * e if t + 1 < m else 0)
                E.insert(0, e)
            E = torch.stack(E)
            before = torch.cat([state[b].double()[None], before_all[at:at + m - 1]])
            other = x[at:at + m].double() if input == "complement" else 0 * before
            eg.append(slope * E * (before - other).abs()), ex.append(c * E), es.append(a[0] * E[0])
            at += m
        for got, tape, value, bound, extra, what in ((dg, g64.grad, vg, bg, torch.cat(eg), "dg"), (dx, x64.grad, vx, bx, torch.cat(ex), "dx"), (ds, s64.grad, vs, bs, torch.stack(es), "dstate")):
            assert torch.allclose(tape, value, rtol=1e-9, atol=1e-11), what
            oracle.close(got, tape, 1.05 * (bound + extra), what)
