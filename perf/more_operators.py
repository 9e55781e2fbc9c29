"""Operators of a decoder with gated recurrent layers and 4-bit weights, as cases that can be timed and compared.

  step      gated linear recurrence row by row: single tokens and windows of drafted ones (`gated.decode_batch`)
  scan      the same over packed sequences (`gated.prefill_varlen`), and with its backward pass (`gated.backward_varlen`)
  matrix    a projection with 4-bit weights, a scale and maybe a zero point for each group of k (`proj.int4`)
  logprobs  log probabilities of given tokens, entropy and top alternatives (`spec.logprobs`), and with gradients (`spec.logprobs_backward`)

`run` computes a case in plain torch operations, or with the library's kernels where `own` is true.  A state is made once; the
kernels' outputs go to buffers of their own, so a pass can be repeated.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

_PKG = "glm53f-afd_b200"


def listed():
    return [
        # One user's next token through a layer's 4,096 channels: latency.
        {"name": "step_1_slot", "kind": "step", "channels": 4096, "lens": "1", "gate": "decay", "input": "plain", "g": "f32", "x": "bf16", "write": True},
        # A busy server's round of drafted windows, gates as the projection leaves them, states read and left as they are.
        {"name": "step_windows_48_slots", "kind": "step", "channels": 8192, "lens": " ".join(str(8 - (i * i) % 5) for i in range(48)), "gate": "sigmoid",
         "input": "complement", "g": "bf16", "x": "bf16", "write": False},
        # A short prompt: launches count.
        {"name": "scan_100_rows", "kind": "scan", "channels": 4096, "lens": "100", "gate": "decay", "input": "plain", "g": "f32", "x": "bf16", "train": False},
        # Packed prompts of unequal lengths that continue carried states, gates as the projection leaves them.
        {"name": "scan_packed_ragged", "kind": "scan", "channels": 8192, "lens": "1 63 64 65 777 1500 2021 3701", "gate": "sigmoid", "input": "complement",
         "g": "bf16", "x": "bf16", "train": False},
        # A long prompt of few channels: the sequence itself has to be divided.
        {"name": "scan_65536_rows", "kind": "scan", "channels": 1024, "lens": "65536", "gate": "decay", "input": "plain", "g": "f32", "x": "bf16", "train": False},
        # A training step's sequences, there and back.
        {"name": "scan_train_4_sequences", "kind": "scan", "channels": 2048, "lens": "4096 4096 4096 4001", "gate": "decay", "input": "complement", "g": "f32",
         "x": "bf16", "train": True},
        # One user's next token through the fused input projection of a layer: latency and the weights' bytes.
        {"name": "matrix_1_row", "kind": "matrix", "rows": 1, "n": 24640, "k": 4096, "group": 128, "zeros": False, "out": "bf16"},
        # A round's odd number of rows through an output projection with zero points and finer groups.
        {"name": "matrix_40_rows", "kind": "matrix", "rows": 40, "n": 4096, "k": 8192, "group": 64, "zeros": True, "out": "f32"},
        # A prefill lane through the same weights: the tensor cores' rate.
        {"name": "matrix_2048_rows", "kind": "matrix", "rows": 2048, "n": 4096, "k": 8192, "group": 128, "zeros": False, "out": "bf16"},
        # One user's next token reported with its 20 best alternatives: latency.
        {"name": "logprobs_1_row", "kind": "logprobs", "rows": 1, "vocab": 131072, "logits": "f32", "temperature": False, "top": 20, "train": False},
        # A busy server's verification round at the users' temperatures.
        {"name": "logprobs_336_rows", "kind": "logprobs", "rows": 336, "vocab": 131072, "logits": "bf16", "temperature": True, "top": 5, "train": False},
        # A policy's training step: log probabilities and entropies of 2,048 tokens, and the logits' gradient.
        {"name": "logprobs_train_2048_rows", "kind": "logprobs", "rows": 2048, "vocab": 131072, "logits": "bf16", "temperature": False, "top": 0, "train": True},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _split(rng: random.Random, total: int, parts: int) -> str:
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return " ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "matrix", "matrix", "logprobs", "logprobs"])
    if kind in ("step", "scan"):
        channels = _log_int(rng, 1, 8192)
        case = {"kind": kind, "channels": channels, "gate": rng.choice(["decay", "sigmoid"]), "input": rng.choice(["plain", "complement"]),
                "g": rng.choice(["f32", "bf16"]), "x": rng.choice(["bf16", "bf16", "f32"])}
        if kind == "step":
            most = rng.choice([1, 4, 8])
            case["lens"] = " ".join(str(rng.randint(1, most)) for _ in range(_log_int(rng, 1, 48)))
            case["write"] = rng.random() < 0.6
        else:
            case["train"] = rng.random() < 0.5
            case["lens"] = _split(rng, _log_int(rng, 1, min(65536, (16384 * 2048 if case["train"] else 65536 * 1024) // channels)), rng.randint(1, 8))
        return case
    if kind == "matrix":
        return {"kind": kind, "rows": _log_int(rng, 1, 2048), "n": _log_int(rng, 64, 8192), "k": 128 * _log_int(rng, 1, 32), "group": rng.choice([32, 64, 128]),
                "zeros": rng.random() < 0.5, "out": rng.choice(["bf16", "f32"])}
    train = rng.random() < 0.4
    vocab = _log_int(rng, 1000, 131072)
    return {"kind": kind, "rows": _log_int(rng, 1, min(2048, 512 * 131072 // vocab)), "vocab": vocab, "logits": rng.choice(["bf16", "f32"]),
            "temperature": rng.random() < 0.5, "top": 0 if train else rng.choice([0, 1, 5, 20, 32]), "train": train}


def _lens(case):
    return [int(x) for x in case["lens"].split()]


def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


# ---- inputs -----------------------------------------------------------------------------------------------------------------


def _prepare_recurrence(case, gen):
    channels, lens = case["channels"], _lens(case)
    rows, batch = sum(lens), len(lens)
    train = case.get("train", False)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    # Channels remember from two to a thousand rows.
    reach = torch.exp2(1 + 9 * torch.rand(channels, generator=gen, device="cuda"))
    if case["gate"] == "decay":
        g = -torch.nn.functional.softplus(normal(rows, channels) + 0.5) / reach
    else:
        g = torch.log(reach) + normal(rows, channels)
    x = normal(rows, channels)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    s = {"lens": lens, "g": g.to(_dtype(case["g"])), "x": x.to(_dtype(case["x"])), "state": 0.5 * normal(batch, channels),
         "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"), "off": torch.arange(batch, dtype=torch.int64, device="cuda") * channels}
    if train:
        s["dout"] = normal(rows, channels).to(s["x"].dtype)
        s["dstate"] = normal(batch, channels)
    return s


def _prepare_matrix(case, gen):
    rows, n, k, group = case["rows"], case["n"], case["k"], case["group"]
    w = (torch.randn((n, k), generator=gen, device="cuda") * k ** -0.5).view(n, k // group, group)
    if case["zeros"]:
        low, high = w.amin(-1), w.amax(-1)
        scales = ((high - low) / 15).bfloat16()
        zeros = torch.round(-low / scales.float()).clamp(0, 15)
    else:
        scales = (w.abs().amax(-1) / 7).bfloat16()
        zeros = torch.full_like(w[..., 0], 8.0)
    codes = (torch.round(w / scales.float()[..., None]) + zeros[..., None]).clamp(0, 15).to(torch.uint8).view(n, k)
    return {"x": torch.randn((rows, k), generator=gen, device="cuda").bfloat16(), "codes": codes[:, 0::2] | (codes[:, 1::2] << 4), "scales": scales,
            "zeros": zeros.to(torch.uint8) if case["zeros"] else None}


def _prepare_logprobs(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    logits = 2.5 * torch.randn((rows, vocab), generator=gen, device="cuda")
    logits[:, rows % 7::11] = -math.inf  # what a grammar rules out
    tokens = (logits + torch.randn((rows, vocab), generator=gen, device="cuda")).argmax(-1)
    s = {"logits": logits.to(_dtype(case["logits"])), "tokens": tokens.int(),
         "temperature": 0.6 + 0.6 * torch.rand(rows, generator=gen, device="cuda") if case["temperature"] else None}
    if case["train"]:
        s["dlogprob"] = torch.randn(rows, generator=gen, device="cuda") / rows
        s["dentropy"] = torch.full((rows,), 0.01 / rows, device="cuda")
    return s


def _buffers(case, s):
    """What the library's calls write to, and what they work in."""
    f32 = {"dtype": torch.float32, "device": "cuda"}
    if case["kind"] == "step":
        s["module"] = importlib.import_module(_PKG + ".gated")
        s["out"], s["state_out"] = torch.empty_like(s["x"]), torch.empty_like(s["state"])
    elif case["kind"] == "scan":
        m = s["module"] = importlib.import_module(_PKG + ".gated")
        rows, batch, channels = s["x"].shape[0], len(s["lens"]), case["channels"]
        s["out"], s["state_out"] = torch.empty_like(s["x"]), torch.empty_like(s["state"])
        s["workspace"] = torch.empty(max(1, m.workspace_bytes(channels, batch, rows)), dtype=torch.uint8, device="cuda")
        if case["train"]:
            s["saves"] = torch.empty(m.saves_rows(batch, rows), channels, **f32)
            s["dg"], s["dx"], s["dstate_in"] = torch.empty_like(s["g"]), torch.empty_like(s["x"]), torch.empty_like(s["state"])
    elif case["kind"] == "matrix":
        m = s["module"] = importlib.import_module(_PKG + ".proj")
        s["weight"] = m.Int4Mat.pack(s["codes"], s["scales"], s["zeros"], group=case["group"])
        s["out"] = torch.empty(case["rows"], case["n"], dtype=_dtype(case["out"]), device="cuda")
    else:
        s["module"] = importlib.import_module(_PKG + ".spec")
        rows, top = case["rows"], case["top"]
        s["logprob"], s["entropy"], s["lse"] = (torch.empty(rows, **f32) for _ in range(3))
        s["top"] = (torch.empty(rows, top, dtype=torch.int32, device="cuda"), torch.empty(rows, top, **f32)) if top else None
        s["dlogits"] = torch.empty_like(s["logits"]) if case["train"] else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"step": _prepare_recurrence, "scan": _prepare_recurrence, "matrix": _prepare_matrix, "logprobs": _prepare_logprobs}[case["kind"]]
    state = make(case, gen)
    state["case"] = case
    if own:
        _buffers(case, state)
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------------


def _plain_gate(case, g):
    """What is kept of the state, what is taken of the input, and the slope of the first."""
    g = g.float()
    if case["gate"] == "decay":
        a = torch.exp(g)
        return a, -torch.expm1(g) if case["input"] == "complement" else torch.ones_like(a), a
    a, rest = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    return a, rest if case["input"] == "complement" else torch.ones_like(a), a * rest


def _plain_rows(a, b, h):
    """h_t = a_t h_(t-1) + b_t over all rows: pieces side by side, then the states between them, then the rows of each."""
    n, channels = a.shape
    if n == 0:
        return a
    size = 1 << ((n - 1).bit_length() + 1) // 2
    parts = -(-n // size)
    more = parts * size - n
    if more:
        a, b = torch.cat([a, a.new_ones(more, channels)]), torch.cat([b, b.new_zeros(more, channels)])
    a, b = a.view(parts, size, channels), b.view(parts, size, channels)
    whole, end = torch.ones_like(a[:, 0]), torch.zeros_like(a[:, 0])
    for i in range(size):
        whole, end = whole * a[:, i], a[:, i] * end + b[:, i]
    starts = torch.empty_like(end)
    for j in range(parts):
        starts[j] = h
        h = whole[j] * h + end[j]
    out = torch.empty_like(a)
    for i in range(size):
        starts = a[:, i] * starts + b[:, i]
        out[:, i] = starts
    return out.view(parts * size, channels)[:n]


def _plain_scan(s):
    case = s["case"]
    out, ends = torch.empty_like(s["x"]), torch.empty_like(s["state"])
    train = case["train"]
    if train:
        dg, dx, dstart = torch.empty_like(s["g"]), torch.empty_like(s["x"]), torch.empty_like(s["state"])
    first = 0
    for i, n in enumerate(s["lens"]):
        at = slice(first, first + n)
        first += n
        start = s["state"][i]
        a, c, slope = _plain_gate(case, s["g"][at])
        x = s["x"][at].float()
        h = _plain_rows(a, c * x, start)
        out[at] = h
        ends[i] = h[-1] if n else start
        if train:
            after = s["dstate"][i]
            if n == 0:
                dstart[i] = after
                continue
            step = torch.cat([torch.ones_like(a[:1]), a.flip(0)[:-1]])
            d = _plain_rows(step, s["dout"][at].float().flip(0), after).flip(0)
            before = torch.cat([start[None], h[:-1]])
            dx[at] = c * d
            dg[at] = d * slope * (before - x if case["input"] == "complement" else before)
            dstart[i] = a[0] * d[0]
    return (out, ends, dg, dx, dstart) if train else (out, ends)


def _plain_step(s):
    case = s["case"]
    a, c, _ = _plain_gate(case, s["g"])
    b = c * s["x"].float()
    lens = s["lens"]
    state, out = s["state"].clone(), torch.empty_like(s["x"])
    starts = [sum(lens[:i]) for i in range(len(lens))]
    for t in range(max(lens)):
        live = [i for i, n in enumerate(lens) if n > t]
        who = torch.tensor(live, device=b.device)
        at = torch.tensor([starts[i] + t for i in live], device=b.device)
        state[who] = a[at] * state[who] + b[at]
        out[at] = state[who].to(out.dtype)
    return (out, state) if case["write"] else out


def _plain_matrix(s):
    n, half = s["codes"].shape
    group = s["case"]["group"]
    q = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(n, -1, group).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    w = ((q - zero) * s["scales"].float()[..., None]).view(n, 2 * half)
    return torch.matmul(s["x"].float(), w.t()).to(_dtype(s["case"]["out"]))


def _plain_logprobs(s):
    case = s["case"]
    x = s["logits"].float()
    heat = 1.0 if s["temperature"] is None else s["temperature"][:, None]
    t = (x - x.amax(-1, keepdim=True)) / heat
    e = torch.exp(t)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    at = s["tokens"].long()[:, None]
    logprob = (t.gather(1, at) - log_total)[:, 0]
    entropy = (log_total - torch.where(e > 0, e * t, 0.0).sum(-1, keepdim=True) / total)[:, 0]
    if case["train"]:
        logp = t - log_total
        p = e / total
        d = -s["dlogprob"][:, None] * p - torch.where(p > 0, s["dentropy"][:, None] * p * (logp + entropy[:, None]), 0.0)
        d.scatter_add_(1, at, s["dlogprob"][:, None])
        return logprob, entropy, (d / heat).to(s["logits"].dtype)
    if not case["top"]:
        return logprob, entropy
    best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    return logprob, entropy, best.int(), t.gather(1, best) - log_total


# ---- the library's operators ------------------------------------------------------------------------------------------------


def _own_step(s):
    case = s["case"]
    s["module"].decode_batch(case["channels"], s["x"].shape[0], s["cu"], s["g"], s["x"], s["state"], s["off"], gate=case["gate"], input=case["input"],
                             state_out=s["state_out"] if case["write"] else None, out=s["out"])
    return (s["out"], s["state_out"]) if case["write"] else s["out"]


def _own_scan(s):
    case = s["case"]
    kinds = {"gate": case["gate"], "input": case["input"], "workspace": s["workspace"]}
    m, rows, longest = s["module"], s["x"].shape[0], max(s["lens"])
    m.prefill_varlen(case["channels"], rows, s["cu"], longest, s["g"], s["x"], s["state"], s["off"], state_out=s["state_out"], out=s["out"],
                     saves=s.get("saves"), **kinds)
    if not case["train"]:
        return s["out"], s["state_out"]
    m.backward_varlen(case["channels"], rows, s["cu"], longest, s["g"], s["x"], s["saves"], s["off"], s["dout"], s["dg"], s["dx"], dstate=s["dstate"],
                      dstate_in=s["dstate_in"], **kinds)
    return s["out"], s["state_out"], s["dg"], s["dx"], s["dstate_in"]


def _own_matrix(s):
    case = s["case"]
    s["module"].int4(s["x"], case["k"], s["weight"], case["rows"], s["out"], case["n"], out_f32=case["out"] == "f32")
    return s["out"]


def _own_logprobs(s):
    case = s["case"]
    s["module"].logprobs(s["logits"], s["tokens"], s["logprob"], temperature=s["temperature"], entropy=s["entropy"], lse=s["lse"] if case["train"] else None,
                         top=s["top"])
    if case["train"]:
        s["module"].logprobs_backward(s["logits"], s["tokens"], s["lse"], s["dlogprob"], s["dlogits"], temperature=s["temperature"], entropy=s["entropy"],
                                      dentropy=s["dentropy"])
        return s["logprob"], s["entropy"], s["dlogits"]
    return (s["logprob"], s["entropy"], *s["top"]) if case["top"] else (s["logprob"], s["entropy"])


def run(state):
    plain = {"step": _plain_step, "scan": _plain_scan, "matrix": _plain_matrix, "logprobs": _plain_logprobs}
    kernels = {"step": _own_step, "scan": _own_scan, "matrix": _own_matrix, "logprobs": _own_logprobs}
    return (kernels if own else plain)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------


def work(case):
    size = {"f32": 4, "bf16": 2}
    if case["kind"] in ("step", "scan"):
        lens = _lens(case)
        values, states = sum(lens) * case["channels"], 4 * len(lens) * case["channels"]
        g, x = size[case["g"]], size[case["x"]]
        if case["kind"] == "step":
            return {"bytes": values * (g + 2 * x) + states * (2 if case["write"] else 1), "flops": 6 * values}
        if case["train"]:  # there: g, x, out; back: g, x, dout, dg, dx
            return {"bytes": values * (3 * g + 5 * x) + 4 * states, "flops": 24 * values}
        return {"bytes": values * (g + 2 * x) + 2 * states, "flops": 6 * values}
    if case["kind"] == "matrix":
        rows, n, k = case["rows"], case["n"], case["k"]
        groups = n * (k // case["group"])
        return {"bytes": n * k // 2 + groups * (3 if case["zeros"] else 2) + 2 * rows * k + rows * n * size[case["out"]], "flops": 2 * rows * n * k}
    values = case["rows"] * case["vocab"]
    return {"bytes": values * size[case["logits"]] * (3 if case["train"] else 1) + case["rows"] * (12 + 8 * case["top"]),
            "flops": values * (14 if case["train"] else 6)}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------------


def _exact_rows(a, b, h):
    """h_t = a_t h_(t-1) + b_t by doubling: after step d every row holds the composition of the 2 d rows up to it."""
    b = b.clone()
    if a.shape[0] == 0:
        return b
    b[0] += a[0] * h
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], a[d:] * b[:-d] + b[d:]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _exact_gate(case, g):
    g = g.double()
    if case["gate"] == "decay":
        return g.exp(), -g.expm1(), g.exp()
    return torch.sigmoid(g), torch.sigmoid(-g), torch.sigmoid(g) * torch.sigmoid(-g)


def _exact_recurrence(s):
    case = s["case"]
    complement = case["input"] == "complement"
    outs, ends, dgs, dxs, dstarts = [], [], [], [], []
    for i, piece in enumerate(torch.split(torch.arange(s["x"].shape[0], device="cuda"), s["lens"])):
        start = s["state"][i].double()
        a, rest, slope = _exact_gate(case, s["g"][piece])
        x = s["x"][piece].double()
        taken = rest if complement else torch.ones_like(rest)
        h = _exact_rows(a, taken * x, start)
        outs.append(h)
        ends.append(h[-1] if len(h) else start)
        if not case.get("train"):
            continue
        d = s["dout"][piece].double()
        if len(h) == 0:
            dgs.append(h), dxs.append(h), dstarts.append(s["dstate"][i].double())
            continue
        d[-1] += s["dstate"][i].double()
        d = _exact_rows(torch.roll(a, -1, 0).flip(0), d.flip(0), torch.zeros_like(start)).flip(0)
        before = torch.roll(h, 1, 0)
        before[0] = start
        dgs.append(d * slope * (before - (x if complement else 0)))
        dxs.append(d * taken)
        dstarts.append(a[0] * d[0])
    out, end = torch.cat(outs), torch.stack(ends)
    if case["kind"] == "step":
        return (out, end) if case["write"] else out
    return (out, end, torch.cat(dgs), torch.cat(dxs), torch.stack(dstarts)) if case["train"] else (out, end)


def _exact_matrix(s):
    group = s["case"]["group"]
    low, high = s["codes"].int() % 16, s["codes"].int() // 16
    n = low.shape[0]
    q = torch.empty(n, 2 * low.shape[1], dtype=torch.float64, device=low.device)
    q[:, ::2], q[:, 1::2] = low.double(), high.double()
    zero = torch.full_like(s["scales"], 8) if s["zeros"] is None else s["zeros"]
    w = (q - zero.double().repeat_interleave(group, 1)) * s["scales"].double().repeat_interleave(group, 1)
    return s["x"].double() @ w.T


def _exact_logprobs(s):
    case = s["case"]
    parts = []
    for first in range(0, case["rows"], 64):
        at = slice(first, min(first + 64, case["rows"]))
        x = s["logits"][at].double()
        heat = torch.ones(len(x), 1, dtype=torch.float64, device=x.device) if s["temperature"] is None else s["temperature"][at].double()[:, None]
        logp = torch.log_softmax(x / heat, -1)
        p = logp.exp()
        finite = logp.masked_fill(logp == -math.inf, 0.0)
        entropy = -(p * finite).sum(-1)
        token = s["tokens"][at].long()
        own_row = torch.arange(len(x), device=x.device)
        row = [logp[own_row, token], entropy]
        if case["train"]:
            d = -s["dentropy"][at].double()[:, None] * p * (finite + entropy[:, None]) - s["dlogprob"][at].double()[:, None] * p
            d[own_row, token] += s["dlogprob"][at].double()
            row.append(d / heat)
        elif case["top"]:
            best = torch.argsort(-x, dim=-1, stable=True)[:, :case["top"]]
            row += [best.int(), torch.take_along_dim(logp, best, 1)]
        parts.append(row)
    return tuple(torch.cat(column) for column in zip(*parts))


def exact(case, seed):
    state = prepare(case, seed)
    return {"step": _exact_recurrence, "scan": _exact_recurrence, "matrix": _exact_matrix, "logprobs": _exact_logprobs}[case["kind"]](state)
