"""Operators of a hybrid decoder beside the KDA layers, as cases that can be timed and compared.

  prefill   linear attention with one decay a head, chunked, over packed prompts (`linear.prefill_varlen`)
  step      the same recurrence row by row: single tokens and windows of drafted ones (`linear.decode_batch`)
  project   a projection with bias, activation and residual in its epilogue (`proj.fused`)
  accept    verification of drafted tokens against the target's distribution from given random numbers (`spec.accept_batch`)

`run` computes a case in plain torch operations, or with the library's kernels where `own` is true.  A state is made once; its
outputs go to buffers of their own, so a pass can be repeated.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

_PKG = "glm53f-afd_b200"
DIM = 128  # channels of a head, keys and values


def listed():
    return [
        # A short prompt of a small shard: launches and the pipeline's fill count.
        {"name": "prefill_100_rows", "kind": "prefill", "heads": 16, "qk_heads": 16, "lens": "100", "state": "f32", "decay": "token"},
        # One prompt through the 64 heads of a layer.
        {"name": "prefill_8192_rows", "kind": "prefill", "heads": 64, "qk_heads": 64, "lens": "8192", "state": "f32", "decay": "token"},
        # Packed prompts of unequal lengths that continue carried bf16 states, keys shared by groups of eight heads.
        {"name": "prefill_packed_ragged", "kind": "prefill", "heads": 64, "qk_heads": 8, "lens": "1 63 64 65 777 1500 2021 3701", "state": "bf16",
         "decay": "token"},
        # A long prompt on one GPU's eight heads, decays fixed for each head.
        {"name": "prefill_long_8_heads", "kind": "prefill", "heads": 8, "qk_heads": 8, "lens": "65536", "state": "f32", "decay": "head"},
        # One user's next token: latency.
        {"name": "step_1_slot", "kind": "step", "heads": 64, "qk_heads": 64, "lens": "1", "state": "bf16", "decay": "token", "write": True},
        # A busy server's decode step on full-precision states.
        {"name": "step_48_slots", "kind": "step", "heads": 64, "qk_heads": 64, "lens": " ".join(["1"] * 48), "state": "f32", "decay": "head", "write": True},
        # Windows of drafted tokens, ragged, the states read and left as they are.
        {"name": "step_windows_16_slots", "kind": "step", "heads": 64, "qk_heads": 8, "lens": "8 5 8 1 7 8 3 8 6 8 2 8 8 4 8 8", "state": "bf16",
         "decay": "token", "write": False},
        # The output projection of a decode step, added to the residual stream.
        {"name": "project_16_rows", "kind": "project", "rows": 16, "n": 4096, "k": 8192, "groups": 1, "act": "none", "bias": "bf16", "residual": True,
         "out": "bf16"},
        # A prefill lane's wide projection with its activation.
        {"name": "project_2048_rows", "kind": "project", "rows": 2048, "n": 8192, "k": 4096, "groups": 1, "act": "silu", "bias": "bf16", "residual": False,
         "out": "bf16"},
        # An odd number of rows through the two stacked second factors of low-rank gates, added to f32 rows.
        {"name": "project_333_rows_2_groups", "kind": "project", "rows": 333, "n": 8192, "k": 128, "groups": 2, "act": "sigmoid", "bias": "f32",
         "residual": True, "out": "f32"},
        # One user's window of eight against probabilities: latency.
        {"name": "accept_1_request", "kind": "accept", "lens": "8", "vocab": 131072, "target": "probs", "draft": True, "greedy": False},
        # A busy server's round against logits, the drafter's distributions at hand, every third request greedy.
        {"name": "accept_48_requests", "kind": "accept", "lens": " ".join(str(8 - (i * i) % 5) for i in range(48)), "vocab": 131072, "target": "logits_bf16",
         "draft": True, "greedy": True},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _split(rng: random.Random, total: int, parts: int) -> str:
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return " ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    kind = rng.choice(["prefill", "step", "project", "accept"])
    if kind in ("prefill", "step"):
        heads = _log_int(rng, 1, 64)
        case = {"kind": kind, "heads": heads, "qk_heads": rng.choice([d for d in range(1, heads + 1) if heads % d == 0]),
                "state": rng.choice(["f32", "bf16"]), "decay": rng.choice(["token", "head"])}
        if kind == "prefill":
            rows = _log_int(rng, 1, min(65536, 8 * 65536 // heads))
            case["lens"] = _split(rng, rows, rng.randint(1, 8))
        else:
            slots = _log_int(rng, 1, 48)
            most = rng.choice([1, 4, 16])
            case["lens"] = " ".join(str(rng.randint(1, most)) for _ in range(slots))
            case["write"] = rng.random() < 0.6
        return case
    if kind == "project":
        return {"kind": kind, "rows": _log_int(rng, 1, 2048), "n": 8 * _log_int(rng, 8, 1024), "k": 64 * _log_int(rng, 1, 64), "groups": rng.choice([1, 1, 2]),
                "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"]), "bias": rng.choice(["none", "bf16", "f32"]),
                "residual": rng.random() < 0.6, "out": rng.choice(["bf16", "f32"])}
    most = rng.randint(1, 8)
    target = rng.choice(["probs", "logits_bf16", "logits_f32"])
    return {"kind": kind, "lens": " ".join(str(rng.randint(1, most)) for _ in range(_log_int(rng, 1, 32))), "vocab": _log_int(rng, 1000, 131072),
            "target": target, "draft": rng.random() < 0.6, "greedy": target != "probs" and rng.random() < 0.5}


def _lens(case):
    return [int(x) for x in case["lens"].split()]


def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


# ---- inputs -----------------------------------------------------------------------------------------------------------------


def _prepare_linear(case, gen):
    heads, qk, lens = case["heads"], case["qk_heads"], _lens(case)
    rows, batch = sum(lens), len(lens)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def unit(t):  # keys and queries of length one, as the layers that use this recurrence normalise them
        return t / t.norm(dim=-1, keepdim=True)

    q, k = (unit(normal(rows, qk, DIM)).bfloat16() for _ in range(2))
    v = (0.5 * normal(rows, heads, DIM)).bfloat16()
    slope = -torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)  # from nearly 1 a row to e^(-1/256)
    if case["decay"] == "token":
        g = (slope * torch.nn.functional.softplus(normal(rows, heads) + 0.5)).contiguous()
    else:
        g = slope.contiguous()
    state = (0.3 * normal(batch, heads, DIM, DIM)).to(_dtype(case["state"]))
    state[::2] *= 0 if case["kind"] == "prefill" and batch > 1 else 1  # half of the packed prompts start afresh
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return {"lens": lens, "q": q, "k": k, "v": v, "g": g, "state": state, "state_out": torch.empty_like(state), "scale": DIM ** -0.5,
            "out": torch.empty(rows, heads, DIM, dtype=torch.bfloat16, device="cuda"), "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
            "off": torch.arange(batch, dtype=torch.int64, device="cuda") * (heads * DIM * DIM)}


def _prepare_project(case, gen):
    groups, rows, n, k = case["groups"], case["rows"], case["n"], case["k"]
    x = torch.randn((groups, rows, k), generator=gen, device="cuda").bfloat16()
    w = (torch.randn((groups, n, k), generator=gen, device="cuda") * k ** -0.5).bfloat16()
    out = torch.empty(groups, rows, n, dtype=_dtype(case["out"]), device="cuda")
    bias = None if case["bias"] == "none" else torch.randn((groups, n), generator=gen, device="cuda").to(_dtype(case["bias"]))
    residual = torch.randn((groups, rows, n), generator=gen, device="cuda").to(out.dtype) if case["residual"] else None
    return {"x": x, "w": w, "out": out, "bias": bias, "residual": residual}


def _prepare_accept(case, gen):
    lens, vocab = _lens(case), case["vocab"]
    rows, batch = sum(lens), len(lens)
    logits = 2.5 * torch.randn((rows, vocab), generator=gen, device="cuda")
    # The drafter sees nearly what the target sees at the row before the token it drafts.
    draft = torch.roll(logits, 1, 0) + 0.4 * torch.randn((rows, vocab), generator=gen, device="cuda")
    if case["draft"]:
        draft = torch.softmax(draft, -1)
        tokens = torch.multinomial(draft, 1, generator=gen)[:, 0].int()
    else:
        tokens, draft = draft.argmax(-1).int(), None
    if case["target"] == "probs":
        target = torch.softmax(logits, -1)
    else:
        target = logits.to(torch.bfloat16 if case["target"] == "logits_bf16" else torch.float32)
    temperature = None
    if case["target"] != "probs":
        temperature = 0.6 + 0.6 * torch.rand(batch, generator=gen, device="cuda")
        if case["greedy"]:
            temperature[::3] = 0.0
            first = 0
            for b, n in enumerate(lens):  # a greedy request's drafts are mostly the target's own choice
                if b % 3 == 0 and n > 1:
                    best = target[first:first + n - 1].float().argmax(-1).int()
                    same = torch.rand(n - 1, generator=gen, device="cuda") < 0.8
                    tokens[first + 1:first + n] = torch.where(same, best, tokens[first + 1:first + n])
                first += n
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return {"lens": lens, "target": target, "draft": draft, "tokens": tokens, "temperature": temperature,
            "u": torch.rand(rows, generator=gen, device="cuda"), "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
            "keep": torch.empty(batch, dtype=torch.int32, device="cuda"), "next": torch.empty(batch, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"prefill": _prepare_linear, "step": _prepare_linear, "project": _prepare_project, "accept": _prepare_accept}[case["kind"]](case, gen)
    state["case"] = case
    if own:
        state["module"] = importlib.import_module(_PKG + {"prefill": ".linear", "step": ".linear", "project": ".proj", "accept": ".spec"}[case["kind"]])
        if case["kind"] == "prefill":
            size = state["module"].prefill_workspace_bytes(case["heads"], len(state["lens"]), max(state["lens"]))
            state["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        if case["kind"] == "project":
            state["weight"] = state["module"].Bf16Mat.dense(state["w"])
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------------


def _plain_prefill(s):
    """Chunks of 64 rows: with G the sum of the log decays up to and with a row,
    y_t = scale (e^G_t S q_t + sum over j <= t of e^(G_t - G_j) (q_t . k_j) v_j),  S' = e^G_C S + sum over j of e^(G_C - G_j) v_j k_j^T."""
    heads = s["v"].shape[1]
    share = heads // s["q"].shape[1]
    q, k, v = (t.float().transpose(0, 1) for t in (s["q"], s["k"], s["v"]))
    if share > 1:
        q, k = q.repeat_interleave(share, 0), k.repeat_interleave(share, 0)
    g = s["g"].double().expand(s["v"].shape[0], heads).t()
    mask = torch.ones(64, 64, dtype=torch.bool, device=q.device).tril()
    first = 0
    for b, n in enumerate(s["lens"]):
        state = s["state"][b].float()
        for at in range(first, first + n, 64):
            end = min(at + 64, first + n)
            c = end - at
            qc, kc, vc = q[:, at:end], k[:, at:end], v[:, at:end]
            total = g[:, at:end].cumsum(1)
            between = torch.exp(torch.where(mask[:c, :c], total[:, :, None] - total[:, None, :], -math.inf)).float()
            y = (torch.matmul(qc, kc.transpose(1, 2)) * between) @ vc
            y += torch.exp(total).float()[:, :, None] * (qc @ state.transpose(1, 2))
            s["out"][at:end] = (s["scale"] * y).transpose(0, 1)
            rest = torch.exp(total[:, -1:] - total).float()
            state = torch.exp(total[:, -1]).float()[:, None, None] * state + (vc * rest[:, :, None]).transpose(1, 2) @ kc
        s["state_out"][b] = state
        first += n
    return s["out"], s["state_out"]


def _plain_step(s):
    """S_t = e^g_t S_(t-1) + v_t k_t^T, y_t = scale S_t q_t; a bf16 state is rounded after each row, as serial steps leave it."""
    heads = s["v"].shape[1]
    share = heads // s["q"].shape[1]
    q, k, v = (t.float() for t in (s["q"], s["k"], s["v"]))
    if share > 1:
        q, k = q.repeat_interleave(share, 1), k.repeat_interleave(share, 1)
    decay = torch.exp(s["g"]).expand(v.shape[0], heads)
    lens, starts = s["lens"], []
    for n in lens:
        starts.append(sum(lens[:len(starts)]))
    state = s["state"].float().clone()
    for t in range(max(lens)):
        live = [b for b, n in enumerate(lens) if n > t]
        rows = [starts[b] + t for b in live]
        at = torch.tensor(rows, device=q.device)
        if len(live) == len(lens):
            new = decay[at][:, :, None, None] * state + v[at][:, :, :, None] * k[at][:, :, None, :]
        else:
            idx = torch.tensor(live, device=q.device)
            new = decay[at][:, :, None, None] * state[idx] + v[at][:, :, :, None] * k[at][:, :, None, :]
        new = new.to(s["state"].dtype).float()
        s["out"][at] = (s["scale"] * (new * q[at][:, :, None, :]).sum(-1)).bfloat16()
        if len(live) == len(lens):
            state = new
        else:
            state[idx] = new
    if not s["case"]["write"]:
        return s["out"]
    s["state_out"].copy_(state)
    return s["out"], s["state_out"]


def _plain_project(s):
    y = torch.matmul(s["x"].float(), s["w"].float().transpose(1, 2))
    if s["bias"] is not None:
        y = y + s["bias"].float()[:, None, :]
    act = s["case"]["act"]
    if act == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif act == "silu":
        y = y / (1 + torch.exp(-y))
    elif act == "sigmoid":
        y = 1 / (1 + torch.exp(-y))
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    s["out"].copy_(y)
    return s["out"]


def _plain_accept(s):
    """Row i of a window holds the target's distribution of the token behind it.  Token i + 1 is kept while u q < p; the next token
    is drawn from the weights max(p - q, 0) of the first row whose token is not kept, or from p behind a whole window.  In 64 bits: sums over a
    vocabulary decide between neighbours."""
    target, lens = s["target"].double(), s["lens"]
    rows, vocab = target.shape
    owner = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)], device=target.device)
    first = torch.tensor([sum(lens[:b]) for b in range(len(lens))], device=target.device)
    width = torch.tensor(lens, device=target.device)
    best = target.argmax(-1)
    if s["temperature"] is None:
        p, greedy = target, torch.zeros(len(lens), dtype=torch.bool, device=target.device)
    else:
        greedy = s["temperature"] == 0
        t = torch.where(greedy, 1.0, s["temperature"]).double()[owner]
        e = torch.exp((target - target.amax(-1, keepdim=True)) / t[:, None])
        p = e / e.sum(-1, keepdim=True)
    tokens = s["tokens"].long()
    at = torch.arange(rows, device=target.device)
    before = (at - 1).clamp(min=0)
    p_token = p[before, tokens]
    q_token = torch.ones_like(p_token) if s["draft"] is None else s["draft"][at, tokens].double()
    kept = torch.where(greedy[owner], best[before] == tokens, s["u"].double() * q_token < p_token)
    keep = torch.ones_like(width)
    alive = torch.ones_like(greedy)
    for i in range(1, max(lens)):
        alive = alive & (width > i) & kept[(first + i).clamp(max=rows - 1)]
        keep = keep + alive
    last = first + keep - 1
    whole = keep == width
    test = (last + 1).clamp(max=rows - 1)
    weight = p[last]
    if s["draft"] is None:
        less = weight.clone()
        less.scatter_(1, tokens[test][:, None], 0.0)
    else:
        less = (weight - s["draft"][test].double()).clamp(min=0)
    less = torch.where(less.sum(-1, keepdim=True) > 0, less, weight)
    weight = torch.where(whole[:, None], weight, less)
    total = weight.cumsum(-1)
    drawn = (total <= (s["u"][first].double() * total[:, -1])[:, None]).sum(-1).clamp(max=vocab - 1)
    s["keep"].copy_(keep)
    s["next"].copy_(torch.where(greedy, best[last], drawn))
    return s["keep"], s["next"]


# ---- the library's operators ------------------------------------------------------------------------------------------------


def _own_prefill(s):
    case = s["case"]
    s["module"].prefill_varlen(case["heads"], s["out"].shape[0], s["cu"], max(s["lens"]), s["q"], s["k"], s["v"], s["g"], s["state"], s["off"],
                               qk_heads=case["qk_heads"], state_out=s["state_out"], scale=s["scale"], out=s["out"], workspace=s["workspace"])
    return s["out"], s["state_out"]


def _own_step(s):
    case = s["case"]
    s["module"].decode_batch(case["heads"], s["out"].shape[0], s["cu"], s["q"], s["k"], s["v"], s["g"], s["state"], s["off"], qk_heads=case["qk_heads"],
                             state_out=s["state_out"] if case["write"] else None, scale=s["scale"], out=s["out"])
    return (s["out"], s["state_out"]) if case["write"] else s["out"]


def _own_project(s):
    case = s["case"]
    n, k, rows = case["n"], case["k"], case["rows"]
    s["module"].fused(s["x"], k, rows * k, s["weight"], rows, s["out"], n, rows * n, out_f32=case["out"] == "f32", bias=s["bias"], activation=case["act"],
                      residual=s["residual"])
    return s["out"]


def _own_accept(s):
    s["module"].accept_batch(s["cu"], s["tokens"], s["target"], s["u"], s["keep"], s["next"], probabilities=s["case"]["target"] == "probs",
                             draft=s["draft"], temperature=s["temperature"])
    return s["keep"], s["next"]


def run(state):
    plain = {"prefill": _plain_prefill, "step": _plain_step, "project": _plain_project, "accept": _plain_accept}
    kernels = {"prefill": _own_prefill, "step": _own_step, "project": _own_project, "accept": _own_accept}
    return (kernels if own else plain)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] in ("prefill", "step"):
        heads, lens = case["heads"], _lens(case)
        rows, size = sum(lens), 4 if case["state"] == "f32" else 2
        passes = 2 if case.get("write", True) else 1
        rows_bytes = rows * 2 * DIM * (2 * heads + 2 * case["qk_heads"]) + 4 * heads * (rows if case["decay"] == "token" else 1)
        return {"bytes": rows_bytes + passes * len(lens) * heads * DIM * DIM * size, "flops": rows * heads * DIM * DIM * 5}
    if case["kind"] == "project":
        groups, rows, n, k = case["groups"], case["rows"], case["n"], case["k"]
        size = 4 if case["out"] == "f32" else 2
        bias = {"none": 0, "bf16": 2, "f32": 4}[case["bias"]]
        return {"bytes": groups * (2 * k * (rows + n) + rows * n * size * (2 if case["residual"] else 1) + n * bias), "flops": 2 * groups * rows * n * k}
    lens, vocab = _lens(case), case["vocab"]
    if case["target"] == "probs":  # the tested tokens' entries, and one row of each distribution for the draw
        size = len(lens) * vocab * (8 if case["draft"] else 4) + 8 * sum(lens)
    else:
        size = sum(lens) * vocab * (2 if case["target"] == "logits_bf16" else 4) + (len(lens) * vocab * 4 if case["draft"] else 0)
    return {"bytes": size, "flops": 4 * size}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------------


def _exact_prefill(s):
    """All chunks of 32 rows side by side, then a scan over the states between them."""
    heads, c = s["v"].shape[1], 32
    group = torch.arange(heads, device=s["v"].device) // (heads // s["q"].shape[1])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["v"].device)
    ends = torch.zeros(s["state"].shape, dtype=torch.float64, device=s["v"].device)
    first = 0
    for b, n in enumerate(s["lens"]):
        if n == 0:
            ends[b] = s["state"][b].double()
            continue
        chunks = -(-n // c)
        for h in range(heads):
            def padded(t):
                z = torch.zeros(chunks * c, *t.shape[1:], dtype=torch.float64, device=t.device)
                z[:n] = t.double()
                return z.view(chunks, c, *t.shape[1:])

            q, k, v = (padded(t[first:first + n, i]) for t, i in ((s["q"], group[h]), (s["k"], group[h]), (s["v"], h)))
            g = padded(s["g"][first:first + n, h] if s["g"].dim() == 2 else s["g"][h].expand(n))
            upto = torch.cumsum(g, 1)
            pair = upto.unsqueeze(2) - upto.unsqueeze(1)
            pair = torch.tril(torch.exp(torch.tril(pair)))
            inside = torch.einsum("ctd,cjd,ctj,cje->cte", q, k, pair, v) if chunks == 1 else torch.bmm(torch.bmm(q, k.mT) * pair, v)
            add = torch.bmm((v * torch.exp(upto[:, -1:] - upto).unsqueeze(2)).mT, k)
            fade = torch.exp(upto[:, -1])
            starts = torch.empty_like(add)
            state = s["state"][b, h].double()
            for i in range(chunks):
                starts[i] = state
                state = fade[i] * state + add[i]
            y = inside + torch.exp(upto).unsqueeze(2) * torch.bmm(q, starts.mT)
            out[first:first + n, h] = s["scale"] * y.reshape(chunks * c, DIM)[:n]
            ends[b, h] = state
        first += n
    return out, ends


def _exact_step(s):
    heads = s["v"].shape[1]
    group = torch.arange(heads, device=s["v"].device) // (heads // s["q"].shape[1])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["v"].device)
    ends = torch.zeros(s["state"].shape, dtype=torch.float64, device=s["v"].device)
    row = 0
    for b, n in enumerate(s["lens"]):
        state = s["state"][b].double()
        for _ in range(n):
            g = (s["g"][row] if s["g"].dim() == 2 else s["g"]).double()
            state = torch.einsum("h,hij->hij", torch.exp(g), state) + torch.einsum("hi,hj->hij", s["v"][row].double(), s["k"][row][group].double())
            if s["state"].dtype == torch.bfloat16:
                state = state.bfloat16().double()
            out[row] = s["scale"] * torch.einsum("hij,hj->hi", state, s["q"][row][group].double())
            row += 1
        ends[b] = state
    return (out, ends) if s["case"]["write"] else out


def _exact_project(s):
    outs = []
    for i in range(s["x"].shape[0]):
        z = s["x"][i].double() @ s["w"][i].double().T
        if s["bias"] is not None:
            z += s["bias"][i].double()
        act = s["case"]["act"]
        if act == "relu":
            z = z.clamp(min=0)
        elif act == "sigmoid":
            z = torch.sigmoid(z)
        elif act == "silu":
            z = z * torch.sigmoid(z)
        elif act == "gelu":
            z = z * (0.5 * torch.erfc(-z / math.sqrt(2)))
        elif act == "gelu_tanh":
            z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        outs.append(z if s["residual"] is None else z + s["residual"][i].double())
    return torch.stack(outs)


def _exact_accept(s):
    keeps, nexts = [], []
    first = 0
    for b, n in enumerate(s["lens"]):
        heat = None if s["temperature"] is None else float(s["temperature"][b])
        tokens, u = s["tokens"][first:first + n].tolist(), s["u"][first:first + n].double().tolist()

        def p_of(i):
            row = s["target"][first + i].double()
            return row if heat is None else torch.softmax(row / heat, 0)

        kept = 1
        if heat == 0:
            best = [int(s["target"][first + i].float().max(0).values.eq(s["target"][first + i].float()).nonzero()[0]) for i in range(n)]
            while kept < n and tokens[kept] == best[kept - 1]:
                kept += 1
            nexts.append(best[kept - 1])
        else:
            while kept < n:
                q = 1.0 if s["draft"] is None else float(s["draft"][first + kept, tokens[kept]])
                if not u[kept] * q < float(p_of(kept - 1)[tokens[kept]]):
                    break
                kept += 1
            weight = p_of(kept - 1)
            if kept < n:
                if s["draft"] is not None:
                    rest = torch.relu(weight - s["draft"][first + kept].double())
                else:
                    rest = weight.clone()
                    rest[tokens[kept]] = 0
                weight = rest if float(rest.sum()) > 0 else weight
            upto = weight.cumsum(0)
            nexts.append(min(int(torch.searchsorted(upto, u[0] * upto[-1], right=True)), weight.numel() - 1))
        keeps.append(kept)
        first += n
    return torch.tensor(keeps, dtype=torch.int32, device="cuda"), torch.tensor(nexts, dtype=torch.int32, device="cuda")


def exact(case, seed):
    state = prepare(case, seed)
    return {"prefill": _exact_prefill, "step": _exact_step, "project": _exact_project, "accept": _exact_accept}[case["kind"]](state)
