"""What the Python entry points of the gated recurrence, the log probabilities and the 4-bit projections refuse of CUDA tensors: nothing is launched, and what would have
been written is as it was."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BF, F32, I32, I64, U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return {n: importlib.import_module("glm53f-afd_b200." + n) for n in ("gated", "spec", "proj", "core")}


def z(*shape, dtype=BF):
    return torch.full(shape, 3, dtype=dtype, device="cuda")


def refused(mods, call, written):
    before = {n: t.clone() for n, t in written.items() if t is not None}
    with pytest.raises(mods["core"].Invalid):
        call()
    torch.cuda.synchronize()
    for n, t in before.items():
        assert torch.equal(written[n], t), n


ROWS = {
    "gates of f16": dict(g=lambda: z(9, 64, dtype=torch.float16)), "too few rows": dict(x=lambda: z(8, 64)), "another width": dict(g=lambda: z(9, 65)), "rows that overlap": dict(x=lambda: z(4096).as_strided((9, 64), (32, 1))),
    "columns apart": dict(g=lambda: z(9, 128)[:, ::2]), "on the host": dict(x=lambda: torch.zeros(9, 64, dtype=BF)), "no inputs": dict(x=lambda: None), "no gates": dict(g=lambda: None),
    "offsets of 32 bits": dict(off=lambda: z(2, dtype=I32)), "too few offsets": dict(off=lambda: z(1, dtype=I64)), "row ranges of 64 bits": dict(cu=lambda: z(3, dtype=I64)), "no channels": dict(channels=lambda: 0),
    "fewer than no rows": dict(rows=lambda: -1), "another gate": dict(gate=lambda: "tanh"), "another input": dict(input=lambda: "half"), "a region beyond the state": dict(far=lambda: 65), "a negative region": dict(far=lambda: -1),
}
STATES = {"a state of bf16": dict(state=lambda: z(2, 64)), "a state with holes": dict(state=lambda: z(2, 128, dtype=F32)[:, ::2]), "a state on the host": dict(state=lambda: torch.zeros(2, 64)), "outputs of another type": dict(out=lambda: z(9, 64, dtype=F32)),
          "too few outputs": dict(out=lambda: z(8, 64)), "a smaller state_out": dict(so=lambda: z(1, 64, dtype=F32)), "a state_out that overlaps": dict(so="overlap")}
LONG = {"a longer sequence than rows": dict(most=lambda: 10), "a workspace on the host": dict(ws=lambda: torch.zeros(1 << 16, dtype=U8)), "a workspace off 16 bytes": dict(ws=lambda: z((1 << 16) + 8, dtype=U8)[8:]), "too few saves": dict(saves=lambda: z(1, 64, dtype=F32)),
        "saves of bf16": dict(saves=lambda: z(9, 64)), "saves off 8 bytes": dict(saves=lambda: z(9 * 64 + 1, dtype=F32)[1:])}
BACK = {"no saves": dict(saves=lambda: None), "a gradient of g of another type": dict(dg=lambda: z(9, 64, dtype=F32)), "a gradient of x of another type": dict(dx=lambda: z(9, 64, dtype=F32)), "too few gradients": dict(dy=lambda: z(8, 64)), "no dout": dict(dy=lambda: None),
        "end states' gradient of bf16": dict(ds=lambda: z(2, 64)), "a dstate_in that overlaps": dict(di="overlap")}


def values(what, **base):
    whole = z(3, 64, dtype=F32)
    a = {k: v for k, v in base.items()}
    for k, v in what.items():
        a[k] = whole[1:] if v == "overlap" else v()
        if v == "overlap":
            a["state" if k == "so" else "ds"] = whole[:2]
    return a


@pytest.mark.parametrize("prefill", [False, True], ids=["step", "prefill"])
@pytest.mark.parametrize("what", [*ROWS, *STATES, *LONG, "nothing to write", "keep of 64 bits"])
def test_scan(mods, what, prefill):
    change = {**ROWS, **STATES, **LONG}.get(what, {})
    if what == "keep of 64 bits" and prefill or what in LONG and not prefill:
        pytest.skip("not an argument of this form")
    a = values(change, channels=64, rows=9, cu=torch.tensor([0, 4, 9], dtype=I32, device="cuda"), most=5, g=z(9, 64), x=z(9, 64), state=z(2, 64, dtype=F32), off=torch.tensor([0, 64], device="cuda"),
               out=z(9, 64), so="in_place", gate="decay", input="plain", far=64, ws=None, saves=None, keep=None)
    if what == "nothing to write":
        a["so"] = a["out"] = None
    if what == "keep of 64 bits":
        a["keep"] = z(2, dtype=I64)
    kinds = dict(gate=a["gate"], input=a["input"], state_out=a["so"], out=a["out"], max_state_off=a["far"])
    if prefill:
        call = lambda: mods["gated"].prefill_varlen(a["channels"], a["rows"], a["cu"], a["most"], a["g"], a["x"], a["state"], a["off"], saves=a["saves"], workspace=a["ws"], **kinds)
    else:
        call = lambda: mods["gated"].decode_batch(a["channels"], a["rows"], a["cu"], a["g"], a["x"], a["state"], a["off"], keep=a["keep"], **kinds)
    refused(mods, call, {"out": a["out"], "state": a["state"], "saves": a["saves"]})


@pytest.mark.parametrize("what", [*ROWS, *LONG, *BACK])
def test_scan_backward(mods, what):
    a = values({**ROWS, **LONG, **BACK}[what], channels=64, rows=9, cu=torch.tensor([0, 4, 9], dtype=I32, device="cuda"), most=5, g=z(9, 64), x=z(9, 64), off=torch.tensor([0, 64], device="cuda"), dy=z(9, 64), dg=z(9, 64), dx=z(9, 64),
               saves=z(4, 64, dtype=F32), ds=z(2, 64, dtype=F32), di=z(2, 64, dtype=F32), gate="decay", input="plain", far=64, ws=None)
    call = lambda: mods["gated"].backward_varlen(a["channels"], a["rows"], a["cu"], a["most"], a["g"], a["x"], a["saves"], a["off"], a["dy"], a["dg"], a["dx"], gate=a["gate"], input=a["input"], dstate=a["ds"], dstate_in=a["di"],
                                                 workspace=a["ws"], max_state_off=a["far"])
    refused(mods, call, {"dg": a["dg"], "dx": a["dx"], "dstate_in": a["di"]})


LOGITS = {
    "logits of f16": dict(logits=lambda: z(3, 50, dtype=torch.float16)), "logits on the host": dict(logits=lambda: torch.zeros(3, 50)), "columns apart": dict(logits=lambda: z(3, 100)[:, ::2]), "one dimension": dict(logits=lambda: z(50)),
    "tokens of 64 bits": dict(tokens=lambda: z(3, dtype=I64)), "too few tokens": dict(tokens=lambda: z(2, dtype=I32)), "temperatures of bf16": dict(heat=lambda: z(3)), "too few temperatures": dict(heat=lambda: z(2, dtype=F32)),
}
FORWARD = {"no tokens": dict(tokens=lambda: None), "nowhere for the tokens'": dict(lp=lambda: None), "too few results": dict(lp=lambda: z(2, dtype=F32)), "entropies of f64": dict(h=lambda: z(3, dtype=torch.float64)), "a list of 33": dict(top=lambda: (z(3, 33, dtype=I32), z(3, 33, dtype=F32))),
           "lists of two lengths": dict(top=lambda: (z(3, 4, dtype=I32), z(3, 5, dtype=F32))), "indices of 64 bits": dict(top=lambda: (z(3, 4, dtype=I64), z(3, 4, dtype=F32))), "lists of fewer rows": dict(top=lambda: (z(2, 4, dtype=I32), z(2, 4, dtype=F32)))}
GRADS = {"no sums": dict(lse=lambda: None), "a gradient of another type": dict(d=lambda: z(3, 50, dtype=F32)), "of another shape": dict(d=lambda: z(3, 51)), "none": dict(d=lambda: None), "no gradient to pass on": dict(dlp=lambda: None), "an entropy's without it": dict(dh=lambda: z(3, dtype=F32)),
         "a gradient that overlaps": dict(d="overlap")}


@pytest.mark.parametrize("what", [*LOGITS, *FORWARD, "nothing to write"])
def test_logprobs(mods, what):
    a = dict(logits=z(3, 50), tokens=z(3, dtype=I32), lp=z(3, dtype=F32), heat=None, h=z(3, dtype=F32), lse=z(3, dtype=F32), top=(z(3, 4, dtype=I32), z(3, 4, dtype=F32)))
    a.update({k: v() for k, v in {**LOGITS, **FORWARD}.get(what, {}).items()})
    if what == "nothing to write":
        a.update(tokens=None, lp=None, h=None, lse=None, top=None)
    call = lambda: mods["spec"].logprobs(a["logits"], a["tokens"], a["lp"], temperature=a["heat"], entropy=a["h"], lse=a["lse"], top=a["top"])
    refused(mods, call, {"lp": a["lp"], "h": a["h"], "lse": a["lse"], **({"ids": a["top"][0], "values": a["top"][1]} if a["top"] else {})})


@pytest.mark.parametrize("what", [*LOGITS, *GRADS])
def test_logprobs_backward(mods, what):
    room = z(4, 50)
    a = dict(logits=room[:3], tokens=z(3, dtype=I32), lse=z(3, dtype=F32), dlp=z(3, dtype=F32), d=z(3, 50), heat=None, h=None, dh=None)
    a.update({k: room[1:] if v == "overlap" else v() for k, v in {**LOGITS, **GRADS}[what].items()})
    call = lambda: mods["spec"].logprobs_backward(a["logits"], a["tokens"], a["lse"], a["dlp"], a["d"], temperature=a["heat"], entropy=a["h"], dentropy=a["dh"])
    refused(mods, call, {"d": a["d"]})


INT4 = {
    "x of f32": dict(x=lambda: z(3, 128, dtype=F32)), "x on the host": dict(x=lambda: torch.zeros(3, 128, dtype=BF)), "x with holes": dict(x=lambda: z(3, 256)[:, ::2]), "too little x": dict(x=lambda: z(2, 128)), "rows of x too short": dict(ldx=lambda: 120),
    "rows of x off 16 bytes": dict(ldx=lambda: 132, x=lambda: z(3, 132)), "x off 16 bytes": dict(xo=lambda: 4, x=lambda: z(4, 128)), "a negative offset": dict(xo=lambda: -8), "rows of out too short": dict(ldo=lambda: 9), "too little out": dict(out=lambda: z(2, 10)),
    "out of f32": dict(out=lambda: z(3, 10, dtype=F32)), "out of bf16": dict(f32=lambda: True), "out beyond its end": dict(oo=lambda: 1), "fewer than no rows": dict(rows=lambda: -1), "a weight cut short": dict(cut=lambda: 1), "more inputs than the weight": dict(k=lambda: 4096, ldx=lambda: 4096, x=lambda: z(3, 4096)),
}


@pytest.mark.parametrize("what", INT4)
def test_int4(mods, what):
    a = dict(x=z(3, 128), ldx=128, rows=3, out=z(3, 10), ldo=10, f32=False, xo=0, oo=0, cut=0, k=128)
    a.update({k: v() for k, v in INT4[what].items()})
    m = mods["proj"].Int4Mat.pack(z(10, 64, dtype=U8), z(10, 2), group=64)
    m = mods["proj"].Int4Mat(m.t[:m.t.numel() - a["cut"]], m.n, a["k"], m.group, m.zeros)
    refused(mods, lambda: mods["proj"].int4(a["x"], a["ldx"], m, a["rows"], a["out"], a["ldo"], a["f32"], a["xo"], a["oo"]), {"out": a["out"]})


PACK = {
    "codes of 16 bits": dict(codes=lambda: z(10, 64, dtype=torch.int16)), "codes on the host": dict(codes=lambda: torch.zeros(10, 64, dtype=U8)), "codes with holes": dict(codes=lambda: z(10, 128, dtype=U8)[:, ::2]), "no rows": dict(codes=lambda: z(0, 64, dtype=U8)),
    "k not of whole pieces": dict(codes=lambda: z(10, 48, dtype=U8)), "scales of f32": dict(scales=lambda: z(10, 2, dtype=F32)), "too few scales": dict(scales=lambda: z(10, 1)), "zero points of 32 bits": dict(zeros=lambda: z(10, 2, dtype=I32)),
    "too few zero points": dict(zeros=lambda: z(9, 2, dtype=U8)), "another group": dict(group=lambda: 48),
}


@pytest.mark.parametrize("what", PACK)
def test_pack(mods, what):
    a = dict(codes=z(10, 64, dtype=U8), scales=z(10, 2), zeros=None, group=64)
    a.update({k: v() for k, v in PACK[what].items()})
    with pytest.raises(mods["core"].Invalid):
        mods["proj"].Int4Mat.pack(a["codes"], a["scales"], a["zeros"], group=a["group"])
    for w in (z(10, 100), z(128), z(10, 128, dtype=BF).cpu()):
        with pytest.raises(mods["core"].Invalid):
            mods["proj"].Int4Mat.quantise(w, group=64)
