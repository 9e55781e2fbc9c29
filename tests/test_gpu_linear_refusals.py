"""What the Python entry points of the linear attention, the verification of drafted tokens and the fused projection refuse of CUDA tensors: nothing is
launched, and what would have been written is as it was."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return {n: importlib.import_module("glm53f-afd_b200." + n) for n in ("linear", "spec", "proj", "core")}


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


LINEAR = {
    "q of f32": dict(q=lambda: z(9, 256, dtype=torch.float32)), "too few rows": dict(k=lambda: z(8, 256)), "another width": dict(v=lambda: z(9, 256)),
    "rows that overlap": dict(q=lambda: z(4096).as_strided((9, 256), (128, 1))), "an odd stride": dict(k=lambda: z(9, 260)[:, :256]),
    "an odd address": dict(v=lambda: z(9 * 512 + 8)[4:-4].view(9, 512)), "columns apart": dict(q=lambda: z(9, 512)[:, ::2]), "on the host": dict(q=lambda: torch.zeros(9, 256, dtype=torch.bfloat16)),
    "decays of bf16": dict(g=lambda: z(9, 4)), "decays of fewer heads": dict(g=lambda: z(9, 3, dtype=torch.float32)), "too few decays": dict(g=lambda: z(8, 4, dtype=torch.float32)),
    "decay columns apart": dict(g=lambda: z(9, 8, dtype=torch.float32)[:, ::2]), "a state of f64": dict(state=lambda: z(2, 4, 128, 128, dtype=torch.float64)),
    "a state on the host": dict(state=lambda: torch.zeros(2, 4, 128, 128)), "a state with holes": dict(state=lambda: z(2, 8, 128, 128, dtype=torch.float32)[:, ::2]),
    "offsets of 32 bits": dict(off=lambda: z(2, dtype=torch.int32)), "too few offsets": dict(off=lambda: z(1, dtype=torch.int64)), "row ranges of 64 bits": dict(cu=lambda: z(3, dtype=torch.int64)),
    "outputs of f32": dict(out=lambda: z(9, 512, dtype=torch.float32)), "too few outputs": dict(out=lambda: z(8, 512)),
    "a region beyond the state": dict(max_state_off=65537), "a negative region": dict(max_state_off=-1), "another type of state_out": dict(state_out=lambda: z(2, 4, 128, 128)),
    "a smaller state_out": dict(state_out=lambda: z(1, 4, 128, 128, dtype=torch.float32)), "heads that do not divide": dict(qk_heads=3),
}


@pytest.mark.parametrize("prefill", [False, True], ids=["step", "prefill"])
@pytest.mark.parametrize("what", LINEAR)
def test_linear(mods, what, prefill):
    a = dict(q=z(9, 256), k=z(9, 256), v=z(9, 512), g=z(9, 4, dtype=torch.float32), state=z(2, 4, 128, 128, dtype=torch.float32), off=z(2, dtype=torch.int64),
             cu=torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda"), out=z(9, 512) + 7, qk_heads=2)
    a.update({k: v() if callable(v) else v for k, v in LINEAR[what].items()})
    before = a["state"].clone(), a["out"].clone()
    rest = {k: a[k] for k in ("out", "qk_heads", "state_out", "max_state_off") if k in a}
    with pytest.raises(mods["linear"].Invalid):
        if prefill:
            mods["linear"].prefill_varlen(4, 9, a["cu"], 5, a["q"], a["k"], a["v"], a["g"], a["state"], a["off"], **rest)
        else:
            mods["linear"].decode_batch(4, 9, a["cu"], a["q"], a["k"], a["v"], a["g"], a["state"], a["off"], **rest)
    torch.cuda.synchronize()
    assert torch.equal(a["state"], before[0]) and torch.equal(a["out"], before[1])


def test_linear_of_one_kind(mods):
    lin, Invalid = mods["linear"], mods["linear"].Invalid
    a = (z(9, 256), z(9, 256), z(9, 512), z(9, 4, dtype=torch.float32), z(2, 4, 128, 128, dtype=torch.float32), z(2, dtype=torch.int64))
    cu, pool = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda"), z(3, 4, 128, 128, dtype=torch.float32)
    with pytest.raises(Invalid, match="neither states nor outputs"):
        lin.decode_batch(4, 9, cu, *a, qk_heads=2, state_out=None)
    with pytest.raises(Invalid, match="keep"):
        lin.decode_batch(4, 9, cu, *a, qk_heads=2, keep=z(1, dtype=torch.int32))
    with pytest.raises(Invalid, match="writes the state"):
        lin.prefill_varlen(4, 9, cu, 5, *a, qk_heads=2, state_out=None, out=z(9, 512))
    with pytest.raises(Invalid, match="memory of its own"):  # one slot further on in the same memory
        lin.prefill_varlen(4, 9, cu, 5, *a[:4], pool[:2], a[5], qk_heads=2, state_out=pool[1:], out=z(9, 512))
    with pytest.raises(Invalid, match="workspace"):
        lin.prefill_varlen(4, 9, cu, 5, *a, qk_heads=2, out=z(9, 512), workspace=torch.zeros(64, dtype=torch.uint8))
    for max_len in (-1, 10):
        with pytest.raises(Invalid, match="max_len"):
            lin.prefill_varlen(4, 9, cu, max_len, *a, qk_heads=2, out=z(9, 512))


ACCEPT = {
    "tokens of 64 bits": dict(tokens=lambda: z(9, dtype=torch.int64)), "probabilities of bf16": dict(target=lambda: z(9, 50), probabilities=True), "logits of f16": dict(target=lambda: z(9, 50, dtype=torch.float16)),
    "too few rows": dict(target=lambda: z(8, 50)), "a flat target": dict(target=lambda: z(450)), "entries apart": dict(target=lambda: z(9, 100)[:, ::2]), "no vocabulary": dict(target=lambda: z(9, 0)),
    "rows that overlap": dict(target=lambda: z(450).as_strided((9, 50), (40, 1))), "another vocabulary drafted": dict(draft=lambda: z(9, 49, dtype=torch.float32)),
    "a draft of bf16": dict(draft=lambda: z(9, 50)), "too few drafted": dict(draft=lambda: z(8, 50, dtype=torch.float32)), "too few numbers": dict(u=lambda: z(8, dtype=torch.float32)),
    "numbers of f64": dict(u=lambda: z(9, dtype=torch.float64)), "too few kept": dict(keep=lambda: z(1, dtype=torch.int32)), "kept of 64 bits": dict(keep=lambda: z(2, dtype=torch.int64)),
    "too few next": dict(next=lambda: z(1, dtype=torch.int32)), "too few temperatures": dict(temperature=lambda: z(1, dtype=torch.float32)),
    "warm probabilities": dict(target=lambda: z(9, 50, dtype=torch.float32), probabilities=True, temperature=lambda: z(2, dtype=torch.float32)),
    "on the host": dict(target=lambda: torch.zeros(9, 50)), "ranges on the host": dict(cu=lambda: torch.zeros(3, dtype=torch.int32)),
}


@pytest.mark.parametrize("what", ACCEPT)
def test_accept(mods, what):
    a = dict(cu=torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda"), tokens=z(9, dtype=torch.int32), target=z(9, 50), u=z(9, dtype=torch.float32), keep=z(2, dtype=torch.int32) - 7,
             next=z(2, dtype=torch.int32) - 7)
    a.update({k: v() if callable(v) else v for k, v in ACCEPT[what].items()})
    before = a["keep"].clone()
    with pytest.raises(mods["spec"].Invalid):
        mods["spec"].accept_batch(a.pop("cu"), a.pop("tokens"), a.pop("target"), a.pop("u"), a["keep"], a["next"], **{k: a[k] for k in ("draft", "temperature", "probabilities") if k in a})
    torch.cuda.synchronize()
    assert torch.equal(a["keep"], before)


FUSED = {
    "an unknown activation": dict(activation="swish"), "a short bias": dict(bias=lambda: z(63)), "a bias with holes": dict(bias=lambda: z(128)[::2]), "a bias of f16": dict(bias=lambda: z(64, dtype=torch.float16)),
    "a bias on the host": dict(bias=lambda: torch.zeros(64)), "a residual of f32": dict(residual=lambda: z(4, 64, dtype=torch.float32)), "a short residual": dict(residual=lambda: z(3, 64)),
    "a residual on the host": dict(residual=lambda: torch.zeros(4, 64, dtype=torch.bfloat16)), "residual rows that overlap": dict(residual=lambda: z(8, 64), ldr=56),
    "a residual before its memory": dict(residual=lambda: z(4, 64), residual_offset=-64), "x on the host": dict(x=lambda: torch.zeros(4, 128, dtype=torch.bfloat16)),
}


@pytest.mark.parametrize("what", FUSED)
def test_fused_projection(mods, what):
    a = {k: v() if callable(v) else v for k, v in FUSED[what].items()}
    out = z(4, 64) + 7
    with pytest.raises(mods["proj"].Invalid):
        mods["proj"].fused(a.pop("x", z(4, 128)), 128, 0, mods["proj"].Bf16Mat.dense(z(64, 128)), 4, out, 64, 0, **a)
    torch.cuda.synchronize()
    assert (out == 7).all()
