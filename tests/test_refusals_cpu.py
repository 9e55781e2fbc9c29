"""What the entry points of the linear attention, the verification of drafted tokens and the fused projection refuse: every refusal comes
before anything touches a device, so none is needed here.  Addresses are numbers that nothing reads."""
import ctypes
import importlib

import pytest

AT = 1 << 20  # an aligned address


@pytest.fixture(scope="module")
def ffi(pkg):
    m = importlib.import_module("glm53f-afd_b200.ffi")
    m.load()
    return m


def call(fn, names, good, **changed):
    assert set(changed) <= set(names), changed
    return fn(*[changed.get(n, good[n]) for n in names])


STEP = ("heads qk_heads batch cu keep q q_stride k k_stride v v_stride g g_stride state_in state_out state_off bf16 scale out out_stride stream").split()
PREFILL = ("heads qk_heads batch cu rows max_len q q_stride k k_stride v v_stride g g_stride state_in state_out state_off bf16 scale out out_stride "
           "workspace nbytes stream").split()
LINEAR = dict(heads=4, qk_heads=2, batch=3, cu=AT, keep=None, rows=100, max_len=90, q=AT, q_stride=256, k=AT, k_stride=256, v=AT, v_stride=512, g=AT, g_stride=4,
              state_in=AT, state_out=AT, state_off=AT, bf16=0, scale=1.0, out=AT, out_stride=512, workspace=None, nbytes=0, stream=None)
BAD_LINEAR = [dict(heads=0, qk_heads=1), dict(heads=65536), dict(qk_heads=0), dict(qk_heads=3), dict(qk_heads=8), dict(batch=-1), dict(heads=65535, qk_heads=1, batch=1 << 20),
              dict(cu=None), dict(q=None), dict(q=AT + 8), dict(q_stride=248), dict(q_stride=260), dict(k=None), dict(k=AT + 2), dict(k_stride=0), dict(v=None), dict(v_stride=256),
              dict(v=AT + 4), dict(g=None), dict(g_stride=3), dict(g_stride=-4), dict(state_in=None), dict(state_off=None), dict(out=AT + 8), dict(out_stride=504), dict(out_stride=516)]


@pytest.mark.parametrize("bad", BAD_LINEAR, ids=str)
def test_linear_attention(ffi, bad):
    assert call(ffi.glm53f_kda_lin_decode_batch, STEP, LINEAR, **bad) == 1
    assert call(ffi.glm53f_kda_lin_prefill_varlen, PREFILL, LINEAR, **bad) == 1


@pytest.mark.parametrize("bad", [dict(rows=-1, max_len=-1), dict(max_len=-1), dict(max_len=101), dict(nbytes=-1), dict(nbytes=4096), dict(workspace=AT + 8, nbytes=4096),
                                 dict(state_out=None), dict(out=None)], ids=str)
def test_linear_prefill(ffi, bad):
    assert call(ffi.glm53f_kda_lin_prefill_varlen, PREFILL, LINEAR, **bad) == 1


def test_linear_steps_that_write_nothing(ffi):
    assert call(ffi.glm53f_kda_lin_decode_batch, STEP, LINEAR, state_out=None, out=None) == 1


@pytest.mark.parametrize("bad", [(0, 1, 100), (65536, 1, 100), (4, 0, 100), (4, 1, 0), (-1, 1, 100), (4, 1, -5)])
def test_linear_workspace_of_nothing(ffi, bad):
    assert ffi.glm53f_kda_lin_prefill_workspace_bytes(*bad) == 0


ACCEPT = "batch cu vocab target kind ld tokens draft draft_ld temperature u keep next stream".split()
JUDGED = dict(batch=2, cu=AT, vocab=100, target=AT, kind=1, ld=100, tokens=AT, draft=None, draft_ld=0, temperature=None, u=AT, keep=AT, next=AT, stream=None)


@pytest.mark.parametrize("bad", [dict(batch=-1), dict(batch=1 << 28), dict(vocab=0), dict(vocab=-3), dict(vocab=0x7fffffc1, ld=1 << 31), dict(ld=99), dict(kind=3), dict(kind=-1), dict(kind=0, temperature=AT),
                                 dict(draft=AT, draft_ld=99), dict(cu=None), dict(target=None), dict(tokens=None), dict(u=None), dict(keep=None), dict(next=None),
                                 dict(target=AT + 2), dict(kind=0, target=AT + 1), dict(kind=2, target=AT + 1), dict(draft=AT + 2, draft_ld=100)], ids=str)
def test_accept(ffi, bad):
    assert call(ffi.glm53f_kda_accept_batch, ACCEPT, JUDGED, **bad) == 1


JOB = dict(x=AT, ldx=128, x_gstride=0, w=AT, ldw=128, w_gstride=0, groups=1, rows=4, n=64, k=128, out=AT, out_f32=0, ldo=64, o_gstride=0)


def job_of(ffi, **changed):
    j = ffi.ProjJob()
    for name, value in {**JOB, **changed}.items():
        setattr(j, name, value)
    return j


@pytest.mark.parametrize("job,epilogue", [
    (dict(), dict(activation=6)), (dict(), dict(activation=-1)), (dict(), dict(bias=AT + 1)), (dict(), dict(bias=AT + 2, bias_f32=1)),
    (dict(groups=2), dict(bias=AT, bias_gstride=-64)), (dict(), dict(residual=AT + 1, ldr=64)), (dict(out_f32=1), dict(residual=AT + 2, ldr=64)),
    (dict(), dict(residual=AT, ldr=63)), (dict(groups=2), dict(residual=AT, ldr=64, r_gstride=-1)), (dict(x=None), dict()), (dict(w=AT + 8), dict()), (dict(n=60), dict()),
    (dict(k=100), dict()), (dict(ldx=120), dict()), (dict(ldo=56), dict()), (dict(rows=-1), dict()), (dict(groups=0), dict())], ids=str)
def test_fused_projection(ffi, job, epilogue):
    j, e = job_of(ffi, **job), ffi.ProjEpilogue(**epilogue)
    assert ffi.glm53f_kda_proj_bf16_fused(j, e, None) == 1


def test_fused_projection_without_arguments(ffi):
    none = lambda kind: ctypes.cast(None, ctypes.POINTER(kind))
    assert ffi.glm53f_kda_proj_bf16_fused(none(ffi.ProjJob), ffi.ProjEpilogue(), None) == 1
    assert ffi.glm53f_kda_proj_bf16_fused(job_of(ffi), none(ffi.ProjEpilogue), None) == 1


def test_the_calls_of_nothing_succeed(ffi):
    """No requests, or no rows of a projection: nothing is read, nothing is launched."""
    nothing = dict(batch=0, cu=None, q=None, k=None, v=None, g=None, state_in=None, state_out=None, state_off=None, out=None)
    assert call(ffi.glm53f_kda_lin_decode_batch, STEP, LINEAR, **nothing) == 0
    assert call(ffi.glm53f_kda_lin_prefill_varlen, PREFILL, LINEAR, **nothing) == 0
    assert call(ffi.glm53f_kda_accept_batch, ACCEPT, JUDGED, batch=0, cu=None, target=None, tokens=None, u=None, keep=None, next=None) == 0
    assert ffi.glm53f_kda_proj_bf16_fused(job_of(ffi, rows=0), ffi.ProjEpilogue(), None) == 0


# ---- the Python entry points: tensors of the host are refused by name --------------------------------------------------------------------

def test_python_refusals(pkg):
    torch = pytest.importorskip("torch")
    linear, spec, proj = (importlib.import_module("glm53f-afd_b200." + n) for n in ("linear", "spec", "proj"))
    cu, off = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    rows = torch.zeros(4, 128, dtype=torch.bfloat16)
    args = (rows, rows, rows, torch.zeros(4, 1), torch.zeros(1, 128, 128), off)
    for fn in (lambda **kw: linear.decode_batch(1, 4, cu, *args, out=rows, **kw), lambda **kw: linear.prefill_varlen(1, 4, cu, 4, *args, out=rows, **kw)):
        with pytest.raises(linear.Invalid):
            fn()
        with pytest.raises(linear.Invalid, match="do not divide"):
            fn(qk_heads=2)
    with pytest.raises(linear.Invalid, match="max_len 5 of 4 rows"):
        linear.prefill_varlen(1, 4, cu, 5, *args, out=rows)
    with pytest.raises(linear.Invalid, match="out is required"):
        linear.prefill_varlen(1, 4, cu, 4, *args)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(spec.Invalid):
        spec.accept_batch(cu, torch.zeros(4, dtype=torch.int32), torch.zeros(4, 9), torch.zeros(4), one, one)
    w = proj.Bf16Mat.dense(torch.zeros(64, 128, dtype=torch.bfloat16))
    x, out = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.bfloat16)
    proj.fused(x, 128, 0, w, 0, out, 64, 0)  # no rows: nothing happens
    for message, kw in (("one of none, relu", dict(activation="swish")), ("bias must be 1 x 64", dict(bias=torch.zeros(63))), ("bias must be", dict(bias=torch.zeros(64).double())),
                        ("out's type", dict(residual=out.float())), ("smaller", dict(residual=out[:3])), ("smaller", dict(residual=out, residual_offset=1)),
                        ("smaller", dict(residual=out, ldr=63))):
        with pytest.raises(proj.Invalid, match=message):
            proj.fused(x, 128, 0, w, 4, out, 64, 0, **kw)
    with pytest.raises(proj.Invalid, match="smaller"):
        proj.fused(x, 128, 0, w, 5, out, 64, 0)
    for kw in (dict(x_offset=-128), dict(out_offset=-64)):  # before the tensor
        with pytest.raises(proj.Invalid, match="not negative"):
            proj.fused(x, 128, 0, w, 2, out, 64, 0, **kw)
    with pytest.raises(proj.Invalid, match="not negative"):
        proj.fused(x, 128, -128, w, 2, out, 64, 0)


def test_accepting_without_a_round(pkg, monkeypatch):
    torch = pytest.importorskip("torch")
    kernel, marks, verify = (importlib.import_module("glm53f-afd_b200." + n) for n in ("kernel", "marks", "verify"))
    monkeypatch.setattr(kernel, "DEVICE", "cpu")
    pool = marks.KvPool(marks.KvConfig(marks.KvLayout.new(1, 0), 2, 2))
    vf = verify.KdaVerify(pool, [None], 8, 2)
    tokens, target, u, one = torch.zeros(5, dtype=torch.int32), torch.zeros(5, 9), torch.zeros(5), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(verify.Invalid, match="no verify is open"):
        vf.accept(tokens, target, u, one, one)
    vf.verify([(pool.slot(), 2), (pool.slot(), 4)])
    with pytest.raises(verify.Invalid, match="5 tokens and 5 rows of the target for 6 rows"):
        vf.accept(tokens, target, u, one, one)
