"""What the fused norm and the epilogue products refuse, on the host before any launch (CPU only)."""
import pytest

from loom_skills_b200 import _lib as L

X, R, W, Y, H, S = 4096, 8192, 12288, 16384, 20480, 24576   # distinct aligned addresses that are never read


def norm(rows=2, k=64, x=X, xd=L.F32, r=None, rd=L.F32, w=W, wd=L.F32, eps=1e-6, h=None, form=L.BF16, y=Y, s=S):
    return L.load().lk_rms_norm(rows, k, x, xd, r, rd, w, wd, eps, h, form, y, s, None)


def mv(fmt=L.Q4_K, n=64, k=256, tokens=2, xq=X, w=W, w2=None, b=None, b2=None, act=L.ACT_NONE, r=None, rd=L.F32, y=Y,
       form=L.F32):
    return L.load().lk_mv_q8_ex(fmt, n, k, tokens, xq, w, w2, b, b2, act, 1.702, 7.0, r, rd, y, form, None)


def gemm(fmt=L.Q4_K, n=64, k=256, rows=2, x=X, s=S, w=W, w2=None, b=None, b2=None, act=L.ACT_NONE, r=None, rd=L.F32,
         y=Y, form=L.F32):
    return L.load().lk_gemm_ex(fmt, rows, k, n, x, s, w, w2, b, b2, act, 1.702, 7.0, r, rd, y, form, None)


EINVAL, EALIGN, EUNSUP, ERANGE = -1, -2, -4, -5


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), EINVAL), (dict(k=0), EINVAL), (dict(eps=-1.0), EINVAL), (dict(eps=float("nan")), EINVAL),
    (dict(xd=99), EINVAL), (dict(wd=L.E4M3), EINVAL), (dict(r=R, rd=99), EINVAL), (dict(form=99), EINVAL),
    (dict(form=L.Q8_ROWS, k=48), EINVAL), (dict(h=H), EINVAL), (dict(k=32769), ERANGE),
    (dict(x=None), EINVAL), (dict(w=None), EINVAL), (dict(y=None), EINVAL),
    (dict(form=L.F16_ROWS, s=None), EINVAL), (dict(form=L.E4M3, s=None), EINVAL),
    (dict(x=X + 2), EALIGN), (dict(w=W + 1, wd=L.BF16), EALIGN), (dict(r=R + 2), EALIGN), (dict(y=Y + 1), EALIGN),
    (dict(r=R, h=H + 2), EALIGN), (dict(form=L.Q8_ROWS, y=Y + 8), EALIGN), (dict(form=L.E4M3, s=S + 2), EALIGN),
    (dict(r=R, rd=L.BF16, h=X), EINVAL),          # h over x of another type
    (dict(y=X, form=L.BF16), EINVAL),             # y over x of another type
    (dict(r=R, y=R), EINVAL), (dict(r=R, h=H, y=H), EINVAL),
])
def test_norm(kw, code):
    assert norm(**kw) == code


@pytest.mark.parametrize("call", [mv, gemm])
@pytest.mark.parametrize("kw,code", [
    (dict(n=0), EINVAL), (dict(n=2**30 + 32), ERANGE), (dict(k=0), EINVAL), (dict(k=128), EINVAL), (dict(form=99), EINVAL), (dict(form=L.E4M3), EINVAL),
    (dict(act=99), EINVAL), (dict(act=-1), EINVAL), (dict(act=L.ACT_SWIGLU_OAI), EINVAL),   # needs a pair
    (dict(b2=16), EINVAL),                        # bias2 without w2
    (dict(r=R, rd=99), EINVAL), (dict(r=Y, rd=L.BF16), EINVAL),   # in place of another type
    (dict(r=R + 2), EALIGN), (dict(b=18), EALIGN), (dict(y=Y + 2), EALIGN), (dict(w=W + 1), EALIGN),
    (dict(w2=W + 1), EALIGN), (dict(x=X + 8), EALIGN), (dict(x=None), EINVAL), (dict(w=None), EINVAL),
    (dict(y=None), EINVAL), (dict(fmt=L.fmt_pair(L.Q4_K, L.Q6_K)), None), (dict(fmt=99), None), (dict(fmt=L.MXFP4S), None),
])
def test_products(call, kw, code):
    if call is mv:
        kw = {("xq" if a == "x" else a): v for a, v in kw.items()}
    rc = call(**kw)
    assert rc == code if code is not None else rc in (EINVAL, EUNSUP)


def test_decode_only():
    assert mv(tokens=-1) == EINVAL
    assert mv(form=L.Q8_ROWS, n=48) == EINVAL
    assert mv(form=L.Q8_ROWS, y=Y + 8) == EALIGN
    assert mv(fmt=L.Q8_0, k=48) == EINVAL
    for fmt in (L.Q3_K, L.IQ3_S, L.MXFP4):        # no integer codes
        assert mv(fmt=fmt) == EUNSUP


def test_prefill_only():
    assert gemm(rows=-1) == EINVAL
    assert gemm(form=L.Q8_ROWS) == EINVAL
    assert gemm(fmt=L.Q8_0, k=32) == EINVAL       # k % 64
    assert gemm(s=None) == EINVAL


def test_empty_calls_succeed():
    assert norm(rows=0, x=None, y=None, w=None) == 0
    assert mv(tokens=0, xq=None, w=None, y=None) == 0
    assert gemm(rows=0, x=None, s=None, w=None, y=None) == 0


def test_ops_take_cuda_tensors_only():
    torch = pytest.importorskip("torch")
    from loom_skills_b200 import ops
    x, w = torch.zeros(2, 64), torch.zeros(64)
    with pytest.raises(L.LkError):
        ops.rms_norm(x, w)
    q = torch.zeros(2 * 64 + 2 * 2 * 8, dtype=torch.uint8)
    with pytest.raises(L.LkError):
        ops.mv_q8_ex("q8_0", torch.zeros(4, 68, dtype=torch.uint8), q, 4, 64, 2)
    with pytest.raises(L.LkError):
        ops.gemm_ex("q8_0", x.half(), torch.ones(2, 2), torch.zeros(4, 68, dtype=torch.uint8), 4)


# operands far apart, of the sizes that the calls below read and write
FX, FW, FW2, FY, FR, FB, FS, FH = (i << 24 for i in range(1, 9))


@pytest.mark.parametrize("at", [FX, FX + 64, FX + 2 * 256 - 256, FW, FW + 64 * 144 - 16, FW2, FB, FB + 128, FR + 256, FR - 256])
def test_products_written_over_their_operands(at):
    assert mv(xq=FX, w=FW, w2=FW2, b=FB, r=FR, y=at) == EINVAL
    assert gemm(x=FX, w=FW, w2=FW2, b=FB, r=FR, s=FS, y=at) == EINVAL


def test_a_product_written_over_its_input_rows():
    assert mv(xq=FX, n=256, w=FW, y=FX, form=L.Q8_ROWS) == EINVAL
    assert gemm(x=FX, s=FS, w=FW, y=FS) == EINVAL and gemm(x=FX, s=FS, w=FW, y=FX, form=L.F16) == EINVAL


@pytest.mark.parametrize("kw", [
    dict(y=FX + 16), dict(y=FX - 16), dict(y=FR), dict(y=FR + 128), dict(y=FW), dict(y=FH), dict(y=FH + 64), dict(h=FX + 64),
    dict(h=FR + 64), dict(h=FW), dict(form=L.F16_ROWS, s=FX), dict(form=L.F16_ROWS, s=FR + 4), dict(form=L.E4M3, s=FW),
    dict(form=L.E4M3, s=FH + 4), dict(form=L.E4M3, s=FY + 4)])
def test_norms_written_over_their_operands(kw):
    args = dict(x=FX, xd=L.BF16, r=FR, rd=L.BF16, w=FW, h=FH, y=FY, s=FS, form=L.BF16)
    assert norm(**{**args, **kw}) == EINVAL
