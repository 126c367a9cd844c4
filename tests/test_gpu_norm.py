"""The fused residual + RMS norm + activation format (lk_rms_norm) against float64, and its quantised forms bit for bit
against the framework's producers run on the same f32 norm."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from oracle import epilogue_oracle as E  # noqa: E402

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from loom_skills_b200 import ops as _ops
    return _ops


def make(rows, k, xd, rd, wd, seed=0, amp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 131 + k)
    x = (torch.randn(rows, k, device="cuda", generator=g) * amp).to(DT[xd])
    r = (torch.randn(rows, k, device="cuda", generator=g) * 3 * amp).to(DT[rd]) if rd else None
    w = (1 + 0.3 * torch.randn(k, device="cuda", generator=g)).to(DT[wd])
    return x, r, w


def f64(t):
    return t.double().cpu().numpy()


SIZES = [(1, 1), (3, 7), (2, 32), (1, 4096), (5, 100), (17, 2880), (257, 256), (3, 8200), (2, 16384), (1, 32768),
         (2, 20001), (4, 8192), (3, 4100),
         # many rows (the kernel that walks them), from several rings an SM to one row a ring
         (5000, 64), (1500, 256), (9000, 8), (900, 2048), (700, 4096), (601, 5120), (400, 16384), (300, 32768),
         # ... of odd widths
         (700, 4097), (1200, 99), (300, 16001), (900, 356), (2000, 33), (256, 32767)]


@pytest.mark.parametrize("rows,k", SIZES)
@pytest.mark.parametrize("xd,rd,wd,form", [("bf16", "bf16", "f32", "bf16"), ("f32", "", "bf16", "f32"),
                                           ("f16", "f32", "f16", "f16"), ("f32", "bf16", "f32", "f32"),
                                           ("bf16", "f16", "f32", "f32")])
def test_plain_forms(ops, rows, k, xd, rd, wd, form):
    x, r, w = make(rows, k, xd, rd, wd)
    got = ops.rms_norm(x, w, 1e-5, residual=r, form=form)
    y, h = got if r is not None else (got, None)
    h64, v64 = E.rms_norm(f64(x), f64(w), np.float32(1e-5), None if r is None else f64(r))
    ok, far = E.within(f64(y), v64, E.NORM_REL * np.abs(v64), form)
    assert ok, far
    if r is not None:
        # one f32 sum and one rounding to the residual's type (which is none for f32)
        assert torch.equal(h, (x.float() + r.float()).to(DT[rd]))


@pytest.mark.parametrize("rows,k", [s for s in SIZES if s[1] % 32 == 0])
@pytest.mark.parametrize("xd,rd", [("bf16", "bf16"), ("f32", ""), ("f16", "f32")])
def test_q8_form_is_quant_q8_of_the_norm(ops, rows, k, xd, rd):
    x, r, w = make(rows, k, xd, rd, "f32", 5)
    x[0, : min(32, k)] = 0
    if r is not None:
        r[0, : min(32, k)] = 0     # an all-zero group
    one = lambda form: (lambda o: o[0] if r is not None else o)(ops.rms_norm(x, w, 1e-6, residual=r, form=form))  # noqa: E731
    assert torch.equal(one("q8"), ops.quant_q8(one("f32")))


@pytest.mark.parametrize("rows,k", SIZES)
@pytest.mark.parametrize("amp", [1.0, 1e-20, 1e12])
def test_row_forms_are_the_producers_of_the_norm(ops, rows, k, amp):
    x, r, w = make(rows, k, "f32", "f32", "f32", 9, amp)
    w = w * 3e4            # row maxima past 2^13: the f16 scale is not 1
    v, _ = ops.rms_norm(x, w, 0.0, residual=r, form="f32")
    (x16, sc), _ = ops.rms_norm(x, w, 0.0, residual=r, form="row_f16")
    (x8, s8), _ = ops.rms_norm(x, w, 0.0, residual=r, form="row_f8")
    e16, esc = ops.row_scale_f16(v)
    e8, es8 = ops.row_scale_f8(v)
    assert torch.equal(x16.view(torch.int16), e16.view(torch.int16)) and torch.equal(sc, esc)
    assert torch.equal(x8, e8) and torch.equal(s8, es8)


def test_zero_rows_infinities_and_nan(ops):
    x, r, w = make(6, 256, "f32", "f32", "f32")
    x[1], r[1] = 0, 0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    x[4] = 1e30                      # squares pass f32
    y, h = ops.rms_norm(x, w, 1e-6, residual=r, form="f32")
    assert (y[1] == 0).all()
    ref, _ = ops.rms_norm(x[[0, 5]].contiguous(), w, 1e-6, residual=r[[0, 5]].contiguous(), form="f32")
    assert torch.equal(y[[0, 5]], ref)          # the other rows are untouched by these
    assert y[3].isnan().all() and y[2, 7].isnan() and (y[2, :7] == 0).all() and (y[4] == 0).all()
    for form in ("q8", "row_f16", "row_f8"):
        out, _ = ops.rms_norm(x, w, 1e-6, residual=r, form=form)
        want = {"q8": ops.quant_q8, "row_f16": ops.row_scale_f16, "row_f8": ops.row_scale_f8}[form](y)
        for a, b in zip(out if isinstance(out, tuple) else (out,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("k,off", [(4096, 1), (4096, 4), (96, 3), (1000, 8)])
@pytest.mark.parametrize("form", ["bf16", "q8", "row_f16", "row_f8"])
def test_operands_off_the_vector_boundary(ops, k, off, form):
    """Contiguous operands that start `off` elements into their storage give what aligned copies give."""
    if form == "q8" and k % 32:
        k = k // 32 * 32
    rows = 3
    def shifted(t):
        big = torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")
        big[off:] = t.reshape(-1)
        return big[off:].view(t.shape)
    x, r, w = make(rows, k, "bf16", "bf16", "f32", 3)
    a, ha = ops.rms_norm(x, w, 1e-6, residual=r, form="f32")
    b, hb = ops.rms_norm(shifted(x), shifted(w), 1e-6, residual=shifted(r), form="f32", h=shifted(torch.zeros_like(r)))
    assert torch.equal(ha, hb)
    # the rows' squares are summed in another order: both are within the bound of the exact value
    h64, v64 = E.rms_norm(f64(x), f64(w), np.float32(1e-6), f64(r))
    for y in (a, b):
        ok, far = E.within(f64(y), v64, E.NORM_REL * np.abs(v64), "f32")
        assert ok, far
    c, _ = ops.rms_norm(shifted(x), shifted(w), 1e-6, residual=shifted(r), form=form)
    if form == "bf16":
        assert E.within(f64(c), v64, E.NORM_REL * np.abs(v64), "bf16")[0]
    elif form == "q8":
        codes, meta = ops.q8_views(c, rows, k)
        val = (codes.view(rows, -1, 32).double() * meta[..., :1].double()).view(rows, k).cpu().numpy()
        d = np.abs(v64).reshape(rows, -1, 32).max(-1, keepdims=True) / 127
        # half a code of rounding, and the scale's f16 rounding times the code
        lim = (0.5 + 127 * 2.0 ** -11 + 1e-3) * d + 2.0 ** -25 * 127
        assert (np.abs(val - v64).reshape(rows, -1, 32) <= lim).all()
    else:
        val = f64(c[0] if form == "row_f16" else c[0].view(torch.float8_e4m3fn))
        s = f64(c[1])[:, :1]
        rel = 2.0 ** -11 if form == "row_f16" else 2.0 ** -4
        tiny = 2.0 ** -25 if form == "row_f16" else 2.0 ** -10
        assert (np.abs(val - v64 * s) <= (rel * 1.001) * np.abs(v64 * s) + tiny).all()


def test_in_place_and_strides(ops):
    x, r, w = make(33, 512, "bf16", "bf16", "bf16", 7)
    y0, h0 = ops.rms_norm(x, w, residual=r, form="f16")
    r1 = r.clone()
    y1, h1 = ops.rms_norm(x, w, residual=r1, form="f16", h=r1)
    assert h1 is r1 and torch.equal(h1, h0) and torch.equal(y1, y0)
    x1 = x.clone()
    y2, h2 = ops.rms_norm(x1, w, residual=r, form="f16", h=x1)
    assert torch.equal(x1, h0) and torch.equal(y2, y0)
    x2 = x.clone()
    y3, h3 = ops.rms_norm(x2, w, residual=r, form="bf16", y=x2)
    assert torch.equal(x2, ops.rms_norm(x, w, residual=r, form="bf16")[0]) and torch.equal(h3, h0)
    xt = torch.empty(512, 33, dtype=x.dtype, device="cuda").t()
    xt.copy_(x)
    y4, _ = ops.rms_norm(xt, w, residual=r, form="f16")
    assert torch.equal(y4, y0)


def test_rows_past_the_last_are_left(ops):
    x, _, w = make(3, 96, "f32", "", "f32")
    big = torch.full((5, 96), 7.0, device="cuda")
    ops.rms_norm(x, w, form="f32", y=big[:3])
    assert (big[3:] == 7).all() and not (big[:3] == 7).any()
    buf = torch.full((3 * 96 + 3 * 3 * 8 + 64,), 9, dtype=torch.uint8, device="cuda")
    ops.rms_norm(x, w, form="q8", y=buf)
    assert (buf[-64:] == 9).all()
    assert ops.rms_norm(x[:0], w, form="f32").shape == (0, 96)


def test_refusals(ops):
    x, r, w = make(2, 64, "f32", "bf16", "f32")
    bad = [dict(form="int4"), dict(h=r), dict(residual=r[:1]), dict(residual=r, h=torch.empty_like(x)),
           dict(residual=r.double()), dict(form="q8", y=torch.empty(8, dtype=torch.uint8, device="cuda")),
           dict(form="row_f16", y=torch.empty_like(x)), dict(form="bf16", y=torch.empty_like(x))]
    for kw in bad:
        with pytest.raises(ops.L.LkError):
            ops.rms_norm(x, w, **kw)
    with pytest.raises(ops.L.LkError):
        ops.rms_norm(x, w[:63])
    with pytest.raises(ops.L.LkError):
        ops.rms_norm(x.double(), w)
    with pytest.raises(ops.L.LkError):
        ops.rms_norm(x[:, :48], w[:48], form="q8")
    with pytest.raises(ops.L.LkError):
        ops.rms_norm(torch.zeros(1, 32769, device="cuda"), torch.zeros(32769, device="cuda"))


def test_captured_replays_and_another_stream(ops):
    x, r, w = make(4, 4096, "bf16", "bf16", "f32", 11)
    want = ops.rms_norm(x, w, residual=r, form="q8")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.rms_norm(x, w, residual=r, form="q8")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0])
    g = torch.cuda.CUDAGraph()
    xs, rs = torch.zeros_like(x), torch.zeros_like(r)
    with torch.cuda.graph(g):
        out, h = ops.rms_norm(xs, w, residual=rs, form="q8")
        out2, h2 = ops.rms_norm(h, w, residual=rs, form="q8", h=h)     # reads what the first launch wrote, in place
    for scale in (1.0, 2.0):
        xs.copy_(x * scale)
        rs.copy_(r)
        g.replay()
        a, ha = ops.rms_norm((x * scale), w, residual=r, form="q8")
        b, hb = ops.rms_norm(ha, w, residual=r, form="q8")
        assert torch.equal(out, a) and torch.equal(out2, b) and torch.equal(h, hb)


@pytest.mark.parametrize("rows,k", [(600, 2048), (300, 8192), (500, 2049), (300, 8190)])
def test_many_rows_in_place(ops, rows, k):
    """The stream updated in its own buffer and the norm written over x, while later rows are already being fetched."""
    x, r, w = make(rows, k, "bf16", "f32", "f32", 31)
    y0, h0 = ops.rms_norm(x, w, 1e-6, residual=r)
    xs, rs = x.clone(), r.clone()
    y, h = ops.rms_norm(xs, w, 1e-6, residual=rs, h=rs, y=xs)
    assert y.data_ptr() == xs.data_ptr() and h.data_ptr() == rs.data_ptr()
    assert torch.equal(y, y0) and torch.equal(h, h0)
    xs = x.clone()                            # h over x
    y, h = ops.rms_norm(xs, w, 1e-6, residual=x * 0.5, h=xs)
    y0, h0 = ops.rms_norm(x, w, 1e-6, residual=x * 0.5)
    assert torch.equal(y, y0) and torch.equal(h, h0)
    # two graphs of one buffer, replayed on two streams one after the other
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.rms_norm(x, w, 1e-6, residual=r)
        graphs.append((g, out))
    for g, out in graphs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        assert torch.equal(out[0], ops.rms_norm(x, w, 1e-6, residual=r)[0])
    assert ops.device_status() == 0
