"""The prefill product with its epilogue (lk_gemm_ex) against float64 of the f16 staging, elementwise, for every format
of the prefill GEMM."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from oracle import epilogue_oracle as E  # noqa: E402
from oracle import qmm_oracle as O  # noqa: E402

FMTS = ["q4_0", "q4_k", "iq4_nl", "q8_0", "q5_0", "q5_k", "q6_k", "iq4_xs", "q3_k", "iq3_s", "mxfp4"]
SCALE_OFFS = {"q5_0": [0], "q8_0": [0], "q5_k": [0, 2], "q6_k": [208], "iq4_xs": [0], "iq4_nl": [0], "q4_0": [0],
              "q4_k": [0, 2], "q3_k": [108], "iq3_s": [0]}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from loom_skills_b200 import ops as _ops
    return _ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def blocks(fmt, rows, k, seed):
    rng = np.random.default_rng(seed)
    nb = rows * k // O.QK[fmt]
    b = rng.integers(0, 256, (nb, O.BLOCK_BYTES[fmt]), dtype=np.uint8)
    if fmt == "mxfp4":
        b[:, 0] = rng.integers(118, 122, nb)
        return b.reshape(rows, -1)
    top = 2e-2 / {"q8_0": 64, "q6_k": 64 * 32, "q4_k": 32, "q5_k": 64, "iq4_xs": 32 * 64, "iq4_nl": 64, "q3_k": 64,
                  "iq3_s": 128}.get(fmt, 8)
    for o in SCALE_OFFS[fmt]:
        b[:, o:o + 2] = (rng.uniform(top / 8, top, nb) * rng.choice([-1, 1], nb)).astype(np.float16).view(np.uint8) \
            .reshape(-1, 2)
    return b.reshape(rows, -1)


def case(fmt, rows, k, n, seed=0, pair=False, bias=False, res=None):
    rng = np.random.default_rng([seed, n, k, rows])
    x = rng.standard_normal((rows, k)).astype(np.float32) * rng.choice([0.1, 1, 6e4], (rows, 1)).astype(np.float32)
    x16, scales = O.row_scale_f16(x)
    c = dict(fmt=fmt, rows=rows, k=k, n=n, x16=x16, scales=scales, w=blocks(fmt, n, k, seed + 1),
             w2=blocks(fmt, n, k, seed + 2) if pair else None)
    c["bias"] = rng.standard_normal(n).astype(np.float32) if bias else None
    c["bias2"] = rng.standard_normal(n).astype(np.float32) if bias and pair else None
    c["res"] = dev(rng.standard_normal((rows, n)).astype(np.float32) * 3).to(DT[res]) if res else None
    return c


def run(ops, c, act=None, out="f32", **kw):
    t = lambda a: None if a is None else dev(a)  # noqa: E731
    return ops.gemm_ex(c["fmt"], dev(c["x16"]), dev(c["scales"]), dev(c["w"]), c["n"], w2=t(c["w2"]), bias=t(c["bias"]),
                       bias2=t(c["bias2"]), act=act, residual=c["res"], out_dtype=DT[out], **kw)


def check(ops, c, act=None, out="f32", rel=None, **kw):
    y = run(ops, c, act, out, **kw)
    g, eg = E.product_f16(c["fmt"], c["w"], c["x16"], c["scales"], c["k"])
    u = eu = None
    if c["w2"] is not None:
        u, eu = E.product_f16(c["fmt"], c["w2"], c["x16"], c["scales"], c["k"])
    res = None if c["res"] is None else c["res"].double().cpu().numpy()
    v, ev = E.epilogue(g, eg, act or ("none" if u is None else "silu"), u, eu, c["bias"], c["bias2"], res)
    got = y.double().cpu().numpy()
    ok, far = E.within(got, v, ev, out)
    assert ok, far
    if rel:   # the plain GEMM's parity bar against the f16-staged product
        assert O.rel_l2(got, v) <= rel
    assert ops.device_status() == 0
    return y


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,k,n", [(1, 256, 1), (5, 256, 33), (64, 1024, 128), (129, 768, 300), (257, 2048, 256),
                                      (300, 512, 515), (31, 4096, 1000), (16, 12288, 48)])
def test_products(ops, fmt, rows, k, n):
    check(ops, case(fmt, rows, k, n, 3), rel=1e-5)


@pytest.mark.parametrize("fmt", ["q4_0", "iq4_nl", "q8_0", "q5_0", "mxfp4"])
@pytest.mark.parametrize("rows,k,n", [(3, 64, 7), (130, 192, 64), (70, 2880, 130), (260, 704, 40)])
def test_widths_of_single_stages(ops, fmt, rows, k, n):
    check(ops, case(fmt, rows, k, n, 5), rel=1e-5)
    check(ops, case(fmt, rows, k, n, 6, pair=True), out="bf16")


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k", "q6_k", "iq4_xs"])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_erf", "relu"])
def test_activation_bias_residual(ops, fmt, act):
    check(ops, case(fmt, 70, 512, 100, 7, bias=True, res="f32"), act, "f32")
    check(ops, case(fmt, 200, 512, 70, 8, bias=True, res="bf16"), act, "bf16")
    check(ops, case(fmt, 300, 256, 65, 9, res="bf16"), act, "f16")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("act", ["silu", "gelu", "swiglu_oai", "none"])
@pytest.mark.parametrize("rows,k,n", [(65, 512, 64), (256, 256, 129), (300, 1024, 200)])
def test_pairs(ops, fmt, act, rows, k, n):
    c = case(fmt, rows, k, n, 11, pair=True, bias=True)
    check(ops, c, act)
    check(ops, case(fmt, rows, k, n, 12, pair=True, res="f16"), act, "bf16")


@pytest.mark.parametrize("rows,k,n", [(2048, 4096, 1024), (1000, 1024, 4100), (4097, 256, 257)])
@pytest.mark.parametrize("pair", [False, True])
def test_many_tiles(ops, rows, k, n, pair):
    check(ops, case("q4_k", rows, k, n, 13, pair=pair, bias=True, res="bf16"), out="bf16")


@pytest.mark.parametrize("fmt", [f for f in FMTS if f != "mxfp4"])
def test_weights_off_the_vector_boundary(ops, fmt):
    c = case(fmt, 70, 512, 50, 15)
    want = run(ops, c)
    w = c["w"]
    big = torch.zeros(w.size + 16, dtype=torch.uint8, device="cuda")
    for off in (2, 6, 8):
        big[off:off + w.size] = dev(w).view(-1)
        got = ops.gemm_ex(fmt, dev(c["x16"]), dev(c["scales"]), big[off:off + w.size], c["n"])
        assert O.rel_l2(got.cpu().numpy(), want.cpu().numpy()) <= 1e-5


def test_rows_do_not_meet(ops):
    """A row of infinities or NaN leaves the others as they are, and nothing past the last row is written."""
    c = case("q4_0", 140, 512, 96, 17, bias=True)
    clean = run(ops, c)
    c["x16"][3, 7] = np.inf
    c["x16"][130, 0] = np.nan
    buf = torch.full((150, 96), 5.0, device="cuda")
    y = run(ops, c, y=buf[:140])
    keep = [i for i in range(140) if i not in (3, 130)]
    assert torch.equal(y[keep], clean[keep])
    assert not torch.isfinite(y[3]).any() and y[130].isnan().all()
    assert (buf[140:] == 5).all()


def test_in_place_residual(ops):
    for rows, k, n in ((100, 4096, 128), (700, 512, 300)):
        c = case("q4_k", rows, k, n, 19, res="bf16")
        want = run(ops, c, out="bf16")
        s = c["res"].clone()
        c["res"] = s
        got = run(ops, c, out="bf16", y=s)
        assert got is s and torch.equal(got, want)
    assert ops.gemm_ex("q4_k", dev(c["x16"])[:0], dev(c["scales"])[:0], dev(c["w"]), c["n"]).shape == (0, 300)


def test_results_repeat_on_other_streams_and_in_graphs(ops):
    for rows in (90, 600):
        c = case("q4_k", rows, 4096, 512, 21, pair=True, bias=True)
        x, sc, w, w2, b, b2 = (dev(c[i]) for i in ("x16", "scales", "w", "w2", "bias", "bias2"))
        call = lambda a: ops.gemm_ex("q4_k", a, sc, w, 512, w2=w2, bias=b, bias2=b2, out_dtype=torch.bfloat16)  # noqa: E731
        want = call(x)
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams * 4:                 # calls that overlap
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(call(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, want) for a in got)
        xs = torch.zeros_like(x)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = call(xs)
            graphs.append((g, y))
        xs.copy_(x)
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for _, y in graphs)
        assert ops.device_status() == 0


def test_refusals(ops):
    c = case("q4_k", 4, 512, 64, 23)
    x, sc, w = dev(c["x16"]), dev(c["scales"]), dev(c["w"])
    bad = [dict(n=65), dict(n=64, bias=torch.zeros(63, device="cuda")), dict(n=64, w2=w[:10]), dict(n=64, act="swiglu_oai"),
           dict(n=64, residual=torch.zeros(3, 64, device="cuda")), dict(n=64, out_dtype="q8"),
           dict(n=64, out_dtype=torch.float64), dict(n=64, y=torch.zeros(4, 64, device="cuda", dtype=torch.half))]
    for kw in bad:
        with pytest.raises(ops.L.LkError):
            ops.gemm_ex("q4_k", x, sc, w, **kw)
    with pytest.raises(ops.L.LkError):
        ops.gemm_ex("q4_k", x.float(), sc, w, 64)
    with pytest.raises(ops.L.LkError):
        ops.gemm_ex("q4_k", x, sc[:3], w, 64)
    with pytest.raises(ops.L.LkError):
        ops.gemm_ex("q4_k", x[:, :500], sc, w, 64)


# row strides of every remainder by 16 bytes: one to eight phases
STRIDES = [("q4_0", 320), ("q4_0", 640), ("iq4_nl", 704), ("q8_0", 320), ("q8_0", 1152), ("q5_0", 320), ("q6_k", 768),
           ("q6_k", 512), ("q3_k", 768), ("iq3_s", 512), ("iq4_xs", 768), ("mxfp4", 320), ("mxfp4", 384)]


@pytest.mark.parametrize("fmt,k", STRIDES)
@pytest.mark.parametrize("rows,n", [(40, 3), (33, 131), (300, 700), (600, 9), (257, 2050)])
def test_row_strides_of_every_phase(ops, fmt, k, rows, n):
    check(ops, case(fmt, rows, k, n, 41, bias=True, res="f32"), "gelu")
    check(ops, case(fmt, rows, k, n, 42, pair=True, bias=True), "silu", "bf16")


@pytest.mark.parametrize("fmt,k,off", [("q4_0", 320, 2), ("q8_0", 320, 6), ("iq4_nl", 704, 14), ("q6_k", 768, 10),
                                       ("mxfp4", 320, 3), ("q4_k", 512, 8)])
def test_weights_off_the_16_byte_boundary(ops, fmt, k, off):
    c = case(fmt, 70, k, 150, 43, pair=True)
    want = run(ops, c)

    def moved(a):
        buf = torch.zeros(a.size + 64, dtype=torch.uint8, device="cuda")
        buf[off:off + a.size] = dev(a).view(-1)
        return buf[off:off + a.size]

    y = ops.gemm_ex(fmt, dev(c["x16"]), dev(c["scales"]), moved(c["w"]), 150, w2=moved(c["w2"]))
    assert torch.equal(y, want)               # the same products in the same order, however the rows are fetched
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt,rows,k,n,pair", [("q4_0", 2048, 896, 4864, False), ("iq4_nl", 1500, 2688, 9000, True),
                                               ("mxfp4", 2048, 384, 6000, False), ("q4_0", 60, 896, 40000, False),
                                               ("iq4_nl", 120, 384, 60000, True), ("q5_0", 30, 640, 60000, False),
                                               ("mxfp4", 64, 2432, 30000, False), ("q8_0", 1024, 896, 4000, True)])
def test_rows_that_end_in_a_chunk_of_two_stages(ops, fmt, rows, k, n, pair):
    """Several tiles a cluster and k % 256 == 128, while another stream keeps the memory busy: bit for bit the quiet result."""
    c = case(fmt, rows, k, n, 51, pair=pair)
    x, sc, w = dev(c["x16"]), dev(c["scales"]), dev(c["w"])
    w2 = dev(c["w2"]) if pair else None
    call = lambda: ops.gemm_ex(fmt, x, sc, w, n, w2=w2)  # noqa: E731
    want = call()
    cols = np.arange(0, n, 61)
    g, eg = E.product_f16(fmt, c["w"][cols], c["x16"], c["scales"], k)
    u, eu = E.product_f16(fmt, c["w2"][cols], c["x16"], c["scales"], k) if pair else (None, None)
    v, ev = E.epilogue(g, eg, "silu" if pair else "none", u, eu)
    ok, far = E.within(want[:, torch.from_numpy(cols).cuda()].double().cpu().numpy(), v, ev, "f32")
    assert ok, far
    a, b = (torch.empty(256 << 20, dtype=torch.uint8, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    busy = torch.cuda.Stream()
    with torch.cuda.stream(busy):
        for _ in range(100):
            b.copy_(a)
    for _ in range(60):
        assert torch.equal(call(), want)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
