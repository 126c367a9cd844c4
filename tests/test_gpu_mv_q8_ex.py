"""The decode product with its epilogue (lk_mv_q8_ex) against float64, elementwise within the f32 roundings it cannot do
without, for every format with integer codes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from oracle import epilogue_oracle as E  # noqa: E402
from oracle import qmm_oracle as O  # noqa: E402

FMTS = ["q4_0", "q4_k", "q8_0", "q5_0", "q5_k", "q6_k", "iq4_nl", "iq4_xs"]
SCALE_OFFS = {"q5_0": [0], "q8_0": [0], "q5_k": [0, 2], "q6_k": [208], "iq4_xs": [0], "iq4_nl": [0], "q4_0": [0],
              "q4_k": [0, 2]}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from loom_skills_b200 import ops as _ops
    return _ops


def blocks(fmt, rows, k, seed):
    """Random blocks of `fmt` (every code and sub-block scale) with finite f16 scales of both signs."""
    rng = np.random.default_rng(seed)
    nb = rows * k // O.QK[fmt]
    b = rng.integers(0, 256, (nb, O.BLOCK_BYTES[fmt]), dtype=np.uint8)
    top = 2e-2 / {"q8_0": 64, "q6_k": 64 * 32, "q4_k": 32, "q5_k": 64, "iq4_xs": 32 * 64, "iq4_nl": 64}.get(fmt, 8)
    for o in SCALE_OFFS[fmt]:
        b[:, o:o + 2] = (rng.uniform(top / 8, top, nb) * rng.choice([-1, 1], nb)).astype(np.float16).view(np.uint8) \
            .reshape(-1, 2)
    return b.reshape(rows, -1)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def case(fmt, n, k, tokens, seed=0, pair=False, bias=False, res=None):
    rng = np.random.default_rng([seed, n, k, tokens])
    x = rng.standard_normal((tokens, k)).astype(np.float32) * rng.choice([0.1, 1, 4], (tokens, 1)).astype(np.float32)
    codes, meta = O.quant_q8(x)
    c = dict(fmt=fmt, n=n, k=k, tokens=tokens, codes=codes, meta=meta, w=blocks(fmt, n, k, seed + 1),
             w2=blocks(fmt, n, k, seed + 2) if pair else None)
    c["bias"] = rng.standard_normal(n).astype(np.float32) if bias else None
    c["bias2"] = rng.standard_normal(n).astype(np.float32) if bias and pair else None
    c["res"] = dev(rng.standard_normal((tokens, n)).astype(np.float32) * 3).to(DT[res]) if res else None
    return c


def xq_of(c):
    return torch.cat([dev(c["codes"]).view(-1).view(torch.uint8), dev(c["meta"]).view(-1).view(torch.uint8)])


def run(ops, c, act=None, out="f32", **kw):
    t = lambda a: None if a is None else dev(a)  # noqa: E731
    return ops.mv_q8_ex(c["fmt"], dev(c["w"]), xq_of(c), c["n"], c["k"], c["tokens"], w2=t(c["w2"]), bias=t(c["bias"]),
                        bias2=t(c["bias2"]), act=act, residual=c["res"], out_dtype=DT.get(out, out), **kw)


def ref(c, act=None, alpha=1.702, limit=7.0):
    g, eg = E.product_q8(c["fmt"], c["w"], c["codes"], c["meta"], c["k"])
    u = eu = None
    if c["w2"] is not None:
        u, eu = E.product_q8(c["fmt"], c["w2"], c["codes"], c["meta"], c["k"])
    res = None if c["res"] is None else c["res"].double().cpu().numpy()
    return E.epilogue(g, eg, act or ("none" if u is None else "silu"), u, eu, c["bias"], c["bias2"], res, alpha, limit)


def check(ops, c, act=None, out="f32", **kw):
    y = run(ops, c, act, out, **kw)
    v, ev = ref(c, act)
    ok, far = E.within(y.double().cpu().numpy(), v, ev, out)
    assert ok, far
    assert ops.device_status() == 0
    return y


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,k,tokens", [(1, 256, 1), (33, 256, 3), (1024, 4096, 1), (100, 2560, 8), (47, 4096, 9),
                                        (96, 12288, 5), (130, 1024, 17), (64, 768, 32), (40, 512, 70), (5, 27648, 8)])
def test_products(ops, fmt, n, k, tokens):
    check(ops, case(fmt, n, k, tokens, 3))


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k", "iq4_nl", "q6_k"])
@pytest.mark.parametrize("n,k", [(1, 4096), (33, 8192), (4745, 4096), (2400, 8192), (512, 12288), (5, 16384), (2400, 16384),
                                 (512, 256), (4745, 2304), (2400, 5120), (33, 6400), (512, 13824), (1, 16128),
                                 (4745, 2048), (64, 6144), (2400, 14336)])
def test_one_token_of_long_rows(ops, fmt, k, n):
    check(ops, case(fmt, n, k, 1, 15, bias=True, res="f32"), "gelu")
    check(ops, case(fmt, n, k, 1, 16, pair=True, bias=True, res="bf16"), "swiglu_oai", "bf16")
    if n % 32 == 0:
        one = case(fmt, n, k, 1, 17, pair=True)
        assert torch.equal(run(ops, one, out="q8"), ops.quant_q8(run(ops, one)))
        single = case(fmt, n, k, 1, 18)
        assert torch.equal(run(ops, single, out="q8"), ops.quant_q8(run(ops, single)))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,k,tokens", [(4809, 256, 1), (4737, 1280, 8), (9500, 512, 3), (4769, 512, 17)])
def test_more_rows_than_one_tile_per_sm(ops, fmt, n, k, tokens):
    check(ops, case(fmt, n, k, tokens, 13))
    check(ops, case(fmt, n // 2 + 1, k, tokens, 14, pair=True, bias=True, res="bf16"), "silu", "bf16")


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0", "q5_0", "iq4_nl"])
@pytest.mark.parametrize("n,k,tokens", [(7, 32, 1), (64, 96, 8), (33, 2880, 5), (20, 1056, 33), (9, 16416, 2)])
def test_widths_of_single_blocks(ops, fmt, n, k, tokens):
    check(ops, case(fmt, n, k, tokens, 5), out="bf16")
    check(ops, case(fmt, n, k, tokens, 6, pair=True))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_erf", "relu"])
def test_activation_bias_residual(ops, fmt, act):
    check(ops, case(fmt, 70, 1024, 6, 7, bias=True, res="f32"), act, "f32")
    check(ops, case(fmt, 70, 1024, 1, 8, bias=True, res="bf16"), act, "bf16")
    check(ops, case(fmt, 70, 512, 11, 9, res="bf16"), act, "f16")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("act", ["silu", "gelu", "swiglu_oai", "none", "gelu_erf", "relu"])
@pytest.mark.parametrize("n,k,tokens", [(48, 1024, 1), (100, 512, 8), (33, 2304, 20)])
def test_pairs(ops, fmt, act, n, k, tokens):
    check(ops, case(fmt, n, k, tokens, 11, pair=True, bias=True), act)
    check(ops, case(fmt, n, k, tokens, 12, pair=True, res="f16"), act, "f16")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("n,k,tokens", [(32, 256, 1), (96, 1024, 8), (320, 4096, 3), (64, 512, 19)])
def test_q8_output_is_quant_q8_of_the_f32_output(ops, fmt, pair, n, k, tokens):
    c = case(fmt, n, k, tokens, 13, pair=pair, bias=True)
    f = run(ops, c, out="f32")
    assert torch.equal(run(ops, c, out="q8"), ops.quant_q8(f))


def test_saturated_activations_and_special_codes(ops):
    """Large products: exp over- and underflows to the limits; codes of -127 and 127 throughout; an all-zero token."""
    c = case("q8_0", 64, 512, 4, 17, pair=True, bias=True)
    c["codes"] = np.where(np.random.default_rng(1).random(c["codes"].shape) < 0.5, -127, 127).astype(np.int8)
    c["codes"][2] = 0
    c["meta"][..., 0] = 40.0
    c["meta"][..., 1] = c["codes"].reshape(4, -1, 32).astype(np.int32).sum(-1)
    for act in ("silu", "gelu", "swiglu_oai"):
        y = check(ops, c, act)
        assert torch.isfinite(y).all()
    for fmt in FMTS:     # the largest dots any format makes
        d = case(fmt, 32, 512, 3, 18)
        d["codes"] = np.full_like(d["codes"], 127)
        d["codes"][1] = -127
        d["meta"][..., 1] = d["codes"].reshape(3, -1, 32).astype(np.int32).sum(-1)
        check(ops, d)


def test_infinite_and_nan_scales_stay_in_their_token(ops):
    c = case("q4_k", 64, 1024, 8, 19)
    clean = run(ops, c)
    c["meta"][3, 5, 0] = np.inf
    c["meta"][6, 0, 0] = np.nan
    y = run(ops, c)
    keep = [0, 1, 2, 4, 5, 7]
    assert torch.equal(y[keep], clean[keep])
    assert not torch.isfinite(y[3]).any() and y[6].isnan().all()


@pytest.mark.parametrize("fmt", FMTS)
def test_weights_off_the_vector_boundary(ops, fmt):
    c = case(fmt, 50, 1024, 4, 21)
    w = c["w"]
    big = torch.zeros(w.size + 16, dtype=torch.uint8, device="cuda")
    want = run(ops, c)
    for off in (2, 6, 8):
        big[off:off + w.size] = dev(w).view(-1)
        got = ops.mv_q8_ex(fmt, big[off:off + w.size], xq_of(c), c["n"], c["k"], c["tokens"])
        assert torch.equal(got, want)


def test_in_place_residual_and_sentinels(ops):
    c = case("q4_k", 100, 512, 3, 23, res="bf16")
    want = run(ops, c, out="bf16")
    stream = torch.full((5, 100), 5.0, dtype=torch.bfloat16, device="cuda")
    stream[:3] = c["res"]
    got = ops.mv_q8_ex("q4_k", dev(c["w"]), xq_of(c), 100, 512, 3, residual=stream[:3], out_dtype=torch.bfloat16,
                       y=stream[:3])
    assert torch.equal(got, want) and (stream[3:] == 5).all()
    buf = torch.full((3 * 96 + 3 * 3 * 8 + 64,), 9, dtype=torch.uint8, device="cuda")
    d = case("q4_k", 96, 512, 3, 24)
    run(ops, d, out="q8", y=buf)
    assert (buf[-64:] == 9).all()
    assert ops.mv_q8_ex("q4_k", dev(c["w"]), xq_of(c), 100, 512, 0).shape == (0, 100)


def test_offsets_past_32_bits(ops):
    """Rows whose byte offset passes 2^32 in one packed weight."""
    n, k = 520000, 8192                       # 520000 * 8704 bytes = 4.5 GB of Q8_0
    c = case("q8_0", 8, k, 1, 25)
    rb = c["w"].shape[1]
    w = torch.zeros(n * rb, dtype=torch.uint8, device="cuda")
    rows = torch.cat([torch.arange(4), torch.arange(n - 4, n)])
    for i, r in enumerate(rows.tolist()):
        w[r * rb:(r + 1) * rb] = dev(c["w"][i])
    y = ops.mv_q8_ex("q8_0", w, xq_of(c), n, k, 1)
    # the split of k follows from n, so the order of the sums does too: each is held to the exact value, not to the other
    v, ev = ref(c)
    ok, far = E.within(y[:, rows.cuda()].double().cpu().numpy(), v, ev, "f32")
    assert ok, far
    assert int((y != 0).sum()) == int((v != 0).sum())


def test_results_repeat_on_other_streams_and_in_graphs(ops):
    c = case("q4_k", 1000, 4096, 8, 27, pair=True, bias=True)
    w, w2, xq, b, b2 = dev(c["w"]), dev(c["w2"]), xq_of(c), dev(c["bias"]), dev(c["bias2"])
    call = lambda q: ops.mv_q8_ex("q4_k", w, q, 1000, 4096, 8, w2=w2, bias=b, bias2=b2)  # noqa: E731
    want = call(xq)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 4:                     # calls that overlap
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call(xq))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) for a in got)
    q = torch.zeros_like(xq)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call(q)
        graphs.append((g, y))
    q.copy_(xq)
    torch.cuda.synchronize()
    for (g, _), s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for _, y in graphs)
    assert ops.device_status() == 0


def test_refusals(ops):
    c = case("q4_k", 64, 512, 2, 29)
    w, xq = dev(c["w"]), xq_of(c)
    ok = dict(n=64, k=512, tokens=2)
    bad = [dict(ok, n=65), dict(ok, tokens=3), dict(ok, k=500), dict(ok, bias=torch.zeros(63, device="cuda")),
           dict(ok, w2=w[:10]), dict(ok, residual=torch.zeros(2, 63, device="cuda")), dict(ok, act="swiglu_oai"),
           dict(ok, out_dtype=torch.float64), dict(ok, y=torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)),
           dict(ok, n=40, out_dtype="q8"), dict(ok, bias2=torch.zeros(64, device="cuda")),
           dict(ok, residual=torch.zeros(2, 64, device="cuda", dtype=torch.float64))]
    for kw in bad:
        with pytest.raises(ops.L.LkError):
            ops.mv_q8_ex("q4_k", w, xq, **kw)
    with pytest.raises(ops.L.LkError):
        ops.mv_q8_ex("q3_k", torch.zeros(64 * 220, dtype=torch.uint8, device="cuda"), xq, 64, 512, 2)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [4768, 9504])
@pytest.mark.parametrize("tokens", [1, 3, 8, 17, 32])
def test_q8_output_of_a_half_filled_last_tile(ops, fmt, n, tokens):
    """Outputs that end in the middle of a 64-row tile: the groups past the last one are nobody's, not the next token's."""
    k = 512
    c = case(fmt, n, k, tokens, 31)
    size = tokens * n + tokens * (n // 32) * 8
    buf = torch.full((size + 256,), 9, dtype=torch.uint8, device="cuda")
    run(ops, c, out="q8", y=buf)
    assert (buf[size:] == 9).all()
    assert torch.equal(buf[:size], ops.quant_q8(run(ops, c)))
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt,n,k,tokens", [("q8_0", 4096, 4096, 12), ("q4_k", 4096, 14336, 8), ("q4_0", 2048, 8192, 3),
                                            ("iq4_nl", 1500, 13824, 5), ("q4_k", 4096, 5120, 16), ("q6_k", 4096, 8192, 10),
                                            ("q5_0", 2048, 11008, 6), ("q5_k", 1024, 14336, 2), ("iq4_xs", 1024, 8192, 7),
                                            ("q5_0", 600, 4640, 4), ("q6_k", 600, 5376, 1)])
def test_rings_whose_slots_change_groups(ops, fmt, n, k, tokens):
    """More stages than an odd number of slots, while another stream keeps the memory busy: bit for bit the quiet result."""
    c = case(fmt, n, k, tokens, 33)
    w, xq = dev(c["w"]), xq_of(c)
    call = lambda: ops.mv_q8_ex(fmt, w, xq, n, k, tokens)  # noqa: E731
    want = call()
    rows = np.arange(0, n, 41)
    d = dict(c, w=c["w"][rows])
    v, ev = ref(d)
    ok, far = E.within(want[:, torch.from_numpy(rows).cuda()].double().cpu().numpy(), v, ev, "f32")
    assert ok, far
    a, b = (torch.empty(256 << 20, dtype=torch.uint8, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    busy = torch.cuda.Stream()
    with torch.cuda.stream(busy):
        for _ in range(100):
            b.copy_(a)
    got = [call() for _ in range(200)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    assert ops.device_status() == 0
