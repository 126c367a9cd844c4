"""The dense gated FFN block (ops.ffn): norm, gate/up and down products onto the residual stream, run together, against
float64; and the fused norm in front of the framework's other products."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from oracle import epilogue_oracle as E  # noqa: E402
from oracle import qmm_oracle as O  # noqa: E402

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
QUANT = {"q4_0": O.quantize_q4_0, "q4_k": O.quantize_q4_k, "iq4_nl": O.quantize_iq4_nl}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from loom_skills_b200 import ops as _ops
    return _ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def weights(fmt, n, k, seed):
    return QUANT[fmt]((np.random.default_rng(seed).standard_normal((n, k)) * 0.05).astype(np.float32))


def f16_rows(a):
    x16, sc = O.row_scale_f16(a.astype(np.float32))
    return x16.astype(np.float64) * sc[:, 1:]


def block_ref(fmt, x, r, nw, wg, wu, wd, h, f, act, bg, bu, bd, decode):
    """float64, with the activations rounded where the path rounds them (codes, or f16 rows) and the weights it
    multiplies (the exact values, or the GEMM's f16 staging, whose own distance from them is the GEMM's to test)."""
    s, v = E.rms_norm(x, nw, np.float32(1e-6), r)
    quantise = (lambda a: O.dequant_q8(*O.quant_q8(a.astype(np.float32)))) if decode else f16_rows
    value = O.dequant if decode else O.dequant_f16
    wv = [value(fmt, w, k).astype(np.float64) for w, k in ((wg, h), (wu, h), (wd, f))]
    v = quantise(v)
    a = E.act_pair(act, v @ wv[0].T + bg, v @ wv[1].T + bu)
    return s + quantise(a) @ wv[2].T + bd


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k", "iq4_nl"])
@pytest.mark.parametrize("tokens,prefill", [(1, None), (7, None), (33, False), (64, None), (200, None), (5, True)])
@pytest.mark.parametrize("dt,act", [("bf16", "silu"), ("f32", "gelu"), ("f32", "swiglu_oai")])
def test_block(ops, fmt, tokens, prefill, dt, act):
    h, f = 512, 768
    rng = np.random.default_rng(tokens)
    x, r = (dev(rng.standard_normal((tokens, h)).astype(np.float32) * a).to(DT[dt]) for a in (1, 2))
    nw = rng.uniform(0.5, 1.5, h).astype(np.float32)
    wg, wu, wd = weights(fmt, f, h, 1), weights(fmt, f, h, 2), weights(fmt, h, f, 3)
    bg, bu, bd = (rng.standard_normal(m).astype(np.float32) for m in (f, f, h))
    y = ops.ffn(fmt, x, dev(nw), dev(wg), dev(wu), dev(wd), h, f, residual=r, act=act, b_gate=dev(bg), b_up=dev(bu),
                b_down=dev(bd), prefill=prefill)
    assert y.dtype == DT[dt] and y.shape == (tokens, h)
    decode = prefill is False or (prefill is None and tokens < 64)
    args = (fmt, x.double().cpu().numpy(), r.double().cpu().numpy(), nw, wg, wu, wd, h, f, act, bg, bu, bd)
    ref = block_ref(*args, decode)
    # a code or an f16 that rounds the other way (f32 against f64 near a tie) moves a value by 1/127 of its group's
    # largest, or 2^-11, for few values: the framework's bar of 1e-3 covers it. A bf16 stream rounds the result, and in
    # prefill the activations between the GEMMs, by at most 2^-8 each.
    tol = 1e-3 + {"f32": 0.0, "bf16": 2.0 ** -8}[dt] * (1 if decode else 2)
    assert O.rel_l2(y.double().cpu().numpy(), ref) <= tol
    assert ops.device_status() == 0


def test_without_a_residual_and_a_wider_down(ops):
    h, f = 512, 512
    rng = np.random.default_rng(5)
    x = dev(rng.standard_normal((3, h)).astype(np.float32))
    nw = np.ones(h, np.float32)
    wg, wu, wd = weights("q4_k", f, h, 1), weights("q4_k", f, h, 2), weights("q4_0", h, f, 3)
    y = ops.ffn("q4_k", x, dev(nw), dev(wg), dev(wu), dev(wd), h, f, fmt_down="q4_0")
    v = O.dequant_q8(*O.quant_q8(E.rms_norm(x.double().cpu().numpy(), nw, np.float32(1e-6))[1].astype(np.float32)))
    a = E.act_pair("silu", v @ O.dequant("q4_k", wg, h).T.astype(np.float64), v @ O.dequant("q4_k", wu, h).T)
    ref = x.double().cpu().numpy() + O.dequant_q8(*O.quant_q8(a.astype(np.float32))) @ O.dequant("q4_0", wd, f).T
    assert O.rel_l2(y.double().cpu().numpy(), ref) <= 1e-3


def test_captured_layers(ops):
    """Two blocks in one graph, the stream updated between them: replays follow new inputs."""
    h, f, fmt = 1024, 1024, "q4_k"
    nw = torch.ones(h, device="cuda")
    ws = [[dev(weights(fmt, *s, seed + 10 * i)) for seed, s in enumerate(((f, h), (f, h), (h, f)))] for i in range(2)]

    def two(x, r):
        for w in ws:
            x = ops.ffn(fmt, x, nw, *w, h, f, residual=r)
        return x

    for tokens in (1, 9, 100):
        x, r = (torch.randn(tokens, h, device="cuda").bfloat16() for _ in range(2))
        want = two(x, r)
        xs, rs = torch.zeros_like(x), torch.zeros_like(r)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = two(xs, rs)
        xs.copy_(x)
        rs.copy_(r)
        for _ in range(3):
            g.replay()
        assert torch.equal(y, want)


def test_norm_before_the_other_products(ops):
    """rms_norm's codes into mv_q8, its f16 rows into gemm, its e4m3 rows into the MXFP4 GEMM: each the product of the
    framework's own producer run on the f32 norm, bit for bit."""
    rng = np.random.default_rng(9)
    h, n = 512, 256
    x, r = (dev(rng.standard_normal((70, h)).astype(np.float32)) for _ in range(2))
    nw = dev(rng.uniform(0.5, 1.5, h).astype(np.float32))
    v, _ = ops.rms_norm(x, nw, residual=r, form="f32")
    w = dev(weights("q4_k", n, h, 4))
    q, _ = ops.rms_norm(x[:5], nw, residual=r[:5], form="q8")
    assert torch.equal(ops.mv_q8("q4_k", w, q, n, h, 5), ops.mv_q8("q4_k", w, ops.quant_q8(v[:5]), n, h, 5))
    (x16, sc), _ = ops.rms_norm(x, nw, residual=r, form="row_f16")
    assert torch.equal(ops.gemm("q4_k", "store", x16, sc, w, n), ops.gemm("q4_k", "store", *ops.row_scale_f16(v), w, n))
    (x8, s8), _ = ops.rms_norm(x, nw, residual=r, form="row_f8")
    nib = torch.randint(0, 256, (n, h // 2), dtype=torch.uint8, device="cuda")
    e8 = torch.randint(118, 124, (n, h // 32), dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.gemm_mxfp4s_f8("store", x8, s8, nib, e8, n),
                       ops.gemm_mxfp4s_f8("store", *ops.row_scale_f8(v), nib, e8, n))


FIRST_CALLS = """
import threading, torch
from loom_skills_b200 import ops
torch.manual_seed(0)
w = torch.randint(0, 255, (512, 144 * 2), dtype=torch.uint8, device="cuda")
w[:, 0::144] = w[:, 2::144] = 0
w[:, 1::144] = w[:, 3::144] = 0x2C          # finite f16 scales and minima
x = torch.randn(300, 512, device="cuda").bfloat16()
nw = torch.ones(512, device="cuda")
def layer(t):
    return ops.ffn("q4_k", x[:t], nw, w, w, w, 512, 512)
sizes = [1, 8, 40, 300]
if MODE == "capture":                       # the first launch of every kernel goes into a graph
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = [layer(t) for t in sizes]
    g.replay()
else:                                       # ... or comes from four threads at once
    got = [None] * 16
    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = layer(sizes[i % 4])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(16)]
    [t.start() for t in threads]
    [t.join() for t in threads]
torch.cuda.synchronize()
for i, y in enumerate(got):
    assert torch.equal(y, layer(sizes[i % 4])) and torch.isfinite(y.float()).all()
assert ops.device_status() == 0
print("same")
"""


@pytest.mark.parametrize("mode", ["capture", "threads"])
def test_first_calls_of_a_process(ops, mode):
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", f"MODE = {mode!r}\n" + FIRST_CALLS], capture_output=True, text=True,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_formats_by_id(ops):
    c = torch.randint(0, 255, (64, 144), dtype=torch.uint8, device="cuda")
    c[:, 0] = c[:, 2] = 0
    c[:, 1] = c[:, 3] = 0x2C
    w = c.repeat(4, 1)
    x, nw = torch.randn(3, 256, device="cuda"), torch.ones(256, device="cuda")
    by_name = ops.ffn("q4_k", x, nw, w, w, w, 256, 256)
    assert torch.equal(ops.ffn(ops.L.Q4_K, x, nw, w, w, w, 256, 256), by_name)
    assert torch.equal(ops.ffn("q4_k", x, nw, w, w, w, 256, 256, prefill=False), by_name)


@pytest.mark.parametrize("fmt", ["q4_0", "iq4_nl"])
@pytest.mark.parametrize("tokens", [64, 100])
@pytest.mark.parametrize("h,f", [(96, 160), (96, 128), (128, 224)])
def test_many_tokens_of_widths_that_are_no_multiple_of_64(ops, fmt, tokens, h, f):
    rng = np.random.default_rng(tokens)
    x, r = (dev(rng.standard_normal((tokens, h)).astype(np.float32)) for _ in range(2))
    nw = np.ones(h, np.float32)
    wg, wu, wd = weights(fmt, f, h, 1), weights(fmt, f, h, 2), weights(fmt, h, f, 3)
    y = ops.ffn(fmt, x, dev(nw), dev(wg), dev(wu), dev(wd), h, f, residual=r)
    ref = block_ref(fmt, x.double().cpu().numpy(), r.double().cpu().numpy(), nw, wg, wu, wd, h, f, "silu", 0, 0, 0, True)
    assert O.rel_l2(y.double().cpu().numpy(), ref) <= 1e-3   # as test_block's f32 stream
    assert ops.device_status() == 0


@pytest.mark.parametrize("tokens", [1, 40, 70])
def test_f16_stream(ops, tokens):
    """Activations past 65504 between the products, a stream that stays in range."""
    h, f = 256, 512
    rng = np.random.default_rng(tokens)
    x, r = (dev(rng.standard_normal((tokens, h)).astype(np.float32)).half() for _ in range(2))
    nw = np.full(h, 200, np.float32)
    wg, wu = weights("q4_k", f, h, 1), weights("q4_k", f, h, 2)
    wd = O.quantize_q4_0((np.random.default_rng(3).standard_normal((h, f)) * 1e-3).astype(np.float32))
    y = ops.ffn("q4_k", x, dev(nw), dev(wg), dev(wu), dev(wd), h, f, residual=r, act="relu", fmt_down="q4_0")
    assert y.dtype == torch.float16 and y.shape == (tokens, h)
    s, v = E.rms_norm(x.double().cpu().numpy(), nw, np.float32(1e-6), r.double().cpu().numpy())
    decode = tokens < 64
    quantise = (lambda a: O.dequant_q8(*O.quant_q8(a.astype(np.float32)))) if decode else f16_rows
    value = O.dequant if decode else O.dequant_f16
    v = quantise(v)
    a = E.act_pair("relu", v @ value("q4_k", wg, h).astype(np.float64).T, v @ value("q4_k", wu, h).astype(np.float64).T)
    assert np.abs(a).max() > 65504
    # h: the sum is rounded once to f16, a second rounding follows at the output; the bar of test_block for the rest
    ref = s + quantise(a) @ value("q4_0", wd, f).astype(np.float64).T
    assert np.abs(ref).max() < 60000
    assert O.rel_l2(y.double().cpu().numpy(), ref) <= 1e-3 + 2 * 2.0 ** -11
    assert ops.device_status() == 0
