"""What the fused norm and the epilogue products cost: the cases, their inputs, and each operator in plain torch.

Three operators of the quantised linear path, as a transformer layer uses them:

  norm      h = x + residual, v = h / sqrt(mean(h^2) + eps) * weight, written in the form the next product reads:
            plain values, int8 codes with a scale per 32 values (q8), f16 rows with a power-of-two scale (row_f16) or
            e4m3 rows with a power-of-two scale (row_f8)
  decode    the product of a few tokens' int8 codes with packed GGUF weights, plus bias, activation (or the product of
            an activated gate and an up projection) and residual
  prefill   the same product and epilogue for many rows of row-scaled f16 activations

run() computes them in elementary torch operations, or (own = True) by the package's entry points.
"""
import math

import torch

own = False

EPS = 1e-6
DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# values and bytes of one block of each weight format
BLOCK = {"q4_0": (32, 18), "q8_0": (32, 34), "iq4_nl": (32, 18), "q4_k": (256, 144), "q6_k": (256, 210)}
IQ4 = (-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113)


# ----------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode token between two layers: latency counts
        dict(name="norm decode q8", op="norm", rows=1, k=4096, x="bf16", res="bf16", w="f32", form="q8"),
        # a small batch of a stream that is kept in f32, a width that is no power of two
        dict(name="norm batch plain", op="norm", rows=17, k=2880, x="f32", res="bf16", w="bf16", form="bf16"),
        # the rows of a prefill on the way to the f16 GEMM
        dict(name="norm prefill row_f16", op="norm", rows=2048, k=4096, x="bf16", res="bf16", w="f32", form="row_f16"),
        # the rows of a long prefill on the way to e4m3 experts
        dict(name="norm prefill row_f8", op="norm", rows=8192, k=2880, x="bf16", res="bf16", w="f32", form="row_f8"),
        # key projection with a bias at one token: the smallest product
        dict(name="decode k bias", op="decode", fmt="q4_0", tokens=1, k=4096, n=1024, pair=False, bias=True,
             act="none", res="", out="f32"),
        # gate and up projections of one token, straight to the down projection's codes
        dict(name="decode gate up", op="decode", fmt="q4_k", tokens=1, k=4096, n=12288, pair=True, bias=False,
             act="silu", res="", out="q8"),
        # down projection of eight sequences, added onto the residual stream
        dict(name="decode down batch", op="decode", fmt="q4_k", tokens=8, k=12288, n=4096, pair=False, bias=False,
             act="none", res="bf16", out="bf16"),
        # odd sizes: five tokens, a width of 90 blocks, an odd number of outputs
        dict(name="decode odd gelu", op="decode", fmt="q8_0", tokens=5, k=2880, n=2883, pair=False, bias=True,
             act="gelu", res="", out="f32"),
        # a gated block of a larger batch
        dict(name="decode gate up batch", op="decode", fmt="iq4_nl", tokens=32, k=5120, n=13824, pair=True, bias=True,
             act="silu", res="", out="bf16"),
        # gate and up projections of a prefill
        dict(name="prefill gate up", op="prefill", fmt="q4_k", tokens=2048, k=4096, n=12288, pair=True, bias=False,
             act="silu", res="", out="bf16"),
        # down projection of a long prefill onto the residual stream: the largest
        dict(name="prefill down", op="prefill", fmt="iq4_nl", tokens=4096, k=27648, n=5120, pair=False, bias=False,
             act="none", res="bf16", out="bf16"),
        # a short prompt, ragged sizes
        dict(name="prefill short", op="prefill", fmt="q6_k", tokens=200, k=4096, n=4100, pair=False, bias=True,
             act="gelu", res="bf16", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "norm", "decode", "decode", "prefill"))
    if op == "norm":
        form = rng.choice(("q8", "row_f16", "row_f8", "bf16", "f32"))
        k = _log(rng, 256, 16384)
        k = max(32, k // 32 * 32) if form == "q8" else k
        rows = _log(rng, 1, min(8192, (8192 * 4096) // k))
        x = rng.choice(("bf16", "bf16", "f32", "f16"))
        return dict(op=op, rows=rows, k=k, x=x, res=rng.choice(("", x, "bf16", "f32")), w=rng.choice(("f32", "bf16")),
                    form=form)
    fmt = rng.choice(tuple(BLOCK))
    pair = rng.random() < 0.4
    act = rng.choice(("silu", "gelu")) if pair else rng.choice(("none", "none", "gelu", "silu"))
    res = "" if pair or act != "none" else rng.choice(("", "bf16", "f32"))
    if op == "decode":
        unit = max(32, BLOCK[fmt][0])
        k = max(unit, _log(rng, 512, 16384) // unit * unit)
        out = rng.choice(("f32", "bf16", "f16")) if res else rng.choice(("f32", "bf16", "q8"))
        n = _log(rng, 64, (12288 * 8192) // (k * (2 if pair else 1)))
        n = n // 32 * 32 if out == "q8" else n
        return dict(op=op, fmt=fmt, tokens=_log(rng, 1, 32), k=k, n=n, pair=pair, bias=rng.random() < 0.5, act=act,
                    res=res, out=out)
    unit = max(64, BLOCK[fmt][0])
    k = max(unit, _log(rng, 512, 16384) // unit * unit)
    n = _log(rng, 256, (12288 * 8192) // (k * (2 if pair else 1)))
    tokens = _log(rng, 33, 4096)
    return dict(op=op, fmt=fmt, tokens=tokens, k=k, n=n, pair=pair, bias=rng.random() < 0.5, act=act, res=res,
                out="bf16")


# --------------------------------------------------------------------------------------------------- packed weights
def _u8(x):
    return x.contiguous().view(torch.uint8)


def _pack(fmt, w):
    """w [n][k] f32 -> packed rows [n][row bytes] of `fmt`, by the plain quantiser of each format."""
    n, k = w.shape
    if fmt == "q8_0":
        b = w.view(n, k // 32, 32)
        d = (b.abs().amax(-1, keepdim=True) / 127).half()
        q = (b / d.float().clamp_min(1e-12)).round().clamp(-127, 127).to(torch.int8)
        return torch.cat([_u8(d), _u8(q)], -1).view(n, -1)
    if fmt in ("q4_0", "iq4_nl"):
        b = w.view(n, k // 32, 32)
        top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
        if fmt == "q4_0":
            d = (top / -8).half()
            q = (b / d.float()).round().add_(8).clamp_(0, 15).to(torch.uint8)
        else:
            d = (top / -127).half()
            book = torch.tensor(IQ4, dtype=torch.float32, device=w.device)
            q = torch.bucketize(b / d.float(), (book[1:] + book[:-1]) / 2).to(torch.uint8)
        return torch.cat([_u8(d), q[..., :16] | (q[..., 16:] << 4)], -1).view(n, -1)
    if fmt == "q4_k":
        b = w.view(n, k // 256, 8, 32)
        low = (-b.amin(-1)).clamp_min(0)
        step = (b.amax(-1) + low) / 15
        d, dm = (step.amax(-1, keepdim=True) / 63).half(), (low.amax(-1, keepdim=True) / 63).half()
        sc = (step / d.float().clamp_min(1e-12)).round().clamp(1, 63).to(torch.uint8)
        m = (low / dm.float().clamp_min(1e-12)).round().clamp(0, 63).to(torch.uint8)
        q = ((b + (dm.float() * m).unsqueeze(-1)) / (d.float() * sc).unsqueeze(-1)).round().clamp_(0, 15).to(torch.uint8)
        head = torch.cat([sc[..., :4] | (sc[..., 4:] >> 4 << 6), m[..., :4] | (m[..., 4:] >> 4 << 6),
                          (sc[..., 4:] & 15) | ((m[..., 4:] & 15) << 4)], -1)
        nib = (q[..., 0::2, :] | (q[..., 1::2, :] << 4)).reshape(n, k // 256, 128)
        return torch.cat([_u8(d), _u8(dm), head, nib], -1).view(n, -1)
    b = w.view(n, k // 256, 16, 16)
    step = b.abs().amax(-1) / 31
    d = (step.amax(-1, keepdim=True) / 127).half()
    sc = (step / d.float().clamp_min(1e-12)).round().clamp(1, 127).to(torch.int8)
    q = (b / (d.float() * sc).unsqueeze(-1)).round().clamp_(-32, 31).add_(32).to(torch.uint8).view(n, k // 256, 2, 4, 32)
    ql = q & 15
    ql = torch.cat([ql[..., 0, :] | (ql[..., 2, :] << 4), ql[..., 1, :] | (ql[..., 3, :] << 4)], -1)
    qh = q >> 4
    qh = qh[..., 0, :] | (qh[..., 1, :] << 2) | (qh[..., 2, :] << 4) | (qh[..., 3, :] << 6)
    return torch.cat([ql.reshape(n, k // 256, 128), qh.reshape(n, k // 256, 64), _u8(sc), _u8(d)], -1).view(n, -1)


def _values(fmt, w, n, k):
    """Packed rows -> the values they stand for, f32 [n][k]."""
    qk, bb = BLOCK[fmt]
    b = w.view(n, k // qk, bb)
    if fmt == "q8_0":
        return (b[..., 2:].view(torch.int8).float() * b[..., :2].view(torch.float16).float()).view(n, k)
    if fmt in ("q4_0", "iq4_nl"):
        q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1)
        if fmt == "q4_0":
            v = q.float() - 8
        else:
            v = torch.tensor(IQ4, dtype=torch.float32, device=w.device)[q.int()]
        return (v * b[..., :2].view(torch.float16).float()).view(n, k)
    if fmt == "q4_k":
        d, dm = b[..., 0:2].view(torch.float16).float(), b[..., 2:4].view(torch.float16).float()
        s = b[..., 4:16]
        sc = torch.cat([s[..., 0:4] & 63, (s[..., 8:12] & 15) | (s[..., 0:4] >> 6 << 4)], -1).float()
        m = torch.cat([s[..., 4:8] & 63, (s[..., 8:12] >> 4) | (s[..., 4:8] >> 6 << 4)], -1).float()
        p = b[..., 16:].reshape(n, k // 256, 4, 1, 32)
        q = torch.cat([p & 15, p >> 4], 3).view(n, k // 256, 8, 32).float()
        return (q * (d * sc).unsqueeze(-1) - (dm * m).unsqueeze(-1)).view(n, k)
    d = b[..., 208:].view(torch.float16).float()
    sc = b[..., 192:208].view(torch.int8).float()
    ql, qh = b[..., :128].reshape(n, k // 256, 2, 1, 64), b[..., 128:192].reshape(n, k // 256, 2, 1, 32)
    lo = torch.cat([ql & 15, ql >> 4], 3).view(n, k // 256, 2, 4, 32)
    hi = torch.cat([qh & 3, (qh >> 2) & 3, (qh >> 4) & 3, qh >> 6], 3)
    q = (lo | (hi << 4)).float() - 32
    return (q.view(n, k // 256, 16, 16) * (d * sc).unsqueeze(-1)).view(n, k)


# ------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = dict(case)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if case["op"] == "norm":
        rows, k = case["rows"], case["k"]
        # hidden rows of differing sizes with a few large channels, as residual streams have
        amp = torch.exp(randn(rows, 1) * 0.5)
        chan = 1 + 20 * (torch.rand(k, device=DEV, generator=g) < 0.003)
        s["vx"] = (randn(rows, k) * amp).to(DT[case["x"]])
        s["vr"] = (randn(rows, k) * amp * chan * 3).to(DT[case["res"]]) if case["res"] else None
        s["vw"] = (1 + 0.2 * randn(k)).to(DT[case["w"]])
        return s
    t, k, n = case["tokens"], case["k"], case["n"]
    x = randn(t, k) * torch.exp(randn(t, 1) * 0.5)
    if case["op"] == "decode":
        # the codes a norm or a quantisation left: [t][k] int8, then (f16-rounded scale, sum of codes) per 32 values
        b = x.view(t, k // 32, 32)
        d = b.abs().amax(-1, keepdim=True) / 127
        c = (b / d).round()
        meta = torch.cat([d.half().float(), c.sum(-1, keepdim=True)], -1)
        s["xq"] = torch.cat([c.to(torch.int8).view(-1).view(torch.uint8), meta.view(-1).view(torch.uint8)])
    else:
        # f16 rows scaled by a power of two (here 1: no value is near the f16 range's end)
        s["x16"] = x.half()
        s["scales"] = torch.ones(t, 2, device=DEV)
    s["w1"] = _pack(case["fmt"], randn(n, k) * 0.02)
    s["w2"] = _pack(case["fmt"], randn(n, k) * 0.02) if case["pair"] else None
    s["b1"] = randn(n) * 0.5 if case["bias"] else None
    s["b2"] = randn(n) * 0.5 if case["bias"] and case["pair"] else None
    s["vr"] = (randn(t, n) * 3).to(DT[case["res"]]) if case["res"] else None
    return s


# ------------------------------------------------------------------------------------------- the operators, plain form
def _q8_values(c, d):
    """int8 codes [t][k/32][32] and their scales -> the values they stand for, in bf16 (one pass)."""
    return torch.mul(c, d, out=torch.empty(c.shape, dtype=torch.bfloat16, device=c.device)).view(c.shape[0], -1)


def _plain_q8(v):
    t, k = v.shape
    b = v.view(t, k // 32, 32)
    d = b.abs().amax(-1, keepdim=True) / 127
    q = b / d
    c = torch.where(d > 0, torch.sign(q) * torch.floor(q.abs() + 0.5), 0)
    return _q8_values(c, d.half().float())


def _exponent(v):
    """floor(log2) of each row's largest magnitude."""
    return torch.frexp(v.abs().amax(-1, keepdim=True)).exponent - 1


def _plain_norm(s):
    h = s["vx"].float()
    if s["vr"] is not None:
        h = h + s["vr"].float()
    v = h * (1 / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS)) * s["vw"].float()
    out = {"h": h.to(s["vr"].dtype)} if s["vr"] is not None else {}
    form = s["form"]
    if form == "q8":
        out["y"] = _plain_q8(v)
    elif form == "row_f16":
        e = (_exponent(v) - 13).clamp(0, 100).float()
        out["y"] = (v * torch.exp2(-e)).half()
        out["scales"] = torch.cat([torch.exp2(-e), torch.exp2(e)], -1)
    elif form == "row_f8":
        e = _exponent(v).float()
        out["y"] = (v * torch.exp2(7 - e)).clamp(-448, 448).to(torch.float8_e4m3fn)
        out["scales"] = torch.cat([torch.exp2(7 - e), torch.exp2(e - 15)], -1)
    else:
        out["y"] = v.to(DT[form])
    return out


def _plain_act(act, g):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    return g


def _plain_product(s, x):
    n, k = s["n"], s["k"]
    g = x @ _values(s["fmt"], s["w1"], n, k).t()
    if s["b1"] is not None:
        g = g + s["b1"]
    y = _plain_act(s["act"], g)
    if s["pair"]:
        u = x @ _values(s["fmt"], s["w2"], n, k).t()
        if s["b2"] is not None:
            u = u + s["b2"]
        y = y * u
    if s["vr"] is not None:
        y = y + s["vr"].float()
    return {"y": _plain_q8(y) if s["out"] == "q8" else y.to(DT[s["out"]])}


def _codes(xq, t, k):
    """int8 codes [t][k/32][32] and scales [t][k/32][1] of a q8 buffer."""
    return (xq[:t * k].view(torch.int8).view(t, k // 32, 32),
            xq[t * k:].view(torch.float32).view(t, k // 32, 2)[..., :1])


def run(s):
    if own:
        return _own(s)
    if s["op"] == "norm":
        return _plain_norm(s)
    if s["op"] == "decode":
        c, d = _codes(s["xq"], s["tokens"], s["k"])
        return _plain_product(s, (c.float() * d).view(s["tokens"], s["k"]))
    return _plain_product(s, s["x16"].float() * s["scales"][:, 1:])


def _own(s):
    from loom_skills_b200 import ops
    if s["op"] == "norm":
        got = ops.rms_norm(s["vx"], s["vw"], EPS, residual=s["vr"], form=s["form"])
        y, h = got if s["vr"] is not None else (got, None)
        out = {} if h is None else {"h": h}
        if s["form"] == "q8":
            out["y"] = _q8_values(*_codes(y, s["rows"], s["k"]))
        elif s["form"] == "row_f16":
            out["y"], out["scales"] = y
        elif s["form"] == "row_f8":
            out["y"], out["scales"] = y[0].view(torch.float8_e4m3fn), y[1]
        else:
            out["y"] = y
        return out
    t, n, k = s["tokens"], s["n"], s["k"]
    epi = dict(w2=s["w2"], bias=s["b1"], bias2=s["b2"], act=s["act"], residual=s["vr"])
    if s["op"] == "prefill":
        return {"y": ops.gemm_ex(s["fmt"], s["x16"], s["scales"], s["w1"], n, out_dtype=DT[s["out"]], **epi)}
    if s["out"] == "q8":
        y = ops.mv_q8_ex(s["fmt"], s["w1"], s["xq"], n, k, t, out_dtype="q8", **epi)
        return {"y": _q8_values(*_codes(y, t, n))}
    return {"y": ops.mv_q8_ex(s["fmt"], s["w1"], s["xq"], n, k, t, out_dtype=DT[s["out"]], **epi)}


def work(case):
    if case["op"] == "norm":
        rows, k = case["rows"], case["k"]
        out = {"q8": 1.25, "row_f16": 2, "row_f8": 1}.get(case["form"]) or SIZE[case["form"]]
        per = SIZE[case["x"]] + out + (2 * SIZE[case["res"]] if case["res"] else 0)
        return {"bytes": rows * k * per + k * SIZE[case["w"]] + (8 * rows if case["form"].startswith("row") else 0),
                "flops": 6.0 * rows * k}
    t, k, n = case["tokens"], case["k"], case["n"]
    qk, bb = BLOCK[case["fmt"]]
    two = 2 if case["pair"] else 1
    bytes_ = two * n * k // qk * bb + t * n * {"q8": 1.25}.get(case["out"], SIZE.get(case["out"], 0))
    bytes_ += t * k * (1.25 if case["op"] == "decode" else 2) + (8 * t if case["op"] == "prefill" else 0)
    bytes_ += two * n * 4 if case["bias"] else 0
    bytes_ += t * n * SIZE[case["res"]] if case["res"] else 0
    return {"bytes": bytes_, "flops": 2.0 * two * t * n * k}


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def _bit_field(block, byte, shift, mask):
    """(block[..., byte[i]] >> shift[i]) & mask for every value i of a block, as f64."""
    byte = torch.as_tensor(byte, device=block.device)
    shift = torch.as_tensor(shift, dtype=torch.uint8, device=block.device)
    return ((block.index_select(-1, byte) >> shift) & mask).double()


def _f64_of_half(block, at):
    return block[..., at:at + 2].contiguous().view(torch.float16).double()


def _exact_weight(fmt, w, n, k):
    """The weights in f64, value i of a block read by its byte and bit position in the format's layout."""
    qk, bb = BLOCK[fmt]
    b = w.view(n, k // qk, bb)
    i = range(qk)
    if fmt == "q8_0":
        q = _bit_field(b, [2 + j for j in i], [0] * qk, 255)
        return (torch.where(q > 127, q - 256, q) * _f64_of_half(b, 0)).view(n, k)
    if fmt in ("q4_0", "iq4_nl"):
        q = _bit_field(b, [2 + j % 16 for j in i], [4 * (j // 16) for j in i], 15)
        if fmt == "iq4_nl":
            book = torch.tensor(IQ4, dtype=torch.float64, device=w.device)
            return (book[q.long()] * _f64_of_half(b, 0)).view(n, k)
        return ((q - 8) * _f64_of_half(b, 0)).view(n, k)
    if fmt == "q4_k":
        q = _bit_field(b, [16 + 32 * (j // 64) + j % 32 for j in i], [4 * (j // 32 % 2) for j in i], 15)
        j8 = range(8)
        low = [_bit_field(b, [4 + at + j % 4 if j < 4 else 12 + j % 4 for j in j8],
                          [0 if j < 4 else 4 * (at // 4) for j in j8], 63) for at in (0, 4)]
        top = [_bit_field(b, [4 + at + j % 4 for j in j8], [6] * 8, 3) for at in (0, 4)]
        first = torch.arange(8, device=w.device) < 4
        sc, m = [torch.where(first, lo, lo.remainder(16) + 16 * hi) for lo, hi in zip(low, top)]
        v = q.view(n, -1, 8, 32) * (_f64_of_half(b, 0) * sc).unsqueeze(-1) - (_f64_of_half(b, 2) * m).unsqueeze(-1)
        return v.view(n, k)
    lo = _bit_field(b, [64 * (j // 128) + j % 64 for j in i], [4 * (j // 64 % 2) for j in i], 15)
    hi = _bit_field(b, [128 + 32 * (j // 128) + j % 32 for j in i], [2 * (j // 32 % 4) for j in i], 3)
    sc = _bit_field(b, [192 + j // 16 for j in i], [0] * qk, 255)
    sc = torch.where(sc > 127, sc - 256, sc)
    return ((lo + 16 * hi - 32) * sc * _f64_of_half(b, 208)).view(n, k)


def _exact_q8(v):
    t, k = v.shape
    b = v.reshape(t, -1, 32)
    d = b.abs().max(-1, keepdim=True).values / 127
    r = torch.where(d > 0, b / torch.where(d > 0, d, 1), 0)
    c = torch.where(r >= 0, (r + 0.5).floor(), (r - 0.5).ceil())
    return (c * d.to(torch.float16).double()).reshape(t, k)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["vx"].double() if s["vr"] is None else s["vx"].double() + s["vr"].double()
        v = h * torch.rsqrt((h * h).sum(-1, keepdim=True) / case["k"] + EPS) * s["vw"].double()
        out = {} if s["vr"] is None else {"h": h}
        top = torch.floor(torch.log2(v.abs().max(-1, keepdim=True).values))
        if case["form"] == "q8":
            out["y"] = _exact_q8(v)
        elif case["form"] == "row_f16":
            e = torch.clamp(top - 13, 0, 100)
            out["y"], out["scales"] = v / 2 ** e, torch.cat([2 ** -e, 2 ** e], -1)
        elif case["form"] == "row_f8":
            out["y"] = torch.clamp(v * 2 ** (7 - top), -448, 448)
            out["scales"] = torch.cat([2 ** (7 - top), 2 ** (top - 15)], -1)
        else:
            out["y"] = v
        return out
    t, k, n = case["tokens"], case["k"], case["n"]
    if case["op"] == "decode":
        raw = s["xq"]
        q = raw[:t * k].view(t, k).double()
        meta = raw[t * k:].view(torch.float32).view(t, -1, 2)
        x = torch.where(q > 127, q - 256, q) * meta[..., 0].double().repeat_interleave(32, -1)
    else:
        x = s["x16"].double() * s["scales"][:, 1].double().view(t, 1)
    p = torch.matmul(x, _exact_weight(case["fmt"], s["w1"], n, k).t())
    p = p if s["b1"] is None else p + s["b1"].double()
    if case["act"] == "silu":
        p = p * torch.sigmoid(p)
    elif case["act"] == "gelu":
        p = p * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3))
    if case["pair"]:
        u = torch.matmul(x, _exact_weight(case["fmt"], s["w2"], n, k).t())
        p = p * (u if s["b2"] is None else u + s["b2"].double())
    if s["vr"] is not None:
        p = p + s["vr"].double()
    return {"y": _exact_q8(p) if case["out"] == "q8" else p}
