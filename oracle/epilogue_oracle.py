"""float64 restatement of the fused norm and the epilogue products (lk_rms_norm, lk_mv_q8_ex, lk_gemm_ex), with the
error each output may have: every function returns (value, slack), slack an elementwise bound on |kernel - value| before
the output's own rounding, from the number of f32 roundings the operation cannot do without."""
import math

import numpy as np

from . import qmm_oracle as O

EPS32 = 2.0 ** -24          # half a step of f32, relative
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}   # half the smallest subnormal (f32: a whole one)

_erf = np.vectorize(math.erf, otypes=[np.float64])


def rms_norm(x, weight, eps, residual=None):
    """(h, v) in float64 from the operands' values."""
    h = np.asarray(x, np.float64) + (0 if residual is None else np.asarray(residual, np.float64))
    v = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    return h, v


# relative error of v in f32: h rounds once (1); the squares and their sum: at most 32 fused steps in a thread and 10
# of the two shuffle trees, and 2 for h's rounding in the square, halved by the root (22); the mean's quotient, + eps, the
# root and its reciprocal (4); two products (2). Sums of squares have no cancellation, so all are relative: 29.
NORM_REL = 30 * EPS32


def act_one(act, g):
    g = np.asarray(g, np.float64)
    with np.errstate(over="ignore"):
        if act == "silu":
            return g / (1 + np.exp(-g))
        if act == "gelu":
            return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))
        if act == "gelu_erf":
            return 0.5 * g * (1 + _erf(g / np.sqrt(2)))
        if act == "relu":
            return np.maximum(g, 0)
    return g


def act_pair(act, g, u, alpha=1.702, limit=7.0):
    if act == "swiglu_oai":
        x, y = np.minimum(g, limit), np.clip(u, -limit, limit)
        with np.errstate(over="ignore"):
            return x / (1 + np.exp(-alpha * x)) * (y + 1)
    return act_one(act, g) * u


# |d act / d g| is at most 1.13 (tanh and erf GELU; SiLU 1.10; with alpha 1.702 1.10 too, its slope being that of
# SiLU at alpha g). Evaluating it in f32 loses at most 16 half steps of |g|: exp, tanh, erf and the division are within 2
# steps (4 half steps) of their value, an argument's rounding moves exp or tanh by at most 2 half steps of |g| where they
# are not yet saturated, and there are up to 5 more products and sums.
SLOPE, ACT_REL = 1.13, 16 * EPS32


def epilogue(g, eg, act, u=None, eu=None, bias=None, bias2=None, residual=None, alpha=1.702, limit=7.0):
    """The epilogue of products g (and u) known to within eg (eu)."""
    if bias is not None:
        g = g + np.asarray(bias, np.float64)
        eg = eg + EPS32 * np.abs(g)
    if u is None:
        v, ev = act_one(act, g), eg
        if act != "none":
            ev = SLOPE * eg + ACT_REL * np.abs(g)
    else:
        if bias2 is not None:
            u = u + np.asarray(bias2, np.float64)
            eu = eu + EPS32 * np.abs(u)
        v = act_pair(act, g, u, alpha, limit)
        a = act_pair(act, g, np.zeros_like(u), alpha, limit) if act == "swiglu_oai" else act_one(act, g)
        up = np.abs(np.clip(u, -limit, limit) + 1) if act == "swiglu_oai" else np.abs(u)
        if act == "none":
            ea = eg
        else:
            ea = SLOPE * eg + ACT_REL * np.abs(g)
        ev = ea * (up + eu) + np.abs(a) * (eu + EPS32 * (up + 1)) + EPS32 * np.abs(v)
    if residual is not None:
        v = v + np.asarray(residual, np.float64)
        ev = ev + EPS32 * np.abs(v)
    return v, ev


def _minimum(fmt, raw, k):
    """|dmin m| of every value of Q4_K / Q5_K rows; zeros for the other formats."""
    raw = np.asarray(raw, np.uint8)
    if fmt not in ("q4_k", "q5_k"):
        return np.zeros(raw.shape[:-1] + (k,))
    b = raw.reshape(-1, O.BLOCK_BYTES[fmt])
    dm = np.abs(np.ascontiguousarray(b[:, 2:4]).view(np.float16).astype(np.float64))
    _, mn = O.q4_k_scale_min(b[:, 4:16])
    return np.repeat(dm * mn, 32, -1).reshape(raw.shape[:-1] + (k,))


def product_q8(fmt, raw, codes, meta, k):
    """x . W^T of int8 codes and its slack. The integer dot of a group is exact; its two or three f32 factors round
    3 times, and the groups' terms (and their minima) are summed in at most k / 32 + 16 steps, so the error is within
    (k / 32 + 20) half steps of the terms' magnitudes, which |W| + 2 |minimum| times |x| bounds. (Q5_0 and Q4_0 may run as
    code * d with a minimum of 16 d or 8 d: four times |d| * 8 bounds both, taken as 2 * 16 d.)"""
    w = O.dequant(fmt, raw, k).astype(np.float64)
    x = O.dequant_q8(codes, meta)
    mag = np.abs(w) + 2 * _minimum(fmt, raw, k)
    if fmt in ("q4_0", "q5_0"):
        d = np.asarray(raw, np.uint8).reshape(-1, O.BLOCK_BYTES[fmt])[:, :2]
        d = np.abs(np.ascontiguousarray(d).view(np.float16).astype(np.float64))
        mag = mag + np.repeat(32 * d, 32, -1).reshape(w.shape)
    return x @ w.T, (k / 32 + 20) * EPS32 * (np.abs(x) @ mag.T)


def product_f16(fmt, raw, x16, scales, k):
    """(x16 . W16^T) * scale of the f16 staging and its slack: f32 accumulation of exact f16 products. The tensor core
    adds 16 products and the running sum at a time, aligned to the largest and cut off below its 24 bits: at most one
    step (2^-23) per term of such a sum, 17 terms, k / 16 sums, each of at most the whole magnitude -- taken as
    (k / 16 + 32) * 2^-21."""
    w = np.asarray(O.dequant_f16(fmt, raw, k), np.float64)
    x = np.asarray(x16, np.float64)
    inv = np.asarray(scales, np.float64)[:, 1:2]
    return (x @ w.T) * inv, (k / 16 + 32) * 2.0 ** -21 * (np.abs(x) @ np.abs(w).T) * np.abs(inv)


def within(got, value, slack, dtype):
    """Elementwise: |got - value| <= slack + half a step of the output type at value's magnitude (and slack's)."""
    got = np.asarray(got, np.float64)
    lim = slack + HALF_STEP[dtype] * (np.abs(value) + slack) + TINY[dtype]
    off = np.abs(got - value)
    # rounding to nearest gives an infinity from half a step past the largest finite f16, 65504 + 16
    over = np.isinf(got) & (np.sign(got) == np.sign(value)) & (np.abs(value) + slack >= 65520) & (dtype == "f16")
    off = np.where(over, 0.0, off)
    return bool((off <= lim).all()), (float(np.max(off / lim)) if got.size else 0.0)
