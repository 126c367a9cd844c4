// What the epilogue products (lk_mv_q8_ex, lk_gemm_ex) and the fused norm share: element loads and stores of the three
// value types, and the activations.
#pragma once
#include <atomic>

#include "lk_common.cuh"

namespace lk {

// Lets `kern` take `bytes` of dynamic shared memory on the current device; `done` (a bit a device) says where that is set
// already. The bit follows the setting: a call that races with the first one sets it again instead of launching without.
template <class Kernel>
bool allow_smem(Kernel kern, int bytes, std::atomic<unsigned>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned bit = 1u << (dev & 31);
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

// element i of an array of LK_F32 / LK_F16 / LK_BF16
LK_DEV float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == LK_BF16) return bf2f(static_cast<const uint16_t*>(p)[i]);
  if (dtype == LK_F16) return h2f(static_cast<const uint16_t*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
// one rounding, to nearest even
LK_DEV void store_elem(void* p, int dtype, int64_t i, float v) {
  if (dtype == LK_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == LK_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// The activation of one product. SiLU and the tanh GELU are g * sigmoid(z) -- 0.5 (1 + tanh(t)) = sigmoid(2 t) -- with
// the fast exponential and quotient: the exponential is off by 2^-21 + |z| 2^-23 of its value, which g * sigmoid turns
// into less than 4 half steps of |g| in f32, and an output costs a dozen instructions where expf and an IEEE division
// cost about 60 (a 2048 x 4096 x 2 * 12288 Q4_K gate/up prefill went from 471 to 424 us, and to 325 us with the
// choices of activation and type outside the loops over outputs).
LK_DEV float swish(float g, float z) { return __fdividef(g, 1.0f + __expf(-z)); }
LK_DEV float act_one(int act, float g) {
  switch (act) {
    case LK_ACT_SILU: return swish(g, g);
    case LK_ACT_GELU: return swish(g, 1.5957691216057308f * fmaf(0.044715f * g, g * g, g));
    case LK_ACT_GELU_ERF: return 0.5f * g * (1.0f + erff(g * 0.7071067811865476f));
    case LK_ACT_RELU: return g < 0.0f ? 0.0f : g;   // keeps a NaN
  }
  return g;
}
// ... of an array, the choice outside the loops
template <int V>
LK_DEV void act_all(int act, float (&v)[V]) {
  if (act == LK_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = act_one(LK_ACT_SILU, v[i]);
  } else if (act == LK_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = act_one(LK_ACT_GELU, v[i]);
  } else if (act == LK_ACT_GELU_ERF) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = act_one(LK_ACT_GELU_ERF, v[i]);
  } else if (act == LK_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = act_one(LK_ACT_RELU, v[i]);
  }
}
// ... and of a gate / up pair
LK_DEV float act_pair(int act, float g, float u, float alpha, float limit) {
  if (act == LK_ACT_SWIGLU_OAI) {
    // comparisons that keep a NaN, as clamp does
    const float x = g > limit ? limit : g, y = u > limit ? limit : (u < -limit ? -limit : u);
    return swish(x, alpha * x) * (y + 1.0f);
  }
  return act_one(act, g) * u;
}

// Everything an epilogue product applies to its f32 sums, in this order: + bias, activation (of one product, or of the
// gate times the up product), + residual, one rounding to the output's type.
struct Epilogue {
  const float* bias;    // [n] or null
  const float* bias2;   // [n] of the up product, or null
  const void* res;      // [rows][n] of res_dtype, or null; may be y
  int res_dtype;
  int act;
  float alpha, limit;
  void* y;              // [rows][n] of y_form; LK_Q8_ROWS: lk_quant_q8's buffer for rows rows of n values
  int y_form;
};

// two f32 multiply-adds (multiplications) in one instruction, each rounded as fmaf rounds
LK_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
LK_DEV float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// k_quant_q8's codes and meta of one 32-value group, one value a lane
LK_DEV void store_q8(uint8_t* y, int64_t total, int64_t at, float v, int lane) {
  float amax = fabsf(v);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  const float d = amax / 127.0f;
  const int q = amax > 0.0f ? int8_t(int(roundf(v / d))) : 0;
  reinterpret_cast<int8_t*>(y)[at] = int8_t(q);
  int sum = q;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0)
    reinterpret_cast<float2*>(y + total)[at / 32] = make_float2(__half2float(__float2half_rn(d)), float(sum));
}

}  // namespace lk
