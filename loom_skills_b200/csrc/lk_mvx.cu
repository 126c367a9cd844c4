// Decode product on int8 activation codes with its epilogue (lk_mv_q8_ex):
//   p[t][n] = sum over 32-value groups g of d[t][g] * sum_i W[n][32 g + i] * c[t][32 g + i]
//   y = act(p + bias) + residual, or act(p_gate + bias, p_up + bias2) + residual
// One warp per output row and 8 tokens: lane l takes the row's groups l, l + 32, ...; a CTA holds 32 consecutive rows,
// the group of the q8 output form.
#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_formats.cuh"
#include "lk_internal.h"

namespace lk {
namespace {

constexpr int kXRows = 32, kXTok = 8;

struct MvxArgs {
  int n, k, tokens;
  const int8_t* codes;   // [tokens][k]
  const float* meta;     // [tokens][k/32][2]
  const uint8_t* w;
  const uint8_t* w2;
  int64_t rb;
  Epilogue e;
};

template <int FMT>
LK_DEV void row_dot(const MvxArgs& p, const uint8_t* row, int t0, int nt, int lane, float (&acc)[kXTok]) {
  constexpr int gpb = fmt_qk(FMT) / 32;
#pragma unroll
  for (int t = 0; t < kXTok; ++t) acc[t] = 0.0f;
  for (int g = lane; g < p.k / 32; g += 32) {
    float v[32];
    group_values<FMT>(row + int64_t(g / gpb) * fmt_block_bytes(FMT), g % gpb, v);
    for (int t = 0; t < nt; ++t) {
      const int8_t* c = p.codes + int64_t(t0 + t) * p.k + 32 * g;
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; ++i) s = fmaf(v[i], float(c[i]), s);
#pragma unroll
      for (int u = 0; u < kXTok; ++u)
        if (u == t) acc[u] = fmaf(s, p.meta[(int64_t(t0 + t) * (p.k / 32) + g) * 2], acc[u]);
    }
  }
#pragma unroll
  for (int t = 0; t < kXTok; ++t)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xFFFFFFFFu, acc[t], o);
}

template <int FMT>
__global__ void __launch_bounds__(32 * kXRows) k_mvx(const MvxArgs p) {
  __shared__ float out[kXTok][kXRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n0 = blockIdx.x * kXRows, t0 = blockIdx.y * kXTok, nt = min(kXTok, p.tokens - t0);
  const int n = n0 + warp;
  if (n < p.n) {
    float g[kXTok], u[kXTok];
    row_dot<FMT>(p, p.w + int64_t(n) * p.rb, t0, nt, lane, g);
    if (p.w2) row_dot<FMT>(p, p.w2 + int64_t(n) * p.rb, t0, nt, lane, u);
    if (lane == 0)
#pragma unroll
      for (int t = 0; t < kXTok; ++t) {
        if (p.e.bias) g[t] += p.e.bias[n];
        if (p.w2 && p.e.bias2) u[t] += p.e.bias2[n];
        out[t][warp] = p.w2 ? act_pair(p.e.act, g[t], u[t], p.e.alpha, p.e.limit) : act_one(p.e.act, g[t]);
      }
  }
  __syncthreads();
  if (warp >= nt) return;
  const int t = t0 + warp;
  const int64_t at = int64_t(t) * p.n + n0 + lane;
  const bool in = n0 + lane < p.n;
  float v = in ? out[warp][lane] : 0.0f;
  if (in && p.e.res) v += load_elem(p.e.res, p.e.res_dtype, at);
  if (p.e.y_form != LK_Q8_ROWS) {
    if (in) store_elem(p.e.y, p.e.y_form, at, v);
    return;
  }
  // n % 32 == 0: a whole group
  float amax = fabsf(v);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  const float d = amax / 127.0f;
  const int q = amax > 0.0f ? int8_t(int(roundf(v / d))) : 0;
  static_cast<int8_t*>(p.e.y)[at] = int8_t(q);
  int sum = q;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0)
    reinterpret_cast<float2*>(static_cast<int8_t*>(p.e.y) + int64_t(p.tokens) * p.n)[at / 32] =
        make_float2(__half2float(__float2half_rn(d)), float(sum));
}

template <int FMT>
int launch(const MvxArgs& a, cudaStream_t s) {
  const dim3 grid((a.n + kXRows - 1) / kXRows, (a.tokens + kXTok - 1) / kXTok);
  k_mvx<FMT><<<grid, 32 * kXRows, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? LK_OK : LK_ECUDA;
}

}  // namespace

int mv_q8_ex(int fmt, int n, int k, int tokens, const uint8_t* xq, const void* w, const void* w2, const Epilogue& e,
             cudaStream_t s) {
  MvxArgs a{};
  a.n = n;
  a.k = k;
  a.tokens = tokens;
  a.codes = reinterpret_cast<const int8_t*>(xq);
  a.meta = reinterpret_cast<const float*>(xq + int64_t(tokens) * k);
  a.w = static_cast<const uint8_t*>(w);
  a.w2 = static_cast<const uint8_t*>(w2);
  a.rb = lk_row_bytes(fmt, k);
  a.e = e;
  switch (fmt) {
    case LK_Q4_0: return launch<LK_Q4_0>(a, s);
    case LK_Q4_K: return launch<LK_Q4_K>(a, s);
    case LK_Q8_0: return launch<LK_Q8_0>(a, s);
    case LK_Q5_0: return launch<LK_Q5_0>(a, s);
    case LK_Q5_K: return launch<LK_Q5_K>(a, s);
    case LK_Q6_K: return launch<LK_Q6_K>(a, s);
    case LK_IQ4_NL: return launch<LK_IQ4_NL>(a, s);
    case LK_IQ4_XS: return launch<LK_IQ4_XS>(a, s);
  }
  return LK_EUNSUPPORTED;
}

}  // namespace lk
