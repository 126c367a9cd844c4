// Prefill product with its epilogue (lk_gemm_ex):
//   p[t][n] = scales[t][1] * sum_k x16[t][k] * W16[n][k],  W16 the GEMM's f16 staging of the packed weights
//   y = act(p + bias) + residual, or act(p_gate + bias, p_up + bias2) + residual
// One CTA per 64 rows x 64 outputs, 32 values of k at a time through shared memory, 4 x 4 outputs a thread.
#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_formats.cuh"
#include "lk_internal.h"

namespace lk {
namespace {

constexpr int kT = 64;

struct GemmxArgs {
  int rows, k, n;
  const __half* x16;
  const float* scales;
  const uint8_t* w;
  const uint8_t* w2;
  int64_t rb;
  Epilogue e;
};

template <int FMT>
__global__ void __launch_bounds__(256) k_gemmx(const GemmxArgs p) {
  __shared__ float xs[32][kT + 1], ws[2][32][kT + 1];
  constexpr int gpb = fmt_qk(FMT) / 32;
  const int t0 = blockIdx.y * kT, n0 = blockIdx.x * kT;
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
  float acc[2][4][4] = {};
  for (int g = 0; g < p.k / 32; ++g) {
    for (int i = threadIdx.x; i < kT * 32; i += 256) {
      const int r = i >> 5, c = i & 31;
      xs[c][r] = t0 + r < p.rows ? __half2float(p.x16[int64_t(t0 + r) * p.k + 32 * g + c]) : 0.0f;
    }
    if (threadIdx.x < 2 * kT) {
      const int r = threadIdx.x & 63, wi = threadIdx.x >> 6;
      const uint8_t* wp = wi ? p.w2 : p.w;
      if (wp) {
        __half h[32] = {};
        if (n0 + r < p.n)
          group_f16<FMT>(wp + int64_t(n0 + r) * p.rb + int64_t(g / gpb) * fmt_block_bytes(FMT), g % gpb, h);
        for (int c = 0; c < 32; ++c) ws[wi][c][r] = __half2float(h[c]);
      }
    }
    __syncthreads();
    for (int c = 0; c < 32; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[0][i][j] = fmaf(xs[c][tr + 16 * i], ws[0][c][tc + 16 * j], acc[0][i][j]);
          if (p.w2) acc[1][i][j] = fmaf(xs[c][tr + 16 * i], ws[1][c][tc + 16 * j], acc[1][i][j]);
        }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + tr + 16 * i, n = n0 + tc + 16 * j;
      if (t >= p.rows || n >= p.n) continue;
      const float inv = p.scales[2 * int64_t(t) + 1];
      float g = acc[0][i][j] * inv, u = acc[1][i][j] * inv;
      if (p.e.bias) g += p.e.bias[n];
      if (p.w2 && p.e.bias2) u += p.e.bias2[n];
      float v = p.w2 ? act_pair(p.e.act, g, u, p.e.alpha, p.e.limit) : act_one(p.e.act, g);
      if (p.e.res) v += load_elem(p.e.res, p.e.res_dtype, int64_t(t) * p.n + n);
      store_elem(p.e.y, p.e.y_form, int64_t(t) * p.n + n, v);
    }
}

template <int FMT>
int launch(const GemmxArgs& a, cudaStream_t s) {
  k_gemmx<FMT><<<dim3((a.n + kT - 1) / kT, (a.rows + kT - 1) / kT), 256, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? LK_OK : LK_ECUDA;
}

}  // namespace

int gemm_ex(int fmt, int rows, int k, int n, const uint16_t* x16, const float* scales, const void* w, const void* w2,
            const Epilogue& e, cudaStream_t s) {
  GemmxArgs a{};
  a.rows = rows;
  a.k = k;
  a.n = n;
  a.x16 = reinterpret_cast<const __half*>(x16);
  a.scales = scales;
  a.w = static_cast<const uint8_t*>(w);
  a.w2 = static_cast<const uint8_t*>(w2);
  a.rb = lk_row_bytes(fmt, k);
  a.e = e;
  switch (fmt) {
    case LK_Q4_0: return launch<LK_Q4_0>(a, s);
    case LK_Q4_K: return launch<LK_Q4_K>(a, s);
    case LK_IQ4_NL: return launch<LK_IQ4_NL>(a, s);
    case LK_Q5_0: return launch<LK_Q5_0>(a, s);
    case LK_Q8_0: return launch<LK_Q8_0>(a, s);
    case LK_Q5_K: return launch<LK_Q5_K>(a, s);
    case LK_Q6_K: return launch<LK_Q6_K>(a, s);
    case LK_IQ4_XS: return launch<LK_IQ4_XS>(a, s);
    case LK_Q3_K: return launch<LK_Q3_K>(a, s);
    case LK_IQ3_S: return launch<LK_IQ3_S>(a, s);
    case LK_MXFP4: return launch<LK_MXFP4>(a, s);
  }
  return LK_EUNSUPPORTED;
}

}  // namespace lk
