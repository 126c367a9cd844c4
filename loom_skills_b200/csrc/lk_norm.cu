// Residual addition, RMS norm and the activation format of the next product in one pass over the row.
//
//   h = x + residual                       (f32; stored rounded once to the residual's type)
//   v = h * rstd * weight,  rstd = 1 / sqrt(mean(h^2) + eps)     (f32, from the unrounded h)
//   y = v rounded to f32 / f16 / bf16, or the codes lk_quant_q8, lk_row_scale_f16 or lk_row_scale_f8 make of v
//
// A CTA works on a row at a time. Thread t holds the 8-value vectors t, t + T, ... of the row in registers from the first
// load to the last store, so x and the residual are read once and h and y written once; the only exchanges are the sum of
// squares (and for the row-scaled forms the row's maximum) through warp shuffles and one shared array.
//
// Few rows, and rows that are not whole 16-byte vectors: a CTA per row, as many threads as vectors, bound by the launch and
// one load latency (1 to 8 rows of 4096: 2.5 to 2.7 us). From 256 rows resident CTAs stream them (k_rms_norm_stream): 2048 x
// 4096 to row-scaled f16 in 15.1 us (4.4 TB/s, 69 % of the measured copy rate) against 17.1 with a CTA per row, 4096 x 5120
// to row-scaled e4m3 29.8 against 37.1; 8192 x 5120 to bf16 66 us (5.1 TB/s).
#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_internal.h"

namespace lk {
namespace {

constexpr int kVec = 8;             // values per vector
constexpr int kNormMaxThreads = 1024;

LK_DEV void nm_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
LK_DEV void nm_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// 8 consecutive values (16-byte aligned)
LK_DEV void load_vec(const void* p, int dtype, int64_t off, float (&v)[kVec]) {
  if (dtype == LK_F32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + off);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + off);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dtype == LK_BF16) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
LK_DEV void store_vec(void* p, int dtype, int64_t off, const float (&v)[kVec]) {
  if (dtype == LK_F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + off);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dtype == LK_BF16) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 b = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + off) = make_uint4(w[0], w[1], w[2], w[3]);
}

LK_DEV float2 pair_of(const float (&v)[kVec], int j) { return make_float2(v[j], v[j + 1]); }
LK_DEV void set_pair(float (&v)[kVec], int j, float2 x) {
  v[j] = x.x;
  v[j + 1] = x.y;
}

// calls f with a value of the element type `dtype` names: the choice is made once for a row, not once an element, whose loads
// would then wait for one another
template <class F>
LK_DEV void with_type(int dtype, const F& f) {
  if (dtype == LK_BF16) f(__nv_bfloat16());
  else if (dtype == LK_F16) f(__half());
  else f(0.0f);
}
// one rounding, to nearest even
template <typename T>
LK_DEV void put(T* p, float v) { *p = T(v); }

struct NormArgs {
  int k;
  const void* x;
  int x_dtype;
  const void* res;
  int res_dtype;
  const void* weight;
  int w_dtype;
  float eps;
  void* h;         // of res_dtype, or null
  void* y;
  float* scales;   // row forms: [rows][2]
  int rows;
};

// Index in the row of element j of a thread's vector u. VEC: rows of whole 16-byte aligned vectors, t, t + T, ... a
// thread's. Otherwise elements are moved one by one: t + (8 u + j) T, so a warp still touches consecutive addresses --
// except for the q8 form, whose 32-value groups stay in four neighbouring lanes.
template <int FORM, bool VEC>
LK_DEV int elem_at(int u, int j) {
  const int t = threadIdx.x, T = blockDim.x;
  return VEC || FORM == LK_Q8_ROWS ? kVec * (t + u * T) + j : t + (kVec * u + j) * T;
}

// From the row's h in registers to its stored output. FORM: LK_F32 (any plain type, y_dtype at run time), LK_Q8_ROWS,
// LK_F16_ROWS or LK_E4M3. weight(u, w): the weight vector u (VEC); own_row(): runs where every thread of the CTA has its
// part of the row in registers; red: [2][32].
template <int FORM, bool VEC, int NV, class Weight, class Own>
LK_DEV void finish_row(const NormArgs& p, int y_dtype, int64_t row, float (&v)[NV][kVec], float (*red)[32],
                       const Weight& weight, const Own& own_row) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, nwarps = blockDim.x >> 5;
  const int64_t base = row * p.k;
  auto at = [](int u, int j) { return elem_at<FORM, VEC>(u, j); };
  float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int j = 0; j < kVec; j += 2) sq = fma2(pair_of(v[u], j), pair_of(v[u], j), sq);
  float ss = sq.x + sq.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
  if (lane == 0) red[0][warp] = ss;
  __syncthreads();
  own_row();
  ss = lane < nwarps ? red[0][lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
  const float rstd = 1.0f / sqrtf(ss / float(p.k) + p.eps);

  float amax = 0.0f;
  if (!VEC)
    with_type(p.w_dtype, [&](auto one) {
      const auto* w = static_cast<const decltype(one)*>(p.weight);
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (at(u, j) < p.k) v[u][j] = v[u][j] * rstd * float(w[at(u, j)]);
    });
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if (VEC) {
      if (at(u, 0) < p.k) {
        float w[kVec];
        weight(u, w);
#pragma unroll
        for (int j = 0; j < kVec; j += 2)
          set_pair(v[u], j, mul2(mul2(pair_of(v[u], j), make_float2(rstd, rstd)), pair_of(w, j)));
      }
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) amax = fmaxf(amax, fabsf(v[u][j]));
  }

  if (FORM == LK_F32) {
    if (VEC) {
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (at(u, 0) < p.k) store_vec(p.y, y_dtype, base + at(u, 0), v[u]);
    } else {
      with_type(y_dtype, [&](auto one) {
        auto* y = static_cast<decltype(one)*>(p.y) + base;
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (at(u, j) < p.k) put(y + at(u, j), v[u][j]);
      });
    }
  } else if (FORM == LK_Q8_ROWS) {
    // k_quant_q8's rounding of each 32-value group, whose values are in four neighbouring lanes
    int8_t* codes = static_cast<int8_t*>(p.y) + base;
    float2* meta = reinterpret_cast<float2*>(static_cast<uint8_t*>(p.y) + int64_t(p.rows) * p.k) + row * (p.k / 32);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      float gmax = fabsf(v[u][0]);   // not from 0: a group of NaN keeps its NaN scale, as k_quant_q8's does
#pragma unroll
      for (int j = 1; j < kVec; ++j) gmax = fmaxf(gmax, fabsf(v[u][j]));
      gmax = fmaxf(gmax, __shfl_xor_sync(0xFFFFFFFFu, gmax, 1));
      gmax = fmaxf(gmax, __shfl_xor_sync(0xFFFFFFFFu, gmax, 2));
      const float d = gmax / 127.0f;
      uint32_t w[2] = {0u, 0u};
      int sum = 0;
      if (gmax > 0.0f) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const int q = int8_t(int(roundf(v[u][j] / d)));
          sum += q;
          w[j >> 2] |= (uint32_t(q) & 255u) << (8 * (j & 3));
        }
      }
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      const int e = at(u, 0);
      if (e < p.k) {
        *reinterpret_cast<uint2*>(codes + e) = make_uint2(w[0], w[1]);
        if ((lane & 3) == 0) meta[e / 32] = make_float2(__half2float(__float2half_rn(d)), float(sum));
      }
    }
  } else {
    // lk_row_scale_f16 / lk_row_scale_f8's exponents from the row's maximum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    if (lane == 0) red[1][warp] = amax;
    __syncthreads();
    amax = lane < nwarps ? red[1][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const int biased = int((__float_as_uint(amax) >> 23) & 255);
    float s, inv;
    if (FORM == LK_F16_ROWS) {
      const int e = min(max(biased - 127 - 13, 0), 100);
      s = __uint_as_float(uint32_t(127 - e) << 23);
      inv = __uint_as_float(uint32_t(127 + e) << 23);
    } else {
      s = __uint_as_float(uint32_t(min(max(261 - biased, 1), 254)) << 23);
      inv = __uint_as_float(uint32_t(min(max(biased - 15, 1), 254)) << 23);
    }
    if (t == 0) {
      p.scales[2 * row] = s;
      p.scales[2 * row + 1] = inv;
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
#pragma unroll
      for (int j = 0; j < kVec; j += 2) set_pair(v[u], j, mul2(pair_of(v[u], j), make_float2(s, s)));
      if (FORM == LK_F16_ROWS) {
        if (VEC) {
          if (at(u, 0) < p.k) store_vec(p.y, LK_F16, base + at(u, 0), v[u]);
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (at(u, j) < p.k) store_elem(p.y, LK_F16, base + at(u, j), v[u][j]);
        }
      } else {
        uint8_t* y8 = static_cast<uint8_t*>(p.y) + base;
        if (VEC) {
          if (at(u, 0) < p.k) {
            uint32_t q[2] = {0u, 0u};
#pragma unroll
            for (int j = 0; j < kVec; j += 2)
              q[j >> 2] |= uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(v[u][j], v[u][j + 1]), __NV_SATFINITE, __NV_E4M3))
                           << (8 * (j & 3));
            *reinterpret_cast<uint2*>(y8 + at(u, 0)) = make_uint2(q[0], q[1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (at(u, j) < p.k) y8[at(u, j)] = __nv_cvt_float_to_fp8(v[u][j], __NV_SATFINITE, __NV_E4M3);
        }
      }
    }
  }
}

// A CTA per row.
template <int FORM, bool VEC, int NV>
__global__ void __launch_bounds__(kNormMaxThreads) k_rms_norm(const NormArgs p, int y_dtype) {
  __shared__ float red[2][32];
  const int64_t base = int64_t(blockIdx.x) * p.k;
  auto at = [](int u, int j) { return elem_at<FORM, VEC>(u, j); };

  nm_launch();
  nm_wait();
  float v[NV][kVec];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if (VEC) {
      const bool in = at(u, 0) < p.k;
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[u][j] = 0.0f;
      if (in) load_vec(p.x, p.x_dtype, base + at(u, 0), v[u]);
    }
  }
  if (!VEC) {
    with_type(p.x_dtype, [&](auto one) {
      const auto* x = static_cast<const decltype(one)*>(p.x) + base;
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[u][j] = at(u, j) < p.k ? float(x[at(u, j)]) : 0.0f;
    });
    if (p.res)
      with_type(p.res_dtype, [&](auto one) {
        using T = decltype(one);
        const T* r = static_cast<const T*>(p.res) + base;
        T* h = static_cast<T*>(p.h) + base;
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (at(u, j) < p.k) v[u][j] += float(r[at(u, j)]);
        if (p.h)
#pragma unroll
          for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j)
              if (at(u, j) < p.k) put(h + at(u, j), v[u][j]);
      });
  }
  if (VEC && p.res) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (VEC) {
        if (at(u, 0) < p.k) {
          float r[kVec];
          load_vec(p.res, p.res_dtype, base + at(u, 0), r);
#pragma unroll
          for (int j = 0; j < kVec; ++j) v[u][j] += r[j];
          if (p.h) store_vec(p.h, p.res_dtype, base + at(u, 0), v[u]);
        }
      }
    }
  }
  finish_row<FORM, VEC, NV>(p, y_dtype, blockIdx.x, v, red,
                            [&](int u, float (&w)[kVec]) { load_vec(p.weight, p.w_dtype, at(u, 0), w); }, [] {});
}

// Many rows: resident CTAs walk the rows, each with a ring of `slots` rows (x, then the residual) that bulk copies fill
// while earlier rows are worked on, so HBM is read without a pause; a CTA per row leaves it idle between a row's loads
// and stores. A slot is free again as soon as the row is in registers, at the barrier of its sum of squares.
constexpr int kMaxSlots = 4;
constexpr uint32_t kNormPolls = 1u << 22;
constexpr int kStreamRows = 256;   // fewer rows than that leave most rings a row or two
// ring bytes of each of n resident CTAs (the system's 1 KB and the kernel's own arrays aside)
constexpr int stream_smem(int n) { return 227 * 1024 / n - 2048; }
template <int NV>
constexpr int stream_threads() { return NV == 1 ? 128 : NV == 2 ? 512 : 1024; }
constexpr int kStreamThreadsPerSm = 1024;   // resident at 64 registers

template <int FORM, int NV>
__global__ void __launch_bounds__(stream_threads<NV>(), kStreamThreadsPerSm / stream_threads<NV>())
    k_rms_norm_stream(const NormArgs p, int y_dtype, int slots, int slot_bytes) {
  constexpr bool kHoldW = NV <= 2;   // the weights stay in registers
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float red[2][32];
  __shared__ uint64_t full[kMaxSlots];
  const int t = threadIdx.x;
  const uint32_t xb = uint32_t(p.k) * (p.x_dtype == LK_F32 ? 4 : 2);
  const uint32_t rb = p.res ? uint32_t(p.k) * (p.res_dtype == LK_F32 ? 4 : 2) : 0;
  auto at = [](int u) { return elem_at<FORM, true>(u, 0); };
  auto fetch = [&](int64_t row, int s) {
    uint8_t* d = ring + s * slot_bytes;
    mbar_expect_tx(&full[s], xb + rb);
    bulk_g2s(d, static_cast<const uint8_t*>(p.x) + row * xb, xb, &full[s]);
    if (rb) bulk_g2s(d + xb, static_cast<const uint8_t*>(p.res) + row * rb, rb, &full[s]);
  };
  nm_launch();
  if (t == 0) {
    for (int i = 0; i < slots; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
    nm_wait();
    for (int i = 0; i < slots; ++i)
      if (int64_t(blockIdx.x) + int64_t(i) * gridDim.x < p.rows) fetch(int64_t(blockIdx.x) + int64_t(i) * gridDim.x, i);
  }
  nm_wait();
  float wt[kHoldW ? NV : 1][kVec];
  if (kHoldW)
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (at(u) < p.k) load_vec(p.weight, p.w_dtype, at(u), wt[u]);
  __syncthreads();
  int s = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    bool in = false;
    for (uint32_t q = 0; q < kNormPolls && !in; ++q) in = mbar_try_wait(&full[s], phase);
    if (!__syncthreads_and(in)) {   // given up: the copies in flight land, then the CTA ends
      if (t == 0) {
        atomicOr(&g_status, 1u);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      }
      __syncthreads();
      return;
    }
    const uint8_t* xs = ring + s * slot_bytes;
    float v[NV][kVec];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[u][j] = 0.0f;
      if (at(u) < p.k) {
        load_vec(xs, p.x_dtype, at(u), v[u]);
        if (p.res) {
          float r[kVec];
          load_vec(xs + xb, p.res_dtype, at(u), r);
#pragma unroll
          for (int j = 0; j < kVec; ++j) v[u][j] += r[j];
          if (p.h) store_vec(p.h, p.res_dtype, row * p.k + at(u), v[u]);
        }
      }
    }
    const int64_t next = row + int64_t(slots) * gridDim.x;
    finish_row<FORM, true, NV>(
        p, y_dtype, row, v, red,
        [&](int u, float (&w)[kVec]) {
          if (kHoldW) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) w[j] = wt[kHoldW ? u : 0][j];
          } else {
            load_vec(p.weight, p.w_dtype, at(u), w);
          }
        },
        [&] {
          if (t == 0 && next < p.rows) fetch(next, s);
        });
    if (++s == slots) {
      s = 0;
      phase ^= 1;
    }
  }
}

template <int FORM, bool VEC, int NV>
int launch(const NormArgs& a, int y_dtype, int threads, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_rms_norm<FORM, VEC, NV>, a, y_dtype) == cudaSuccess ? LK_OK : LK_ECUDA;
}

template <int FORM, int NV>
int launch_stream(const NormArgs& a, int y_dtype, int threads, cudaStream_t s) {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int slot = a.k * ((a.x_dtype == LK_F32 ? 4 : 2) + (!a.res ? 0 : a.res_dtype == LK_F32 ? 4 : 2));
  int per_sm = kStreamThreadsPerSm / threads;
  while (per_sm > 1 && stream_smem(per_sm) < 2 * slot) --per_sm;
  int slots = stream_smem(per_sm) / slot;
  slots = slots < kMaxSlots ? slots : kMaxSlots;
  auto kern = k_rms_norm_stream<FORM, NV>;
  static std::atomic<unsigned> allowed{0};
  if (!allow_smem(kern, stream_smem(1), allowed)) return LK_ECUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows < sms * per_sm ? a.rows : sms * per_sm, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = slots * slot;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, y_dtype, slots, slot) == cudaSuccess ? LK_OK : LK_ECUDA;
}

template <int FORM, bool VEC>
int pick(const NormArgs& a, int y_dtype, cudaStream_t s) {
  const int nvec = (a.k + kVec - 1) / kVec;
  const int slot = a.k * ((a.x_dtype == LK_F32 ? 4 : 2) + (!a.res ? 0 : a.res_dtype == LK_F32 ? 4 : 2));
  if (VEC && a.rows >= kStreamRows && slot <= stream_smem(1)) {
    const int nv = nvec <= 128 ? 1 : nvec <= 1024 ? 2 : 4, threads = ((nvec + nv - 1) / nv + 31) / 32 * 32;
    if (nv == 1) return launch_stream<FORM, 1>(a, y_dtype, threads, s);
    if (nv == 2) return launch_stream<FORM, 2>(a, y_dtype, threads, s);
    return launch_stream<FORM, 4>(a, y_dtype, threads, s);
  }
  const int nv = nvec <= kNormMaxThreads ? 1 : nvec <= 2 * kNormMaxThreads ? 2 : 4;
  const int threads = ((nvec + nv - 1) / nv + 31) / 32 * 32;
  if (nv == 1) return launch<FORM, VEC, 1>(a, y_dtype, threads, s);
  if (nv == 2) return launch<FORM, VEC, 2>(a, y_dtype, threads, s);
  return launch<FORM, VEC, 4>(a, y_dtype, threads, s);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int rms_norm(int rows, int k, const void* x, int x_dtype, const void* res, int res_dtype, const void* weight,
             int w_dtype, float eps, void* h, int form, void* y, float* scales, cudaStream_t s) {
  const NormArgs a{k, x, x_dtype, res, res_dtype, weight, w_dtype, eps, h, y, scales, rows};
  // 16-byte vectors of whole rows; e4m3 and q8 rows are stored 8 bytes at a time, which an 8-byte aligned y allows
  const bool vec = k % kVec == 0 && al16(x) && al16(res) && al16(weight) && al16(h) &&
                   (form == LK_E4M3 ? (reinterpret_cast<uintptr_t>(y) & 7) == 0 : al16(y));
  switch (form) {
    case LK_Q8_ROWS: return vec ? pick<LK_Q8_ROWS, true>(a, 0, s) : pick<LK_Q8_ROWS, false>(a, 0, s);
    case LK_F16_ROWS: return vec ? pick<LK_F16_ROWS, true>(a, 0, s) : pick<LK_F16_ROWS, false>(a, 0, s);
    case LK_E4M3: return vec ? pick<LK_E4M3, true>(a, 0, s) : pick<LK_E4M3, false>(a, 0, s);
  }
  return vec ? pick<LK_F32, true>(a, form, s) : pick<LK_F32, false>(a, form, s);
}

LK_STATUS_READER(status_norm)

}  // namespace lk
