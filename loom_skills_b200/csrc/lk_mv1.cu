// lk_mv_q8_ex for one token of Q4_K, Q4_0, IQ4_NL and Q6_K rows of up to 16384 values (multiples of 256).
//
// One token fills one of the eight columns of an int8 MMA, and what feeds the MMA -- nibbles to operand layout, scales to
// the lanes that need them -- is what lk_mvx.cu's kernel then spends its time on. Here a lane owns two units of 64
// values of every row (lk_q8.cuh): its activation codes stay in registers, the unit's scales are its own, and a unit
// costs 3 or 9 shared loads (Q6_K: 18), 16 masks and 16 dp4a. The Q4_K pair of 4096 -> 12288 takes 10.4 us (5.4 TB/s, 86 % of the
// measured copy rate) against 14.0 on the MMA form, Q4_0 4096 -> 4096 4.3 against 4.6, 4096 -> 1024 3.3 against 3.6.
//
// A CTA an SM: a producer streams whole rows (they are contiguous: one bulk copy for a stage's rows of a weight) into a
// ring of 160 to 216 KB; consumer warps, each the owner of 4096 values of two rows of a stage (a gate row and its up row, or two
// outputs), leave their sums in shared memory; a finisher warp adds the slices in order, applies the epilogue and
// stores, and only then frees the stage, so no consumer waits for an output.
#include <type_traits>

#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_internal.h"
#include "lk_q8.cuh"

namespace lk {
namespace {

constexpr int kSliceChunks = 16;   // 4096 values of a row: a warp's part of it
constexpr int chunk_bytes(int fmt) { return fmt == LK_Q6_K ? 210 : kChunkBytes; }
constexpr int slice_bytes(int fmt) { return kSliceChunks * chunk_bytes(fmt); }
constexpr uint32_t kWaitPolls = 1u << 22;

// row groups of a stage for rows of S slices: 16 consumer warps (12 of S = 3); each group takes two rows
constexpr int groups_of(int s) { return s == 1 ? 16 : s == 2 ? 8 : 4; }
constexpr int stages_of(int fmt, int s) { return fmt == LK_Q6_K ? 2 : s == 3 ? 4 : 3; }

LK_DEV void m1_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
LK_DEV void m1_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
LK_DEV bool poll(uint64_t* bar, uint32_t phase) {
  for (uint32_t q = 0; q < kWaitPolls; ++q)
    if (mbar_try_wait(bar, phase)) return true;
  return false;
}

// Two consecutive IQ4_NL blocks (Q4_0's layout): 8 codes of a word at once come out as values 4j, 16 + 4j, 4j + 1, ..., so
// the unit's activation words are mixed alike when they are loaded.
LK_DEV void mix(uint32_t (&x)[8]) {
  uint32_t y[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[2 * j] = prmt(x[j], x[4 + j], 0x5140u);
    y[2 * j + 1] = prmt(x[j], x[4 + j], 0x7362u);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = y[j];
}
LK_DEV float iq4_unit_dot(const uint8_t* sb, const q8::XUnit& u, int pg) {
  const uint32_t* bw = reinterpret_cast<const uint32_t*>(sb + 36 * pg);
  uint32_t v[9];
#pragma unroll
  for (int j = 0; j < 9; ++j) v[j] = bw[j];
  int i0 = 0, i1 = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t a, b;
    iq4_lookup8<0x80808080u>(__funnelshift_r(v[j], v[j + 1], 16), a, b);
    i0 = __dp4a(int(b), int(u.xa[2 * j + 1]), __dp4a(int(a), int(u.xa[2 * j]), i0));
    iq4_lookup8<0x80808080u>(v[5 + j], a, b);
    i1 = __dp4a(int(b), int(u.xb[2 * j + 1]), __dp4a(int(a), int(u.xb[2 * j]), i1));
  }
  return h2f(uint16_t(v[0] & 0xffffu)) * u.dx0 * q8::i2f_small(i0) + h2f(uint16_t(v[4] >> 16)) * u.dx1 * q8::i2f_small(i1);
}

// Q6_K: unit pg of a super-block is values 16 i .. 16 i + 15 of the four groups of half h (pg = 2 h + i): 16 bytes of low
// nibbles for two groups each and 16 of high bits, four scales. Super-blocks start at even bytes.
struct XUnit6 {
  uint32_t x[16];
  float dx[4];
  int s32[4];   // 32 x the sum of the 16 codes: the weights are q - 32
};
LK_DEV void load_x6(const uint8_t* codes, const float* meta, int c, int pg, XUnit6& u) {
  const int h = pg >> 1, i = pg & 1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(codes + c * 256 + 128 * h + 32 * j + 16 * i));
    u.x[4 * j] = v.x;
    u.x[4 * j + 1] = v.y;
    u.x[4 * j + 2] = v.z;
    u.x[4 * j + 3] = v.w;
    u.dx[j] = __ldg(meta + 2 * (c * 8 + 4 * h + j));
    int s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) s = __dp4a(int(u.x[4 * j + k]), 0x01010101, s);
    u.s32[j] = 32 * s;
  }
}
template <int N>
LK_DEV void ld_even(uint32_t a, uint32_t (&w)[N]) {
  const uint32_t base = a & ~3u, sh = (a & 2u) * 8u;
  uint32_t v[N + 1];
#pragma unroll
  for (int i = 0; i <= N; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i]) : "r"(base + 4u * i));
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], sh);
}
LK_DEV float q6_unit_dot(const uint8_t* sb, const XUnit6& u, int pg) {
  const uint32_t a = smem_u32(sb), h = pg >> 1, i = pg & 1;
  uint32_t q0[4], q1[4], qh[4], sc[2];
  ld_even(a + 64 * h + 16 * i, q0);
  ld_even(a + 64 * h + 32 + 16 * i, q1);
  ld_even(a + 128 + 32 * h + 16 * i, qh);
  ld_even(a + 192 + 8 * h, sc);   // bytes 2 j + i: the scale of group j
  int dot[4] = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    constexpr uint32_t kLow = 0x0F0F0F0Fu, kTwo = 0x30303030u;
    dot[0] = q8::dp4a_us((q0[k] & kLow) | ((qh[k] << 4) & kTwo), u.x[k], dot[0]);
    dot[1] = q8::dp4a_us((q1[k] & kLow) | ((qh[k] << 2) & kTwo), u.x[4 + k], dot[1]);
    dot[2] = q8::dp4a_us(((q0[k] >> 4) & kLow) | (qh[k] & kTwo), u.x[8 + k], dot[2]);
    dot[3] = q8::dp4a_us(((q1[k] >> 4) & kLow) | ((qh[k] >> 2) & kTwo), u.x[12 + k], dot[3]);
  }
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int scale = int(int8_t((sc[j >> 1] >> (16 * (j & 1) + 8 * i)) & 255u));
    s = fmaf(u.dx[j] * float(scale), q8::i2f_small(dot[j] - u.s32[j]), s);
  }
  return h2f(*reinterpret_cast<const uint16_t*>(sb + 208)) * s;
}

struct Mv1Args {
  int n, k;
  const uint8_t* xq;   // codes, then meta
  const uint8_t* w;
  const uint8_t* w2;
  int units;           // of `spu` stages each, dealt to the CTAs in turn (the q8 form: a group of 32 outputs)
  int spu;
  Epilogue e;
};

template <int FMT, bool PAIR, int S>
__global__ void __launch_bounds__(32 * (2 + groups_of(S) * S), 1) k_mv1(const Mv1Args p) {
  constexpr int kG = groups_of(S), kCW = kG * S, kNst = stages_of(FMT, S), kRowsT = 2 * kG;
  constexpr int kOut = PAIR ? kG : 2 * kG;   // outputs of a stage
  constexpr int kStage = kRowsT * S * slice_bytes(FMT), kCB = chunk_bytes(FMT);
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float part[kNst][kRowsT][S];
  __shared__ uint64_t full[kNst], done[kNst], empty[kNst];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunks = p.k >> 8, row_b = chunks * chunk_bytes(FMT);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kNst; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&done[i], kCW);
      mbar_init(&empty[i], 1);
    }
    fence_mbar_init();
  }
  __syncthreads();
  m1_launch();
  const int spu = p.spu, my = (p.units - int(blockIdx.x) + int(gridDim.x) - 1) / int(gridDim.x) * spu;   // this CTA's stages
  // first output of this CTA's stage i
  auto first_of = [&](int i) { return (int64_t(blockIdx.x) + int64_t(i / spu) * gridDim.x) * (spu * kOut) + i % spu * kOut; };

  if (warp == 0) {
    // ------------------------------------------------------------------ producer (one lane)
    if (lane == 0) {
      bool live = true;
      for (int i = 0; i < my; ++i) {
        const int s = i % kNst;
        if (i == 1) m1_wait();   // one stage of weights goes out before the previous kernel ends
        if (i >= kNst && !poll(&empty[s], ((i / kNst) - 1) & 1)) {
          atomicOr(&g_status, 1u);
          live = false;
          break;
        }
        const int64_t o0 = first_of(i);
        const int64_t left = p.n - o0;
        const int outs = left <= 0 ? 0 : left < kOut ? int(left) : kOut;
        uint8_t* dst = ring + s * kStage;
        mbar_expect_tx(&full[s], uint32_t(outs) * row_b * (PAIR ? 2 : 1));
        if (outs > 0) {
          bulk_g2s(dst, p.w + o0 * row_b, uint32_t(outs) * row_b, &full[s]);
          if (PAIR) bulk_g2s(dst + kG * row_b, p.w2 + o0 * row_b, uint32_t(outs) * row_b, &full[s]);
        }
      }
      if (!live)   // let the copies in flight land before the CTA ends
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    return;
  }
  m1_wait();
  bool live = true;   // a warp whose wait gave up still walks its stages, so that the others end too
  if (warp == 1) {
    // ------------------------------------------------------------------ finisher: a lane an output
    float v = 0.0f;
    for (int i = 0; i < my; ++i) {
      const int s = i % kNst, j = i % spu, mine = lane - j * kOut;
      if (live && !__all_sync(0xFFFFFFFFu, poll(&done[s], (i / kNst) & 1))) {
        if (lane == 0) atomicOr(&g_status, 1u);
        live = false;
      }
      const int64_t n = first_of(i) + mine;
      if (mine >= 0 && mine < kOut && n < p.n) {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int q = 0; q < S; ++q) {
          a += part[s][mine][q];
          if (PAIR) b += part[s][kG + mine][q];
        }
        if (p.e.bias) a += __ldg(p.e.bias + n);
        if (PAIR && p.e.bias2) b += __ldg(p.e.bias2 + n);
        v = PAIR ? act_pair(p.e.act, a, b, p.e.alpha, p.e.limit) : act_one(p.e.act, a);
        if (p.e.res) v += load_elem(p.e.res, p.e.res_dtype, n);
        if (p.e.y_form != LK_Q8_ROWS) store_elem(p.e.y, p.e.y_form, n, v);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (p.e.y_form == LK_Q8_ROWS && j == spu - 1)   // a unit is a group of 32 outputs
        store_q8(static_cast<uint8_t*>(p.e.y), p.n, first_of(i) - j * kOut + lane, v, lane);
    }
    return;
  }
  // -------------------------------------------------------------------- consumers
  const int g = (warp - 2) / S, sl = (warp - 2) % S, pg = lane & 3;
  const int ra = PAIR ? g : 2 * g, rb = PAIR ? kG + g : 2 * g + 1;   // this warp's rows of a stage
  constexpr int kLike = FMT == LK_IQ4_NL ? LK_Q4_0 : FMT;
  std::conditional_t<FMT == LK_Q6_K, XUnit6, q8::XUnit> xu[2];
  const int c0 = kSliceChunks * sl + (lane >> 2);   // this lane's units: page pg of chunks c0 and c0 + 8, inside the row
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (c0 + 8 * u >= chunks) break;
    const float* meta = reinterpret_cast<const float*>(p.xq + p.k);
    if constexpr (FMT == LK_Q6_K) load_x6(p.xq, meta, c0 + 8 * u, pg, xu[u]);
    else q8::load_xunit<kLike, false>(p.xq, meta, c0 + 8 * u, pg, xu[u]);
    if constexpr (FMT == LK_IQ4_NL) {
      mix(xu[u].xa);
      mix(xu[u].xb);
    }
  }
  const uint32_t hsel = q8::q4k_hsel(pg), big = q8::q4k_big(pg);
  for (int i = 0; i < my; ++i) {
    const int s = i % kNst;
    if (live && !__all_sync(0xFFFFFFFFu, poll(&full[s], (i / kNst) & 1))) {
      if (lane == 0) atomicOr(&g_status, 1u);
      live = false;
    }
    const uint8_t* base = ring + s * kStage + c0 * kCB;
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (c0 + 8 * u >= chunks) break;
      const uint8_t* wa = base + ra * row_b + 8 * u * kCB;
      const uint8_t* wb = base + rb * row_b + 8 * u * kCB;
      if constexpr (FMT == LK_Q6_K) {
        a += q6_unit_dot(wa, xu[u], pg);
        b += q6_unit_dot(wb, xu[u], pg);
      } else if constexpr (FMT == LK_IQ4_NL) {
        a += iq4_unit_dot(wa, xu[u], pg);
        b += iq4_unit_dot(wb, xu[u], pg);
      } else {
        a += q8::unit_dot<FMT>(wa, xu[u], pg, hsel, big);
        b += q8::unit_dot<FMT>(wb, xu[u], pg, hsel, big);
      }
    }
    // both rows' sums at once: lanes 0 .. 15 go on with row a's, 16 .. 31 with row b's
    const float give = lane < 16 ? b : a, keep = lane < 16 ? a : b;
    float t = keep + __shfl_xor_sync(0xFFFFFFFFu, give, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    if ((lane & 15) == 0) part[s][lane == 0 ? ra : rb][sl] = t;
    __syncwarp();
    if (lane == 0) mbar_arrive(&done[s]);
  }
}

template <int FMT, bool PAIR, int S>
int launch(Mv1Args a, cudaStream_t s) {
  constexpr int kOut = PAIR ? groups_of(S) : 2 * groups_of(S);
  constexpr int smem = stages_of(FMT, S) * 2 * groups_of(S) * S * slice_bytes(FMT);
  static_assert(smem + 2048 <= 227 * 1024, "the ring");
  auto kern = k_mv1<FMT, PAIR, S>;
  static std::atomic<unsigned> allowed{0};
  if (!allow_smem(kern, smem, allowed)) return LK_ECUDA;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t cfg = {};
  // full stages: evener ones (14 of 16 outputs for the pair's 12288, 7 of 32 for 1024) gained nothing, 10.4 -> 11.1 and 3.3
  // -> 3.4 us
  a.spu = a.e.y_form == LK_Q8_ROWS ? 32 / kOut : 1;
  a.units = (a.n + a.spu * kOut - 1) / (a.spu * kOut);
  cfg.gridDim = dim3(a.units < sms ? a.units : sms, 1, 1);
  cfg.blockDim = dim3(32 * (2 + groups_of(S) * S), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? LK_OK : LK_ECUDA;
}

template <int FMT>
int launch_f(const Mv1Args& a, cudaStream_t s) {
  switch ((a.k + 4095) / 4096) {
    case 1: return a.w2 ? launch<FMT, true, 1>(a, s) : launch<FMT, false, 1>(a, s);
    case 2: return a.w2 ? launch<FMT, true, 2>(a, s) : launch<FMT, false, 2>(a, s);
    case 3: return a.w2 ? launch<FMT, true, 3>(a, s) : launch<FMT, false, 3>(a, s);
    case 4: return a.w2 ? launch<FMT, true, 4>(a, s) : launch<FMT, false, 4>(a, s);
  }
  return LK_EUNSUPPORTED;
}

}  // namespace

// Q4_K and Q4_0: faster than the MMA form at every k tried (1024 to 16384). IQ4_NL, whose code lookups weigh more than the
// MMA's overhead: where at least 3/4 of the lanes of the row's slices have units (pair of 4096 -> 12288 17.3 us against
// 19.8, 13824 -> 5120 15.0 against 20.7, 12288 -> 4096 11.2 against 11.0; a pair of 5120 -> 13824 28.1 against 25.5). Q6_K:
// where rows start at 16-byte multiples (pair of 4096 -> 12288 18.9 against 23.6, 12288 -> 4096 12.1 against 13.0, 2048 ->
// 4096 4.0 against 4.6).
bool mv_q8_one_takes(int fmt, int k, const void* xq, const void* w, const void* w2) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(w2);
  const bool full = 4 * k >= 3 * ((k + 4095) / 4096 * 4096);
  const bool taken = fmt == LK_Q4_K || fmt == LK_Q4_0 || (fmt == LK_IQ4_NL && full) || (fmt == LK_Q6_K && k % 2048 == 0);
  return taken && k % 256 == 0 && k <= 16384 && (all & 15) == 0;
}

int mv_q8_one(int fmt, int n, int k, const uint8_t* xq, const void* w, const void* w2, const Epilogue& e, cudaStream_t s) {
  Mv1Args a{};
  a.n = n;
  a.k = k;
  a.xq = xq;
  a.w = static_cast<const uint8_t*>(w);
  a.w2 = static_cast<const uint8_t*>(w2);
  a.e = e;
  switch (fmt) {
    case LK_Q4_K: return launch_f<LK_Q4_K>(a, s);
    case LK_Q4_0: return launch_f<LK_Q4_0>(a, s);
    case LK_IQ4_NL: return launch_f<LK_IQ4_NL>(a, s);
    case LK_Q6_K: return launch_f<LK_Q6_K>(a, s);
  }
  return LK_EUNSUPPORTED;
}

LK_STATUS_READER(status_mv1)

}  // namespace lk
