// lk_mv_q8_ex for one token of Q4_K, Q4_0 and IQ4_NL rows of up to 16384 values (multiples of 256).
//
// One token fills one of the eight columns of an int8 MMA, and what feeds the MMA -- nibbles to operand layout, scales to
// the lanes that need them -- is what lk_mvx.cu's kernel then spends its time on. Here a lane owns two units of 64
// values of every row (lk_q8.cuh): its activation codes stay in registers, the unit's scales are its own, and a unit
// costs 3 or 9 shared loads, 16 masks and 16 dp4a. The Q4_K pair of 4096 -> 12288 takes 10.4 us (5.4 TB/s, 86 % of the
// measured copy rate) against 14.0 on the MMA form, Q4_0 4096 -> 4096 4.3 against 4.6, 4096 -> 1024 3.3 against 3.6.
//
// A CTA an SM: a producer streams whole rows (they are contiguous: one bulk copy for a stage's rows of a weight) into a
// ring of 216 KB; consumer warps, each the owner of 4096 values of two rows of a stage (a gate row and its up row, or two
// outputs), leave their sums in shared memory; a finisher warp adds the slices in order, applies the epilogue and
// stores, and only then frees the stage, so no consumer waits for an output.
#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_internal.h"
#include "lk_q8.cuh"

namespace lk {
namespace {

constexpr int kSliceChunks = 16, kRowSlice = kSliceChunks * kChunkBytes;   // 4096 values of a row: a warp's part of it
constexpr uint32_t kWaitPolls = 1u << 22;

// row groups of a stage for rows of S slices: 16 consumer warps (12 of S = 3); each group takes two rows
constexpr int groups_of(int s) { return s == 1 ? 16 : s == 2 ? 8 : 4; }
constexpr int stages_of(int s) { return s == 3 ? 4 : 3; }

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
  constexpr int kG = groups_of(S), kCW = kG * S, kNst = stages_of(S), kRowsT = 2 * kG;
  constexpr int kOut = PAIR ? kG : 2 * kG;   // outputs of a stage
  constexpr int kStage = kRowsT * S * kRowSlice;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float part[kNst][kRowsT][S];
  __shared__ uint64_t full[kNst], done[kNst], empty[kNst];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunks = p.k >> 8, row_b = chunks * kChunkBytes;
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
  q8::XUnit xu[2];
  const int c0 = kSliceChunks * sl + (lane >> 2);   // this lane's units: page pg of chunks c0 and c0 + 8, inside the row
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (c0 + 8 * u >= chunks) break;
    q8::load_xunit<kLike, false>(p.xq, reinterpret_cast<const float*>(p.xq + p.k), c0 + 8 * u, pg, xu[u]);
    if (FMT == LK_IQ4_NL) {
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
    const uint8_t* base = ring + s * kStage + c0 * kChunkBytes;
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (c0 + 8 * u >= chunks) break;
      const uint8_t* wa = base + ra * row_b + 8 * u * kChunkBytes;
      const uint8_t* wb = base + rb * row_b + 8 * u * kChunkBytes;
      if constexpr (FMT == LK_IQ4_NL) {
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
  constexpr int smem = stages_of(S) * 2 * groups_of(S) * S * kRowSlice;
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
// 19.8, 13824 -> 5120 15.0 against 20.7, 12288 -> 4096 11.2 against 11.0; a pair of 5120 -> 13824 28.1 against 25.5).
bool mv_q8_one_takes(int fmt, int k, const void* xq, const void* w, const void* w2) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(w2);
  const bool full = 4 * k >= 3 * ((k + 4095) / 4096 * 4096);
  return (fmt == LK_Q4_K || fmt == LK_Q4_0 || (fmt == LK_IQ4_NL && full)) && k % 256 == 0 && k <= 16384 && (all & 15) == 0;
}

int mv_q8_one(int fmt, int n, int k, const uint8_t* xq, const void* w, const void* w2, const Epilogue& e, cudaStream_t s) {
  Mv1Args a{};
  a.n = n;
  a.k = k;
  a.xq = xq;
  a.w = static_cast<const uint8_t*>(w);
  a.w2 = static_cast<const uint8_t*>(w2);
  a.e = e;
  return fmt == LK_Q4_K ? launch_f<LK_Q4_K>(a, s) : fmt == LK_Q4_0 ? launch_f<LK_Q4_0>(a, s) : launch_f<LK_IQ4_NL>(a, s);
}

LK_STATUS_READER(status_mv1)

}  // namespace lk
