// Decode product on int8 activation codes with its epilogue (lk_mv_q8_ex):
//   p[t][n] = sum over 32-value groups g of d[t][g] * sum_i W[n][32 g + i] * c[t][32 g + i]
//   y = act(p + bias) + residual, or act(p_gate + bias) * (p_up + bias2) + residual
//
// The dot of a group runs on the int8 tensor cores: mma m16n8k32 takes 16 rows' weight codes and 8 tokens' activation
// codes of one group and gives the exact integer dots, which are then scaled in f32. An instruction costs the same for 1
// token as for 8, and the packed 4-bit words are already in its operand order (byte i of a block holds values i and
// 16 + i: one word gives a thread its low and its high half), so a weight is unpacked once for all tokens of the call.
//
// A CTA walks tiles of 32 weight rows (of a pair: 16 gate and 16 up rows) over all of k in stages of 1024 values. A
// producer warp bulk-copies each row's 16-byte aligned window and the tokens' codes and group meta into a ring; 16
// consumer warps take a row half and one of 8 k slices of 128 values each, so a warp's f32 sums are 4 per 8 tokens, and
// meet at the tile's end in shared memory. There every output is finished by one thread, in a fixed order of sums.
#include <mutex>

#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_formats.cuh"
#include "lk_internal.h"

namespace lk {
namespace {

constexpr int kRows = 32;              // weight rows of a tile
constexpr int kSlices = 8;             // k slices of a stage
constexpr int kSliceG = 4;             // 32-value groups of a slice
constexpr int kStageV = kSlices * kSliceG * 32;
constexpr int kCWarps = 2 * kSlices;   // consumer warps
constexpr int kThreads = 32 * (1 + kCWarps);
constexpr int kTokStride = 36;         // floats between tokens of the partial sums: conflict-free stores
constexpr int kSmemMax = 227 * 1024;
constexpr uint32_t kWaitPolls = 1u << 22;

LK_DEV void mx_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
LK_DEV void mx_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// row slots of the shared stages: 16 bytes past a multiple of 128, so that the 8 rows x 4 words a warp reads at once
// fall into 32 banks; with room for a window's 15 leading bytes and a realigning load's trailing word
__host__ __device__ constexpr int slot_of(int bytes) { return (bytes + 32 + 111) / 128 * 128 + 16; }
__host__ __device__ constexpr int stage_bytes(int fmt) { return kStageV / fmt_qk(fmt) * fmt_block_bytes(fmt); }
constexpr int kXSlot = slot_of(kStageV), kMetaSlot = slot_of(kStageV / 32 * 8);
constexpr int slot_bytes(int fmt, int nt) { return kRows * slot_of(stage_bytes(fmt)) + 8 * nt * (kXSlot + kMetaSlot); }
constexpr int red_bytes(int nt) { return kSlices * 8 * nt * kTokStride * 4; }
constexpr int kTailBytes = 256 + 16 * 32 * 4;   // barriers; the first tile of a pair of tiles (q8 output of a pair)
constexpr int stages_of(int fmt, int nt) {
  const int s = (kSmemMax - red_bytes(nt) - kTailBytes) / slot_bytes(fmt, nt);
  return s > 8 ? 8 : s;
}

struct MvxArgs {
  int n, k, tokens;
  const uint8_t* codes;  // [tokens][k] int8
  const uint8_t* meta;   // [tokens][k/32][2] f32
  const uint8_t* w;
  const uint8_t* w2;
  int64_t rb;
  int units;             // tiles, or pairs of tiles (q8 output of a gate / up pair), of one token tile
  int tiles_per_unit;
  Epilogue e;
};

// bytes of the 16-byte aligned window around [src, src + len)
LK_DEV uint32_t window(uintptr_t src, uint32_t len) {
  return uint32_t(((src + len + 15) & ~uintptr_t(15)) - (src & ~uintptr_t(15)));
}
LK_DEV uint32_t lds(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
LK_DEV uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
// the word at a 2-byte aligned address (AL: 4-byte aligned)
template <bool AL>
LK_DEV uint32_t ldw(uint32_t a) {
  if (AL) return lds(a);
  const uint32_t b = a & ~3u;
  return __funnelshift_r(lds(b), lds(b + 4), (a & 3u) * 8u);
}
LK_DEV float lds_f16(uint32_t a) { return h2f(uint16_t(lds16(a))); }

// One weight row's slice of 4 groups: the packed words a thread (t = lane & 3) contributes to the MMAs. For group j,
// lo(j) holds the codes of values 4t .. 4t + 3 and hi(j) those of 16 + 4t .. 16 + 4t + 3, one per byte, as UNSIGNED ? u8 :
// s8 times 2^SHIFT.
template <int FMT, bool AL>
struct Slice {
  static constexpr bool kUnsigned = FMT == LK_Q4_K || FMT == LK_Q5_K;
  static constexpr int kQk = fmt_qk(FMT), kBb = fmt_block_bytes(FMT);
  uint32_t r[FMT == LK_Q8_0 || FMT == LK_Q5_0 ? 8 : FMT == LK_Q5_K || FMT == LK_Q6_K ? 6 : 4];

  // p: the row's chunk in shared memory; ks: the slice
  LK_DEV void load(uint32_t p, int ks, int t) {
    if (kQk == 32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = p + (4 * ks + j) * kBb;
        if (FMT == LK_Q8_0) {
          r[2 * j] = ldw<AL>(b + 2 + 4 * t);
          r[2 * j + 1] = ldw<AL>(b + 18 + 4 * t);
        } else if (FMT == LK_Q5_0) {
          r[2 * j] = ldw<AL>(b + 6 + 4 * t);
          // bits 4t .. 4t + 3 and 16 + 4t .. of qh, in one word: bits 0-3 and 16-19
          r[2 * j + 1] = (ldw<AL>(b + 2) >> (4 * t)) & 0x000F000Fu;
        } else {
          r[j] = ldw<AL>(b + 2 + 4 * t);
        }
      }
    } else {
      const uint32_t b = p + (ks >> 1) * kBb;   // the slice is half a super-block: groups 4 h .. 4 h + 3
      const int h = ks & 1;
      if (FMT == LK_Q4_K) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = ldw<AL>(b + 16 + 64 * h + 16 * i + 4 * t);
      } else if (FMT == LK_Q5_K) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = ldw<AL>(b + 48 + 64 * h + 16 * i + 4 * t);
#pragma unroll
        for (int i = 0; i < 2; ++i) r[4 + i] = ldw<AL>(b + 16 + 16 * i + 4 * t) >> (4 * h);
      } else if (FMT == LK_Q6_K) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = ldw<AL>(b + 64 * h + 16 * i + 4 * t);
#pragma unroll
        for (int i = 0; i < 2; ++i) r[4 + i] = ldw<AL>(b + 128 + 32 * h + 16 * i + 4 * t);
      } else {   // IQ4_XS
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = ldw<AL>(b + 8 + 64 * h + 16 * i + 4 * t);
      }
    }
  }

  // the codes of group j (0..3)
  LK_DEV void codes(int j, uint32_t& lo, uint32_t& hi) const {
    constexpr uint32_t kLow = 0x0F0F0F0Fu, kHigh = 0xF0F0F0F0u, kTop = 0x80808080u;
    if (FMT == LK_Q4_0) {            // 16 (q - 8)
      lo = ((r[j] << 4) & kHigh) ^ kTop;
      hi = (r[j] & kHigh) ^ kTop;
    } else if (FMT == LK_IQ4_NL || FMT == LK_IQ4_XS) {
      lo = iq4_lookup4(r[j] & kLow) ^ kTop;
      hi = iq4_lookup4((r[j] >> 4) & kLow) ^ kTop;
    } else if (FMT == LK_Q8_0) {
      lo = r[2 * j];
      hi = r[2 * j + 1];
    } else if (FMT == LK_Q5_0) {     // 8 (q - 16): the nibble at bit 3, the fifth bit at 7
      const uint32_t q = r[2 * j], b = r[2 * j + 1];
      lo = (((q & kLow) << 3) | spread(b)) ^ kTop;
      hi = (((q >> 1) & 0x78787878u) | spread(b >> 16)) ^ kTop;
    } else if (FMT == LK_Q4_K) {     // page j / 2: even groups q, odd groups 16 q
      const uint32_t m = (j & 1) ? kHigh : kLow;
      lo = r[2 * (j >> 1)] & m;
      hi = r[2 * (j >> 1) + 1] & m;
    } else if (FMT == LK_Q5_K) {     // nibble | bit j << 4
      lo = ((r[2 * (j >> 1)] >> (4 * (j & 1))) & kLow) | (((r[4] >> j) & 0x01010101u) << 4);
      hi = ((r[2 * (j >> 1) + 1] >> (4 * (j & 1))) & kLow) | (((r[5] >> j) & 0x01010101u) << 4);
    } else if (FMT == LK_Q6_K) {     // 4 (q - 32): nibble at bit 2, the two high bits at 6
      lo = six(r[2 * (j & 1)], r[4], j);
      hi = six(r[2 * (j & 1) + 1], r[5], j);
    }
  }
  // factor of the codes' scale
  static constexpr float kInv0 = FMT == LK_Q4_0 ? 0.0625f : FMT == LK_Q5_0 ? 0.125f : FMT == LK_Q6_K ? 0.25f : 1.0f;
  static constexpr float kInv1 = FMT == LK_Q4_K ? 0.0625f : kInv0;   // odd groups

  // scale s of group t, and its minimum (Q4_K, Q5_K) or its second 16 values' scale (Q6_K) in m: this lane's share of
  // what the four lanes of a row exchange
  LK_DEV static void scales(uint32_t p, int ks, int t, float& s, float& m) {
    m = 0.0f;
    if (kQk == 32) {
      s = lds_f16(p + (4 * ks + t) * kBb) * kInv0;
      return;
    }
    const uint32_t b = p + (ks >> 1) * kBb;
    const int j = 4 * (ks & 1) + t;
    if (FMT == LK_Q4_K || FMT == LK_Q5_K) {
      const uint32_t dd = ldw<AL>(b), s0 = ldw<AL>(b + 4), s1 = ldw<AL>(b + 8), s2 = ldw<AL>(b + 12);
      uint32_t sc, mn;
      q4k_scale_min_w(s0, s1, s2, j, sc, mn);
      s = h2f(uint16_t(dd & 0xffffu)) * float(sc) * ((t & 1) ? kInv1 : kInv0);
      m = h2f(uint16_t(dd >> 16)) * float(mn);
    } else if (FMT == LK_Q6_K) {
      const uint32_t two = lds16(b + 192 + 2 * j);
      const float d = lds_f16(b + 208) * kInv0;
      s = d * float(int8_t(two & 255u));
      m = d * float(int8_t(two >> 8));
    } else {   // IQ4_XS
      const uint32_t sh = lds16(b + 2), sl = ldw<AL>(b + 4);
      const int ls = int(((sl >> (4 * j)) & 15u) | (((sh >> (2 * j)) & 3u) << 4));
      s = lds_f16(b) * float(ls - 32);
    }
  }

 private:
  // bits 0..3 -> bit 7 of bytes 0..3
  LK_DEV static uint32_t spread(uint32_t b) { return ((b & 15u) * 0x10204080u) & 0x80808080u; }
  LK_DEV static uint32_t six(uint32_t ql, uint32_t qh, int j) {
    const uint32_t n = j < 2 ? (ql << 2) & 0x3C3C3C3Cu : (ql >> 2) & 0x3C3C3C3Cu;
    const uint32_t t = j == 0 ? qh << 6 : j == 1 ? qh << 4 : j == 2 ? qh << 2 : qh;
    return (n | (t & 0xC0C0C0C0u)) ^ 0x80808080u;
  }
};

// c = A . B over 32 (k16: the first 16) values, starting from 1.5 * 2^23: the bits of the float 12582912 + dot
constexpr int kMagicBits = 0x4B400000;
constexpr float kMagic = 12582912.0f;
template <bool UNSIGNED>
LK_DEV void mma_k32(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float (&f)[4]) {
  int c[4];
  if (UNSIGNED)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kMagicBits));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kMagicBits));
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __int_as_float(c[i]) - kMagic;   // exact: |dot| < 2^22
}
LK_DEV void mma_k16(uint32_t a0, uint32_t a1, uint32_t b0, float (&f)[4]) {
  int c[4];
  asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(b0), "r"(kMagicBits));
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __int_as_float(c[i]) - kMagic;
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

template <int FMT, bool AL, bool PAIR, int NT>
__global__ void __launch_bounds__(kThreads, 1) k_mvx(const MvxArgs p) {
  constexpr int kS = stages_of(FMT, NT), kSlot = slot_bytes(FMT, NT), kWSlot = slot_of(stage_bytes(FMT));
  constexpr int kCB = stage_bytes(FMT), kT = 8 * NT;
  constexpr int kOut = PAIR ? kRows / 2 : kRows;   // outputs of a tile
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem + kS * kSlot);            // [slice][token][36]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kS * kSlot + red_bytes(NT));
  uint64_t* empty = full + kS;
  float* first = reinterpret_cast<float*>(full) + 64;                  // [32 tokens][16]: a unit's first tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.y * kT, ntok = min(kT, p.tokens - t0);
  const int nst = (p.k + kStageV - 1) / kStageV, groups = p.k / 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kS; ++i) {
      mbar_init(&full[i], 2);   // the weights' bytes and the activations' are announced apart
      mbar_init(&empty[i], kCWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  mx_launch();
  // tile row r: gate or up weight and its row (rows past n read row 0's bytes and are never stored)
  auto row_src = [&](int tile, int r, int st) {
    const int n = PAIR ? tile * kOut + (r & 15) : tile * kOut + r;
    const uint8_t* b = PAIR && r >= 16 ? p.w2 : p.w;
    return reinterpret_cast<uintptr_t>(b) + uintptr_t(int64_t(n < p.n ? n : 0) * p.rb + int64_t(st) * kCB);
  };
  const int ntile = (p.n + kOut - 1) / kOut;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    bool live = true, waited = false;
    int s = 0;
    uint32_t turn = 0;
    bool used = false;   // the ring has been round once
    for (int u = blockIdx.x; u < p.units && live; u += gridDim.x) {
      for (int i = 0; i < p.tiles_per_unit && live; ++i) {
        const int tile = u * p.tiles_per_unit + i;
        if (tile >= ntile) break;
        for (int st = 0; st < nst; ++st) {
          if (used && !__all_sync(0xFFFFFFFFu, [&] {
                for (uint32_t q = 0; q < kWaitPolls; ++q)
                  if (mbar_try_wait(&empty[s], turn ^ 1)) return true;
                return false;
              }())) {
            atomicOr(&g_status, 1u);
            live = false;
            break;
          }
          uint8_t* dst = smem + s * kSlot;
          {
            const uintptr_t src = row_src(tile, lane, st);
            const uint32_t len = uint32_t(min(int64_t(kCB), p.rb - int64_t(st) * kCB)), bytes = window(src, len);
            uint32_t total = bytes;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
            if (lane == 0) mbar_expect_tx(&full[s], total);
            __syncwarp();
            bulk_g2s(dst + lane * kWSlot, reinterpret_cast<const void*>(src & ~uintptr_t(15)), bytes, &full[s]);
          }
          if (!waited) {   // the weights of the first stage go out before the previous kernel ends; its output after
            mx_wait();
            waited = true;
          }
          {
            const int gc = min(kStageV / 32, groups - st * (kStageV / 32));
            const int64_t g0 = int64_t(t0 + lane) * groups + st * (kStageV / 32);
            const uintptr_t cs = reinterpret_cast<uintptr_t>(p.codes) + g0 * 32, ms = reinterpret_cast<uintptr_t>(p.meta) + g0 * 8;
            const uint32_t mb = window(ms, gc * 8);
            uint32_t total = lane < ntok ? gc * 32 + mb : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
            if (lane == 0) mbar_expect_tx(&full[s], total);
            __syncwarp();
            if (lane < ntok) {
              uint8_t* xd = dst + kRows * kWSlot;
              bulk_g2s(xd + lane * kXSlot, reinterpret_cast<const void*>(cs), gc * 32, &full[s]);
              bulk_g2s(xd + kT * kXSlot + lane * kMetaSlot, reinterpret_cast<const void*>(ms & ~uintptr_t(15)), mb, &full[s]);
            }
          }
          if (++s == kS) {
            s = 0;
            turn ^= 1;
            used = true;
          }
        }
      }
    }
    if (!live)   // let the copies in flight land before the CTA ends
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    return;
  }

  // ------------------------------------------------------------------ consumers
  mx_wait();
  const int cw = warp - 1, half = cw >> 3, ks = cw & 7, g = lane >> 2, t = lane & 3;
  const uint32_t sbase = smem_u32(smem);
  int s = 0;
  uint32_t turn = 0;
  bool live = true;
  for (int u = blockIdx.x; u < p.units && live; u += gridDim.x) {
    for (int i = 0; i < p.tiles_per_unit && live; ++i) {
      const int tile = u * p.tiles_per_unit + i;
      if (tile >= ntile) break;
      float acc[NT][4];
#pragma unroll
      for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[q][c] = 0.0f;
      // low address bits of the two rows' windows: (row start + stage offset) mod 16
      const uint32_t r0 = uint32_t(row_src(tile, 16 * half + g, 0)), r1 = uint32_t(row_src(tile, 16 * half + g + 8, 0));
      const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>(p.meta)) + uint32_t(t0) * uint32_t(groups) * 8u;
      for (int st = 0; st < nst; ++st) {
        bool ok = false;
        for (uint32_t q = 0; q < kWaitPolls && !ok; ++q) ok = mbar_try_wait(&full[s], turn);
        if (!__all_sync(0xFFFFFFFFu, ok)) {
          atomicOr(&g_status, 1u);
          live = false;
          break;
        }
        const int gc = min(kStageV / 32, groups - st * (kStageV / 32)) - 4 * ks;   // groups of this slice
        if (gc > 0) {
          const uint32_t sb = sbase + s * kSlot;
          const uint32_t p0 = sb + (16 * half + g) * kWSlot + ((r0 + uint32_t(st) * kCB) & 15u);
          const uint32_t p1 = sb + (16 * half + g + 8) * kWSlot + ((r1 + uint32_t(st) * kCB) & 15u);
          const uint32_t xb = sb + kRows * kWSlot + ks * 128 + 4 * t;                 // + token * kXSlot
          const uint32_t mb = sb + kRows * kWSlot + kT * kXSlot + ks * 32;            // + token * kMetaSlot + window
          Slice<FMT, AL> w0, w1;
          w0.load(p0, ks, t);
          w1.load(p1, ks, t);
          float s0, z0, s1, z1;
          Slice<FMT, AL>::scales(p0, ks, t, s0, z0);
          Slice<FMT, AL>::scales(p1, ks, t, s1, z1);
#pragma unroll
          for (int j = 0; j < kSliceG; ++j) {
            if (j >= gc) break;
            const int from = (lane & 28) | j;
            const float a0 = __shfl_sync(0xFFFFFFFFu, s0, from), a1 = __shfl_sync(0xFFFFFFFFu, s1, from);
            float b0 = 0.0f, b1 = 0.0f;
            constexpr bool kTwo = FMT == LK_Q6_K, kMin = FMT == LK_Q4_K || FMT == LK_Q5_K;
            if (kTwo || kMin) {
              b0 = __shfl_sync(0xFFFFFFFFu, z0, from);
              b1 = __shfl_sync(0xFFFFFFFFu, z1, from);
            }
            uint32_t lo0, hi0, lo1, hi1;
            w0.codes(j, lo0, hi0);
            w1.codes(j, lo1, hi1);
#pragma unroll
            for (int q = 0; q < NT; ++q) {
              const int tok = 8 * q + g;
              uint32_t x0 = 0, x1 = 0;
              if (tok < ntok) {
                x0 = lds(xb + tok * kXSlot + 32 * j);
                x1 = lds(xb + tok * kXSlot + 32 * j + 16);
              }
              float d[2] = {0.0f, 0.0f}, xs[2] = {0.0f, 0.0f};
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int tk = 8 * q + 2 * t + c;
                if (tk < ntok) {
                  const uint32_t a = mb + tk * kMetaSlot + ((m0 + uint32_t(tk) * uint32_t(groups) * 8u) & 15u) + 8 * j;
                  d[c] = __uint_as_float(lds(a));
                  if (kMin) xs[c] = d[c] * __uint_as_float(lds(a + 4));
                }
              }
              float f[4];
              if (kTwo) {
                float h[4];
                mma_k16(lo0, lo1, x0, f);
                mma_k16(hi0, hi1, x1, h);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  acc[q][c] = fmaf(fmaf(h[c], c < 2 ? b0 : b1, f[c] * (c < 2 ? a0 : a1)), d[c & 1], acc[q][c]);
              } else {
                mma_k32<Slice<FMT, AL>::kUnsigned>(lo0, lo1, hi0, hi1, x0, x1, f);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  acc[q][c] = fmaf(f[c] * d[c & 1], c < 2 ? a0 : a1, acc[q][c]);
                  if (kMin) acc[q][c] = fmaf(-(c < 2 ? b0 : b1), xs[c & 1], acc[q][c]);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == kS) {
          s = 0;
          turn ^= 1;
        }
      }
      if (!__all_sync(0xFFFFFFFFu, live)) live = false;
      // the slices' sums meet: [slice][token][row]
      asm volatile("bar.sync 1, 512;" ::: "memory");   // the last tile's have been read
#pragma unroll
      for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          red[(ks * kT + 8 * q + 2 * t + (c & 1)) * kTokStride + 16 * half + g + (c >= 2 ? 8 : 0)] = acc[q][c];
      asm volatile("bar.sync 1, 512;" ::: "memory");
      const int ctid = threadIdx.x - 32;
      for (int o = ctid; o < kT * kOut; o += 32 * kCWarps) {   // whole warps: kOut * 8 is a multiple of 32
        const int tk = o / kOut, r = o % kOut, n = tile * kOut + r;
        const bool in = tk < ntok && n < p.n;
        float v = 0.0f;
        if (in) {
          float a = 0.0f, b = 0.0f;
#pragma unroll
          for (int q = 0; q < kSlices; ++q) {
            a += red[(q * kT + tk) * kTokStride + r];
            if (PAIR) b += red[(q * kT + tk) * kTokStride + 16 + r];
          }
          if (p.e.bias) a += __ldg(p.e.bias + n);
          if (PAIR && p.e.bias2) b += __ldg(p.e.bias2 + n);
          v = PAIR ? act_pair(p.e.act, a, b, p.e.alpha, p.e.limit) : act_one(p.e.act, a);
          if (p.e.res) v += load_elem(p.e.res, p.e.res_dtype, int64_t(t0 + tk) * p.n + n);
        }
        if (p.e.y_form != LK_Q8_ROWS) {
          if (in) store_elem(p.e.y, p.e.y_form, int64_t(t0 + tk) * p.n + n, v);
        } else if (!PAIR) {
          if (tk < ntok)   // n % 32 == 0: a warp is a whole group of one token
            store_q8(static_cast<uint8_t*>(p.e.y), int64_t(p.tokens) * p.n, int64_t(t0 + tk) * p.n + n, v, lane);
        } else if (i == 0) {
          first[tk * 16 + r] = v;   // the unit's second tile finishes the group
        } else {
          // lanes 0-15 hold token tk's second half (this lane's first half from shared memory), 16-31 token tk + 1's
          const float f = first[tk * 16 + r];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int src = 16 * k + (lane & 15);
            const float lo = __shfl_sync(0xFFFFFFFFu, f, src), hi = __shfl_sync(0xFFFFFFFFu, v, src);
            const int tok = (o - lane) / kOut + k;
            if (tok < ntok)
              store_q8(static_cast<uint8_t*>(p.e.y), int64_t(p.tokens) * p.n,
                       int64_t(t0 + tok) * p.n + (tile - 1) * kOut + lane, lane < 16 ? lo : hi, lane);
          }
        }
      }
    }
  }
}

template <int FMT, bool AL, bool PAIR, int NT>
int launch(const MvxArgs& a, cudaStream_t s) {
  constexpr int kS = stages_of(FMT, NT);
  static_assert(kS >= 2, "two stages at least");
  static_assert(kS * 16 <= 256 && kTailBytes >= 256 + 32 * 16 * 4, "the tail");
  constexpr int smem = kS * slot_bytes(FMT, NT) + red_bytes(NT) + kTailBytes;
  auto kern = k_mvx<FMT, AL, PAIR, NT>;
  static unsigned configured = 0;
  if (!once_per_device(configured)) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.units < sms ? a.units : sms, (a.tokens + 8 * NT - 1) / (8 * NT), 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? LK_OK : LK_ECUDA;
}

template <int FMT, bool AL>
int launch_f(const MvxArgs& a, cudaStream_t s) {
  if (a.w2) {
    if (a.tokens <= 8) return launch<FMT, AL, true, 1>(a, s);
    if (a.tokens <= 16) return launch<FMT, AL, true, 2>(a, s);
    return launch<FMT, AL, true, 4>(a, s);
  }
  if (a.tokens <= 8) return launch<FMT, AL, false, 1>(a, s);
  if (a.tokens <= 16) return launch<FMT, AL, false, 2>(a, s);
  return launch<FMT, AL, false, 4>(a, s);
}

}  // namespace

int mv_q8_ex(int fmt, int n, int k, int tokens, const uint8_t* xq, const void* w, const void* w2, const Epilogue& e,
             cudaStream_t s) {
  MvxArgs a{};
  a.n = n;
  a.k = k;
  a.tokens = tokens;
  a.codes = xq;
  a.meta = xq + int64_t(tokens) * k;
  a.w = static_cast<const uint8_t*>(w);
  a.w2 = static_cast<const uint8_t*>(w2);
  a.rb = lk_row_bytes(fmt, k);
  a.e = e;
  const int outs = w2 ? kRows / 2 : kRows, tiles = (n + outs - 1) / outs;
  a.tiles_per_unit = w2 && e.y_form == LK_Q8_ROWS ? 2 : 1;
  a.units = (tiles + a.tiles_per_unit - 1) / a.tiles_per_unit;
  if (int64_t(tokens) > 65535 * 32) return LK_ERANGE;
  // whole words where blocks and rows are multiples of 4 bytes (Q4_K, Q5_K, IQ4_XS) from a 4-byte aligned start
  const bool al = ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(w2)) & 3) == 0;
  switch (fmt) {
    case LK_Q4_0: return launch_f<LK_Q4_0, false>(a, s);
    case LK_Q8_0: return launch_f<LK_Q8_0, false>(a, s);
    case LK_Q5_0: return launch_f<LK_Q5_0, false>(a, s);
    case LK_Q6_K: return launch_f<LK_Q6_K, false>(a, s);
    case LK_IQ4_NL: return launch_f<LK_IQ4_NL, false>(a, s);
    case LK_Q4_K: return al ? launch_f<LK_Q4_K, true>(a, s) : launch_f<LK_Q4_K, false>(a, s);
    case LK_Q5_K: return al ? launch_f<LK_Q5_K, true>(a, s) : launch_f<LK_Q5_K, false>(a, s);
    case LK_IQ4_XS: return al ? launch_f<LK_IQ4_XS, true>(a, s) : launch_f<LK_IQ4_XS, false>(a, s);
  }
  return LK_EUNSUPPORTED;
}

LK_STATUS_READER(status_mvx)

}  // namespace lk
