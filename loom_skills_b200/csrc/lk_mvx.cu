// Decode product on int8 activation codes with its epilogue (lk_mv_q8_ex):
//   p[t][n] = sum over 32-value groups g of d[t][g] * sum_i W[n][32 g + i] * c[t][32 g + i]
//   y = act(p + bias) + residual, or act(p_gate + bias) * (p_up + bias2) + residual
//
// The dot of a group runs on the int8 tensor cores: mma m16n8k32 takes 16 rows' weight codes and 8 tokens' activation
// codes of one group and gives the exact integer dots, which are then scaled in f32. An instruction costs the same for 1
// token as for 8, and the packed 4-bit words are already in its operand order (byte i of a block holds values i and
// 16 + i: one word gives a thread its low and its high half), so a weight is unpacked once for all tokens of the call.
//
// A CTA walks tiles of weight rows over all of k in stages. A producer fills a ring; 16 consumer warps are two groups of
// 8, a warp taking 32 rows (of a pair: 16 gate and 16 up rows) of one of 8 k slices. Many tiles: a tile is 64 rows, each
// group takes 32 of them. At most one tile an SM: a tile is 32 rows and the groups take its stages in turn. The warps'
// f32 sums meet at the tile's end in shared memory, where one thread finishes each output, in a fixed order of sums.
//
// The minima of Q4_K and Q5_K, sum_g dmin m[n][g] * d[t][g] sum_c[t][g], are a product over groups of their own: mma
// m16n8k4 with the 6-bit m (exact in tf32) and d * sum as the sum of two tf32 parts (22 bits), then one FMA by dmin.
//
// Two ways into shared memory. Box form (rows, codes and meta at 16-byte strides): TMA boxes of 128 bytes x 32 rows in
// the 128-byte swizzle, which puts the 8 rows x 4 words a warp reads at once into 32 banks; the activations stay in
// shared memory after a CTA's first tile where they leave three stages of weights. Row form (anything else): a bulk copy
// per row and token into padded slots; a copy costs about 85 clocks whatever its size, which bounds this form.
//
// Measured, a Q4_K pair of 4096 -> 12288 (56.6 MB, 8.8 us at the measured copy rate): 16.1 us at 8 tokens (3.5 TB/s), 23.9 at
// 16, 35.9 at 32; the loads alone 10.9, 13.1 and 15.7. The rest is instruction issue: one scale per 32 values, row and
// token. One token of the 4-bit formats is lk_mv1.cu's.
#include <cstring>

#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_formats.cuh"
#include "lk_internal.h"
#include "lk_rings.cuh"

namespace lk {

int make_map(CUtensorMap* map, const void* base, CUtensorMapDataType dt, int elem_bytes, int64_t rows, int64_t cols,
             int box_cols, int box_rows, CUtensorMapSwizzle swz);

namespace {

using namespace mvx;

// 16 consumer warps and a warpgroup whose first warp is the producer: launched at 96 registers a thread (the most that 640
// threads can have), of which the producer's 128 threads give 64 each to the consumers' 512 (61440 in all, before and
// after). The consumers' loop needs about 110: with 96 and a lone producer warp, spills cost 5% (Q4_K) to 30% (Q6_K).
// The build holds every instantiation to the 96 (build.py): launched with fewer, the consumers' would never come free.
constexpr int kThreads = 32 * kCWarps + 128, kLaunchRegs = 96, kProducerRegs = 32, kConsumerRegs = 112;
static_assert(128 * kProducerRegs + 32 * kCWarps * kConsumerRegs <= kThreads * kLaunchRegs, "a split that waits forever");
constexpr uint32_t kWaitPolls = 1u << 22;

LK_DEV void mx_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
LK_DEV void mx_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct MvxArgs {
  int n, k, tokens;
  const uint8_t* codes;  // [tokens][k] int8
  const uint8_t* meta;   // [tokens][k/32][2] f32
  const uint8_t* w;
  const uint8_t* w2;
  int64_t rb;
  int units;             // tiles, or pairs of tiles (q8 output of a gate / up pair), of one token tile
  int tiles_per_unit;
  int stages;            // ring slots
  int resident;          // the activations of all of k stay in shared memory
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
LK_DEV uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
// four 8 x 16-byte matrices: lane l supplies the address of row l % 8 of matrix l / 8, and gets word l % 4 of row l / 4 of
// each -- the operand layout of the MMAs
LK_DEV void ldmatrix4(uint32_t a, uint32_t& m0, uint32_t& m1, uint32_t& m2, uint32_t& m3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(m0), "=r"(m1), "=r"(m2), "=r"(m3)
               : "r"(a));
}

// Where byte b of a stage of this thread's four tile rows (g, g + 8, g + 16, g + 24) sits in shared memory, and loads of
// all four. Row form: linear from each row's window, at any 2-byte alignment.
struct RowAt {
  static constexpr bool kBoxes = false;
  uint32_t p[4];
  template <int LOW>
  LK_DEV void word(uint32_t b, uint32_t (&u)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = p[i] + b, c = a & ~3u;
      u[i] = __funnelshift_r(lds(c), lds(c + 4), (a & 3u) * 8u);
    }
  }
  LK_DEV void half(uint32_t b, uint32_t (&u)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = lds16(p[i] + b);
  }
};
// Box form: 128-byte segments, PITCH bytes apart, of swizzled rows (16-byte chunk c of row r at c ^ (r & 7)). Row g + 8 is
// 1024 bytes on, rows g + 16 and g + 24 UP bytes (the second half of the box, or the up weight's box), all with the same
// swizzle, so one address serves four rows.
template <int PITCH, int UP>
struct BoxAt {
  static constexpr bool kBoxes = true;
  uint32_t p, off, x;      // row g in segment 0; the stage's first byte in it; (g & 7) << 4
  uint32_t mp, mx, mb;     // the row, its swizzle and the 16-byte step this lane supplies to ldmatrix4
  LK_DEV uint32_t at(uint32_t b) const {
    b += off;
    return p + (b >> 7) * PITCH + ((b & 0x7Fu) ^ x);
  }
  LK_DEV static constexpr uint32_t row_offset(int i) { return (i & 1) * 1024 + (i >> 1) * UP; }
  LK_DEV static void four(uint32_t a, uint32_t (&u)[4]) {
    u[0] = lds(a);
    u[1] = lds(a + 1024);
    u[2] = lds(a + UP);
    u[3] = lds(a + UP + 1024);
  }
  // words t of the 16-byte chunks at b (u) and b + 16 (v)
  LK_DEV void chunks(uint32_t b, uint32_t (&u)[4], uint32_t (&v)[4]) const {
    b += off + mb;
    const uint32_t a = mp + (b >> 7) * PITCH + ((b & 0x7Fu) ^ mx);
    ldmatrix4(a, u[0], u[1], v[0], v[1]);
    ldmatrix4(a + UP, u[2], u[3], v[2], v[3]);
  }
  // LOW: b mod 4 where it is known, else -1 (even)
  template <int LOW>
  LK_DEV void word(uint32_t b, uint32_t (&u)[4]) const {
    if (LOW == 0) {
      four(at(b), u);
      return;
    }
    uint32_t lo[4], hi[4];
    four(at(b & ~3u), lo);
    four(at((b & ~3u) + 4), hi);
    const uint32_t sh = LOW == 2 ? 16u : (b & 3u) * 8u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __funnelshift_r(lo[i], hi[i], sh);
  }
  LK_DEV void half(uint32_t b, uint32_t (&u)[4]) const {
    const uint32_t a = at(b);
    u[0] = lds16(a);
    u[1] = lds16(a + 1024);
    u[2] = lds16(a + UP);
    u[3] = lds16(a + UP + 1024);
  }
};

// 128 values (4 groups) of a thread's four tile rows: the packed words it contributes to the MMAs (t = lane & 3). For
// group j and row i, lo holds the codes of values 4t .. 4t + 3 and hi those of 16 + 4t .. 16 + 4t + 3, one per byte, u8 or
// s8, times the power of two that its scale divides by.
template <int FMT>
struct Slice {
  static constexpr bool kUnsigned = FMT == LK_Q4_K || FMT == LK_Q5_K;
  // lo and hi hold values 4t, 16 + 4t, 4t + 1, 16 + 4t + 1 and 4t + 2, ...: the activations' words are mixed alike
  static constexpr bool kMixed = FMT == LK_IQ4_NL || FMT == LK_IQ4_XS;
  static constexpr int kQk = fmt_qk(FMT), kBb = fmt_block_bytes(FMT);
  // byte c of block j, mod 4 (blocks start at a multiple of 8 for j = 0)
  static constexpr int low(int c, int j) { return (j * kBb + c) % 4; }
  uint32_t r[FMT == LK_Q8_0 || FMT == LK_Q5_0 ? 8 : FMT == LK_Q5_K || FMT == LK_Q6_K ? 6 : 4][4];   // [word][row]

  template <int J, class At>
  LK_DEV void load_block(const At& at, uint32_t b, int t) {
    if constexpr (FMT == LK_Q8_0) {
      at.template word<low(2, J)>(b + 2 + 4 * t, r[2 * J]);
      at.template word<low(2, J)>(b + 18 + 4 * t, r[2 * J + 1]);
    } else if constexpr (FMT == LK_Q5_0) {
      at.template word<low(6, J)>(b + 6 + 4 * t, r[2 * J]);
      // bits 4t .. 4t + 3 and 16 + 4t .. of qh, in one word: bits 0-3 and 16-19
      at.template word<low(2, J)>(b + 2, r[2 * J + 1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[2 * J + 1][i] = (r[2 * J + 1][i] >> (4 * t)) & 0x000F000Fu;
    } else {
      at.template word<low(2, J)>(b + 2 + 4 * t, r[J]);
    }
  }
  // part: which 128 values of the stage
  template <class At>
  LK_DEV void load(const At& at, int part, int t) {
    if constexpr (kQk == 32) {
      const uint32_t b = 4 * part * kBb;
      load_block<0>(at, b, t);
      load_block<1>(at, b + kBb, t);
      load_block<2>(at, b + 2 * kBb, t);
      load_block<3>(at, b + 3 * kBb, t);
    } else {
      const uint32_t b = (part >> 1) * kBb;   // half a super-block: groups 4 h .. 4 h + 3
      const int h = part & 1;
      if constexpr ((FMT == LK_Q4_K || FMT == LK_Q5_K) && At::kBoxes) {
        constexpr int kQs = FMT == LK_Q4_K ? 16 : 48;
        at.chunks(b + kQs + 64 * h, r[0], r[1]);
        at.chunks(b + kQs + 64 * h + 32, r[2], r[3]);
        if constexpr (FMT == LK_Q5_K) at.chunks(b + 16, r[4], r[5]);
      } else if constexpr (FMT == LK_Q4_K || FMT == LK_Q5_K || FMT == LK_IQ4_XS) {
        constexpr int kQs = FMT == LK_Q4_K ? 16 : FMT == LK_Q5_K ? 48 : 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) at.template word<0>(b + kQs + 64 * h + 16 * i + 4 * t, r[i]);
        if constexpr (FMT == LK_Q5_K) {
          at.template word<0>(b + 16 + 4 * t, r[4]);
          at.template word<0>(b + 32 + 4 * t, r[5]);
        }
      } else {   // Q6_K
#pragma unroll
        for (int i = 0; i < 4; ++i) at.template word<-1>(b + 64 * h + 16 * i + 4 * t, r[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) at.template word<-1>(b + 128 + 32 * h + 16 * i + 4 * t, r[4 + i]);
      }
      if constexpr (FMT == LK_Q5_K) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          r[4][i] >>= 4 * h;
          r[5][i] >>= 4 * h;
        }
      }
    }
  }

  // the codes of group j (0..3) of row i
  LK_DEV void codes(int i, int j, uint32_t& lo, uint32_t& hi) const {
    constexpr uint32_t kLow = 0x0F0F0F0Fu, kHigh = 0xF0F0F0F0u, kTop = 0x80808080u;
    if constexpr (FMT == LK_Q4_0) {            // 16 (q - 8)
      lo = ((r[j][i] << 4) & kHigh) ^ kTop;
      hi = (r[j][i] & kHigh) ^ kTop;
    } else if constexpr (FMT == LK_IQ4_NL || FMT == LK_IQ4_XS) {
      iq4_lookup8<0x80808080u>(r[j][i], lo, hi);   // values 4t, 16 + 4t, 4t + 1, 16 + 4t + 1 | 4t + 2, ... (kMixed)
    } else if constexpr (FMT == LK_Q8_0) {
      lo = r[2 * j][i];
      hi = r[2 * j + 1][i];
    } else if constexpr (FMT == LK_Q5_0) {     // 8 (q - 16): the nibble at bit 3, the fifth bit at 7
      const uint32_t q = r[2 * j][i], b = r[2 * j + 1][i];
      lo = (((q & kLow) << 3) | spread(b)) ^ kTop;
      hi = (((q >> 1) & 0x78787878u) | spread(b >> 16)) ^ kTop;
    } else if constexpr (FMT == LK_Q4_K) {     // page j / 2: even groups q, odd groups 16 q
      const uint32_t m = (j & 1) ? kHigh : kLow;
      lo = r[2 * (j >> 1)][i] & m;
      hi = r[2 * (j >> 1) + 1][i] & m;
    } else if constexpr (FMT == LK_Q5_K) {     // nibble | bit j << 4
      lo = ((r[2 * (j >> 1)][i] >> (4 * (j & 1))) & kLow) | (((r[4][i] >> j) & 0x01010101u) << 4);
      hi = ((r[2 * (j >> 1) + 1][i] >> (4 * (j & 1))) & kLow) | (((r[5][i] >> j) & 0x01010101u) << 4);
    } else {                                   // Q6_K: 4 (q - 32): nibble at bit 2, the two high bits at 6
      lo = six(r[2 * (j & 1)][i], r[4][i], j);
      hi = six(r[2 * (j & 1) + 1][i], r[5][i], j);
    }
  }
  // factor of the codes' scale, of even and of odd groups
  static constexpr float inv(int odd) {
    return FMT == LK_Q4_0 || (FMT == LK_Q4_K && odd) ? 0.0625f : FMT == LK_Q5_0 ? 0.125f : FMT == LK_Q6_K ? 0.25f : 1.0f;
  }

  // This lane's share of what the four lanes of a row exchange: scales s of group t of its four rows, and in m the second
  // 16 values' scales (Q6_K) or the 6-bit minima (Q4_K, Q5_K; dmin: their rows' factor).
  template <class At>
  LK_DEV static void scales(const At& at, int part, int t, float (&s)[4], float (&m)[4], float (&dmin)[4]) {
    uint32_t d[4];
    if constexpr (kQk == 32) {
      at.half((4 * part + t) * kBb, d);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = h2f(uint16_t(d[i])) * inv(0);
    } else {
      const uint32_t b = (part >> 1) * kBb;
      const int h = part & 1, j = 4 * h + t;
      if constexpr (FMT == LK_Q4_K || FMT == LK_Q5_K) {
        uint32_t s0[4], s1[4], s2[4];
        if constexpr (At::kBoxes) {
          const uint32_t a = at.at(b);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 q = lds128(a + at.row_offset(i));
            d[i] = q.x;
            s0[i] = q.y;
            s1[i] = q.z;
            s2[i] = q.w;
          }
        } else {
          at.template word<0>(b, d);
          at.template word<0>(b + 4, s0);
          at.template word<0>(b + 8, s1);
          at.template word<0>(b + 12, s2);
        }
        const float f = (t & 1) ? inv(1) : inv(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // q4k_scale_min_w with the half h, uniform in a warp, outside
          uint32_t sc = s0[i] >> (8 * t), mn = s1[i] >> (8 * t);
          if (h == 0) {
            sc &= 63u;
            mn &= 63u;
          } else {
            const uint32_t lo = s2[i] >> (8 * t);
            sc = (lo & 15u) | ((sc >> 2) & 48u);
            mn = ((lo >> 4) & 15u) | ((mn >> 2) & 48u);
          }
          s[i] = h2f(uint16_t(d[i] & 0xffffu)) * u2f(sc) * f;
          m[i] = u2f(mn);
          dmin[i] = h2f(uint16_t(d[i] >> 16));
        }
      } else if constexpr (FMT == LK_Q6_K) {
        uint32_t two[4];
        at.half(b + 192 + 2 * j, two);
        at.half(b + 208, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = h2f(uint16_t(d[i])) * inv(0);
          s[i] = f * float(int8_t(two[i] & 255u));
          m[i] = f * float(int8_t(two[i] >> 8));
        }
      } else {   // IQ4_XS
        uint32_t sh[4], sl[4];
        at.half(b, d);
        at.half(b + 2, sh);
        at.template word<0>(b + 4, sl);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ls = int(((sl[i] >> (4 * j)) & 15u) | (((sh[i] >> (2 * j)) & 3u) << 4));
          s[i] = h2f(uint16_t(d[i])) * float(ls - 32);
        }
      }
    }
  }

 private:
  LK_DEV static float u2f(uint32_t v) { return __uint_as_float(0x4B000000u | v) - 8388608.0f; }   // v < 2^23, exact
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
  for (int i = 0; i < 4; ++i) f[i] = __int_as_float(c[i]);   // |dot| < 2^22
}
LK_DEV void mma_k16(uint32_t a0, uint32_t a1, uint32_t b0, float (&f)[4]) {
  int c[4];
  asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(b0), "r"(kMagicBits));
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __int_as_float(c[i]);
}

// D += A . B of 16 x 4 by 4 x 8 in tf32 (the low 13 bits of the operands are not read)
LK_DEV void mma_tf32(float a0, float a1, float b, float (&d)[4]) {
  asm("mma.sync.aligned.m16n8k4.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(b)));
}

// 4 groups of 32 rows x 8 NT tokens: the warp's sums grow by the groups' dots. acc[q][4 h + 2 i + c]: row 16 h + 8 i + g,
// token 8 q + 2 t + c. x(q, pr, w): the codes' words of groups 2 pr and 2 pr + 1 for token 8 q + g; m(q, c, pr): (scale, sum of
// codes) of those groups for token 8 q + 2 t + c; xs(q): of group t for token 8 q + g. COLS: the columns a thread keeps (1
// where the call has one token).
template <int FMT, int NT, int COLS, class At, class XAt, class MAt, class SAt>
LK_DEV void slice_dot(const At& at, int part, int gc, int lane, const XAt& x, const MAt& m, const SAt& xs,
                      float (&acc)[NT][8]) {
  constexpr bool kTwo = FMT == LK_Q6_K, kMin = FMT == LK_Q4_K || FMT == LK_Q5_K;
  const int t = lane & 3;
  Slice<FMT> w;
  w.load(at, part, t);
  float s[4], z[4], dmin[4];
  Slice<FMT>::scales(at, part, t, s, z, dmin);
  if (kMin) {   // k is whole super-blocks: all 4 groups
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      const float v = xs(q), hi = __uint_as_float(__float_as_uint(v) & 0xFFFFE000u), lo = v - hi;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_tf32(z[2 * h], z[2 * h + 1], hi, p);
        mma_tf32(z[2 * h], z[2 * h + 1], lo, p);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float* a = &acc[q][4 * h + 2 * i];
          const float dm = -dmin[2 * h + i];
          if (COLS == 2) {
            const float2 v = fma2(make_float2(dm, dm), make_float2(p[2 * i], p[2 * i + 1]), make_float2(a[0], a[1]));
            a[0] = v.x;
            a[1] = v.y;
          } else {
            a[0] = fmaf(dm, p[2 * i], a[0]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int pr = 0; pr < 2; ++pr) {
    if (2 * pr >= gc) break;
    uint32_t lo[2][4], hi[2][4];   // [group][row]
    float a[2][4], b[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = 2 * pr + k, from = (lane & 28) | j;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[k][i] = __shfl_sync(0xFFFFFFFFu, s[i], from);
        if (kTwo) b[k][i] = __shfl_sync(0xFFFFFFFFu, z[i], from);
        w.codes(i, j, lo[k][i], hi[k][i]);
      }
    }
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      uint32_t xw[4];
      x(q, pr, xw);
      if (Slice<FMT>::kMixed) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t lo8 = xw[2 * k], hi8 = xw[2 * k + 1];
          xw[2 * k] = prmt(lo8, hi8, 0x5140u);
          xw[2 * k + 1] = prmt(lo8, hi8, 0x7362u);
        }
      }
      uint4 mt[2];
#pragma unroll
      for (int c = 0; c < COLS; ++c) mt[c] = m(q, c, pr);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (!At::kBoxes && 2 * pr + k >= gc) break;   // box form: an even number of groups
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[4], e[4];
          if (kTwo) {
            mma_k16(lo[k][2 * h], lo[k][2 * h + 1], xw[2 * k], f);
            mma_k16(hi[k][2 * h], hi[k][2 * h + 1], xw[2 * k + 1], e);
          } else {
            mma_k32<Slice<FMT>::kUnsigned>(lo[k][2 * h], lo[k][2 * h + 1], hi[k][2 * h], hi[k][2 * h + 1], xw[2 * k],
                                           xw[2 * k + 1], f);
          }
          if (COLS == 2) {   // both columns at once, the same sums as below
            const float2 d = k ? make_float2(__uint_as_float(mt[0].z), __uint_as_float(mt[1].z))
                               : make_float2(__uint_as_float(mt[0].x), __uint_as_float(mt[1].x));
            const float2 off = mul2(make_float2(-kMagic, -kMagic), d);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = 2 * h + i;
              float* p = &acc[q][4 * h + 2 * i];
              float2 v = make_float2(p[0], p[1]);
              v = fma2(fma2(make_float2(f[2 * i], f[2 * i + 1]), d, off), make_float2(a[k][r], a[k][r]), v);
              if (kTwo) v = fma2(fma2(make_float2(e[2 * i], e[2 * i + 1]), d, off), make_float2(b[k][r], b[k][r]), v);
              p[0] = v.x;
              p[1] = v.y;
            }
            continue;
          }
#pragma unroll
          for (int c = 0; c < COLS; ++c) {
            // dot * d as (12582912 + dot) * d - 12582912 * d: the scale has the 11 bits of an f16, so the second product
            // is exact and the whole rounds once (an infinite scale gives NaN)
            const float d = __uint_as_float(k ? mt[c].z : mt[c].x), off = -kMagic * d;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float& v = acc[q][4 * h + 2 * i + c];
              const int r = 2 * h + i;
              v = fmaf(fmaf(f[2 * i + c], d, off), a[k][r], v);
              if (kTwo) v = fmaf(fmaf(e[2 * i + c], d, off), b[k][r], v);
            }
          }
        }
      }
    }
  }
}

LK_DEV bool poll(uint64_t* bar, uint32_t phase) {
  for (uint32_t q = 0; q < kWaitPolls; ++q)
    if (mbar_try_wait(bar, phase)) return true;
  return false;
}

template <int FMT, int FORM, bool PAIR, int NT, int RG>
__global__ void __launch_bounds__(kThreads, 1)
    k_mvx(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap w2map,
          const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap mmap, const MvxArgs p) {
  constexpr int kV = stage_values(FMT, FORM, RG, NT), kCB = stage_bytes(FMT, kV), kWB = w_bytes(FMT, FORM, RG, kV);
  constexpr int kXB = x_bytes(FORM, NT, kV), kWSlot = slot_of(kCB), kT = 8 * NT;
  constexpr int kXSlot = slot_of(kV), kMetaSlot = slot_of(kV / 4);   // row form
  constexpr int kOutG = PAIR ? kRows / 2 : kRows, kOut = RG * kOutG;   // outputs of a row group, of a tile
  constexpr int kPitch = kOut * 128;                                   // a box: kOut rows of one weight
  constexpr int kRed = red_slices(NT);
  constexpr int kSub = kV / 1024;                  // 128-value parts of a warp's slice
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nst = (p.k + kV - 1) / kV, groups = p.k / 32, kS = p.stages;
  const int slot = kWB + (p.resident ? 0 : kXB);
  uint8_t* xres = smem + kS * slot;                                    // resident activations
  float* red = reinterpret_cast<float*>(xres + (p.resident ? nst * kXB : 0));   // [slice][token][36]
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(red) + red_bytes(NT));
  uint64_t* empty = full + kMaxStages;
  float* first = reinterpret_cast<float*>(full) + 64;                  // [32 tokens][16]: a unit's first tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.y * kT, ntok = min(kT, p.tokens - t0);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kS; ++i) {
      mbar_init(&full[i], 2);   // the weights' bytes and the activations' are announced apart
      mbar_init(&empty[i], releases(RG, kS));
    }
    fence_mbar_init();
  }
  __syncthreads();
  mx_launch();
  // row form: tile row r, gate or up weight (rows past n read row 0's bytes and are never stored)
  auto row_src = [&](int tile, int r, int st) {
    const int n = tile * kOut + (PAIR ? r & 15 : r);
    const uint8_t* b = PAIR && r >= 16 ? p.w2 : p.w;
    return reinterpret_cast<uintptr_t>(b) + uintptr_t(int64_t(n < p.n ? n : 0) * p.rb + int64_t(st) * kCB);
  };
  const int ntile = (p.n + kOut - 1) / kOut;

  if (warp >= kCWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    if (warp != kCWarps) return;
    // ------------------------------------------------------------------ producer
    bool live = true, waited = false, used = false;   // used: the ring has been round once
    int s = 0, round = 0;                              // round: tiles so far
    uint32_t turn = 0;
    if (lane == 0 && FORM != kRowForm) {
      prefetch_tensormap(&wmap);
      if (PAIR) prefetch_tensormap(&w2map);
    }
    for (int u = blockIdx.x; u < p.units && live; u += gridDim.x) {
      for (int i = 0; i < p.tiles_per_unit && live; ++i, ++round) {
        const int tile = u * p.tiles_per_unit + i;
        if (tile >= ntile) break;
        for (int st = 0; st < nst; ++st) {
          if (used && !__all_sync(0xFFFFFFFFu, poll(&empty[s], turn ^ 1))) {
            atomicOr(&g_status, 1u);
            live = false;
            break;
          }
          uint8_t* dst = smem + s * slot;
          const int64_t b0 = int64_t(st) * kCB;
          const uint32_t len = uint32_t(min(int64_t(kCB), p.rb - b0));
          if (FORM != kRowForm) {
            if (lane == 0) {
              const int seg0 = int(b0 >> 7), segs = int((b0 + len + 127) >> 7) - seg0;
              mbar_expect_tx(&full[s], uint32_t(segs) * RG * kRows * 128);
              for (int g = 0; g < segs; ++g) {
                tma_load_2d(dst + g * kPitch, &wmap, (seg0 + g) * 32, tile * kOut, &full[s]);
                if (PAIR) tma_load_2d(dst + kWB / 2 + g * kPitch, &w2map, (seg0 + g) * 32, tile * kOut, &full[s]);
              }
            }
          } else {
            const uintptr_t src = row_src(tile, lane, st);
            const uint32_t bytes = window(src, len);
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
          const int gc = min(kV / 32, groups - st * (kV / 32));   // groups of the stage
          uint8_t* xd = p.resident ? xres + st * kXB : dst + kWB;
          if (p.resident && round > 0) {
            if (lane == 0) mbar_arrive(&full[s]);
          } else if (FORM == kBox1) {
            if (lane == 0) {
              const int64_t g0 = int64_t(t0) * groups + st * (kV / 32);
              mbar_expect_tx(&full[s], gc * 40);
              bulk_g2s(xd, p.codes + g0 * 32, gc * 32, &full[s]);
              bulk_g2s(xd + kV, p.meta + g0 * 8, gc * 8, &full[s]);
            }
          } else if (FORM == kBox) {
            if (lane == 0) {
              const int nc = (gc + 3) / 4, nm = (gc + 15) / 16;   // boxes of 128 codes, of 16 groups' meta
              mbar_expect_tx(&full[s], uint32_t(nc + nm) * kT * 128);
              for (int g = 0; g < nc; ++g) tma_load_2d(xd + g * kT * 128, &xmap, st * kV + g * 128, t0, &full[s]);
              for (int g = 0; g < nm; ++g)
                tma_load_2d(xd + kT * kV + g * kT * 128, &mmap, st * (kV / 16) + g * 32, t0, &full[s]);
            }
          } else {
            const int64_t g0 = int64_t(t0 + lane) * groups + st * (kV / 32);
            const uintptr_t cs = reinterpret_cast<uintptr_t>(p.codes) + g0 * 32, ms = reinterpret_cast<uintptr_t>(p.meta) + g0 * 8;
            const uint32_t mb = window(ms, gc * 8);
            uint32_t total = lane < ntok ? gc * 32 + mb : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
            if (lane == 0) mbar_expect_tx(&full[s], total);
            __syncwarp();
            if (lane < ntok) {
              bulk_g2s(xd + lane * kXSlot, reinterpret_cast<const void*>(cs), gc * 32, &full[s]);
              bulk_g2s(xd + kT * kXSlot + lane * kMetaSlot, reinterpret_cast<const void*>(ms & ~uintptr_t(15)), mb, &full[s]);
            }
          }
          __syncwarp();
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
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  mx_wait();
  const int group = warp / kSlices, ks = warp % kSlices, g = lane >> 2, t = lane & 3;
  const uint32_t sbase = smem_u32(smem), xbase = smem_u32(xres);
  // this thread's activations inside a stage: the codes it loads or supplies the address of (box forms: row lane % 8 and
  // 16-byte chunk lane / 8 of ldmatrix4), and the meta of tokens 8 q + 2 t and 8 q + 2 t + 1. Columns past the call's
  // tokens repeat the last one (row form) or hold zeros (boxes), and are never stored.
  uint32_t xoff[NT], moff[NT][2], soff[NT];
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    xoff[q] = FORM == kBox1 ? (lane >> 3) * 16 : FORM == kBox ? (8 * q + (lane & 7)) * 128 : min(8 * q + g, ntok - 1) * kXSlot + 4 * t;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int tk = 8 * q + 2 * t + c, tr = min(tk, ntok - 1);
      const uint32_t a = uint32_t(reinterpret_cast<uintptr_t>(p.meta)) + uint32_t(t0 + tr) * uint32_t(groups) * 8u;
      moff[q][c] = FORM == kBox1 ? kV : FORM == kBox ? kT * kV + tk * 128 : kT * kXSlot + tr * kMetaSlot + (a & 15u);
    }
    // the meta of group t of token 8 q + g
    const int tr = min(8 * q + g, ntok - 1);
    const uint32_t a = uint32_t(reinterpret_cast<uintptr_t>(p.meta)) + uint32_t(t0 + tr) * uint32_t(groups) * 8u;
    soff[q] = FORM == kBox1 ? kV + 8 * t : FORM == kBox ? kT * kV + (8 * q + g) * 128 + 8 * (t & 1)
                                                        : kT * kXSlot + tr * kMetaSlot + (a & 15u) + 8 * t;
  }
  int s = 0;
  uint32_t turn = 0;
  bool live = true;
  int round = 0;   // tiles so far
  // a warp whose wait gave up skips the stages left but comes to every barrier, so that the others end too
  for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
    for (int i = 0; i < p.tiles_per_unit; ++i, ++round) {
      const int tile = u * p.tiles_per_unit + i;
      if (tile >= ntile) break;
      float acc[NT][8];
#pragma unroll
      for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[q][c] = 0.0f;
      uint32_t low[4];   // row form: low address bits of the four rows' windows
#pragma unroll
      for (int r = 0; r < 4; ++r) low[r] = FORM == kRowForm ? uint32_t(row_src(tile, 8 * r + g, 0)) : 0u;
      auto next = [&] {
        if (++s == kS) {
          s = 0;
          turn ^= 1;
        }
      };
      for (int st = 0; st < nst && live; ++st) {
        const bool mine = takes(RG, group, st, round);
        if (!mine && !follows(RG, kS)) {
          next();
          continue;
        }
        if (!__all_sync(0xFFFFFFFFu, poll(&full[s], turn))) {
          atomicOr(&g_status, 1u);
          live = false;
          break;
        }
        if (!mine) {
          if (lane == 0) mbar_arrive(&empty[s]);
          next();
          continue;
        }
        const uint32_t sb = sbase + s * slot, xb = p.resident ? xbase + st * kXB : sb + kWB;
        const int gst = min(kV / 32, groups - st * (kV / 32));
#pragma unroll 1
        for (int sub = 0; sub < kSub; ++sub) {
          const int part = ks * kSub + sub, gc = gst - 4 * part;   // which 128 values; groups left there
          if (gc <= 0) break;
          // words of groups 4 part + 2 pr and + 1: values 4t.. and 16 + 4t.. of each
          auto xa = [&](int q, int pr, uint32_t (&w)[4]) {
            if constexpr (FORM == kBox) {   // one box per 128 values
              ldmatrix4(xb + part * kT * 128 + (xoff[q] ^ uint32_t(((4 * pr + (lane >> 3)) ^ (lane & 7)) << 4)), w[0], w[1],
                        w[2], w[3]);
            } else if constexpr (FORM == kBox1) {
              ldmatrix4(xb + xoff[q] + part * 128 + 64 * pr, w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = lds(xb + xoff[q] + part * 128 + 64 * pr + 16 * i);
            }
          };
          auto ma = [&](int q, int c, int pr) {
            if constexpr (FORM == kBox)   // one box per 16 groups: 16-byte chunk (group / 2) of the token's row
              return lds128(xb + (part >> 2) * kT * 128 + moff[q][c] +
                            uint32_t(((2 * (part & 3) + pr) ^ (2 * t + c)) << 4));
            if constexpr (FORM == kBox1) return lds128(xb + moff[q][c] + part * 32 + 16 * pr);
            const uint32_t a = xb + moff[q][c] + part * 32 + 16 * pr;
            return make_uint4(lds(a), lds(a + 4), lds(a + 8), lds(a + 12));
          };
          auto sa = [&](int q) {
            const uint32_t a = FORM == kBox ? xb + (part >> 2) * kT * 128 + soff[q] + uint32_t(((2 * (part & 3) + (t >> 1)) ^ g) << 4)
                                            : xb + soff[q] + part * 32;
            return __uint_as_float(lds(a)) * __uint_as_float(lds(a + 4));
          };
          constexpr int kCols = FORM == kBox1 ? 1 : 2;
          if constexpr (FORM == kRowForm) {
            RowAt at;
#pragma unroll
            for (int r = 0; r < 4; ++r) at.p[r] = sb + (8 * r + g) * kWSlot + ((low[r] + uint32_t(st) * kCB) & 15u);
            slice_dot<FMT, NT, kCols>(at, part, gc, lane, xa, ma, sa, acc);
          } else {
            const uint32_t base = sb + (RG == 2 ? group * kOutG * 128 : 0);
            const BoxAt<kPitch, PAIR ? kWB / 2 : 16 * 128> at{base + g * 128, uint32_t(int64_t(st) * kCB) & 127u,
                                                              uint32_t(g) << 4, base + (lane & 15) * 128,
                                                              uint32_t(lane & 7) << 4, uint32_t(lane >> 4) << 4};
            slice_dot<FMT, NT, kCols>(at, part, gc, lane, xa, ma, sa, acc);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        next();
      }
      // the warps' sums meet: [warp][token][row]. Where half of the warps write and the other half adds, the first are
      // group 1 (one row group) or slices 4 .. 7 of both (two).
      const bool late = kRed == kCWarps ? false : RG == 1 ? group == 0 : ks < kSlices / 2;
      const int at = kRed == kCWarps ? group * kSlices + ks : RG == 1 ? ks : group * (kSlices / 2) + ks % (kSlices / 2);
      float* mine = red + at * kT * kTokStride + 2 * t * kTokStride + g;
      asm volatile("bar.sync 1, 512;" ::: "memory");   // the last tile's have been read
      if (!late) {
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int c = 0; c < 8; ++c) mine[(8 * q + (c & 1)) * kTokStride + 8 * (c >> 1)] = acc[q][c];
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");
      if (kRed != kCWarps) {
        if (late) {
#pragma unroll
          for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int c = 0; c < 8; ++c) mine[(8 * q + (c & 1)) * kTokStride + 8 * (c >> 1)] += acc[q][c];
        }
        asm volatile("bar.sync 1, 512;" ::: "memory");
      }
      const int ctid = threadIdx.x;
      for (int o = ctid; o < kT * kOut; o += 32 * kCWarps) {   // whole warps: kOut * 8 is a multiple of 32
        const int tk = o / kOut, r = o % kOut, n = tile * kOut + r;
        const bool in = tk < ntok && n < p.n;
        float v = 0.0f;
        if (in) {
          float a = 0.0f, b = 0.0f;
#pragma unroll
          for (int q = 0; q < kRed / 2; ++q) {
            // one row group: warps q and q + kRed / 2 hold this output's sums; two: the group's own kRed / 2 warps
            const float* e = red + ((RG == 2 ? r / kOutG * (kRed / 2) : 0) + q) * kT * kTokStride + tk * kTokStride + r % kOutG;
            constexpr int kOther = kRed / 2 * kT * kTokStride;
            a += RG == 1 ? e[0] + e[kOther] : e[0];
            if (PAIR) b += RG == 1 ? e[16] + e[kOther + 16] : e[16];
          }
          if (p.e.bias) a += __ldg(p.e.bias + n);
          if (PAIR && p.e.bias2) b += __ldg(p.e.bias2 + n);
          v = PAIR ? act_pair(p.e.act, a, b, p.e.alpha, p.e.limit) : act_one(p.e.act, a);
          if (p.e.res) v += load_elem(p.e.res, p.e.res_dtype, int64_t(t0 + tk) * p.n + n);
        }
        if (p.e.y_form != LK_Q8_ROWS) {
          if (in) store_elem(p.e.y, p.e.y_form, int64_t(t0 + tk) * p.n + n, v);
        } else if (kOut % 32 == 0) {
          if (in)   // n % 32 == 0: a warp is a whole group of one token, inside or past the last output
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

struct Maps {
  CUtensorMap w, w2, x, m;
};

template <int FMT, int FORM, bool PAIR, int NT, int RG>
int launch(const Maps& m, MvxArgs a, cudaStream_t s) {
  constexpr int kV = stage_values(FMT, FORM, RG, NT), kXB = x_bytes(FORM, NT, kV);
  static_assert(two_stages(FMT, FORM, RG, NT, kV), "two stages at least");
  static_assert(2 * kMaxStages * 8 <= 256, "the barriers");
  const Ring ring = ring_of(FMT, FORM, RG, NT, a.k);
  a.resident = ring.resident;
  a.stages = ring.stages;
  const int smem = fixed_bytes(NT) + ring.stages * ring.slot + (ring.resident ? ring.nst * kXB : 0);
  auto kern = k_mvx<FMT, FORM, PAIR, NT, RG>;
  static std::atomic<unsigned> allowed{0};
  if (!allow_smem(kern, kSmemMax, allowed)) return LK_ECUDA;
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
  return cudaLaunchKernelEx(&cfg, kern, m.w, m.w2, m.x, m.m, a) == cudaSuccess ? LK_OK : LK_ECUDA;
}

template <int FMT, int FORM, bool PAIR, int NT>
int launch_r(const Maps& m, const MvxArgs& a, int rg, cudaStream_t s) {
  if constexpr (two_groups(FMT, FORM, NT)) {
    if (rg == 2) return launch<FMT, FORM, PAIR, NT, 2>(m, a, s);
  }
  return launch<FMT, FORM, PAIR, NT, 1>(m, a, s);
}
template <int FMT, int FORM, bool PAIR>
int launch_t(const Maps& m, const MvxArgs& a, int rg, cudaStream_t s) {
  if (FORM == kBox1 || a.tokens <= 8) return launch_r<FMT, FORM, PAIR, 1>(m, a, rg, s);
  if (a.tokens <= 16) return launch_r<FMT, FORM == kBox1 ? kBox : FORM, PAIR, 2>(m, a, rg, s);
  return launch_r<FMT, FORM == kBox1 ? kBox : FORM, PAIR, 4>(m, a, rg, s);
}

template <int FMT>
int launch_f(MvxArgs a, cudaStream_t s) {
  auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool pair = a.w2 != nullptr;
  // boxes: rows, codes and meta at 16-byte strides from 16-byte aligned starts
  const bool box = a.rb % 16 == 0 && al16(a.w) && al16(a.w2) && a.k % 64 == 0 && a.k >= 256;
  const int form = !box ? kRowForm : a.tokens == 1 ? kBox1 : kBox, nt = a.tokens <= 8 ? 1 : a.tokens <= 16 ? 2 : 4;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int outs = pair ? kRows / 2 : kRows;
  // 64-row tiles where there are more 32-row ones than SMs
  const int rg = (a.n + outs - 1) / outs > sms && two_groups(FMT, form, nt) ? 2 : 1;
  const int tiles = (a.n + rg * outs - 1) / (rg * outs);
  a.tiles_per_unit = rg == 1 && pair && a.e.y_form == LK_Q8_ROWS ? 2 : 1;   // 32 outputs: a group of the q8 form
  a.units = (tiles + a.tiles_per_unit - 1) / a.tiles_per_unit;
  Maps m;
  if (!box) {
    memset(&m, 0, sizeof(m));
    return pair ? launch_t<FMT, kRowForm, true>(m, a, rg, s) : launch_t<FMT, kRowForm, false>(m, a, rg, s);
  }
  const int rows = rg * outs;
  int rc = make_map(&m.w, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, a.n, a.rb / 4, 32, rows, CU_TENSOR_MAP_SWIZZLE_128B);
  m.w2 = m.x = m.m = m.w;
  if (rc == LK_OK && pair)
    rc = make_map(&m.w2, a.w2, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, a.n, a.rb / 4, 32, rows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == LK_OK && form == kBox)
    rc = make_map(&m.x, a.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.tokens, a.k, 128, 8 * nt, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == LK_OK && form == kBox)
    rc = make_map(&m.m, a.meta, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, a.tokens, a.k / 16, 32, 8 * nt, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != LK_OK) return rc;
  if (form == kBox1) return pair ? launch_t<FMT, kBox1, true>(m, a, rg, s) : launch_t<FMT, kBox1, false>(m, a, rg, s);
  return pair ? launch_t<FMT, kBox, true>(m, a, rg, s) : launch_t<FMT, kBox, false>(m, a, rg, s);
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
  if (int64_t(tokens) > 65535 * 32) return LK_ERANGE;
  if (tokens == 1 && mv_q8_one_takes(fmt, k, xq, w, w2)) return mv_q8_one(fmt, n, k, xq, w, w2, e, s);
  switch (fmt) {
    case LK_Q4_0: return launch_f<LK_Q4_0>(a, s);
    case LK_Q4_K: return launch_f<LK_Q4_K>(a, s);
    case LK_Q8_0: return launch_f<LK_Q8_0>(a, s);
    case LK_Q5_0: return launch_f<LK_Q5_0>(a, s);
    case LK_Q5_K: return launch_f<LK_Q5_K>(a, s);
    case LK_Q6_K: return launch_f<LK_Q6_K>(a, s);
    case LK_IQ4_NL: return launch_f<LK_IQ4_NL>(a, s);
    case LK_IQ4_XS: return launch_f<LK_IQ4_XS>(a, s);
  }
  return LK_EUNSUPPORTED;
}

LK_STATUS_READER(status_mvx)

}  // namespace lk
