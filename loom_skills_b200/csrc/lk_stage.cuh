// The prefill GEMMs' weight staging: packed chunks of 256 values in shared memory -> f16 rows of a K-major tile in the
// 128-byte swizzle the tensor core reads, one 32-value group at a time, with the reference's one-rounding rules
// (lk_gemm.cu, lk_gemmx.cu).
#pragma once
#include "lk_common.cuh"
#include "lk_formats.cuh"

namespace lk {

// packed bytes of one 256-value chunk of a row, and the bytes a window of it takes in shared memory: the chunk
// copied from its 16-byte aligned start, so up to 15 bytes before and after it
__host__ __device__ constexpr int chunk_bytes(int fmt) { return 256 / fmt_qk(fmt) * fmt_block_bytes(fmt); }
__host__ __device__ constexpr int window_bytes(int fmt) { return (chunk_bytes(fmt) + 15 + 15) / 16 * 16; }
// shared-memory bytes of one row's chunk: the TMA box form's 144, a window of the format's chunk, or for a format pair
// the largest window of any format (Q8_0's)
__host__ __device__ constexpr int row_slot_bytes(int fmt, bool win) {
  return !win ? kChunkBytes : fmt == kFmtPair ? window_bytes(LK_Q8_0) : window_bytes(fmt);
}

LK_DEV uint32_t hsub2u(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
LK_DEV uint32_t hmul2u(uint32_t a, __half2 b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), b);
  return *reinterpret_cast<uint32_t*>(&r);
}
LK_DEV uint32_t hfma2u(uint32_t a, __half2 b, __half2 c) {
  __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), b, c);
  return *reinterpret_cast<uint32_t*>(&r);
}

// N little-endian words from a 2-byte aligned shared-memory address: N + 1 aligned loads and funnel shifts (the
// load past the end stays inside the CTA's shared memory: the row windows are followed by the staging buffers)
template <int N>
LK_DEV void ld_words_2a(const uint8_t* p, uint32_t (&w)[N]) {
  // explicit shared-memory loads: the aligned address is formed as an integer, and a generic load through it would
  // not be known to be shared
  const uint32_t a = smem_u32(p), base = a & ~3u, sh = (a & 3u) * 8u;
  uint32_t v[N + 1];
#pragma unroll
  for (int i = 0; i <= N; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i]) : "r"(base + 4u * i));
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], sh);
}

// Word-wise f16 staging of one 32-value group for the formats whose codes sit in whole bytes or nibble/bit planes
// (Q8_0, Q5_0, Q5_K, Q6_K): 4 codes per 32-bit word, f16(1024 + code) by a byte permute, the exact code (or centred
// code) by one f16 subtraction, then the reference's single rounding -- one f16 multiply by d (Q8_0, Q5_0), or the
// f16 fma of the K-quants with f16(d sc) and f16(-dmin m) / f16(-32 d sc) -- the same operations group_f16 does value
// by value. words[i] = codes of values 4i..4i+3; s / o: the scale and offset of values 0..15 (s[0], o[0]) and 16..31.
LK_DEV void stage_words(const uint32_t (&c)[8], uint32_t bias, const __half2 (&s)[2], const __half2 (&o)[2], bool fma,
                        uint8_t* b_tile, int r, int c0) {
#pragma unroll
  for (int cc = 0; cc < 4; ++cc) {
    const __half2 sc = s[cc >> 1], of = o[cc >> 1];
    uint32_t h[4] = {prmt(c[2 * cc], 0x64646464u, 0x4140u), prmt(c[2 * cc], 0x64646464u, 0x4342u),
                     prmt(c[2 * cc + 1], 0x64646464u, 0x4140u), prmt(c[2 * cc + 1], 0x64646464u, 0x4342u)};
    uint4 out;
    uint32_t* po = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
    for (int t = 0; t < 4; ++t) po[t] = fma ? hfma2u(hsub2u(h[t], bias), sc, of) : hmul2u(hsub2u(h[t], bias), sc);
    *reinterpret_cast<uint4*>(b_tile + sw128(r, c0 + cc)) = out;
  }
}

template <int FMT>
LK_DEV void dequant_group_words(const uint8_t* chunk, int j, uint8_t* b_tile, int r, int c0) {
  uint32_t c[8];
  __half2 s[2], o[2];
  if (FMT == LK_Q8_0) {   // int8 codes: code ^ 0x80 = code + 128; f16(1152 + code) - 1152 = code; f16(d code)
    const uint8_t* b = chunk + 34 * j;
    ld_words_2a(b + 2, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] ^= 0x80808080u;
    const __half d = __ushort_as_half(*reinterpret_cast<const uint16_t*>(b));
    s[0] = s[1] = __halves2half2(d, d);
    stage_words(c, 0x64806480u, s, s, false, b_tile, r, c0);
  } else if (FMT == LK_Q5_0) {   // nibble | bit i of qh << 4; f16(1024 + code) - 1040 = code - 16; f16(d (code - 16))
    const uint8_t* b = chunk + 22 * j;
    uint32_t qh[1], qs[4];
    ld_words_2a(b + 2, qh);
    ld_words_2a(b + 6, qs);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t hb = (qh[0] >> (4 * i)) & 15u;
      c[i] = ((i < 4 ? qs[i] : qs[i - 4] >> 4) & 0x0F0F0F0Fu) |
             ((hb & 1u) << 4) | ((hb & 2u) << 11) | ((hb & 4u) << 18) | ((hb & 8u) << 25);
    }
    const __half d = __ushort_as_half(*reinterpret_cast<const uint16_t*>(b));
    s[0] = s[1] = __halves2half2(d, d);
    stage_words(c, 0x64106410u, s, s, false, b_tile, r, c0);
  } else if (FMT == LK_Q5_K) {   // Q4_K's nibble pages | bit j of qh[l] << 4; fma(code, f16(d sc), f16(-dmin m))
    int sc, m;
    q4k_scale_min(chunk + 4, j, sc, m);
    uint32_t qs[8], qh[8];
    ld_words_2a(chunk + 48 + 32 * (j >> 1), qs);
    ld_words_2a(chunk + 16, qh);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[i] = ((qs[i] >> (4 * (j & 1))) & 0x0F0F0F0Fu) | (((qh[i] >> j) & 0x01010101u) << 4);
    s[0] = s[1] = __float2half2_rn(f16_at(chunk) * float(sc));
    o[0] = o[1] = __float2half2_rn(-(f16_at(chunk + 2) * float(m)));
    stage_words(c, 0x64006400u, s, o, true, b_tile, r, c0);
  } else {   // Q6_K: ql nibble | 2 bits of qh << 4 (0..63); fma(code, f16(d sc), f16(-32 d sc)) per 16 values
    const int h = j >> 2, jj = j & 3;
    uint32_t ql[8], qh[8];
    ld_words_2a(chunk + 64 * h + 32 * (jj & 1), ql);
    ld_words_2a(chunk + 128 + 32 * h, qh);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[i] = ((ql[i] >> (4 * (jj >> 1))) & 0x0F0F0F0Fu) | (((qh[i] >> (2 * jj)) & 0x03030303u) << 4);
    const float d = f16_at(chunk + 208);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float a = d * float(int8_t(chunk[192 + 2 * j + t]));
      s[t] = __float2half2_rn(a);
      o[t] = __float2half2_rn(-32.0f * a);
    }
    stage_words(c, 0x64006400u, s, o, true, b_tile, r, c0);
  }
}

// One 32-value group (j of the 256-value chunk) of any format into 4 swizzled 16-byte chunks of the B tile, with the
// reference's staging (group_f16: one rounding, or the K-quants' f16 fma)
template <int FMT>
LK_DEV void dequant_group_any(const uint8_t* chunk, int j, uint8_t* b_tile, int r, int c0) {
  if (FMT == LK_Q8_0 || FMT == LK_Q5_0 || FMT == LK_Q5_K || FMT == LK_Q6_K) {
    dequant_group_words<FMT>(chunk, j, b_tile, r, c0);
    return;
  }
  __half h[32];
  if (fmt_qk(FMT) == 32) group_f16<FMT>(chunk + j * fmt_block_bytes(FMT), 0, h);
  else group_f16<FMT>(chunk, j, h);
#pragma unroll
  for (int cc = 0; cc < 4; ++cc)
    *reinterpret_cast<uint4*>(b_tile + sw128(r, c0 + cc)) = reinterpret_cast<const uint4*>(h)[cc];
}

// 8 codes (bytes of t0, t1; low nibble only) -> 8 f16 (1024 + code), natural k order
LK_DEV void magic8(uint32_t t0, uint32_t t1, uint32_t (&h)[4]) {
  h[0] = prmt(t0, 0x64646464u, 0x4140u);
  h[1] = prmt(t0, 0x64646464u, 0x4342u);
  h[2] = prmt(t1, 0x64646464u, 0x4140u);
  h[3] = prmt(t1, 0x64646464u, 0x4342u);
}

// Dequantise one 32-value group of one weight row into 4 swizzled 16-byte chunks of the B tile.
//   raw    : the row's 144-byte packed chunk (256 values) in shared memory
//   j      : group within the chunk (0..7); b_tile: the B stage; r: tile row; c0: first 16-byte chunk (0 or 4)
// Register arithmetic only: scales are formed in f16 (exact products rounded once), no conversion instructions.
template <int FMT>
LK_DEV void dequant_group(const uint8_t* raw, int j, uint8_t* b_tile, int r, int c0) {
  if (FMT == LK_Q4_K) {
    const uint8_t* qs = raw + 16 + 32 * (j >> 1);
    uint4 a = *reinterpret_cast<const uint4*>(qs);
    uint4 b = *reinterpret_cast<const uint4*>(qs + 16);
    uint4 hd = *reinterpret_cast<const uint4*>(raw);
    uint32_t sh = (j & 1) * 4;
    uint32_t c[8] = {(a.x >> sh) & 0x0F0F0F0Fu, (a.y >> sh) & 0x0F0F0F0Fu, (a.z >> sh) & 0x0F0F0F0Fu,
                     (a.w >> sh) & 0x0F0F0F0Fu, (b.x >> sh) & 0x0F0F0F0Fu, (b.y >> sh) & 0x0F0F0F0Fu,
                     (b.z >> sh) & 0x0F0F0F0Fu, (b.w >> sh) & 0x0F0F0F0Fu};
    uint32_t sc, m;
    q4k_scale_min_w(hd.y, hd.z, hd.w, j, sc, m);
    // f16(d * sc) and f16(-dmin * m): the f16 product of exact operands rounds once, like the f32 product + fptrunc
    __half a16 = __hmul(__ushort_as_half(uint16_t(hd.x & 0xffffu)), small_int_half(sc));
    __half c16 = __hneg(__hmul(__ushort_as_half(uint16_t(hd.x >> 16)), small_int_half(m)));
    __half2 scale = __halves2half2(a16, a16), offset = __halves2half2(c16, c16);
    const uint32_t k1024 = 0x64006400u;
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {
      uint32_t h[4];
      magic8(c[2 * cc], c[2 * cc + 1], h);
      uint4 out;
      out.x = hfma2u(hsub2u(h[0], k1024), scale, offset);
      out.y = hfma2u(hsub2u(h[1], k1024), scale, offset);
      out.z = hfma2u(hsub2u(h[2], k1024), scale, offset);
      out.w = hfma2u(hsub2u(h[3], k1024), scale, offset);
      *reinterpret_cast<uint4*>(b_tile + sw128(r, c0 + cc)) = out;
    }
    return;
  }
  // Q4_0 / IQ4_NL: 18-byte block j at raw + 18j: f16 d, then 16 code bytes (2-byte aligned)
  const uint16_t* p16 = reinterpret_cast<const uint16_t*>(raw + 18 * j);
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = uint32_t(p16[1 + 2 * i]) | (uint32_t(p16[2 + 2 * i]) << 16);
  __half dh = __ushort_as_half(p16[0]);
  __half2 scale = __halves2half2(dh, dh);
  const uint32_t koff = FMT == LK_Q4_0 ? 0x64086408u : 0x64806480u;   // f16 1032 (1024 + 8) | 1152 (1024 + 128)
#pragma unroll
  for (int cc = 0; cc < 4; ++cc) {
    // chunk cc: values 8cc .. 8cc+7 = (cc < 2 ? low : high) nibbles of bytes 8*(cc&1) .. +7
    uint32_t w0 = q[2 * (cc & 1)], w1 = q[2 * (cc & 1) + 1];
    uint32_t t0 = ((cc >= 2) ? (w0 >> 4) : w0) & 0x0F0F0F0Fu;
    uint32_t t1 = ((cc >= 2) ? (w1 >> 4) : w1) & 0x0F0F0F0Fu;
    if (FMT == LK_IQ4_NL) {
      t0 = iq4_lookup4(t0);
      t1 = iq4_lookup4(t1);
    }
    uint32_t h[4];
    magic8(t0, t1, h);
    uint4 out;
    // exact centred code (q - 8, or the kvalue), then one f16 multiply by d: the reference's single rounding
    out.x = hmul2u(hsub2u(h[0], koff), scale);
    out.y = hmul2u(hsub2u(h[1], koff), scale);
    out.z = hmul2u(hsub2u(h[2], koff), scale);
    out.w = hmul2u(hsub2u(h[3], koff), scale);
    *reinterpret_cast<uint4*>(b_tile + sw128(r, c0 + cc)) = out;
  }
}

// dequant_group / dequant_group_any of the format `fmt` read at run time (format pairs)
LK_DEV void dequant_group_rt(int fmt, const uint8_t* chunk, int j, uint8_t* b_tile, int r, int c0) {
  switch (fmt) {
    case LK_Q4_0: dequant_group<LK_Q4_0>(chunk, j, b_tile, r, c0); return;
    case LK_IQ4_NL: dequant_group<LK_IQ4_NL>(chunk, j, b_tile, r, c0); return;
    case LK_Q4_K:   // the box form's register decode where the window left the 144-byte chunk 16-byte aligned
      if ((reinterpret_cast<uintptr_t>(chunk) & 15) == 0) dequant_group<LK_Q4_K>(chunk, j, b_tile, r, c0);
      else dequant_group_any<LK_Q4_K>(chunk, j, b_tile, r, c0);
      return;
    case LK_Q5_0: dequant_group_any<LK_Q5_0>(chunk, j, b_tile, r, c0); return;
    case LK_Q8_0: dequant_group_any<LK_Q8_0>(chunk, j, b_tile, r, c0); return;
    case LK_Q5_K: dequant_group_any<LK_Q5_K>(chunk, j, b_tile, r, c0); return;
    case LK_Q6_K: dequant_group_any<LK_Q6_K>(chunk, j, b_tile, r, c0); return;
    case LK_IQ4_XS: dequant_group_any<LK_IQ4_XS>(chunk, j, b_tile, r, c0); return;
    case LK_Q3_K: dequant_group_any<LK_Q3_K>(chunk, j, b_tile, r, c0); return;
    case LK_IQ3_S: dequant_group_any<LK_IQ3_S>(chunk, j, b_tile, r, c0); return;
    case LK_MXFP4: dequant_group_any<LK_MXFP4>(chunk, j, b_tile, r, c0); return;
  }
}

}  // namespace lk
