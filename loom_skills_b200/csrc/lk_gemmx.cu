// Prefill product with its epilogue (lk_gemm_ex) on the 5th-generation tensor cores:
//   p[t][n] = scales[t][1] * sum_k x16[t][k] * W16[n][k],  W16 the GEMM's f16 staging of the packed weights
//   y = act(p + bias) + residual, or act(p_gate + bias) * (p_up + bias2) + residual
//
// The tile is computed transposed, D^T = W X^T: the weight rows are the M side of the MMA and the tokens its N side. A
// lane of TMEM then holds one output column n and its columns hold tokens, so the epilogue's bias is one value per lane,
// a store of one token is 32 consecutive outputs of its row without a detour through shared memory, and a short batch
// pads nothing but the N side (32 to 256 tokens). Gate and up rows of a pair alternate in the tile (row 2i gate, 2i + 1
// up), so both products of an output sit in neighbouring lanes: one shuffle brings them together.
//
// Two forms of one kernel:
//   CG = 2  two CTAs of a cluster share a 256 x 256 tile (tcgen05 cta_group::2): each stages 128 weight rows and loads
//           128 tokens, so a stage of 64 k moves 16 KB of activations and 4.5 KB of packed Q4 per SM for 2 x 128 x 256 x 64
//           products -- half of what a one-CTA 256 x 128 tile moves, which L2 bandwidth bounded. Persistent over the
//           tiles, two TMEM accumulators, so the epilogue of one tile runs under the next one's MMAs.
//   CG = 1  few tiles: 128 weight rows x NT tokens per cluster of S CTAs, each over its own range of k; the partial
//           tiles meet through distributed shared memory, each CTA finishing every S-th group of tokens. The order of
//           the sum is fixed, so results repeat bit for bit, and nothing waits on a CTA that may not be running.
//
// Measured (Q4_K, device time): a gate / up pair of 2048 x 4096 x 2 12288 309 to 320 us in a short burst from cold clocks (1.29 to
// 1.33 PFLOP/s), 362 where calls follow one another for seconds and the power limit holds (1.14; sustained cuBLAS bf16 is 1.42);
// IQ4_NL 4096 x 27648 x 5120 1028 to 1091 cold, 1170 sustained; the pair of 2048 rows in other formats (cold) IQ4_NL 338,
// Q5_0 383, Q8_0 380 to 430, Q6_K 415 to 463, IQ4_XS 606, MXFP4 618, Q5_K 761, IQ3_S 1168, Q3_K 3540: staging, by the value where
// the format has no word-wise decode.
// Many tokens: a stage moves 74 KB through shared memory (about 580 clocks) for 512 clocks of MMA. Few: staging a stage of
// weights and issuing its MMAs each take a warp 600 to 700 clocks of latency (64 x 4096 x 2 12288 47 to 55 us); more staging
// warps, deeper rings and looking ahead of the MMA warp's waits gained nothing.
//
// Warps: 0 loads token tiles and 2 packed weights (TMA), 1 issues the MMAs, 4.. stage weights (packed chunk -> f16 in
// the swizzled A tile), the last four run the epilogue.
#include "lk_common.cuh"
#include "lk_epi.cuh"
#include "lk_internal.h"
#include "lk_rings.cuh"
#include "lk_stage.cuh"

namespace lk {

int make_map(CUtensorMap* map, const void* base, CUtensorMapDataType dt, int elem_bytes, int64_t rows, int64_t cols,
             int box_cols, int box_rows, CUtensorMapSwizzle swz);
int encode_tiled(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const cuuint64_t* dims,
                 const cuuint64_t* strides, const cuuint32_t* box, const cuuint32_t* estr, CUtensorMapSwizzle swz);

namespace {

using namespace gx;

constexpr uint32_t kWaitPolls = 1u << 22;

struct GxArgs {
  int rows, k, n;
  const float* scales;
  const uint8_t* wp;
  const uint8_t* w2p;
  int64_t rb;
  int mt, nt;      // token tiles, weight tiles
  int band;        // token tiles walked together (see tile_of)
  int cpr;         // packed chunks (256 values) per k range
  int splits;      // CG = 1: CTAs per cluster
  int boxed;       // window form: the windows of a stage come in TMA boxes, one of a weight's rows of each phase
  int lp;          // log2 of the phases (see WeightMaps)
  Epilogue e;
};

// The packed weights' tensor maps: w, w2 of every phase. A row stride that is no multiple of 16 bytes is one after P = 2, 4
// or 8 rows: rows of one phase, r = P j + f, are a tensor of their own from the 16-byte boundary at or before row f.
struct WeightMaps {
  CUtensorMap w[8], w2[8];
};

LK_DEV void gx_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
LK_DEV void gx_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
LK_DEV uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
LK_DEV void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
LK_DEV uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
LK_DEV bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
// Arrive on a barrier of another CTA of the cluster. What the arrival vouches for is in this SM's own shared memory or
// TMEM -- staged weights, which the proxy fence before it has made visible to the tensor core that reads them here, a
// token tile that the TMA wrote here, an accumulator read to its end -- so nothing has to become visible to the other
// SM's threads. A release at cluster scope would drain the thread's global accesses too and took about 1000 clocks an
// arrival (517 -> 369 us on 2048 x 4096 x 24576 Q4_K without it).
LK_DEV void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
LK_DEV void st_peer(uint32_t cluster_addr, float x, float y, float z, float w) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "f"(x), "f"(y), "f"(z), "f"(w)
               : "memory");
}
// Bounded wait
LK_DEV bool wait_bar(uint64_t* bar, uint32_t phase) {
  for (uint32_t i = 0; i < kWaitPolls; ++i)
    if (mbar_try_wait(bar, phase)) return true;
  return false;
}
// A wait of a whole warp (wait_one: of a lane that works alone). One that gave up sets the status bit and `live` to
// false; the warp then leaves its loops, and every other warp follows at its own next wait, so the kernel ends.
LK_DEV void wait_one(uint64_t* bar, uint32_t phase, bool& live) {
  if (wait_bar(bar, phase)) return;
  live = false;
  atomicOr(&g_status, 1u);
}
LK_DEV void wait_for(uint64_t* bar, uint32_t phase, bool& live) {
  if (__all_sync(0xFFFFFFFFu, wait_bar(bar, phase))) return;
  live = false;
  atomicOr(&g_status, 1u);
}
// A place in a ring of N stages: the stage, and the parity of its use
template <int N>
struct Place {
  int s = 0;
  uint32_t turn = 0;
  LK_DEV void next(int by = 1) {
    s += by;
    while (s >= N) {   // once, but for rings shorter than a step
      s -= N;
      turn ^= 1;
    }
  }
  LK_DEV Place ahead(int by) const {
    Place q = *this;
    q.next(by);
    return q;
  }
};

template <int CG>
LK_DEV void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if (CG == 1) {
    umma_f16(d, ad, bd, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// arrives on `bar` (in both CTAs of a pair) when the MMAs issued so far are done
template <int CG>
LK_DEV void commit(uint64_t* bar) {
  if (CG == 1)
    umma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(uint16_t(3))
        : "memory");
}
template <int CG>
LK_DEV void talloc(uint32_t* slot, uint32_t cols) {
  if (CG == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
LK_DEV void tfree(uint32_t addr, uint32_t cols) {
  if (CG == 1)
    tmem_dealloc(addr, cols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
// 32 lanes x 16 consecutive columns
LK_DEV void tmem_ld(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// residual and store of V outputs of one lane: output n of tokens t, t + step, ... (the type switches outside the loops)
template <int V, typename T>
LK_DEV void add_as(const T* r, int64_t step, int count, float (&o)[V]) {
  T x[V];
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < count) x[i] = r[i * step];
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < count) o[i] += float(x[i]);
}
template <int V, typename T>
LK_DEV void store_as(T* y, int64_t step, int count, const float (&o)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < count) {
      if constexpr (sizeof(T) == 4) *y = o[i];
      else *y = T(o[i]);   // to nearest even
      y += step;
    }
}
template <int V>
LK_DEV void add_and_store(const Epilogue& e, float (&o)[V], int64_t at, int64_t step, int count) {
  if (e.res) {
    if (e.res_dtype == LK_BF16) add_as(static_cast<const __nv_bfloat16*>(e.res) + at, step, count, o);
    else if (e.res_dtype == LK_F16) add_as(static_cast<const __half*>(e.res) + at, step, count, o);
    else add_as(static_cast<const float*>(e.res) + at, step, count, o);
  }
  if (e.y_form == LK_BF16) store_as(static_cast<__nv_bfloat16*>(e.y) + at, step, count, o);
  else if (e.y_form == LK_F16) store_as(static_cast<__half*>(e.y) + at, step, count, o);
  else store_as(static_cast<float*>(e.y) + at, step, count, o);
}

// The epilogue of C tokens (columns) of one tile row. v: the lane's sums; sc: the tokens' scales (shared memory); t:
// the first token; row: the lane's row of the CTA's tile; n0: the tile's first output. All 32 lanes take part.
template <bool PAIR, int C>
LK_DEV void finish(const GxArgs& p, float (&v)[C], const float* sc, int t, int n0, int row) {
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] *= sc[i];   // the row scale: a power of two, exact
  const int left = p.rows - t;
  if (!PAIR) {
    const int n = n0 + row;
    if (n >= p.n) return;
    if (p.e.bias) {
      const float b = __ldg(p.e.bias + n);
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] += b;
    }
    if (p.e.act != LK_ACT_NONE) act_all(p.e.act, v);
    add_and_store(p.e, v, int64_t(t) * p.n + n, p.n, left);
  } else {
    // even lanes hold the gate, odd lanes the up product of output n; even lanes finish the even tokens
    const int n = n0 + (row >> 1), odd = row & 1;
    const float b = p.e.bias && n < p.n ? __ldg(p.e.bias + n) : 0.0f;
    const float b2 = p.e.bias2 && n < p.n ? __ldg(p.e.bias2 + n) : 0.0f;
    float g[C / 2], u[C / 2];
#pragma unroll
    for (int j = 0; j < C / 2; ++j) {
      const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2 * j] : v[2 * j + 1], 1);
      const float own = odd ? v[2 * j + 1] : v[2 * j];
      g[j] = (odd ? other : own) + b;
      u[j] = (odd ? own : other) + b2;
    }
    if (n >= p.n) return;
    if (p.e.act == LK_ACT_SWIGLU_OAI) {
#pragma unroll
      for (int j = 0; j < C / 2; ++j) g[j] = act_pair(LK_ACT_SWIGLU_OAI, g[j], u[j], p.e.alpha, p.e.limit);
    } else {
      act_all(p.e.act, g);
#pragma unroll
      for (int j = 0; j < C / 2; ++j) g[j] *= u[j];
    }
    add_and_store(p.e, g, int64_t(t + odd) * p.n + n, 2 * int64_t(p.n), (left - odd + 1) >> 1);
  }
}

// One thread's 32 values of a 64-value stage (page `sub` of a 144-byte chunk at a 16-byte aligned row, half h), the
// packed words in registers between load and store: dequant_group's rounding, value by value.
template <int FMT>
struct BoxItem {
  uint4 hd, a, b;   // Q4_K: header and the page's 32 bytes; else words 4h .. 4h + 4 of the page's 36 bytes in a, b.x
  LK_DEV void load(const uint8_t* chunk, int sub, int h) {
    if (FMT == LK_Q4_K) {
      const uint4* q = reinterpret_cast<const uint4*>(chunk + 16 + 32 * sub);
      hd = *reinterpret_cast<const uint4*>(chunk);
      a = q[0];
      b = q[1];
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(chunk + 36 * sub) + 4 * h;
      a = make_uint4(w[0], w[1], w[2], w[3]);
      b.x = w[4];
    }
  }
  LK_DEV void store(uint8_t* tile, int r, int h, int sub) const {
    if (FMT == LK_Q4_K) {
      const uint32_t sh = 4 * h, w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      uint32_t sc, m;
      q4k_scale_min_w(hd.y, hd.z, hd.w, 2 * sub + h, sc, m);
      const __half a16 = __hmul(__ushort_as_half(uint16_t(hd.x & 0xffffu)), small_int_half(sc));
      const __half c16 = __hneg(__hmul(__ushort_as_half(uint16_t(hd.x >> 16)), small_int_half(m)));
      const __half2 scale = __halves2half2(a16, a16), offset = __halves2half2(c16, c16);
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        uint32_t x[4];
        magic8((w[2 * cc] >> sh) & 0x0F0F0F0Fu, (w[2 * cc + 1] >> sh) & 0x0F0F0F0Fu, x);
        uint4 out;
        out.x = hfma2u(hsub2u(x[0], 0x64006400u), scale, offset);
        out.y = hfma2u(hsub2u(x[1], 0x64006400u), scale, offset);
        out.z = hfma2u(hsub2u(x[2], 0x64006400u), scale, offset);
        out.w = hfma2u(hsub2u(x[3], 0x64006400u), scale, offset);
        *reinterpret_cast<uint4*>(tile + sw128(r, 4 * h + cc)) = out;
      }
    } else {
      // blocks 2 sub (h = 0: d in the low half of its first word, codes from byte 2) and 2 sub + 1 (h = 1: d in the high
      // half of the word both blocks share, codes from the next word)
      const uint32_t w[5] = {a.x, a.y, a.z, a.w, b.x};
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = __funnelshift_rc(w[i], w[i + 1], h ? 32 : 16);
      const __half dh = __ushort_as_half(uint16_t(h ? w[0] >> 16 : w[0] & 0xffffu));
      const __half2 scale = __halves2half2(dh, dh);
      const uint32_t off = FMT == LK_Q4_0 ? 0x64086408u : 0x64806480u;   // f16 1024 + 8 | 1024 + 128
      uint32_t lk[8];   // IQ4_NL: word i's codebook bytes of values 4i, 16 + 4i, 4i + 1, 16 + 4i + 1 | 4i + 2, ...
      if (FMT == LK_IQ4_NL)
#pragma unroll
        for (int i = 0; i < 4; ++i) iq4_lookup8<0>(q[i], lk[2 * i], lk[2 * i + 1]);
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        uint32_t x[4];
        if (FMT == LK_IQ4_NL) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = prmt(lk[4 * (cc & 1) + i], 0x64646464u, cc >= 2 ? 0x4341u : 0x4240u);
        } else {
          const uint32_t t0 = ((cc >= 2) ? (q[2 * (cc & 1)] >> 4) : q[2 * (cc & 1)]) & 0x0F0F0F0Fu;
          const uint32_t t1 = ((cc >= 2) ? (q[2 * (cc & 1) + 1] >> 4) : q[2 * (cc & 1) + 1]) & 0x0F0F0F0Fu;
          magic8(t0, t1, x);
        }
        uint4 out;
        out.x = hmul2u(hsub2u(x[0], off), scale);
        out.y = hmul2u(hsub2u(x[1], off), scale);
        out.z = hmul2u(hsub2u(x[2], off), scale);
        out.w = hmul2u(hsub2u(x[3], off), scale);
        *reinterpret_cast<uint4*>(tile + sw128(r, 4 * h + cc)) = out;
      }
    }
  }
};
// one warp's part of a stage is staged: tells the MMA warp (of the pair's leader)
template <int CG>
LK_DEV void staged(uint64_t* bar) {
  if (CG == 2) arrive_at(peer_addr(bar, 0));
  else mbar_arrive(bar);
}
template <int FMT>
LK_DEV void dequant_group_win(const uint8_t* chunk, int j, uint8_t* tile, int r, int c0) {
  if (FMT == LK_Q4_0 || FMT == LK_IQ4_NL) dequant_group<FMT>(chunk, j, tile, r, c0);
  else dequant_group_any<FMT>(chunk, j, tile, r, c0);
}

template <int FMT, bool WIN, bool PAIR, int CG, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    k_gemmx(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ WeightMaps wm, const GxArgs p) {
  constexpr Rings kG = rings_of(FMT, WIN, CG, NT);
  constexpr int kB = kG.b_bytes, kRaw = kG.raw_bytes, kS = kG.s, kR = kG.r, kBatch = batch_of(kS);
  constexpr int kRW = row_slot_bytes(FMT, WIN);
  constexpr int kCB = WIN ? chunk_bytes(FMT) : kChunkBytes;
  constexpr int kBuf = 2;                                // accumulators
  constexpr int kOut = PAIR ? kRows / 2 : kRows;         // outputs of a CTA's tile
  constexpr int kEp0 = 4 + 8 * kDqG;   // first epilogue warp
  constexpr uint32_t kCols = kBuf * NT;
  constexpr int kC = 16;   // columns the epilogue holds in registers
  constexpr uint32_t kIdesc = idesc_f16(kRows * CG, NT, 0);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + kS * kABytes;
  uint8_t* sR = sB + kS * kB;
  uint8_t* tail = smem + body_bytes(FMT, WIN, CG, NT);
  float* stok = reinterpret_cast<float*>(tail);                      // [2][256] token scales
  // full (the leader's): a stage's token tiles have landed and its weights are staged, in both CTAs of a pair. x_in
  // (the other CTA's): its own token tile has landed, which its warp 1 passes on.
  uint64_t* full = reinterpret_cast<uint64_t*>(tail + 2 * 256 * 4);
  uint64_t* x_in = full + kS;
  uint64_t* empty = x_in + kS;        // the stage's MMAs are done
  uint64_t* full_r = empty + kS;
  uint64_t* empty_r = full_r + kR;
  uint64_t* acc_full = empty_r + kR;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  static_assert(2 * 256 * 4 + (3 * kS + 2 * kR + 4) * 8 + 4 <= kTailBytes, "the tail");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(cta_rank());
  const int csize = CG == 2 ? 2 : p.splits;
  const int cluster = int(blockIdx.x) / csize, nclusters = int(gridDim.x) / csize;
  const int half = CG == 2 ? rank : 0;   // which half of the pair's weight rows and tokens
  const int ntiles = p.mt * p.nt;
  const int my_tiles = ntiles > cluster ? (ntiles - 1 - cluster) / nclusters + 1 : 0;
  const int kst = p.k / kStageK;
  const int ks0 = CG == 2 ? 0 : rank * p.cpr * 4, ks1 = CG == 2 ? kst : min(kst, ks0 + p.cpr * 4);

  // tile t -> first token and first output of this CTA's half. Tiles go band by band of `band` token tiles, the token
  // tiles of a band fastest, so the tiles in flight reuse both the band's activations and few weight tiles from L2.
  auto tile_of = [&](int t, int& t0, int& n0) {
    const int per = p.band * p.nt, b = t / per, r = t - b * per;
    const int h = min(p.band, p.mt - b * p.band);
    t0 = (b * p.band + r % h) * NT;
    n0 = (r / h) * (kOut * CG) + half * kOut;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < kS; ++i) {
      mbar_init(&full[i], 8 * CG + CG);
      mbar_init(&x_in[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kR; ++i) {
      mbar_init(&full_r[i], 1);
      mbar_init(&empty_r[i], 8 * kDqG);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpW * CG);
    }
    fence_mbar_init();
  }
  if (warp == 1) talloc<CG>(tslot, kCols);
  tc_fence_before();
  if (CG == 2 || p.splits > 1) cluster_barrier();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  gx_launch();
  gx_wait();
  bool live = true;   // no wait of this warp has given up

  // window form: the packed bytes of tile row r's chunk at k stage ks
  auto win_src = [&](int r, int n0, int ks, uintptr_t& src, uint32_t& len, bool& in) {
    const int n = n0 + (PAIR ? r >> 1 : r);
    in = n < p.n;
    const int64_t c0 = int64_t(ks >> 2) * kCB;
    len = uint32_t(min(int64_t(kCB), p.rb - c0));
    src = reinterpret_cast<uintptr_t>(PAIR && (r & 1) ? p.w2p : p.wp) + uintptr_t(int64_t(in ? n : 0) * p.rb + c0);
  };

  const bool lead = CG == 1 || rank == 0;
  if (warp == 0) {
    // ------------------------------------------------------------------ token tiles (one lane)
    if (lane == 0) {
      prefetch_tensormap(&xmap);
      uint64_t* bars = lead ? full : x_in;
      Place<kS> at;
      bool first = true;   // the first use of every stage waits for nothing
      for (int li = 0; li < my_tiles && live; ++li) {
        int t0, n0;
        tile_of(cluster + li * nclusters, t0, n0);
        for (int ks = ks0; ks < ks1; ++ks) {
          if (!first) wait_one(&empty[at.s], at.turn ^ 1, live);
          if (!live) break;
          mbar_expect_tx(&bars[at.s], kB);
          tma_load_2d(sB + at.s * kB, &xmap, ks * kStageK, t0 + half * (NT / CG), &bars[at.s]);
          at.next();
          if (at.s == 0) first = false;
        }
      }
      if (!live)   // let the copies in flight land before the CTA ends
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ packed weights
    if (lane == 0 && (!WIN || p.boxed)) {
      prefetch_tensormap(&wm.w[0]);
      if (PAIR) prefetch_tensormap(&wm.w2[0]);
    }
    Place<kR> at;
    bool first = true;
    for (int li = 0; li < my_tiles && live; ++li) {
      int t0, n0;
      tile_of(cluster + li * nclusters, t0, n0);
      for (int ks = ks0; ks < ks1; ks += 4) {
        if (!first) wait_for(&empty_r[at.s], at.turn ^ 1, live);
        if (!live) break;
        uint8_t* dst = sR + at.s * kRaw;
        uint64_t* bar = &full_r[at.s];
        if (WIN && p.boxed) {
          // the windows of a phase start at the same byte of their rows: a box kRW wide from there
          if (lane == 0) {
            const int64_t c0 = int64_t(ks >> 2) * kCB;
            mbar_expect_tx(bar, kRaw);
            for (int f = 0; f < 1 << p.lp; ++f) {
              uint8_t* d = dst + f * (kOut >> p.lp) * kRW;
              const int64_t lead = (reinterpret_cast<uintptr_t>(p.wp) + uintptr_t(f * p.rb)) & 15;
              tma_load_2d(d, &wm.w[f], int((c0 + lead) & ~int64_t(15)) / 4, n0 >> p.lp, bar);
              if (PAIR) {
                const int64_t lead2 = (reinterpret_cast<uintptr_t>(p.w2p) + uintptr_t(f * p.rb)) & 15;
                tma_load_2d(d + kRaw / 2, &wm.w2[f], int((c0 + lead2) & ~int64_t(15)) / 4, n0 >> p.lp, bar);
              }
            }
          }
        } else if (WIN) {
          // each lane copies the 16-byte aligned window around its rows' chunk; the stage's bytes are announced first
          uint32_t total = 0;
#pragma unroll
          for (int i = 0; i < kRows / 32; ++i) {
            uintptr_t src;
            uint32_t len;
            bool in;
            win_src(lane + 32 * i, n0, ks, src, len, in);
            if (in) total += uint32_t(((src + len + 15) & ~uintptr_t(15)) - (src & ~uintptr_t(15)));
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
          if (lane == 0) mbar_expect_tx(bar, total);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kRows / 32; ++i) {
            uintptr_t src;
            uint32_t len;
            bool in;
            const int r = lane + 32 * i;
            win_src(r, n0, ks, src, len, in);
            const uintptr_t a0 = src & ~uintptr_t(15);
            if (in)
              bulk_g2s(dst + r * kRW, reinterpret_cast<const void*>(a0),
                       uint32_t(((src + len + 15) & ~uintptr_t(15)) - a0), bar);
          }
        } else if (lane == 0) {
          mbar_expect_tx(bar, kRaw);
          tma_load_2d(dst, &wm.w[0], (ks >> 2) * (kChunkBytes / 4), n0, bar);
          if (PAIR) tma_load_2d(dst + kRaw / 2, &wm.w2[0], (ks >> 2) * (kChunkBytes / 4), n0, bar);
        }
        __syncwarp();
        at.next();
        if (at.s == 0) first = false;
      }
    }
    if (!live)
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  } else if (warp == 1 && !lead) {
    // ------------------------------------------------------------------ tells the leader of this CTA's token tiles
    if (lane == 0) {
      Place<kS> at;
      for (int g = my_tiles * (ks1 - ks0); g > 0; --g) {
        wait_one(&x_in[at.s], at.turn, live);
        if (!live) break;
        arrive_at(peer_addr(&full[at.s], 0));
        at.next();
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue (the leader's)
    // The whole warp walks the loop and one elected lane issues: descriptors and barrier addresses then stay in uniform
    // registers (369 -> 308 us on 2048 x 4096 x 24576 Q4_K against a loop of lane 0 alone).
    const uint64_t ad0 = sdesc_k128(smem_u32(sA)), bd0 = sdesc_k128(smem_u32(sB));
    const bool issue = elect_one();
    Place<kS> at;
    for (int li = 0; li < my_tiles && live; ++li) {
      const int buf = li % kBuf;
      if (li >= kBuf) wait_for(&acc_empty[buf], ((li / kBuf) - 1) & 1, live);
      uint32_t more = 0;
#pragma unroll 1
      for (int ks = ks0; ks < ks1; ++ks) {
        wait_for(&full[at.s], at.turn, live);
        if (!live) break;
        tc_fence_after();
        if (issue) {
          const uint64_t ad = ad0 + uint32_t(at.s * (kABytes >> 4)), bd = bd0 + uint32_t(at.s * (kB >> 4));
          mma<CG>(tmem + buf * NT, ad, bd, kIdesc, more);
#pragma unroll
          for (int kk = 1; kk < kStageK / 16; ++kk) mma<CG>(tmem + buf * NT, ad + 2 * kk, bd + 2 * kk, kIdesc, 1);
          commit<CG>(&empty[at.s]);
          if (ks == ks1 - 1) commit<CG>(&acc_full[buf]);
        }
        more = 1;
        at.next();
      }
    }
  } else if (warp >= 4 && warp < kEp0) {
    // ------------------------------------------------------------------ weight staging
    const int group = (warp - 4) >> 3, dt = (threadIdx.x - 128) & 255;
    const int r = dt >> 1, h = dt & 1;   // tile row, which 32 of the stage's 64 values
    // where the row's packed chunk sits in a raw stage: boxes of a pair, gate rows then up rows; of a weight, phase by phase
    const bool split = PAIR && (!WIN || p.boxed);
    const int ro = split ? r >> 1 : r, lp = WIN && p.boxed ? p.lp : 0;
    const int slot = (split ? (r & 1) * (kRows / 2) : 0) + (ro & ((1 << lp) - 1)) * (kOut >> lp) + (ro >> lp);
    Place<kS> at;   // the chunk's first stage
    Place<kR> ar;
    int used = 0;   // stages before the chunk's: the first use of a stage waits for nothing
    for (int li = 0; li < my_tiles && live; ++li) {
      int t0, n0;
      tile_of(cluster + li * nclusters, t0, n0);
      for (int ks = ks0; ks < ks1 && live; ks += 4) {
        const int subs = min(4, ks1 - ks);
        const uint8_t* chunk = sR + ar.s * kRaw + slot * kRW;
        if (WIN) {
          uintptr_t src;
          uint32_t len;
          bool in;
          win_src(r, n0, ks, src, len, in);
          chunk += src & 15;
        }
        wait_for(&full_r[ar.s], ar.turn, live);
        // this group's stages of the chunk. Both sets of packed words are loaded before either is decoded (a wait that is
        // already satisfied still takes 100 to 250 clocks here, and one item's dependent chain about 500); or, where the
        // ring is too short for that, every other stage by itself
        const Turn turn = turn_of(kBatch, group, WIN ? subs : 4);
        if (kBatch == 2) {
          if (turn.count > 0) {
            const int sub = turn.first;
            const bool two = turn.count == 2;
            const Place<kS> st = at.ahead(sub), su = at.ahead(sub + 1);
            uint8_t* d0 = sA + st.s * kABytes;
            uint8_t* d1 = sA + su.s * kABytes;
            // the MMAs end in order: the later stage being free says that the earlier one is
            auto stages_free = [&] {
              if (two && used + sub + 1 >= kS) wait_for(&empty[su.s], su.turn ^ 1, live);
              else if (used + sub >= kS) wait_for(&empty[st.s], st.turn ^ 1, live);
              return live;
            };
            if (WIN) {
              if (!stages_free()) break;
              dequant_group_win<FMT>(chunk, 2 * sub + h, d0, r, 4 * h);
              if (two) dequant_group_win<FMT>(chunk, 2 * sub + 2 + h, d1, r, 4 * h);
            } else {   // whole chunks only: always two
              BoxItem<FMT> i0, i1;
              i0.load(chunk, sub, h);
              i1.load(chunk, sub + 1, h);
              if (!stages_free()) break;
              i0.store(d0, r, h, sub);
              i1.store(d1, r, h, sub + 1);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              staged<CG>(&full[st.s]);
              if (two) staged<CG>(&full[su.s]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (i >= turn.count) break;
            const int sub = turn.first + 2 * i;
            const Place<kS> st = at.ahead(sub);
            if (used + sub >= kS) wait_for(&empty[st.s], st.turn ^ 1, live);
            if (!live) break;
            uint8_t* dst = sA + st.s * kABytes;
            if (WIN) {
              dequant_group_win<FMT>(chunk, 2 * sub + h, dst, r, 4 * h);
            } else {
              BoxItem<FMT> item;
              item.load(chunk, sub, h);
              item.store(dst, r, h, sub);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) staged<CG>(&full[st.s]);
          }
        }
        if (lane == 0) mbar_arrive(&empty_r[ar.s]);
        ar.next();
        at.next(subs);
        used += subs;
      }
    }
  } else if (warp >= kEp0 && (CG == 2 || p.splits == 1)) {
    // ------------------------------------------------------------------ epilogue from TMEM
    const int q = warp & 3, row = 32 * q + lane;   // the lane quarter a warp may read
    int t0, n0;
    epilogue_tiles(
        my_tiles, live,
        [&](int li) {
          tile_of(cluster + li * nclusters, t0, n0);
          float* sc = stok + (li & 1) * 256;
          for (int i = threadIdx.x - 32 * kEp0; i < NT; i += 32 * kEpW)
            sc[i] = t0 + i < p.rows ? __ldg(p.scales + 2 * int64_t(t0 + i) + 1) : 0.0f;
        },
        [] { asm volatile("bar.sync 3, 128;" ::: "memory"); },   // the four epilogue warps
        [&](int li) { wait_for(&acc_full[li % kBuf], (li / kBuf) & 1, live); },
        [&](int li) {
          const int buf = li % kBuf;
          const float* sc = stok + (li & 1) * 256;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < NT && t0 + c < p.rows; c += kC) {
            float v[kC];
            tmem_ld(tmem + buf * NT + c + (uint32_t(32 * q) << 16), v);
            finish<PAIR, kC>(p, v, sc + c, t0 + c, n0, row);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) arrive_at(peer_addr(&acc_empty[buf], 0));
            else mbar_arrive(&acc_empty[buf]);
          }
        });
  }
  __syncwarp();

  if (CG == 1 && p.splits > 1) {
    // The partial tiles of the k ranges meet. Groups of 8 tokens are dealt to the CTAs in turn; every CTA stores its sums
    // of a group straight from TMEM into the shared memory of the group's owner (the rings: idle once all MMAs of the
    // cluster are done, hence the first barrier), which adds them in range order and finishes. Stores of 16 bytes that
    // nobody waits for: reading the peers' tiles took 7000 clocks of a 200 x 4096 x 4100 call, pushing them 1400 and
    // the wait for the stores about 3000.
    uint8_t* part = smem;   // [range][own group][half][128 rows][4 tokens] f32
    int t0, n0;
    tile_of(cluster, t0, n0);
    constexpr int kGroups = kThreads / 128;   // all warps take part: a quarter of the lanes each, as TMEM is read
    const int q = warp & 3, row = 32 * q + lane, own = (NT / 8 + p.splits - 1) / p.splits;
    wait_for(&acc_full[0], 0, live);
    tc_fence_after();
    for (int i = threadIdx.x; i < NT; i += kThreads)
      stok[i] = t0 + i < p.rows ? __ldg(p.scales + 2 * int64_t(t0 + i) + 1) : 0.0f;
    __syncwarp();
    cluster_barrier();
#pragma unroll 1
    for (int c = 16 * (warp >> 2); c < NT && t0 + c < p.rows; c += 16 * kGroups) {
      float v[16];
      tmem_ld(tmem + c + (uint32_t(32 * q) << 16), v);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int g = (c >> 3) + h;
        const uint32_t a = peer_addr(part, uint32_t(g % p.splits)) + (int(rank) * own + g / p.splits) * 4096 + row * 16;
        st_peer(a, v[8 * h], v[8 * h + 1], v[8 * h + 2], v[8 * h + 3]);
        st_peer(a + 2048, v[8 * h + 4], v[8 * h + 5], v[8 * h + 6], v[8 * h + 7]);
      }
    }
    __syncwarp();
    cluster_barrier();   // the last word between the CTAs
#pragma unroll 1
    for (int l = warp >> 2; l < own; l += kGroups) {
      const int c = 8 * (int(rank) + p.splits * l);
      if (c >= NT || t0 + c >= p.rows) break;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      for (int s = 0; s < p.splits; ++s) {
        const float4* f = reinterpret_cast<const float4*>(part + (s * own + l) * 4096) + row;
        const float4 x = f[0], y = f[128];
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      }
      finish<PAIR, 8>(p, v, stok + c, t0 + c, n0, row);
    }
    __syncwarp();
  }
  // nobody of a pair leaves while the other may still signal its barriers
  tc_fence_before();
  if (CG == 2) cluster_barrier();
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tfree<CG>(tmem, kCols);
}

template <int FMT, bool WIN, bool PAIR, int CG, int NT>
int launch_t(const CUtensorMap& xm, const WeightMaps& m, const GxArgs& a, int grid, cudaStream_t s) {
  constexpr int smem = 1024 + body_bytes(FMT, WIN, CG, NT) + kTailBytes;
  static_assert(smem <= kSmemMax, "the CTA exceeds shared memory");
  static_assert(rings_of(FMT, WIN, CG, NT).s >= 3 && rings_of(FMT, WIN, CG, NT).r >= 2, "the rings");
  auto kern = k_gemmx<FMT, WIN, PAIR, CG, NT>;
  static std::atomic<unsigned> allowed{0};
  if (!allow_smem(kern, smem, allowed)) return LK_ECUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG == 2 ? 2 : a.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, xm, m, a) == cudaSuccess ? LK_OK : LK_ECUDA;
}

struct Plan {
  int cg, nt, splits, grid;
};

template <int FMT, bool WIN>
int launch_f(const Plan& pl, bool pair, const CUtensorMap& xm, const WeightMaps& m, const GxArgs& a, cudaStream_t s) {
#define LK_GX(CG, NT)                                             \
  if (pl.cg == CG && pl.nt == NT)                                 \
    return pair ? launch_t<FMT, WIN, true, CG, NT>(xm, m, a, pl.grid, s) : launch_t<FMT, WIN, false, CG, NT>(xm, m, a, pl.grid, s);
  LK_GX(2, 256)
  LK_GX(1, 256)
  LK_GX(1, 128)
  LK_GX(1, 64)
  LK_GX(1, 32)
#undef LK_GX
  return LK_EUNSUPPORTED;
}

// The form of a call, by the time each is expected to take in units of 10 ns (fitted to Q4_K calls of 32 to 4096 rows,
// k 4096 and 12288, 1024 to 24576 outputs; the chosen form was within 6 % of the best of the forms tried):
//   CG = 2                rounds of whole-k tiles on sms / 2 pairs, 0.43 us a stage
//   CG = 1, the smallest token tile that holds all rows (256 at most)
//     one CTA a tile      rounds on all SMs, 0.27 to 0.51 us a stage by the token tile
//     k split S ways      one tile a cluster, 8 us to start and fill, 2 to meet. Clusters of up to 2 fill the chip; of 4,
//                         9 tenths of it, of 8, 8 tenths (a cluster lies within one GPC).
Plan choose(int rows, int n, int kchunks, bool pair, int sms) {
  const int outs = pair ? kRows / 2 : kRows, stages = 4 * kchunks;
  const int64_t tiles2 = int64_t((rows + 255) / 256) * ((n + 2 * outs - 1) / (2 * outs));
  const int pairs = sms / 2;
  Plan best{2, 256, 1, 2 * int(tiles2 < pairs ? tiles2 : pairs)};
  int64_t cost = (tiles2 + pairs - 1) / pairs * stages * 43 + 1000;
  const int nt = rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  const int stage = nt == 32 ? 27 : nt == 64 ? 30 : nt == 128 ? 35 : 51;
  const int64_t tiles1 = int64_t((rows + nt - 1) / nt) * ((n + outs - 1) / outs);
  for (int sp = 1; sp <= 8 && sp <= kchunks; ++sp) {
    const int per = (kchunks + sp - 1) / sp;
    if ((kchunks + per - 1) / per != sp) continue;   // no empty range
    const int64_t slots = sp <= 2 ? sms / sp : sp <= 4 ? sms * 9 / (10 * sp) : sms * 8 / (10 * sp);
    const int64_t rounds = (tiles1 + slots - 1) / slots;
    const int64_t c = sp == 1 ? rounds * stages * stage + 800 : rounds * (4 * per * stage + 1000);
    if (c < cost && tiles1 * sp < (int64_t(1) << 31)) {
      cost = c;
      best = Plan{1, nt, sp, int(sp == 1 ? (tiles1 < sms ? tiles1 : sms) : tiles1 * sp)};
    }
  }
  return best;
}

}  // namespace

int gemm_ex(int fmt, int rows, int k, int n, const uint16_t* x16, const float* scales, const void* w, const void* w2,
            const Epilogue& e, cudaStream_t s) {
  const bool pair = w2 != nullptr;
  const int outs = pair ? kRows / 2 : kRows, kchunks = (k + 255) / 256;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const Plan pl = choose(rows, n, kchunks, pair, sms);
  GxArgs a{};
  a.rows = rows;
  a.k = k;
  a.n = n;
  a.scales = scales;
  a.wp = static_cast<const uint8_t*>(w);
  a.w2p = static_cast<const uint8_t*>(w2);
  a.rb = lk_row_bytes(fmt, k);
  a.mt = (rows + pl.nt - 1) / pl.nt;
  a.nt = (n + outs * pl.cg - 1) / (outs * pl.cg);
  a.band = a.mt < 8 ? a.mt : 8;
  a.splits = pl.splits;
  a.cpr = (kchunks + pl.splits - 1) / pl.splits;
  a.e = e;
  // Rows come by TMA boxes: the Q4 family's 144-byte chunks as they are, of other chunks the window around them, a box for
  // each phase of the row stride. A copy takes the SM about 85 clocks whatever its size: 4 boxes instead of 128 row copies
  // took 430 x 2688 x 20615 Q8_0 from 170 to 75 us, 3201 x 10880 x 947 IQ4_NL from 231 to 103. Row by row: fewer rows than
  // phases, and strides of 16 bytes from a start that is not a multiple of 16.
  const bool al16 = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && (reinterpret_cast<uintptr_t>(w2) & 15) == 0;
  const bool win = !((fmt == LK_Q4_0 || fmt == LK_Q4_K || fmt == LK_IQ4_NL) && k % 256 == 0 && al16);
  a.lp = a.rb % 16 == 0 ? 0 : a.rb % 8 == 0 ? 1 : a.rb % 4 == 0 ? 2 : 3;
  const int phases = 1 << a.lp;
  // (of one phase an aligned start, so that no row reaches into the next one's stride; n rows at least one of each)
  const bool boxes = a.rb % 2 == 0 && n >= phases && (a.lp > 0 || al16);
  a.boxed = win && boxes;
  CUtensorMap xm;
  int rc = make_map(&xm, x16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, rows, k, kStageK, pl.nt / pl.cg,
                    CU_TENSOR_MAP_SWIZZLE_128B);
  WeightMaps m;
  for (int f = 0; f < 8; ++f) m.w[f] = m.w2[f] = xm;   // row by row: none is read
  if (boxes)
    for (int f = 0; f < phases && rc == LK_OK; ++f) {
      const cuuint32_t box[2] = {cuuint32_t(row_slot_bytes(fmt, win) / 4), cuuint32_t(outs / phases)}, estr[2] = {1, 1};
      const cuuint64_t strides[1] = {cuuint64_t(a.rb) * phases};
      for (int q = 0; q < (pair ? 2 : 1) && rc == LK_OK; ++q) {
        const uintptr_t row = reinterpret_cast<uintptr_t>(q ? w2 : w) + uintptr_t(a.rb) * f;
        const cuuint64_t dims[2] = {cuuint64_t(((row & 15) + a.rb + 3) / 4), cuuint64_t((n - f + phases - 1) / phases)};
        rc = encode_tiled(q ? &m.w2[f] : &m.w[f], CU_TENSOR_MAP_DATA_TYPE_UINT32, 2,
                          reinterpret_cast<const void*>(row & ~uintptr_t(15)), dims, strides, box, estr,
                          CU_TENSOR_MAP_SWIZZLE_NONE);
      }
    }
  if (rc != LK_OK) return rc;
  if (!win) {
    switch (fmt) {
      case LK_Q4_0: return launch_f<LK_Q4_0, false>(pl, pair, xm, m, a, s);
      case LK_Q4_K: return launch_f<LK_Q4_K, false>(pl, pair, xm, m, a, s);
      case LK_IQ4_NL: return launch_f<LK_IQ4_NL, false>(pl, pair, xm, m, a, s);
    }
    return LK_EUNSUPPORTED;
  }
  switch (fmt) {
    case LK_Q4_0: return launch_f<LK_Q4_0, true>(pl, pair, xm, m, a, s);
    case LK_Q4_K: return launch_f<LK_Q4_K, true>(pl, pair, xm, m, a, s);
    case LK_IQ4_NL: return launch_f<LK_IQ4_NL, true>(pl, pair, xm, m, a, s);
    case LK_Q5_0: return launch_f<LK_Q5_0, true>(pl, pair, xm, m, a, s);
    case LK_Q8_0: return launch_f<LK_Q8_0, true>(pl, pair, xm, m, a, s);
    case LK_Q5_K: return launch_f<LK_Q5_K, true>(pl, pair, xm, m, a, s);
    case LK_Q6_K: return launch_f<LK_Q6_K, true>(pl, pair, xm, m, a, s);
    case LK_IQ4_XS: return launch_f<LK_IQ4_XS, true>(pl, pair, xm, m, a, s);
    case LK_Q3_K: return launch_f<LK_Q3_K, true>(pl, pair, xm, m, a, s);
    case LK_IQ3_S: return launch_f<LK_IQ3_S, true>(pl, pair, xm, m, a, s);
    case LK_MXFP4: return launch_f<LK_MXFP4, true>(pl, pair, xm, m, a, s);
  }
  return LK_EUNSUPPORTED;
}

LK_STATUS_READER(status_gemmx)

}  // namespace lk
