// The shared-memory rings of the epilogue products: their lengths, and which stages each reader of a ring takes, as functions
// that the kernels and a walk of the rings on the host both call.
//
// mbarrier.try_wait.parity tells a phase from its two neighbours only: a wait for use m of a slot returns at once while use
// m - 1 is still open. So a reader that lets a use of a slot go by must know in another way that it is over before it waits
// for the next one.
#pragma once
#include "lk_formats.cuh"
#include "lk_stage.cuh"

namespace lk {

// ---------------------------------------------------------------------------------------------------------------
// lk_mvx.cu: 16 consumer warps in two groups of 8 (a warp for each k slice of a stage)
// ---------------------------------------------------------------------------------------------------------------
namespace mvx {

constexpr int kRows = 32;              // weight rows of a warp
constexpr int kSlices = 8;             // k slices of a stage, a warp of each group for each
constexpr int kCWarps = 2 * kSlices;   // consumer warps
constexpr int kTokStride = 36;         // floats between tokens of the partial sums: conflict-free stores
constexpr int kSmemMax = 227 * 1024;
constexpr int kMaxStages = 8;

// How a call's operands reach shared memory, and its tokens: kBox1 is the box form of one token, whose codes need no
// swizzle (all rows read the same words) and come by plain bulk copies.
enum { kRowForm = 0, kBox = 1, kBox1 = 2 };
// packed bytes of a row's stage; 128-byte segments that can hold them wherever they start
__host__ __device__ constexpr int stage_bytes(int fmt, int v) { return v / fmt_qk(fmt) * fmt_block_bytes(fmt); }
__host__ __device__ constexpr int segments(int fmt, int v) {
  return stage_bytes(fmt, v) % 128 == 0 ? stage_bytes(fmt, v) / 128 : (stage_bytes(fmt, v) + 126) / 128 + 1;
}
// row form slots: 16 bytes past a multiple of 128, so that 8 rows x 4 words fall into 32 banks; with room for a window's
// 15 leading bytes and a realigning load's trailing word
__host__ __device__ constexpr int slot_of(int bytes) { return (bytes + 32 + 111) / 128 * 128 + 16; }
// weight bytes of a stage in shared memory, and a stage's activations (box forms: multiples of 1024, which the swizzle's
// pattern is aligned to)
__host__ __device__ constexpr int w_bytes(int fmt, int form, int rg, int v) {
  return rg * kRows * (form == kRowForm ? slot_of(stage_bytes(fmt, v)) : segments(fmt, v) * 128);
}
__host__ __device__ constexpr int x_bytes(int form, int nt, int v) {
  return form == kRowForm ? 8 * nt * (slot_of(v) + slot_of(v / 4)) : form == kBox1 ? (v + v / 4 + 1023) / 1024 * 1024 : 8 * nt * (v + v / 4);
}
// partial sums of all 16 warps; for 32 tokens of half of them, to which the other half adds
__host__ __device__ constexpr int red_slices(int nt) { return nt <= 2 ? kCWarps : kCWarps / 2; }
__host__ __device__ constexpr int red_bytes(int nt) { return red_slices(nt) * 8 * nt * kTokStride * 4; }
constexpr int kTailBytes = 256 + 16 * 32 * 4;   // barriers; the first tile of a unit of two (q8 output of a pair)
__host__ __device__ constexpr int fixed_bytes(int nt) { return 1024 + red_bytes(nt) + kTailBytes; }
__host__ __device__ constexpr bool two_stages(int fmt, int form, int rg, int nt, int v) {
  return 2 * (w_bytes(fmt, form, rg, v) + x_bytes(form, nt, v)) + fixed_bytes(nt) <= kSmemMax;
}
// values of a stage: 2048 for up to 8 tokens where two such stages fit (a stage's waits and addresses cost a warp as much as
// a third of its 128 values' work: 16.9 -> 16.1 us on the Q4_K pair of 4096 -> 12288 at 8 tokens), else 1024. The same in
// both forms of one row group, so that those sum in the same order.
__host__ __device__ constexpr int stage_values(int fmt, int form, int rg, int nt) {
  return nt == 1 && (rg == 1 || two_stages(fmt, form, rg, nt, 2048)) ? 2048 : 1024;
}
// whether two stages of 64-row tiles fit beside the sums
__host__ __device__ constexpr bool two_groups(int fmt, int form, int nt) {
  return form != kRowForm && two_stages(fmt, form, 2, nt, stage_values(fmt, form, 2, nt));
}

// A call's ring: stages of k, ring slots, and whether the activations of all of k stay in shared memory, which they do where
// they leave three stages of weights (two for the widest rows of 8 tokens and fewer).
struct Ring {
  int nst, stages, slot, resident;
};
__host__ __device__ constexpr Ring ring_of(int fmt, int form, int rg, int nt, int k) {
  const int v = stage_values(fmt, form, rg, nt), wb = w_bytes(fmt, form, rg, v), xb = x_bytes(form, nt, v);
  Ring r{(k + v - 1) / v, 0, 0, 0};
  r.resident = form != kRowForm && int64_t(r.nst) * xb + (nt == 1 ? 2 : 3) * wb + fixed_bytes(nt) <= kSmemMax;
  r.slot = wb + (r.resident ? 0 : xb);
  r.stages = (kSmemMax - fixed_bytes(nt) - (r.resident ? r.nst * xb : 0)) / r.slot;
  if (r.stages > kMaxStages) r.stages = kMaxStages;
  return r;
}

// Whether group `group` multiplies stage `st` of a CTA's tile number `round`. Two row groups: each takes its rows of every
// stage. One: the groups take the stages in turn; starting a tile with the other group swaps two summands.
__host__ __device__ constexpr bool takes(int rg, int group, int st, int round) {
  return rg == 2 || ((st + round) & 1) == group;
}
// Whether a group also waits for the stages it does not multiply, and releases them. In a ring of an even number of slots a
// slot stays with one group for the whole of a tile, and at the tile's end the sums' barrier says that every stage has been
// read, so a group never lets a use of its own slots go by. In an odd ring the slots change hands from one use to the next:
// both groups then follow every stage, and a slot is free when both have.
__host__ __device__ constexpr bool follows(int rg, int stages) { return rg == 1 && stages % 2 == 1; }
// warps that release a stage
__host__ __device__ constexpr int releases(int rg, int stages) { return rg == 2 || follows(rg, stages) ? kCWarps : kSlices; }

}  // namespace mvx

// ---------------------------------------------------------------------------------------------------------------
// lk_gemmx.cu: a ring of stages of 64 k (a staged weight tile and a token tile) and one of packed chunks of 256
// ---------------------------------------------------------------------------------------------------------------
namespace gx {

constexpr int kRows = 128;       // weight rows of a CTA's tile (the M side)
constexpr int kStageK = 64;      // k values per MMA stage: one 128-byte swizzled row
constexpr int kEpW = 4;          // epilogue warps
constexpr int kABytes = kRows * kStageK * 2;
constexpr int kSmemMax = 227 * 1024;

// Staging warps: groups of 8 that take the stages in turn.
constexpr int kDqG = 2;
constexpr int kThreads = 32 * (4 + 8 * kDqG + kEpW);

// Two rings: stages (a staged weight tile and a token tile, one barrier for both, so the MMA warp waits once a stage) and
// packed chunks. Few tokens: the weights stream from HBM once, and the packed ring gets what keeps that many bytes in
// flight (110 KB a SM for the 4-bit formats); many: both operands come from L2 and the stages get it.
constexpr int kTailBytes = 2 * 256 * 4 + 512;   // token scales of two tiles, barriers, the TMEM address
struct Rings {
  int s, r, b_bytes, raw_bytes;
  __host__ __device__ constexpr int bytes() const { return s * (kABytes + b_bytes) + r * raw_bytes; }
};
__host__ __device__ constexpr int at_most(int a, int b) { return a < b ? a : b; }
__host__ __device__ constexpr Rings rings_of(int fmt, bool win, int cg, int nt) {
  Rings g{0, 0, nt / cg * kStageK * 2, kRows * row_slot_bytes(fmt, win)};
  const int room = kSmemMax - 1024 - kTailBytes;
  if (cg == 2) {
    g.r = at_most(3, (room - 3 * (kABytes + g.b_bytes)) / g.raw_bytes);
    g.s = at_most(6, (room - g.r * g.raw_bytes) / (kABytes + g.b_bytes));
  } else {
    g.r = at_most(nt <= 64 ? 5 : 3, (room - 3 * (kABytes + g.b_bytes)) / g.raw_bytes);
    g.s = at_most(6, (room - g.r * g.raw_bytes) / (kABytes + g.b_bytes));
  }
  return g;
}
// the partial sums of a split reuse the rings: splits x ceil(nt / 8 / splits) groups of 8 tokens, at most 7 more than nt / 8
__host__ __device__ constexpr int body_bytes(int fmt, bool win, int cg, int nt) {
  const int ring = rings_of(fmt, win, cg, nt).bytes(), part = cg == 1 ? (nt + 56) * kRows * 4 : 0;
  return ring > part ? ring : part;
}

// The stages of a chunk of `subs` (4, fewer in a row's last chunk) that a staging group takes: `count` from `first`, next to
// each other with a batch of 2 (every other one with a batch of 1). A group waits for the slot of its last stage (batch 2;
// of each stage, batch 1), which says that the MMAs up to the slot's last use are done; for its next wait to find the
// barrier no more than one phase behind, its waits must be at most the ring's length apart. With a batch of 2 they
// are up to 5 stages apart (group 1 around a last chunk of 1), because a last chunk of 2 is shared: taken whole by group 0
// it would leave group 1 6 stages without a wait. With a batch of 1, up to 3.
__host__ __device__ constexpr int batch_of(int stages) { return stages >= 5 ? 2 : 1; }
struct Turn {
  int first, count;
};
__host__ __device__ constexpr Turn turn_of(int batch, int group, int subs) {
  if (batch == 2 && subs > 2) return Turn{2 * group, at_most(2, subs - 2 * group)};
  if (batch == 2) return Turn{group, group < subs ? 1 : 0};
  return Turn{group, (subs - group + 1) / 2};
}

// An epilogue warp's tiles: the four warps share the token scales that fill() loads, so each comes to sync() once a tile,
// also after its own wait() has given up (live is false then) while another warp's passed.
#pragma nv_exec_check_disable
template <class Fill, class Sync, class Wait, class Work>
__host__ __device__ __forceinline__ void epilogue_tiles(int tiles, const bool& live, const Fill& fill, const Sync& sync,
                                                        const Wait& wait, const Work& work) {
  for (int li = 0; li < tiles; ++li) {
    fill(li);
    sync();
    if (live) wait(li);
    if (live) work(li);
  }
}

}  // namespace gx

}  // namespace lk
