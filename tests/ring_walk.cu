// Walks the shared-memory rings of the epilogue products on the host: the warps of a CTA as actors that a random scheduler
// advances one step at a time, copies that land in any order, and barriers that answer a parity wait as the hardware does.
// Ring lengths and who takes which stage come from the kernels' own functions (lk_rings.cuh). Reported: a wait that passes
// for another use of its slot than the waiter's, a slot refilled while it is read, and a state nobody can leave.
//
// Planted mistakes, for the test of the walk:
//   ring_walk mvx [alone]     alone: the groups never follow each other's stages
//   ring_walk gemmx [whole]   whole: a last chunk of two stages is group 0's alone
//   ring_walk epilogue        waits that give up in some of the epilogue warps
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "lk_rings.cuh"

namespace {

struct Bar {
  int count = 0, pending = 0, done = 0;   // done: phases completed
  void init(int n) { count = pending = n; }
  void arrive() {
    if (--pending == 0) {
      ++done;
      pending = count;
    }
  }
  bool passes(int parity) const { return (done & 1) != parity; }   // mbarrier.try_wait.parity
};

struct Fault {
  const char* what = nullptr;
  void set(const char* w) {
    if (!what) what = w;
  }
};

using Rng = std::mt19937;
int below(Rng& r, int n) { return int(r() % unsigned(n)); }
// some actors run much more slowly than others in each walk
struct Speeds {
  std::vector<int> w;
  int total = 0;
  Speeds(Rng& r, int actors) {
    for (int i = 0; i < actors; ++i) {
      w.push_back(below(r, 3) ? 64 : below(r, 2) ? 8 : 1);
      total += w.back();
    }
  }
  int pick(Rng& r) const {
    int x = below(r, total), i = 0;
    while (x >= w[i]) x -= w[i++];
    return i;
  }
};

// ------------------------------------------------------------------------------------------------------------ lk_mvx.cu
const char* walk_mvx(int rg, int kS, int nst, int tiles, bool alone, unsigned seed) {
  using namespace lk::mvx;
  Rng rng(seed);
  Fault f;
  const bool follow = !alone && follows(rg, kS);
  std::vector<Bar> full(kS), empty(kS);
  std::vector<int> reading(kS, 0);
  for (int i = 0; i < kS; ++i) {
    full[i].init(1);   // the landing of a stage's copies
    empty[i].init(alone ? kSlices * rg : releases(rg, kS));
  }
  std::vector<int> flight;   // stages whose copies are under way
  int issued = 0;
  const int total = nst * tiles;
  struct Warp {
    int tile = 0, st = 0, s = 0, turn = 0, step = 0;   // step 1: multiplying; 2: at the tile's sums
    bool over = false;
  };
  std::vector<Warp> w(kCWarps);
  int at_sums = 0, sums = 0;
  const Speeds speed(rng, kCWarps + 2);
  long idle = 0;
  for (;;) {
    bool all = issued == total && flight.empty();
    for (auto& x : w) all = all && x.over;
    if (all || f.what) return f.what;
    if (++idle > 2000000) return "nobody can go on";
    const int a = speed.pick(rng);
    if (a == kCWarps) {   // producer
      if (issued == total) continue;
      const int s = issued % kS, use = issued / kS;
      if (use > 0) {
        if (!empty[s].passes((use & 1) ^ 1)) continue;
        if (empty[s].done != use) f.set("the producer passed for another use");
      }
      if (reading[s]) f.set("a slot was refilled while it was read");
      flight.push_back(issued++);
      idle = 0;
    } else if (a == kCWarps + 1) {   // a copy lands
      if (flight.empty()) continue;
      const int i = below(rng, int(flight.size()));
      full[flight[i] % kS].arrive();
      flight.erase(flight.begin() + i);
      idle = 0;
    } else {
      Warp& x = w[a];
      if (x.over) continue;
      const int group = a / kSlices;
      auto next = [&] {
        ++x.st;
        if (++x.s == kS) x.s = 0, x.turn ^= 1;
      };
      if (x.step == 2) {   // the barriers of the sums
        if (sums <= x.tile) continue;
        ++x.tile;
        x.st = x.step = 0;
        x.over = x.tile == tiles;
      } else if (x.step == 1) {
        --reading[x.s];
        empty[x.s].arrive();
        next();
        x.step = 0;
      } else if (x.st == nst) {
        x.step = 2;
        if (++at_sums == kCWarps) at_sums = 0, ++sums;
      } else {
        const bool mine = takes(rg, group, x.st, x.tile);
        if (!mine && !follow) {
          next();
        } else {
          if (!full[x.s].passes(x.turn)) continue;
          if (full[x.s].done != (x.tile * nst + x.st) / kS + 1) f.set("a consumer passed for another use");
          if (mine) {
            ++reading[x.s];
            x.step = 1;
          } else {
            empty[x.s].arrive();
            next();
          }
        }
      }
      idle = 0;
    }
  }
}

// every ring the size rules can give, of rows up to 40960 values (longer rows only repeat a ring that is not resident)
int run_mvx(bool alone) {
  using namespace lk::mvx;
  const int fmts[] = {LK_Q4_0, LK_Q4_K, LK_Q8_0, LK_Q5_0, LK_Q5_K, LK_Q6_K, LK_IQ4_NL, LK_IQ4_XS};
  std::set<std::tuple<int, int, int>> rings;
  for (int fmt : fmts)
    for (int form : {kRowForm, kBox, kBox1})
      for (int nt : {1, 2, 4})
        for (int rg : {1, 2}) {
          if ((form == kBox1 && nt > 1) || (rg == 2 && !two_groups(fmt, form, nt))) continue;
          const int unit = lk::fmt_qk(fmt);
          for (int k = unit; k <= 40960; k += unit) {
            const Ring r = ring_of(fmt, form, rg, nt, k);
            if (r.stages < 2) return printf("a ring of %d slots\n", r.stages), 1;
            rings.insert(std::make_tuple(rg, r.stages, r.nst));
          }
        }
  int faults = 0, odd = 0;
  for (auto& t : rings) {
    const int rg = std::get<0>(t), kS = std::get<1>(t), nst = std::get<2>(t);
    odd += rg == 1 && kS % 2 == 1 && nst > kS;
    for (int tiles = 1; tiles <= 3; ++tiles)
      for (unsigned seed = 0; seed < 8; ++seed)
        if (const char* what = walk_mvx(rg, kS, nst, tiles, alone, seed * 7919 + nst * 31 + kS)) {
          if (!faults) printf("groups %d, slots %d, stages %d, tiles %d: %s\n", rg, kS, nst, tiles, what);
          ++faults;
        }
  }
  printf("mvx: %d rings, %d of them odd and shared, %d faults\n", int(rings.size()), odd, faults);
  return faults != 0;
}

// ---------------------------------------------------------------------------------------------------------- lk_gemmx.cu
const char* walk_gemmx(int cg, int kS, int kR, int kst, int tiles, bool whole, unsigned seed) {
  using namespace lk::gx;
  const int batch = batch_of(kS), total = kst * tiles, per_tile = (kst + 3) / 4, chunks = per_tile * tiles;
  Rng rng(seed);
  Fault f;
  // a wait for the `use`-th completed phase of a barrier (parity of use - 1)
  auto pass = [&](const Bar& b, int use, const char* who) {
    if (!b.passes((use & 1) ^ 1)) return false;
    if (b.done != use) f.set(who);
    return true;
  };
  struct Cta {
    std::vector<Bar> x_in, empty, full_r, empty_r, acc_full;
    std::vector<int> tok, raw;   // copies under way
    int tok_at = 0, raw_at = 0, tell_at = 0;
  };
  std::vector<Cta> cta(cg);
  std::vector<Bar> full(kS), acc_empty(2);
  for (auto& b : full) b.init(8 * cg + cg);
  for (auto& b : acc_empty) b.init(kEpW * cg);
  for (auto& c : cta) {
    auto make = [](std::vector<Bar>& v, int n, int count) {
      v.resize(n);
      for (auto& b : v) b.init(count);
    };
    make(c.x_in, kS, 1);
    make(c.empty, kS, 1);
    make(c.full_r, kR, 1);
    make(c.empty_r, kR, 8 * kDqG);
    make(c.acc_full, 2, 1);
  }
  std::vector<int> queue;   // MMAs under way
  int mma_at = 0, mma_done = 0, finished = 0;
  bool mma_open = false;    // the tile's accumulator is free
  std::vector<std::function<bool()>> actors;   // one step: whether it could
  for (int ci = 0; ci < cg; ++ci) {
    Cta* c = &cta[ci];
    const bool lead = ci == 0;
    actors.push_back([&, c] {   // token tiles
      const int i = c->tok_at, s = i % kS;
      if (i == total || (i >= kS && !pass(c->empty[s], i / kS, "the token tiles passed for another use"))) return false;
      if (i >= kS && mma_done <= i - kS) f.set("a token tile was overwritten before its MMA");
      c->tok.push_back(c->tok_at++);
      return true;
    });
    actors.push_back([&, c, lead] {
      if (c->tok.empty()) return false;
      const int j = below(rng, int(c->tok.size())), s = c->tok[j] % kS;
      (lead ? full : c->x_in)[s].arrive();
      c->tok.erase(c->tok.begin() + j);
      return true;
    });
    if (!lead)
      actors.push_back([&, c] {   // tells the leader
        const int i = c->tell_at;
        if (i == total || !pass(c->x_in[i % kS], i / kS + 1, "x_in passed for another use")) return false;
        full[i % kS].arrive();
        ++c->tell_at;
        return true;
      });
    actors.push_back([&, c] {   // packed chunks
      const int j = c->raw_at;
      if (j == chunks || (j >= kR && !pass(c->empty_r[j % kR], j / kR, "the packed ring passed for another use"))) return false;
      c->raw.push_back(c->raw_at++);
      return true;
    });
    actors.push_back([&, c] {
      if (c->raw.empty()) return false;
      const int j = below(rng, int(c->raw.size()));
      c->full_r[c->raw[j] % kR].arrive();
      c->raw.erase(c->raw.begin() + j);
      return true;
    });
    for (int w = 0; w < 8 * kDqG; ++w) {   // staging warps
      struct State {
        int chunk = 0, i = 0;
        bool open = false;
      };
      auto st = std::make_shared<State>();
      actors.push_back([&, c, st, w] {
        if (st->chunk == chunks) return false;
        const int group = w / 8, tile = st->chunk / per_tile, part = st->chunk % per_tile;
        const int base = tile * kst + 4 * part, subs = at_most(4, kst - 4 * part);
        Turn t = turn_of(batch, group, subs);
        if (whole && batch == 2 && subs == 2) t = Turn{0, group == 0 ? 2 : 0};
        if (!st->open) {
          if (!pass(c->full_r[st->chunk % kR], st->chunk / kR + 1, "full_r passed for another use")) return false;
          st->open = true;
          return true;
        }
        if (st->i < t.count) {
          const int n = batch == 2 ? t.count : 1, first = base + t.first + (batch == 2 ? 0 : 2 * st->i), last = first + n - 1;
          if (last >= kS && !pass(c->empty[last % kS], last / kS, "a staging group passed for another use")) return false;
          for (int i = first; i <= last; ++i) {
            if (i >= kS && mma_done <= i - kS) f.set("a weight tile was overwritten before its MMA");
            full[i % kS].arrive();
          }
          st->i += n;
          return true;
        }
        c->empty_r[st->chunk % kR].arrive();
        ++st->chunk;
        st->i = 0;
        st->open = false;
        return true;
      });
    }
    for (int w = 0; w < kEpW; ++w) {   // epilogue warps
      auto tile = std::make_shared<int>(0);
      actors.push_back([&, c, tile] {
        if (*tile == tiles || !pass(c->acc_full[*tile % 2], *tile / 2 + 1, "the epilogue passed for another tile")) return false;
        acc_empty[*tile % 2].arrive();
        finished += ++*tile == tiles;
        return true;
      });
    }
  }
  actors.push_back([&] {   // issues the MMAs
    if (mma_at == total) return false;
    const int tile = mma_at / kst;
    if (mma_at % kst == 0 && !mma_open) {
      if (tile >= 2 && !pass(acc_empty[tile % 2], tile / 2, "the MMA warp passed for another accumulator")) return false;
      mma_open = true;
      return true;
    }
    if (!pass(full[mma_at % kS], mma_at / kS + 1, "the MMA warp passed for another use")) return false;
    queue.push_back(mma_at++);
    if (mma_at % kst == 0) mma_open = false;
    return true;
  });
  actors.push_back([&] {   // an MMA ends: in order
    if (queue.empty()) return false;
    const int i = queue.front();
    queue.erase(queue.begin());
    mma_done = i + 1;
    for (auto& c : cta) {
      c.empty[i % kS].arrive();
      if (i % kst == kst - 1) c.acc_full[i / kst % 2].arrive();
    }
    return true;
  });
  const Speeds speed(rng, int(actors.size()));
  for (long idle = 0; idle < 2000000; ++idle) {
    if (f.what || finished == kEpW * cg) return f.what;
    if (actors[speed.pick(rng)]()) idle = 0;
  }
  return "nobody can go on";
}

int run_gemmx(bool whole) {
  using namespace lk::gx;
  const int fmts[] = {LK_Q4_0, LK_Q4_K, LK_IQ4_NL, LK_Q5_0, LK_Q8_0, LK_Q5_K, LK_Q6_K, LK_IQ4_XS, LK_Q3_K, LK_IQ3_S, LK_MXFP4};
  std::set<std::tuple<int, int, int, bool>> rings;   // the last: rows of whole chunks only
  for (int fmt : fmts)
    for (bool win : {false, true})
      for (int nt : {32, 64, 128, 256, 512}) {
        if (!win && fmt != LK_Q4_0 && fmt != LK_Q4_K && fmt != LK_IQ4_NL) continue;
        const int cg = nt == 512 ? 2 : 1;
        const Rings g = rings_of(fmt, win, cg, cg == 2 ? 256 : nt);
        rings.insert(std::make_tuple(cg, g.s, g.r, !win || lk::fmt_qk(fmt) == 256));
      }
  int faults = 0, walks = 0;
  for (auto& t : rings)
    for (int kst = 1; kst <= 22; ++kst) {
      if (std::get<3>(t) && kst % 4) continue;
      for (int tiles : {1, 2, 5})
        for (unsigned seed = 0; seed < 6; ++seed, ++walks)
          if (const char* what = walk_gemmx(std::get<0>(t), std::get<1>(t), std::get<2>(t), kst, tiles, whole, seed * 7919 + kst)) {
            if (!faults)
              printf("CTAs %d, stages %d, packed %d, k stages %d, tiles %d: %s\n", std::get<0>(t), std::get<1>(t),
                     std::get<2>(t), kst, tiles, what);
            ++faults;
          }
    }
  printf("gemmx: %d rings, %d walks, %d faults\n", int(rings.size()), walks, faults);
  return faults != 0;
}

// Each warp meets the others once a tile, whichever of its waits gives up, and neither waits nor works after that.
int run_epilogue() {
  for (int tiles = 0; tiles <= 6; ++tiles)
    for (int gives_up = 0; gives_up <= tiles; ++gives_up) {   // at this tile; at `tiles`: never
      bool live = true;
      int fills = 0, syncs = 0, waits = 0, works = 0;
      lk::gx::epilogue_tiles(
          tiles, live, [&](int li) { fills += li == syncs; }, [&] { ++syncs; },
          [&](int li) {
            ++waits;
            if (li == gives_up) live = false;
          },
          [&](int li) { works += li == waits - 1; });
      if (fills != tiles || syncs != tiles || works != gives_up || waits != (gives_up < tiles ? gives_up + 1 : tiles))
        return printf("%d tiles, given up at %d: %d barriers, %d waits, %d tiles finished\n", tiles, gives_up, syncs, waits, works), 1;
    }
  return 0;
}

}  // namespace

int main(int argc, char** argv) {
  const bool plant = argc > 2;
  if (argc > 1 && !strcmp(argv[1], "mvx")) return run_mvx(plant);
  if (argc > 1 && !strcmp(argv[1], "gemmx")) return run_gemmx(plant);
  if (argc > 1 && !strcmp(argv[1], "epilogue")) return run_epilogue();
  return 2;
}
