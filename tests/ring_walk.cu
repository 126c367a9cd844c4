// Walks the shared-memory rings of the epilogue products on the host: the warps of a CTA as actors that a random scheduler
// advances one step at a time, copies that land in any order, and barriers that answer a parity wait as the hardware does.
// Ring lengths and who takes which stage come from the kernels' own functions (lk_rings.cuh). Reported: a wait that passes
// for another use of its slot than the waiter's, a slot refilled while it is read, and a state nobody can leave.
//
//   ring_walk mvx [alone]     alone: the groups never follow each other's stages (a planted mistake, for the test of the walk)
#include <cstdio>
#include <cstdlib>
#include <cstring>
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

}  // namespace

int main(int argc, char** argv) {
  const bool plant = argc > 2;
  if (argc > 1 && !strcmp(argv[1], "mvx")) return run_mvx(plant);
  return 2;
}
