"""CPU: the 4-bit head's hidden stages (csrc/ring.cuh) under every order of
loads and consumers: a lane that passes its wait finds its own block.

The barriers are modelled as the hardware has them: a wait by parity passes
unless the phase at hand has that parity.  Loads land in any order and each
lane runs as far as its waits let it, so that a ring whose stages change lanes
shows what it does (one such is run beside, as a check of the model)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MODEL = r"""
#define __host__
#define __device__
#define __forceinline__ inline
#include "ring.cuh"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace mstar;

static uint64_t state;
static uint32_t rnd(uint32_t n) {
  state = state * 6364136223846793005ull + 1442695040888963407ull;
  return (uint32_t)(state >> 33) % n;
}

// What a lane would do that counts the other lane's blocks without waiting for them.
struct Shared {
  Ring r;
  uint32_t stage(int) const { return r.i; }
  uint32_t parity(int) const { return r.parity; }
  void next(int, uint32_t stages) { r.next(stages); }
};

struct Barrier {
  uint32_t phase = 0, pending = 0, need;
  explicit Barrier(uint32_t n) : need(n) {}
  void arrive() { if (++pending == need) pending = 0, ++phase; }
  bool passes(uint32_t parity) const { return (phase & 1u) != parity; }
};

// One run over `tiles` of nblk blocks each (block b of a tile belongs to lane b
// mod LANES): the number of waits that passed on another block's stage, or -1 if
// nothing could go on.
template <int LANES, typename Rings, bool SHARED>
static int run(uint32_t stages, int nblk, int tiles, uint64_t seed) {
  state = seed * 977 + 13;
  const int total = nblk * tiles, ISS = 2;  // two issuers per lane (halves of a tile)
  std::vector<Barrier> full(stages, Barrier(1)), empty(stages, Barrier(ISS));
  std::vector<int> holds(stages, -1);
  std::vector<std::pair<int, int>> flying;  // loads: stage, block
  auto lane_of = [&](int b) { return LANES == 2 ? (b % nblk) & 1 : 0; };
  Rings pr;
  int pb = 0;
  std::vector<uint32_t> used(LANES, 0);
  const uint32_t per = SHARED ? stages : stages / LANES;
  Rings cr[LANES * ISS];
  int cb[LANES * ISS] = {}, wrong = 0;
  int idle = 0;
  for (long step = 0;; ++step) {
    bool done = pb == total && flying.empty();
    for (int c = 0; c < LANES * ISS; ++c) done = done && cb[c] >= total;
    if (done) return wrong;
    if (++idle > 100000) return -1;
    const uint32_t who = rnd(2 + LANES * ISS);
    if (who == 0) {  // the producer
      if (pb == total) continue;
      const int lane = lane_of(pb), u = SHARED ? 0 : lane;
      const uint32_t at = pr.stage(lane);
      if (used[u] == per && !empty[at].passes(pr.parity(lane) ^ 1u)) continue;
      flying.push_back({(int)at, pb++});
      pr.next(lane, stages);
      if (used[u] < per) ++used[u];
    } else if (who == 1) {  // a load lands: now and then the oldest waits long
      if (flying.empty()) continue;
      const size_t k = flying.size() > 1 && rnd(16) ? 1 + rnd((uint32_t)flying.size() - 1) : 0;
      holds[flying[k].first] = flying[k].second;
      full[flying[k].first].arrive();
      flying.erase(flying.begin() + k);
    } else {  // an issuer
      const int c = (int)who - 2, lane = c / ISS;
      Rings &r = cr[c];
      int &b = cb[c];
      while (b < total && lane_of(b) != lane) {
        if (SHARED) r.next(lane, stages);
        ++b;
      }
      if (b >= total) continue;
      const uint32_t at = r.stage(lane);
      if (!full[at].passes(r.parity(lane))) continue;
      if (holds[at] != b) ++wrong;
      empty[at].arrive();
      r.next(lane, stages);
      ++b;
    }
    idle = 0;
  }
}

int main() {
  int bad = 0, stuck = 0, seen = 0;
  for (int nblk : {1, 2, 3, 5, 6, 9, 11})
    for (uint64_t seed = 0; seed < 60; ++seed) {
      for (uint32_t stages : {6u, 8u}) {
        const int w = run<2, LaneRings<2>, false>(stages, nblk, 24, seed);
        bad += w > 0, stuck += w < 0;
        seen += run<2, Shared, true>(stages, nblk, 24, seed) != 0;
      }
      for (uint32_t stages : {3u, 4u}) {
        const int w = run<1, LaneRings<1>, false>(stages, nblk, 24, seed);
        bad += w > 0, stuck += w < 0;
      }
    }
  std::printf("%d %d %d\n", bad, stuck, seen);
}
"""


@pytest.fixture(scope="module")
def counts(tmp_path_factory):
    d = tmp_path_factory.mktemp("rings")
    src, exe = d / "model.cpp", d / "model"
    src.write_text(MODEL)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "mstar_rs_b200", "csrc"), "-o", str(exe),
                           str(src)])
    return [int(x) for x in subprocess.check_output([str(exe)], timeout=120).split()]


def test_no_lane_takes_another_blocks_stage(counts):
    assert counts[0] == 0


def test_the_rings_never_stop(counts):
    assert counts[1] == 0


def test_the_model_shows_a_stage_that_changes_lanes(counts):
    assert counts[2] > 0
