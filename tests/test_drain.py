"""A tensor-core kernel that gives up: its copies land before its shared memory
goes (csrc/drain.h), run on the CPU against a model of the barriers."""
import os
import re
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "maxim-rs_b200", "csrc")

MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "drain.h"

// An mbarrier of one arrival: a phase ends when it has arrived and no bytes are owed.
struct Barrier {
  int phase = 0, pending = 1;
  long owed = 0;
  void settle() { if (pending == 0 && owed == 0) ++phase, pending = 1; }
  void arm(long bytes) { if (pending == 0) abort(); owed += bytes; --pending; settle(); }
  void bytes(long n) { owed -= n; settle(); }
  bool ended(unsigned parity) const { return unsigned(phase & 1) != parity; }
};

// `mine` rounds armed and issued, `peers` issued on the same barriers (shared)
// or none of the peer's; of the copies on their way, those in `late` land only
// while the drain waits. Checks that afterwards all have landed.
static int run(unsigned mine, unsigned peers, bool shared, unsigned stages, unsigned late_bits, bool stuck) {
  const long B = 24576;
  std::vector<Barrier> bars(stages);
  struct Copy { unsigned stage; bool landed; };
  std::vector<Copy> copies;
  unsigned k = 0;
  const unsigned hi = mine > peers ? mine : peers, lo = mine < peers ? mine : peers;
  for (unsigned i = 0; i < hi; ++i) {
    // Rounds a whole ring ago have been used, so they have landed.
    const bool old = i + stages < hi || i + stages < lo;
    if (i < mine) bars[i % stages].arm((shared ? 2 : 1) * B);
    for (int who = 0; who < (shared ? 2 : 1); ++who) {
      if (i >= (who ? peers : mine)) continue;
      const bool late = !old && (late_bits >> (k++ % 16) & 1);
      copies.push_back({i % stages, !late});
      if (!late) bars[i % stages].bytes(B);
    }
  }
  unsigned waits = 0;
  const bool ok = mx::land_copies(
      mine, shared ? peers : mine, stages, [&](unsigned s) { bars[s].arm(B); },
      [&](unsigned s) { bars[s].bytes(B); },
      [&](unsigned s, unsigned parity) {
        ++waits;
        if (!stuck)
          for (auto& c : copies)
            if (!c.landed && c.stage == s) c.landed = true, bars[s].bytes(B);
        return bars[s].ended(parity);
      });
  const unsigned expect = hi < stages ? hi : stages;
  if (waits != expect) return printf("mine %u peers %u: %u waits of %u\n", mine, peers, waits, expect), 1;
  bool all = true;
  for (auto& c : copies) all = all && c.landed;
  if (ok != all) return printf("mine %u peers %u late %x: said %d, is %d\n", mine, peers, late_bits, ok, all), 1;
  if (!stuck && !all) return printf("mine %u peers %u late %x: left one in flight\n", mine, peers, late_bits), 1;
  return 0;
}

int main() {
  int bad = 0;
  for (unsigned stages : {2u, 5u, 8u})
    for (unsigned mine = 0; mine <= 3 * stages; ++mine)
      for (unsigned late = 0; late < 1u << 16; late += 977)
        for (int stuck = 0; stuck < 2; ++stuck) {
          bad += run(mine, mine, false, stages, late, stuck);
          for (unsigned peers = mine < stages ? 0 : mine - stages; peers <= mine + stages; ++peers)
            bad += run(mine, peers, true, stages, late, stuck);
        }
  return bad != 0;
}
"""


def test_every_copy_has_landed(tmp_path):
    src = tmp_path / "drain.cpp"
    src.write_text(MODEL)
    exe = tmp_path / "drain"
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[:2000]


def test_the_flag_does_not_cut_the_drain_short():
    """The waits of the drain take no abort flag: it is up by then, and would end them at once."""
    text = open(os.path.join(CSRC, "kernels_dense.cuh")).read()
    drains = re.findall(r"mbar_wait(?:<[^;]*?>)?\((?:drained|&full\[s\]),[^;]*?;", text)
    assert len(drains) == 2 and all("nullptr" in d for d in drains), drains
    assert not re.search(r"\bwait(_pair|_order)?\(drained", text)
