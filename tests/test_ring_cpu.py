"""CPU: the arithmetic by which a kernel that gives up waits for exactly the copies that it has under way (csrc/ring.h), on
a model of the barriers."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascendnpu-ir_b200", "csrc")

MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "ring.h"
using namespace bsir;

// one arrival a phase; a phase is over when the arrival is there and as many bytes came as were announced
struct Barrier {
  unsigned phase = 0;
  bool arrived = false;
  long bytes = 0;                      // announced and not yet here
  void turn() { if (arrived && bytes == 0) { ++phase; arrived = false; } }
  void expect(long n) { arrived = true; bytes += n; turn(); }
  void land(long n) { bytes -= n; turn(); }
  bool passes(unsigned parity) const { return (phase & 1u) != parity; }       // the phase of this parity is over
};
static void check(bool ok, const char *what, int a, int b, int c) {
  if (!ok) { std::printf("%s: %d %d %d\n", what, a, b, c); std::exit(1); }
}

// a ring of one CTA: of each slot the last load may still be under way
static void single(int slots, int issued, unsigned flying) {
  std::vector<Barrier> bar(slots);
  for (int i = 0; i < issued; ++i) {
    bar[i % slots].expect(8);
    if (i + slots < issued || !(flying >> (i % slots) & 1u)) bar[i % slots].land(8);
  }
  const int slot = issued % slots;
  const unsigned phase = issued / slots & 1u;
  for (int s = 0; s < slots; ++s) {
    const bool under_way = s < issued && (flying >> s & 1u);
    check(bar[s].passes(ring_last_parity(s, slot, phase)) == !under_way, "single", slots, issued, s);
    check(bar[s].passes(0) || bar[s].passes(1), "one parity always passes", slots, issued, s);
  }
  if (issued > 0) check(ring_last_slot(slots, slot) == (issued - 1) % slots, "last", slots, issued, slot);
}

// two CTAs on the leader's barriers, which issued different numbers of loads
struct Pair {
  std::vector<Barrier> bar;
  std::vector<int> left[2];            // copies under way of the leader and of the peer, by slot
  bool late = false;                   // which of the two lands first
  void complete(unsigned s, unsigned n) { bar[s].land(n); }
  void expect(unsigned s, unsigned n) { bar[s].expect(n); }
  void wait(unsigned s, unsigned parity) {
    for (int k = 0; k < 2; ++k) {
      const int who = late ? 1 - k : k;
      if (!left[who][s]) continue;
      check(!bar[s].passes(parity), "let through with a copy under way", s, parity, who);
      left[who][s] = 0;
      bar[s].land(8);
    }
    check(bar[s].passes(parity), "never over", s, parity, 0);
  }
};
struct Operations {
  Pair &p;
  void complete(unsigned s, unsigned n) { p.complete(s, n); }
  void expect(unsigned s, unsigned n) { p.expect(s, n); }
  void wait(unsigned s, unsigned parity) { p.wait(s, parity); }
};
static void pair(int slots, int leader, int peer, unsigned flying, bool late) {
  Pair p;
  p.bar.resize(slots);
  p.left[0].assign(slots, 0);
  p.left[1].assign(slots, 0);
  p.late = late;
  const int most = leader > peer ? leader : peer;
  for (int i = 0; i < most; ++i) {
    const int s = i % slots;
    const bool last = i + slots >= most;
    if (i < leader) p.bar[s].expect(16);
    for (int who = 0; who < 2; ++who) {
      if (i >= (who ? peer : leader)) continue;
      if (last && (flying >> (2 * s + who) & 1u)) p.left[who][s] = 1;
      else p.bar[s].land(8);
    }
  }
  ring_settle_pair(slots, leader, peer, 8, Operations{p});
}
int main() {
  for (int slots = 1; slots <= 9; ++slots)
    for (int issued = 0; issued <= 5 * slots; ++issued)
      for (unsigned flying = 0; flying < (1u << slots); ++flying) single(slots, issued, flying);
  for (int slots = 1; slots <= 5; ++slots)
    for (int leader = 0; leader <= 4 * slots + 1; ++leader)
      for (int peer = leader - slots < 0 ? 0 : leader - slots; peer <= leader + slots; ++peer)
        for (unsigned flying = 0; flying < (1u << 2 * slots); ++flying) {
          pair(slots, leader, peer, flying, false);
          pair(slots, leader, peer, flying, true);
        }
  std::printf("held\n");
}
"""

@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_ring_waits_for_what_is_under_way(tmp_path):
    cpp, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    cpp.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", CSRC, str(cpp), "-o", str(exe)], check=True, timeout=120)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "held", r.stdout


@pytest.mark.parametrize("name", ["mxfp4_gemm.cu", "mxfp4_quant.cu", "gemm_dense.cu", "gemm_w4a16.cu", "cumulative.cu"])
def test_waits_on_the_way_out_go_by_the_ring(name):
    """A wait that either parity of a barrier ends is over at once, whatever is under way; one for a load that was never
    issued spins to its limit."""
    text = open(os.path.join(CSRC, name)).read()
    assert not re.search(r"try_wait\([^;]*, 0\) \|\| mbar_try_wait\([^;]*, 1\)", text)
    assert not re.search(r"i < 200000", text) and re.search(r"ring_drain\(", text)


@pytest.mark.parametrize("name", ["fused_rows.cu", "chain_jit.cu"])
def test_streamed_rows_stop_after_a_wait_that_gave_up(name):
    """No load into a buffer whose last one is not known to have landed, and a wait for the last loads at the end."""
    text = open(os.path.join(CSRC, name)).read()
    for line in re.findall(r".*\bissue\(k \+ .*", text):
        assert "ok &&" in line
    assert re.search(r"ring_last_parity\(|each buffer's last row", text)


@pytest.mark.parametrize("name", ["mxfp4_gemm.cu", "gemm_dense.cu", "gemm_w4a16.cu"])
def test_next_kernel_is_let_in_after_tensor_memory_is_allocated(name):
    """One that is let in earlier may take the tensor memory that this one is still waiting for, and then wait for it."""
    text = open(os.path.join(CSRC, name)).read()
    kernels = re.split(r"\n__global__ ", text)[1:]
    seen = 0
    for body in kernels:
        body = body.split("\n}\n", 1)[0]
        alloc, let_in = re.search(r"tmem_alloc\(smem|tcgen05\.alloc", body), body.find("pdl_launch_dependents()")
        if alloc and let_in >= 0:
            seen += 1
            assert alloc.start() < let_in
    assert seen
