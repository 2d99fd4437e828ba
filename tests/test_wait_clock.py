"""The clock of a bounded wait (csrc/wait_clock.cuh), compiled for the host: a wait gives up when its time is over, and never
before, whatever the tick it began in and across the wrap of its 32 bits."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(__file__), "..", "larder_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "wait_clock.cuh"

int main() {
  const uint64_t tick = 1u << 16, limits[] = {2000000000ull, 64 * 2000000000ull};
  long long bad = 0, seen = 0;
  auto expect = [&](bool ok, uint64_t first, uint64_t later) {
    ++seen;
    if (!ok && bad++ < 10) std::printf("began at %llu, looked %llu ns later\n", (unsigned long long)first, (unsigned long long)later);
  };
  // beginnings: consecutive ticks, about the wraps of the stamp (2^30 ticks) and of 32 bits of ticks, and far on
  const uint64_t about[] = {0, 1ull << 29, 1ull << 30, 1ull << 32, (1ull << 32) + 12345, 0x18c0123456789abull};
  for (uint64_t a : about)
    for (int k = -20; k < 20; ++k)
      for (uint64_t part : {uint64_t(0), tick / 2, tick - 1}) {
        const uint64_t t = (a + uint64_t(int64_t(k))) % (1ull << 48), first = t * tick + part;
        const uint32_t s = lb2::wait_look(0, first, limits[0]);
        expect(s != 0 && s != 1, first, 0);
        for (uint64_t limit : limits) {
          for (uint64_t later : {uint64_t(0), uint64_t(1), tick / 2, tick, 2 * tick, 3 * tick, 4 * tick, 5 * tick, uint64_t(1000000),
                                 limit / 2, limit - tick})
            expect(lb2::wait_look(s, first + later, limit) == s, first, later);
          for (uint64_t later : {limit + 2 * tick, 2 * limit, 100 * limit})
            expect(lb2::wait_look(s, first + later, limit) == 1, first, later);
        }
      }
  std::printf("%lld of %lld wrong\n", bad, seen);
  return bad != 0;
}
"""


def test_a_wait_gives_up_when_its_time_is_over(tmp_path):
    src, exe = tmp_path / "clock.cpp", tmp_path / "clock"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
