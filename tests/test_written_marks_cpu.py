"""Streams whose weights the library has just written (csrc/written.h), compiled and run on the host: the product that follows on a stream
must find its mark, however many streams, devices and captures there are."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vq_gemm_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include <thread>
#include "written.h"
using vqg::WrittenMarks;
#define EXPECT(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  WrittenMarks m;
  static char streams[5000];
  EXPECT(!m.maybe(0, nullptr) && !m.take({0, nullptr, 0}));
  // many streams at once, each marked twice: every product finds its mark, once
  for (char& s : streams) { m.note({0, &s, 0}); m.note({0, &s, 0}); }
  for (char& s : streams) EXPECT(m.maybe(0, &s) && m.take({0, &s, 0}) && !m.take({0, &s, 0}));
  EXPECT(!m.maybe(0, streams));
  // the default streams of two devices
  m.note({0, nullptr, 0});
  EXPECT(!m.maybe(1, nullptr) && !m.take({1, nullptr, 0}) && m.take({0, nullptr, 0}));
  // a captured product leaves an eager mark, and an eager one a captured mark
  m.note({0, streams, 0});
  EXPECT(m.maybe(0, streams) && !m.take({0, streams, 7}) && m.take({0, streams, 0}));
  m.note({0, streams, 7});
  EXPECT(!m.take({0, streams, 0}) && !m.take({0, streams, 8}) && m.take({0, streams, 7}));
  // threads with streams of their own
  int lost[8] = {};
  std::thread t[8];
  for (int i = 0; i < 8; ++i)
    t[i] = std::thread([&, i] {
      for (int n = 0; n < 2000; ++n) {
        m.note({0, streams + i, 0});
        lost[i] += !(m.maybe(0, streams + i) && m.take({0, streams + i, 0}));
      }
    });
  for (auto& x : t) x.join();
  for (int n : lost) EXPECT(n == 0);
  return 0;
}
"""


def test_every_mark_is_found_once(tmp_path):
    source, program = tmp_path / "marks.cpp", tmp_path / "marks"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-pthread", f"-I{CSRC}", str(source), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout
