"""How a call that is too large for one launch is cut (pieces.h, host only): every piece lies inside the call, up to the largest
number of sequences or tokens that the entry points take.  Compiled with the host compiler, overflow checked."""
import os
import shutil
import subprocess

import pytest

HIP = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pccl_amd", "csrc", "hip")

PROGRAM = r'''
#include <climits>
#include <cstdio>
#include <cstdlib>
#include "pieces.h"
int main(int argc, char **argv) {
  for (int k = 1; k + 1 < argc; k += 2) {
    const long total = atol(argv[k]), most = atol(argv[k + 1]);
    long pieces = 0, next = 0;
    const int rc = pccl_host::in_pieces(total, most, [&](long first, long n) {
      if (first != next || first < 0 || n < 1 || n > most || n > total - first || first > INT_MAX) return 1;
      next = first + n;
      return ++pieces > total ? 2 : 0;
    });
    printf("%d %ld %d\n", rc, pieces, next == total);
  }
  const long tokens[][4] = {{0, 5, 16, 0}, {8, 0, 16, 0}, {80, 5, 16, 80}, {79, 5, 16, 79}, {81, 5, 16, 80}, {INT_MAX, 5, 16, 80}, {15, 1, 16, 15},
                            {INT_MAX, LONG_MAX, 1 << 20, INT_MAX}, {INT_MAX, INT_MAX, 1, INT_MAX}, {INT_MAX, 2047, 1 << 20, 2047l << 20}, {INT_MAX, 2048, 1 << 20, INT_MAX}};
  for (auto &t : tokens)
    if (pccl_host::tokens_in_pages(t[0], t[1], t[2]) != t[3]) return 2;
  return pccl_host::in_pieces(10, 3, [](long first, long) { return first == 3 ? 7 : first > 3 ? 8 : 0; }) == 7 ? 0 : 1;
}
'''


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_pieces_stay_inside(tmp_path):
    (tmp_path / "t.cc").write_text(PROGRAM)
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", HIP, str(tmp_path / "t.cc"), "-o", str(exe)],
                   check=True)
    cases = [(0, 5), (1, 5), (5, 5), (6, 5), (70000, 65535), (2147450880, 65535), (2147450881, 65535), (2147483647, 65535), (2147483647, 1 << 26),
             (2147483647, (1 << 26) - 1), ((1 << 26) + 1, 1 << 26)]
    out = subprocess.run([str(exe)] + [str(x) for c in cases for x in c], check=True, capture_output=True, text=True, timeout=60).stdout
    assert out.split("\n")[:-1] == ["0 %d 1" % -(-total // most) for total, most in cases]


def test_the_entry_points_cut_by_it():
    """No loop of its own over sequences or tokens in the cache's entry points."""
    with open(os.path.join(HIP, "block_cache.hip")) as f:
        text = f.read()
    entry = text[text.index('extern "C"'):]
    assert entry.count("in_pieces(") == 3 and "for (int seq" not in entry and "for (long lo" not in entry
