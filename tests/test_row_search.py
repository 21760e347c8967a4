"""The search for a row's first token (``probed_bound``, landmark_b200/csrc/gnr_embedding.cu), compiled for the host from its source with
the 32 probes of a warp counted in a loop: every answer of every length, also those that a gradient's long lists have."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HOST = """
#include <stdint.h>
#define __device__
#define __forceinline__ inline
%s
// positions below `answer` hold a smaller key, the others none
static int64_t bound(int64_t n, int64_t answer) {
  return probed_bound(n, [&](int64_t lo, int64_t hi, int64_t step) {
    int count = 0;
    for (int lane = 0; lane < 32; ++lane) {
      const int64_t at = lo + (lane + 1) * step - 1;
      count += at < hi && at < answer;
    }
    return count;
  });
}
// answers from `first` on, `hop` apart, that are not found
extern "C" int64_t wrong(int64_t n, int64_t first, int64_t hop) {
  int64_t count = 0;
  for (int64_t answer = first; answer <= n; answer += hop) count += bound(n, answer) != answer;
  return count;
}
"""


@pytest.fixture(scope="module")
def wrong(tmp_path_factory):
    text = open(os.path.join(ROOT, "landmark_b200", "csrc", "gnr_embedding.cu")).read()
    beg = text.index("template <typename Below> __device__ __forceinline__ int64_t probed_bound")
    folder = tmp_path_factory.mktemp("search")
    src, lib = folder / "search.cpp", folder / "search.so"
    src.write_text(HOST % text[beg:text.index("\n}\n", beg) + 3])
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", str(src), "-o", str(lib)], check=True)
    f = C.CDLL(str(lib)).wrong
    f.argtypes, f.restype = [C.c_int64] * 3, C.c_int64
    return f


def test_every_answer_of_short_lists(wrong):
    assert [n for n in range(4500) if wrong(n, 0, 1)] == []


@pytest.mark.parametrize("n", [9009, 33 * 33 * 33, 33 * 33 * 33 - 1, 33 * 33 * 33 + 1, 65536, 65537, 131072, 1500007])
def test_every_answer_of_long_lists(wrong, n):
    assert wrong(n, 0, 1) == 0


@pytest.mark.parametrize("n", [20_000_003, 2 ** 31 - 1])
def test_answers_of_the_longest_lists(wrong, n):
    assert wrong(n, 0, 4099) == 0 and wrong(n, n - 2000, 1) == 0
