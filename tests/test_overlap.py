"""CPU test: whether strided tensors share memory (csrc/sphkv_overlap.h), held to an
enumeration of their bytes."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spherical-kv_amd", "csrc")

SOURCE = r"""
#include "sphkv_overlap.h"
#include <cstdio>
#include <random>
#include <set>
using namespace sphkv;
template <class F> void bytes(const Rows& r, F f) {
  int64_t n = 1;
  for (int i = 0; i < r.dims; ++i) n *= r.count[i];
  for (int64_t k = 0; k < n; ++k) {
    int64_t j = k, at = r.at;
    for (int i = 0; i < r.dims; j /= r.count[i++]) at += (j % r.count[i]) * r.stride[i];
    for (int64_t b = 0; b < r.bytes; ++b) f(at + b);
  }
}
int main() {
  std::mt19937 g(1);
  auto in = [&](int a, int b) { return (int64_t)a + (int64_t)(g() % (unsigned)(b - a + 1)); };
  long wrong = 0, both[2] = {0, 0}, self[2] = {0, 0};
  for (int it = 0; it < 100000; ++it) {
    Rows a, b;
    for (Rows* r : {&a, &b}) {
      r->bytes = in(1, 6), r->at = in(0, 60), r->dims = (int)in(0, 3);
      for (int i = 0; i < r->dims; ++i) r->count[i] = in(it % 50 ? 1 : 0, 4), r->stride[i] = in(-12, it % 2 ? 40 : 12);
    }
    if (it % 3 == 0) {                         // of equal strides, as two halves of one buffer
      b.dims = a.dims;
      for (int i = 0; i < a.dims; ++i) b.stride[i] = a.stride[i], b.count[i] = it % 50 ? a.count[i] : in(0, 4);
    }
    std::set<int64_t> of_a;
    bool twice = false, common = false;
    bytes(a, [&](int64_t x) { twice |= !of_a.insert(x).second; });
    bytes(b, [&](int64_t x) { common |= of_a.count(x) > 0; });
    wrong += share(a, b) != common || share(b, a) != common || (of_a.size() && shares_itself(a) != twice);
    ++both[common], ++self[twice];
  }
  // sizes of caches: two halves of each page, of each token, and a buffer that reaches one byte into the next
  const int64_t G = (int64_t)1 << 32;
  const Rows k{G, 256, 3, {2000000, 8, 16}, {65536, 256, 2048}}, v{G + 32768, 256, 3, {2000000, 8, 16}, {65536, 4096, 256}};
  const Rows t{G, 256, 3, {2000000, 8, 16}, {65536, 512, 4096}}, u{G + 256, 256, 3, {2000000, 8, 16}, {65536, 512, 4096}};
  wrong += share(k, v) || share(t, u) || shares_itself(k) || shares_itself(v) || shares_itself(t);
  Rows w = u;
  w.at -= 1;
  wrong += !share(t, w);
  w = t;
  w.stride[2] = 128;
  wrong += !shares_itself(w);
  printf("%ld wrong, %ld and %ld pairs, %ld and %ld alone\n", wrong, both[0], both[1], self[0], self[1]);
  return wrong != 0 || !both[0] || !both[1] || !self[0] || !self[1];
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_shared_memory_by_enumeration(tmp_path):
    (tmp_path / "t.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", CSRC, "-o", str(tmp_path / "t"), str(tmp_path / "t.cpp")], check=True)
    done = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
