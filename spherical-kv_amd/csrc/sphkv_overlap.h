// Do strided tensors share memory?  Host code in plain C++ (no HIP), so that a CPU
// test can hold it to an enumeration.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace sphkv {

// Rows of `bytes` consecutive bytes, one at `at` plus a multiple of each stride (in
// bytes, of either sign) below its count.
struct Rows {
  __int128 at;
  int64_t bytes;
  int dims;
  int64_t count[3], stride[3];
};

// Is there a sum of x_i stride_i with 0 <= x_i <= most_i in [lo, hi]?  Strides positive,
// largest first: of each, only multiples from which the smaller ones can still reach
// the interval.  Beyond `budget` steps the answer is yes (strides that are neither
// multiples of each other nor far apart; tensors in use need a few).
struct Sums {
  int dims = 0;
  __int128 stride[6], most[6], rest[7];
  int budget = 4096;
  void add(int64_t s, int64_t m) {
    if (m <= 0 || s == 0) return;
    for (int i = 0; i < dims; ++i)
      if (stride[i] == s) {
        most[i] += m;
        return;
      }
    int i = dims++;
    for (; i > 0 && stride[i - 1] < s; --i) {
      stride[i] = stride[i - 1];
      most[i] = most[i - 1];
    }
    stride[i] = s;
    most[i] = m;
  }
  bool reach(__int128 lo, __int128 hi) {
    rest[dims] = 0;
    for (int i = dims; i-- > 0;) rest[i] = rest[i + 1] + stride[i] * most[i];
    return from(0, lo, hi);
  }
  bool from(int i, __int128 lo, __int128 hi) {
    if (hi < 0 || lo > rest[i]) return false;
    if (lo <= 0) return true;
    if (i == dims) return false;
    const __int128 s = stride[i], least = lo - rest[i + 1];
    const __int128 a = least > 0 ? (least + s - 1) / s : 0, b = std::min(most[i], hi / s);
    for (__int128 x = a; x <= b; ++x) {
      if (--budget < 0) return true;
      if (from(i + 1, lo - x * s, hi - x * s)) return true;
    }
    return false;
  }
};

// every stride that takes part as a positive one
inline Rows positive(Rows r) {
  int n = 0;
  for (int i = 0; i < r.dims; ++i) {
    if (r.count[i] <= 1) continue;
    int64_t s = r.stride[i];
    if (s < 0) {
      r.at += (__int128)s * (r.count[i] - 1);
      s = -s;
    }
    r.count[n] = r.count[i];
    r.stride[n++] = s;
  }
  r.dims = n;
  return r;
}

// Do two of a tensor's rows share a byte?
inline bool shares_itself(const Rows& rows) {
  Rows r = positive(rows);
  for (int i = 1; i < r.dims; ++i)                                   // (at most three)
    for (int j = i; j > 0 && r.stride[j - 1] > r.stride[j]; --j) {
      std::swap(r.stride[j - 1], r.stride[j]);
      std::swap(r.count[j - 1], r.count[j]);
    }
  bool apart = true;                                                 // each stride passes all that the smaller ones reach
  __int128 size = r.bytes;
  for (int i = 0; i < r.dims; ++i) {
    apart = apart && r.stride[i] >= size;
    size += (__int128)r.stride[i] * (r.count[i] - 1);
  }
  if (apart) return false;
  // rows that differ in index i (the first by more), not before, anyhow behind
  for (int i = 0; i < r.dims; ++i) {
    if (r.stride[i] == 0) return true;
    Sums s;
    __int128 off = r.stride[i];
    s.add(r.stride[i], r.count[i] - 2);
    for (int j = i + 1; j < r.dims; ++j) {
      s.add(r.stride[j], 2 * (r.count[j] - 1));
      off -= (__int128)r.stride[j] * (r.count[j] - 1);
    }
    if (s.reach(-r.bytes + 1 - off, r.bytes - 1 - off)) return true;
  }
  return false;
}

// Does a row of one tensor share a byte with a row of the other?
inline bool share(const Rows& one, const Rows& two) {
  for (const Rows* r : {&one, &two})
    for (int i = 0; i < r->dims; ++i)
      if (r->count[i] <= 0) return false;
  const Rows a = positive(one), b = positive(two);
  // (a's offset + b's offset from its end back) in the interval
  Sums s;
  __int128 off = a.at - b.at;
  for (int i = 0; i < a.dims; ++i) s.add(a.stride[i], a.count[i] - 1);
  for (int i = 0; i < b.dims; ++i) {
    s.add(b.stride[i], b.count[i] - 1);
    off -= (__int128)b.stride[i] * (b.count[i] - 1);
  }
  return s.reach(-a.bytes + 1 - off, b.bytes - 1 - off);
}

// The same rows at the same places?
inline bool same(const Rows& a, const Rows& b) {
  if (a.at != b.at || a.bytes != b.bytes || a.dims != b.dims) return false;
  for (int i = 0; i < a.dims; ++i)
    if (a.count[i] != b.count[i] || (a.count[i] > 1 && a.stride[i] != b.stride[i])) return false;
  return true;
}

}  // namespace sphkv
