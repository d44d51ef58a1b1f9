// Device-side helpers of attention over paged caches, shared by the 8-bit and the
// 16-bit cache (sphkv_kv8.hip, sphkv_kv16.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include "sphkv_common.h"
#include "sphkv_internal.h"

namespace sphkv {
namespace {

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int clampi(int64_t x, int64_t lo, int64_t hi) {
  return (int)(x < lo ? lo : (x > hi ? hi : x));
}

// rows of sequence s, whatever the list holds: begin..end within [0, num_rows]
__device__ __forceinline__ void rows_of(const Cache8Batch& b, int s, int& begin, int& end) {
  if (!b.cu) {
    begin = s;
    end = s + 1;
    return;
  }
  begin = clampi(b.cu[s], 0, b.num_rows);
  end = clampi(b.cu[s + 1], begin, b.num_rows);
}

// Work slots of a ragged batch without its lengths on the host: sequence s
// starts at slot (cu[s] * mul >> shift) + extra * s, so n rows get more than
// n * mul / 2^shift - 1 + extra slots.  The last sequence whose first slot is
// at most j: 64 probes at a time, one step up to 64 sequences.  j is uniform
// over the wave.
__device__ __forceinline__ int64_t first_slot(const Cache8Batch& b, int s, int mul, int shift, int extra) {
  return (((int64_t)clampi(b.cu[s], 0, b.num_rows) * mul) >> shift) + (int64_t)extra * s;
}

__device__ __forceinline__ int seq_of_slot(const Cache8Batch& b, int64_t j, int mul, int shift, int extra) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0, hi = b.num_seqs;
  while (hi - lo > 1) {
    const int step = (hi - lo + kWave - 1) / kWave, p = lo + lane * step;
    const bool le = p < hi && first_slot(b, p < hi ? p : lo, mul, shift, extra) <= j;
    const int cnt = __popcll(__ballot(le));
    lo += (cnt > 0 ? cnt - 1 : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

template <int TYPE>
__device__ __forceinline__ void store1(void* p, int64_t i, float x) {
  if constexpr (TYPE == kFp16) ((_Float16*)p)[i] = (_Float16)x;
  else if constexpr (TYPE == kBf16) ((__bf16*)p)[i] = (__bf16)x;
  else ((float*)p)[i] = x;
}

template <int TYPE> struct Elem { typedef uint16_t T; static constexpr int kVec = 8; };
template <> struct Elem<kFp32> { typedef float T; static constexpr int kVec = 4; };

template <int TYPE>
__device__ __forceinline__ float value_of(typename Elem<TYPE>::T x) {
  if constexpr (TYPE == kFp16) return (float)__builtin_bit_cast(_Float16, x);
  else if constexpr (TYPE == kBf16) return __builtin_bit_cast(float, (uint32_t)x << 16);
  else return x;
}

// N consecutive elements at any alignment that theirs allows
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned { T x[N]; };

// over the 16 lanes of each row by rotation, then over the rows
template <int N>
__device__ __forceinline__ float row_rotated(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + N, 0xF, 0xF, true));
}
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, row_rotated<8>(x));
  x = fmaxf(x, row_rotated<4>(x));
  x = fmaxf(x, row_rotated<2>(x));
  x = fmaxf(x, row_rotated<1>(x));
  return rows_max(x);
}

// two numbers as fp16, half to even
__device__ __forceinline__ half2v fp16_pair(float x, float y) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  return __builtin_convertvector(float2v{x, y}, half2v);
}

__device__ __forceinline__ float log2_of(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float kTopWeight = 8.0f;      // log2 of the weight at the reference, ...
constexpr float kSlackWeight = 4.0f;    // ... which moves once a weight passes 2^4 times that
constexpr float kNoScore = -3.0e38f;    // reference before the first score
// A row's reference for the largest exponent `top` that it has seen, and whether it is
// to move there: by the difference, for past 2^27 an fp32 step is 16 and more, and
// a weight of 2^16 is no fp16 number.  top - kTopWeight, or top where that would round
// further down.  (Not contracted: `top` may be a product, and its rounded value counts.)
__device__ __forceinline__ bool moves_to(float top, float ref) {
#pragma clang fp contract(off)
  return top - ref > kTopWeight + kSlackWeight;
}
__device__ __forceinline__ float reference_at(float top) {
#pragma clang fp contract(off)
  const float to = top - kTopWeight;
  return top - to > kTopWeight ? top : to;
}

__device__ __forceinline__ float wave_sum(float x) {
  x += row_rotated<8>(x);
  x += row_rotated<4>(x);
  x += row_rotated<2>(x);
  x += row_rotated<1>(x);
  return rows_sum(x);
}

// Partials first, first + step, ... before end of one output row, joined by the
// wave, CH (up to 16) at a time whose loads are all on the way at once: R, l and
// the lane's DH / 64 outputs.  `at(i)`: partial i's reference (its sum `sums` floats on) and
// its row.  A reference times `scale` is a power of two's exponent.
template <int DPL, int CH, class AT>
__device__ __forceinline__ void join(int64_t first, int64_t end, int64_t step, int sums, AT at, float& R, float& l,
                                     float (&acc)[DPL], float scale = 1.0f) {
  const int lane = threadIdx.x & 63;
  R = kNoScore;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
  for (int64_t g = first; g < end; g += CH * step) {
    float a[CH][DPL], r = kNoScore, ls = 0.f;
    if (lane < CH && g + lane * step < end) {
      const float* ref = at(g + lane * step).ref;
      r = ref[0];
      ls = ref[sums];
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int64_t k = g + i * step;
      const float* row = at(k < end ? k : g).row + lane * DPL;        // (a missing one's weight is 0)
#pragma unroll
      for (int d = 0; d < DPL; ++d) a[i][d] = row[d];
    }
    const float M = fmaxf(R, wave_max(r)), f = exp2_of((r - M) * scale), was = exp2_of((R - M) * scale);
    const bool has = lane < CH && g + lane * step < end;
    const float w = has ? f : 0.f;
    l = fmaf(l, was, wave_sum(ls * w));
#pragma unroll
    for (int d = 0; d < DPL; ++d) acc[d] *= was;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
      if (g + i * step < end)
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[d] = fmaf(a[i][d], wi, acc[d]);
    }
    R = M;
  }
}
struct Partial { const float* ref; const float* row; };

__device__ __forceinline__ float halves_max(float x) {
  float a = x, b = x;
  swap32(a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float halves_sum(float x) {
  float a = x, b = x;
  swap32(a, b);
  return a + b;
}

typedef float floatx16 __attribute__((ext_vector_type(16)));
template <int N> struct Int { static constexpr int value = N; };

}  // namespace
}  // namespace sphkv
