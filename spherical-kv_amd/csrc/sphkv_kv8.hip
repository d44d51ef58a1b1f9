// The 8-bit KV cache: write, read back and attention (include/sphkv.h, "8-bit
// KV cache").  No reference counterpart: the reference keeps angle codes and
// fp16 values.
#include <hip/hip_runtime.h>

#include "sphkv_attend.h"

namespace sphkv {
namespace {

constexpr float kLeastScale = 0x1p-60f, kMostScale = 0x1p60f;

// the page of block blk of sequence s, or -1
__device__ __forceinline__ int page_of(const Cache8& c, const Cache8Batch& b, int s, int64_t blk) {
  if (blk < 0 || blk >= b.max_blocks) return -1;
  const int p = b.table[s * b.table_stride + blk];
  return p >= 0 && p < c.num_pages ? p : -1;
}

template <int FMT>
__device__ __forceinline__ float decode1(uint8_t c) {
  if constexpr (FMT == kCache8Int8) return (float)(int8_t)c;
  return __builtin_amdgcn_cvt_f32_fp8(c, 0);
}

// the lowest n bytes of a dword (none below 1, all from 4 on)
__device__ __forceinline__ uint32_t low_bytes(int n) {
  n = min(max(n, 0), 4);
  return (uint32_t)((1ull << (8 * n)) - 1);
}

// byte k (a constant after unrolling) of four codes
template <int FMT>
__device__ __forceinline__ float decode_byte(uint32_t x, int k) {
  if constexpr (FMT == kCache8Int8) return (float)(int8_t)(x >> (8 * k));
  switch (k) {
    case 0: return __builtin_amdgcn_cvt_f32_fp8(x, 0);
    case 1: return __builtin_amdgcn_cvt_f32_fp8(x, 1);
    case 2: return __builtin_amdgcn_cvt_f32_fp8(x, 2);
    default: return __builtin_amdgcn_cvt_f32_fp8(x, 3);
  }
}

// The scale of a block whose largest finite magnitude is a.
template <int FMT>
__device__ __forceinline__ float block_scale(float a) {
  float s;
  if constexpr (FMT == kCache8Int8) {
    s = __fdiv_rn(a, 127.0f);
  } else {
    // a = m 2^e, m in [1/2, 1): a / 2^(e-9) = 512 m <= 448 up to m = 7/8
    int e;
    const float m = frexpf(a, &e);
    s = a > 0.f ? ldexpf(1.0f, m <= 0.875f ? e - 9 : e - 8) : 0.f;
  }
  return fminf(fmaxf(s, kLeastScale), kMostScale);
}

// The code nearest to x / s, half to even; inv = 1 / s.
// int8: r = rint(x * inv) is at most one off, and x - r s is exact (it is a
// multiple of the smaller of the two last places and below 1.5 s), so its
// comparison with s / 2 puts r right.  e4m3: s is a power of two, so x * inv is
// exact and rounded once.
template <int FMT>
__device__ __forceinline__ float scaled(float x, float s, float inv) {
  x = x == x ? x : 0.f;
  if constexpr (FMT == kCache8Int8) {
    float r = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
    const float d = fmaf(-r, s, x), h = 0.5f * s, a = fabsf(d);
    const bool off = (a > h) | ((a == h) & ((int)r & 1));
    r += off ? __builtin_copysignf(1.f, d) : 0.f;
    return fminf(fmaxf(r, -127.f), 127.f);
  }
  return fminf(fmaxf(x * inv, -448.f), 448.f);
}
template <int FMT>
__device__ __forceinline__ uint32_t code4(float x, float y, float z, float w, float s, float inv) {
  x = scaled<FMT>(x, s, inv);
  y = scaled<FMT>(y, s, inv);
  z = scaled<FMT>(z, s, inv);
  w = scaled<FMT>(w, s, inv);
  if constexpr (FMT == kCache8Int8)
    return ((uint32_t)(int)x & 255u) | ((uint32_t)(int)y & 255u) << 8 | ((uint32_t)(int)z & 255u) << 16 | (uint32_t)(int)w << 24;
  return __builtin_amdgcn_cvt_pk_fp8_f32(z, w, __builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false), true);
}

// A code of scale s as a code of scale t > s (both exact in 64 bits).
template <int FMT>
__device__ __forceinline__ uint8_t recode(uint8_t c, float s, float t) {
  const double y = (double)decode1<FMT>(c) * s / t;
  if constexpr (FMT == kCache8Int8) return (uint8_t)(int)fmin(fmax(rint(y), -127.), 127.);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32((float)y, (float)y, 0, false);
}

// ---- write and read ------------------------------------------------------------
//
// Both move bytes: 2 * 16 * DH elements of a run of 16 tokens in and out per
// wave, once.  A lane takes 16 bytes of a key row at a time; of the values, which
// lie token-minor, two dims of all its tokens (of 8 at DH 64, the lane's half
// saying which), so that the transposition is the lane's own.  100K fp16 tokens of
// 8 heads x 128 are written as int8 in 136 us and read back in 122 (626 MB each way:
// 4.6 and 5.1 TB/s, a large copy has 4.9).

template <int TYPE>
__device__ __forceinline__ typename Elem<TYPE>::T element_of(float x) {
  if constexpr (TYPE == kFp16) return __builtin_bit_cast(uint16_t, (_Float16)x);
  else if constexpr (TYPE == kBf16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  else return x;
}

// |x|, or 0 where x is not finite
__device__ __forceinline__ float finite_abs(float x) {
  x = fabsf(x);
  return x < INFINITY ? x : 0.f;
}

// Largest magnitude of a lane's elements by their bits (two at a time where they
// have 16), infinities and NaN at the top.
typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
template <int TYPE>
struct Top {
  uint32_t bits = 0;
  template <int N>
  __device__ __forceinline__ void add(const typename Elem<TYPE>::T (&x)[N]) {
    if constexpr (TYPE == kFp32) {
#pragma unroll
      for (int i = 0; i < N; ++i) bits = max(bits, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const uint32_t y = ((uint32_t)x[i] | (uint32_t)x[i + 1] << 16) & 0x7FFF7FFFu;
        bits = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, bits), __builtin_bit_cast(ushort2v, y)));
      }
    }
  }
  __device__ __forceinline__ float value() const {
    if constexpr (TYPE == kFp32) return __builtin_bit_cast(float, bits);
    else return value_of<TYPE>((uint16_t)max(bits & 0xFFFFu, bits >> 16));
  }
};

// Four codes in the plain case (finite values that the scale reaches), and
// `worst`, to which they raise |x - code s|.  int8: x / s + 1.5 * 2^23 has the
// rounded quotient in its low byte; where `worst` stays below s / 2 by more than
// the product can be off, all are the nearest.  e4m3: exact.
constexpr float kRoundInt = 12582912.f;
template <int FMT>
__device__ __forceinline__ uint32_t plain_code4(const float (&x)[4], float s, float inv, float& worst) {
  if constexpr (FMT == kCache8Int8) {
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = fmaf(x[i], inv, kRoundInt);
      y[i] = __builtin_bit_cast(uint32_t, r);
      worst = fmaxf(worst, fabsf(fmaf(kRoundInt - r, s, x[i])));
    }
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0C0C0400u), __builtin_amdgcn_perm(y[1], y[0], 0x0C0C0400u), 0x05040100u);
  }
  return __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false), true);
}
// whether plain_code4's codes hold
template <int FMT>
__device__ __forceinline__ bool plain_holds(float top, float s, float worst) {
  return top < INFINITY && s < kMostScale && (FMT == kCache8E4M3 || worst < s * (0.5f - 0x1p-14f));
}

// Workgroups of whole pages: RUNS waves a page, at least four waves.
template <int TYPE, int FMT, int DH, int RUNS>
__global__ __launch_bounds__(RUNS == 8 ? 512 : 256) void cache8_write_kernel(Cache8RowsLaunch L, uint32_t items) {
  constexpr int kWaves = RUNS == 8 ? 8 : 4, kPages = kWaves / RUNS;
  constexpr int VEC = Elem<TYPE>::kVec, LPR = DH / VEC, RPL = 64 / LPR, KN = 16 / RPL;   // lanes a row, rows a load, loads
  constexpr int VT = DH / 8;                                         // tokens of a lane's values: 16 (DH 128) or 8
  typedef typename Elem<TYPE>::T E;
  __shared__ float s_top[2][kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, run = wave % RUNS;
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  const uint32_t item = blockIdx.x * kPages + wave / RUNS;
  const uint32_t j = item / c.num_kv;
  const int h = (int)(item - j * c.num_kv);
  constexpr int ps = 16 * RUNS;
  int o = 0, e = 0, page = -1;                                        // the page's new slots o .. e - 1
  int64_t row0 = 0;                                                   // row of slot o
  if (item < items) {
    int s = (int)j, begin, end;
    int64_t jj = 0;
    if (b.cu) {
      s = uniform(seq_of_slot(b, j, 1, c.page_shift, 2));
      jj = j - first_slot(b, s, 1, c.page_shift, 2);
    }
    rows_of(b, s, begin, end);
    const int64_t start = b.at[s], blk = start / ps + jj, left = start + (end - begin) - blk * ps;
    if (start >= 0 && jj >= 0 && left > 0) {                          // (jj < 0: row starts that decrease)
      o = jj ? 0 : (int)(start & (ps - 1));
      e = left < ps ? (int)left : ps;
      if (o < e) page = uniform(page_of(c, b, s, blk));
      row0 = begin + (blk * ps + o - start);
    }
  }
  const bool any = page >= 0 && o < e;
  const int lo = any ? min(max(o - 16 * run, 0), 16) : 0, hi = any ? min(max(e - 16 * run, 0), 16) : 0;
  const int64_t ph = (int64_t)(any ? page : 0) * c.num_kv + h;
  const int64_t first = row0;
  row0 += 16 * run - o;                                               // row of this run's token 0
  uint8_t* kc = c.k + (ph * ps + 16 * run) * DH;
  uint8_t* vc = c.v + (ph * ps + 16 * run) * DH;
  const int krow = lane / LPR, kdim = VEC * (lane % LPR);             // key rows krow + RPL i, dims kdim ..
  const int vdim = 2 * (lane & (DH / 2 - 1)), vtok = DH == 128 ? 0 : 8 * (lane >> 5);
  // every lane loads, the page's first new row where its own is none (a branch
  // around a load would wait for each, and that row changes no maximum)
  const int64_t other = any ? first : 0;
  Unaligned<E, VEC> kx[KN];
  Unaligned<E, 2> vx[VT];
#pragma unroll
  for (int i = 0; i < KN; ++i) {
    const int t = krow + RPL * i;
    const int64_t row = t >= lo && t < hi ? row0 + t : other;
    kx[i] = *(const Unaligned<E, VEC>*)((const E*)L.k + row * L.k_row + h * L.k_head + kdim);
  }
#pragma unroll
  for (int i = 0; i < VT; ++i) {
    const int t = vtok + i;
    const int64_t row = t >= lo && t < hi ? row0 + t : other;
    vx[i] = *(const Unaligned<E, 2>*)((const E*)L.v + row * L.v_row + h * L.v_head + vdim);
  }
  float kold = 0.f, vold = 0.f;
  if (any) {
    kold = c.scales[2 * ph];
    vold = c.scales[2 * ph + 1];
  }
  Top<TYPE> km, vm;
#pragma unroll
  for (int i = 0; i < KN; ++i) km.add(kx[i].x);
#pragma unroll
  for (int i = 0; i < VT; ++i) vm.add(vx[i].x);
  float ktop = km.value(), vtop = vm.value();
  const bool kfine = !__any(!(ktop < INFINITY)), vfine = !__any(!(vtop < INFINITY));
  if (!kfine) {
    ktop = 0.f;
#pragma unroll
    for (int i = 0; i < KN; ++i)
#pragma unroll
      for (int v = 0; v < VEC; ++v) ktop = fmaxf(ktop, finite_abs(value_of<TYPE>(kx[i].x[v])));
  }
  if (!vfine) {
    vtop = 0.f;
#pragma unroll
    for (int i = 0; i < VT; ++i) vtop = fmaxf(vtop, fmaxf(finite_abs(value_of<TYPE>(vx[i].x[0])), finite_abs(value_of<TYPE>(vx[i].x[1]))));
  }
  ktop = wave_max(ktop);
  vtop = wave_max(vtop);
  if constexpr (RUNS > 1) {
    if (lane == 0) {
      s_top[0][wave] = ktop;
      s_top[1][wave] = vtop;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < RUNS; ++w) {
      ktop = fmaxf(ktop, s_top[0][wave - run + w]);
      vtop = fmaxf(vtop, s_top[1][wave - run + w]);
    }
  }
  if (!any) return;
  float ks = block_scale<FMT>(ktop), vs = block_scale<FMT>(vtop);
  if (o > 0 && kold >= ks) ks = kold;
  if (o > 0 && vold >= vs) vs = vold;
  if (run == 0 && lane == 0) *(float2*)(c.scales + 2 * ph) = float2{ks, vs};
  // (every wave of a page has read the old scales: before the barrier, or itself)
  const float kinv = __fdiv_rn(1.0f, ks), vinv = __fdiv_rn(1.0f, vs);
  uint32_t ky[KN][VEC / 4], vy[2][VT / 4];
  float kworst = 0.f, vworst = 0.f;
#pragma unroll
  for (int i = 0; i < KN; ++i)
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) {
      const float x[4] = {value_of<TYPE>(kx[i].x[4 * k]), value_of<TYPE>(kx[i].x[4 * k + 1]),
                          value_of<TYPE>(kx[i].x[4 * k + 2]), value_of<TYPE>(kx[i].x[4 * k + 3])};
      ky[i][k] = plain_code4<FMT>(x, ks, kinv, kworst);
    }
#pragma unroll
  for (int d = 0; d < 2; ++d)
#pragma unroll
    for (int k = 0; k < VT / 4; ++k) {
      const float x[4] = {value_of<TYPE>(vx[4 * k].x[d]), value_of<TYPE>(vx[4 * k + 1].x[d]),
                          value_of<TYPE>(vx[4 * k + 2].x[d]), value_of<TYPE>(vx[4 * k + 3].x[d])};
      vy[d][k] = plain_code4<FMT>(x, vs, vinv, vworst);
    }
  if (!kfine || __any(!plain_holds<FMT>(ktop, ks, kworst)))
#pragma unroll
    for (int i = 0; i < KN; ++i)
#pragma unroll
      for (int k = 0; k < VEC / 4; ++k)
        ky[i][k] = code4<FMT>(value_of<TYPE>(kx[i].x[4 * k]), value_of<TYPE>(kx[i].x[4 * k + 1]),
                              value_of<TYPE>(kx[i].x[4 * k + 2]), value_of<TYPE>(kx[i].x[4 * k + 3]), ks, kinv);
  if (!vfine || __any(!plain_holds<FMT>(vtop, vs, vworst)))
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
      for (int k = 0; k < VT / 4; ++k)
        vy[d][k] = code4<FMT>(value_of<TYPE>(vx[4 * k].x[d]), value_of<TYPE>(vx[4 * k + 1].x[d]),
                              value_of<TYPE>(vx[4 * k + 2].x[d]), value_of<TYPE>(vx[4 * k + 3].x[d]), vs, vinv);
#pragma unroll
  for (int i = 0; i < KN; ++i) {
    const int t = krow + RPL * i;
    if (t < lo || t >= hi) continue;
    if constexpr (VEC == 8) *(uint2*)(kc + t * DH + kdim) = uint2{ky[i][0], ky[i][1]};
    else *(uint32_t*)(kc + t * DH + kdim) = ky[i][0];
  }
  // Codes held before, under a larger scale, a byte a lane at a time.  int8 tokens
  // alike in size grow 16 % of the scales per token appended to pages of 16, so most
  // calls wait for a wave that does this (256 sequences of 8 heads: 13.4 us a call, 8.0
  // where no scale grows); e4m3's powers of two grow 2.5 % at pages of 32 (17.1 and 8.9).
  if (lo > 0 && ks > kold)
#pragma unroll 1
    for (int i = lane; i < lo * DH; i += kWave) kc[i] = recode<FMT>(kc[i], kold, ks);
  if (lo > 0 && vs > vold)
#pragma unroll 1
    for (int i = 0; i < 2 * VT; ++i) {
      uint8_t* p = vc + (vdim + i / VT) * 16 + vtok + i % VT;
      if (vtok + i % VT < lo) *p = recode<FMT>(*p, vold, vs);
    }
  if (lo < hi) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      uint32_t (&y)[VT / 4] = vy[d];
      uint32_t* p = (uint32_t*)(vc + (vdim + d) * 16 + vtok);
      if (lo > 0 || hi < 16) {                                        // the run's other tokens keep their bytes
#pragma unroll
        for (int k = 0; k < VT / 4; ++k) {
          const uint32_t was = p[k];
          const int a = lo - vtok - 4 * k, z = hi - vtok - 4 * k;    // the dword's new bytes: a .. z - 1
          const uint32_t fresh = low_bytes(z) & ~low_bytes(a);
          y[k] = (y[k] & fresh) | (was & ~fresh);
        }
      }
      if constexpr (VT == 16) *(uintx4*)p = uintx4{y[0], y[1], y[2], y[3]};
      else *(uint2*)p = uint2{y[0], y[1]};
    }
  }
}

// One wave per (16-token run, kv head).
template <int TYPE, int FMT, int DH>
__global__ __launch_bounds__(256) void cache8_read_kernel(Cache8RowsLaunch L, uint32_t items) {
  constexpr int LPR = DH / 16, RPL = 64 / LPR, KN = 16 / RPL, VT = DH / 8;
  typedef typename Elem<TYPE>::T E;
  const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  if (item >= items) return;
  const uint32_t j = item / c.num_kv;
  const int h = (int)(item - j * c.num_kv), ps = 1 << c.page_shift;
  int s = (int)j, begin, end;
  int64_t jj = 0;
  if (b.cu) {
    s = uniform(seq_of_slot(b, j, 1, 4, 2));
    jj = j - first_slot(b, s, 1, 4, 2);
  }
  rows_of(b, s, begin, end);
  const int64_t start = b.at[s], pos0 = ((start >> 4) + jj) << 4, left = start + (end - begin) - pos0;
  const int lo = jj ? 0 : (int)(start & 15), hi = left < 16 ? (int)left : 16;
  if (lo >= hi || jj < 0) return;                                     // (jj < 0: row starts that decrease)
  const int page = uniform(page_of(c, b, s, pos0 >> c.page_shift));
  const int64_t row0 = begin + (pos0 - start);                        // row of the run's token 0
  uintx4 kx[KN], vx[2];
  float sk = 0.f, sv = 0.f;
  const int krow = lane / LPR, kdim = 16 * (lane % LPR);
  const int vdim = 2 * (lane & (DH / 2 - 1)), vtok = DH == 128 ? 0 : 8 * (lane >> 5);
#pragma unroll
  for (int i = 0; i < KN; ++i) kx[i] = uintx4{0, 0, 0, 0};
  vx[0] = vx[1] = uintx4{0, 0, 0, 0};
  if (page >= 0) {
    const int64_t ph = (int64_t)page * c.num_kv + h, at = (ph * ps + (pos0 & (ps - 1))) * DH;
    if (L.k)
#pragma unroll
      for (int i = 0; i < KN; ++i) kx[i] = *(const uintx4*)(c.k + at + (krow + RPL * i) * DH + kdim);
    if (L.v) {
      if constexpr (VT == 16) {
#pragma unroll
        for (int d = 0; d < 2; ++d) vx[d] = *(const uintx4*)(c.v + at + (vdim + d) * 16);
      } else {
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const uint2 x = *(const uint2*)(c.v + at + (vdim + d) * 16 + vtok);
          vx[d].x = x.x;
          vx[d].y = x.y;
        }
      }
    }
    const float2 sc = *(const float2*)(c.scales + 2 * ph);
    sk = sc.x;
    sv = sc.y;
  }
  if (L.k) {
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const int t = krow + RPL * i;
      if (t < lo || t >= hi) continue;
      constexpr int N = 16 / sizeof(E);                               // elements of a 16-byte store
      E* p = (E*)L.k + (row0 + t) * L.k_row + h * L.k_head + kdim;
#pragma unroll
      for (int k = 0; k < 16 / N; ++k) {
        struct __attribute__((aligned(16))) { E x[N]; } y;
#pragma unroll
        for (int n = 0; n < N; ++n) y.x[n] = element_of<TYPE>(decode_byte<FMT>(kx[i][(k * N + n) / 4], n & 3) * sk);
        *(decltype(y)*)(p + k * N) = y;
      }
    }
  }
  if (L.v) {
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      const int t = vtok + i;
      if (t < lo || t >= hi) continue;
      struct __attribute__((aligned(2 * sizeof(E)))) { E x[2]; } y;
#pragma unroll
      for (int d = 0; d < 2; ++d) y.x[d] = element_of<TYPE>(decode_byte<FMT>(vx[d][i / 4], i & 3) * sv);
      *(decltype(y)*)((E*)L.v + (row0 + t) * L.v_row + h * L.v_head + vdim) = y;
    }
  }
}

// ---- decode ------------------------------------------------------------------
//
// out = sum_t w_t c_t / sum_t (w_t / sv_t),  w_t = 2^(s_t + log2 sv_t - R),
// s_t = sm_scale log2(e) sk_t <q, k_t>, c_t the value codes, R a reference near
// the largest s_t + log2 sv_t.  With the value scale inside the exponent, the
// largest weight that meets the codes is near 2^8 wherever the scales lie, so
// weights fit fp16 (11 bits) and the products run on raw codes.
//
// A tile is 64 tokens, one wave's step: S^T = K Q^T as four 16x16 blocks
// (v_mfma_f32_16x16x32_f16: int8 and e4m3 are exact in fp16), O^T += V^T P^T as
// DH/16 blocks of 32 tokens.  Token 16 g + 4 i + j of a tile is row 4 g + j of
// score block i, so lane (g, column) ends up with the scores of the 16 tokens
// 16 g .. 16 g + 15 of one page run, in order: they are its part of the second
// product's B operand as they stand, and the 16 bytes that it loads per value
// row are its part of the A operand.  Nothing passes through LDS.
// A column is a query head; up to 8 heads use two columns each, the second one
// for what the first one's fp16 weight leaves out.  More heads fill the columns, and
// that rest is a product of its own, hidden behind the loads (32 contexts of 2K to 8K
// tokens, 4 heads x 16 queries x 128, 45.5 us with it and 45.9 without; 16 contexts
// of 2K to 16K, 2 x 64, 55.2 and 56.3).
//
// Work: the tiles of all (sequence, kv head) pairs in a row, cut into equal
// runs, one per workgroup; its four waves take the tiles of a pair in turn and
// join their sums in LDS.  A pair that one workgroup holds is written out there;
// the others leave a partial per workgroup (two at most: its first and its last
// pair) for the merge kernel.  HBM-bound: 64 contexts of 2K..32K tokens, 8 heads x
// 128 in e4m3, 2.28 GB in 400 us (5.7 TB/s); one of 32K in int8 20 us, about 4 of them
// the merge.
constexpr int kTileTokens = 64;
// Workgroups: two of four waves per CU at DH 128, three at DH 64, whose registers
// allow it (256 contexts of 100 to 900 tokens 50.7 us, 58.0 with two).  Their tiles
// are a multiple of their waves.
__host__ __device__ constexpr int decode_groups(int dh) { return dh == 128 ? 512 : 768; }
constexpr int kDecodeWaves = 4;
// An exponent is one multiply-add, s_t + (log2 sv_t - R), whose rounding differs
// from that of R by up to 2^-24 R: from this on they are rounded alike, s_t + log2
// sv_t first, so that the largest weight is exactly that at any magnitude (always: 3
// to 5 % of the prefill).
constexpr float kPlainScore = 0x1p18f;

// heads handled together: a kv head's first 16, next 16, ...
__host__ __device__ __forceinline__ int head_parts(int gqa) { return (gqa + 15) / 16; }
__host__ __device__ __forceinline__ int part_cols(int gqa, int part) { return gqa - part * 16 < 16 ? gqa - part * 16 : 16; }
// floats of one partial: reference and sum per column, then acc[cols][DH]
__host__ __device__ __forceinline__ int64_t partial8_floats(int gqa, int dh) { return 32 + (int64_t)(gqa < 16 ? gqa : 16) * dh; }
__host__ __device__ __forceinline__ int64_t plan_bytes(int num_seqs) { return (16 + 8 * ((int64_t)num_seqs + 1) + 255) / 256 * 256; }

__device__ __forceinline__ int seq_tokens(const Cache8& c, const Cache8Batch& b, int s) {
  return clampi(b.at[s], 0, (int64_t)b.max_blocks << c.page_shift);
}

__device__ __forceinline__ int64_t shfl64(int64_t x, int lane) {
  const int lo = __shfl((int)x, lane, kWave), hi = __shfl((int)(x >> 32), lane, kWave);
  return ((int64_t)hi << 32) | (uint32_t)lo;
}

// inclusive scan over the wave
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t y = shfl64(x, lane - d);
    if (lane >= d) x += y;
  }
  return x;
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return ((int64_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x);
}

// Four codes as two pairs of fp16 (exact).  int8: the byte + 128 below 1024,
// whose fp16 last place is 1, less 1152.
template <int FMT>
__device__ __forceinline__ void codes4(uint32_t x, half2v& a, half2v& b) {
  if constexpr (FMT == kCache8Int8) {
    x ^= 0x80808080u;
    const half2v off = {(_Float16)1152.f, (_Float16)1152.f};
    a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - off;
    b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - off;
  } else {
    a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true);
  }
}

template <int FMT>
__device__ __forceinline__ half8 codes8(uint32_t x, uint32_t y) {
  half2v a, b, c, d;
  codes4<FMT>(x, a, b);
  codes4<FMT>(y, c, d);
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A query row's part in a lane as fp16.  fp16 rows as they are.  bf16 rows times
// a power of two that brings their largest magnitude (row_max joins the lanes
// that share a row) into [2^14, 2^15): what lies 2^-29 below it or higher is
// exact, the rest within 2^-40 of it.  `back` undoes it on the scores.
template <int TYPE, int N, class MAX>
__device__ __forceinline__ void query_fp16(const uintx4 (&raw)[N], MAX row_max, half8 (&out)[N], int& back) {
  back = 0;
  if constexpr (TYPE == kFp16) {
    // (used here, so that their wait is here: a wait at the first product, inside
    // the loop, would in every turn be for the loads of the next tile too)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uintx4 x = raw[i];
      asm volatile("" : "+v"(x));
      out[i] = __builtin_bit_cast(half8, x);
    }
  } else {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m = fmaxf(m, fabsf(__builtin_bit_cast(float, raw[i][e] << 16)));
        m = fmaxf(m, fabsf(__builtin_bit_cast(float, raw[i][e] & 0xFFFF0000u)));
      }
    m = row_max(m);
    int e = 0;
    frexpf(m, &e);                                    // m in [2^(e-1), 2^e)
    back = m > 0.f && m < INFINITY ? e - 15 : 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        out[i][2 * k] = (_Float16)ldexpf(__builtin_bit_cast(float, raw[i][k] << 16), -back);
        out[i][2 * k + 1] = (_Float16)ldexpf(__builtin_bit_cast(float, raw[i][k] & 0xFFFF0000u), -back);
      }
  }
}

// a tile's bytes in a lane
template <int DH>
struct Tile {
  uintx4 k[4][DH / 64];       // score block i, dims 64 j + 16 kb ..: token 16 (r >> 2) + 4 i + (r & 3), r = lane & 15
  uintx4 v[DH / 16];          // value row 16 d + (lane & 15), tokens 16 g .. 16 g + 15, g = lane >> 4
  float sk, sv;               // the scales of the tokens of run g
  int page;                   // their page, or -1
};

// TWIN: up to 8 heads, in columns 0..7 and again in 8..15
template <int FMT, int TYPE, int DH, bool TWIN>
__global__ __launch_bounds__(256, 2) void cache8_decode_kernel(Cache8AttendLaunch L, float* partials, int64_t* base_of) {
  constexpr int DT = DH / 16;
  __shared__ float s_ref[4][16], s_sum[4][16];
  __shared__ float s_acc[4][16][DH + 4];
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int parts = head_parts(L.gqa), HV = c.num_kv * parts, n = b.num_seqs;

  // this workgroup's tiles
  int64_t total = 0;
  for (int i = lane; i < n; i += kWave) total += (seq_tokens(c, b, i) + kTileTokens - 1) / kTileTokens;
  total = uniform64(shfl64(wave_scan(total), 63)) * HV;
  constexpr int64_t kShare = (int64_t)decode_groups(DH) * kDecodeWaves;
  const int64_t per = total > kShare ? (total + kShare - 1) / kShare * kDecodeWaves : kDecodeWaves;
  int64_t p = (int64_t)blockIdx.x * per;
  const int64_t pend = p + per < total ? p + per : total;
  const bool writes_plan = blockIdx.x == 0 && wave == 3;
  int s = 0;
  int64_t sbase = 0;                                  // tile at which sequence s starts
  if (p < pend || writes_plan) {
    int64_t before = 0;
    bool found = false;
    for (int i0 = 0; i0 < n && (!found || writes_plan); i0 += kWave) {
      const int i = i0 + lane;
      const int64_t t = i < n ? (int64_t)((seq_tokens(c, b, i) + kTileTokens - 1) / kTileTokens) * HV : 0;
      const int64_t incl = before + wave_scan(t);
      if (writes_plan && i < n) base_of[1 + i] = incl - t;
      const uint64_t past = __ballot(incl > p);
      if (!found && past) {
        const int l = __ffsll((unsigned long long)past) - 1;
        found = true;
        s = i0 + l;
        sbase = uniform64(shfl64(incl - t, l));
      }
      before = uniform64(shfl64(incl, 63));
    }
    if (writes_plan && lane == 0) {
      base_of[0] = per;
      base_of[1 + n] = total;
    }
  }
  const float qscale = L.sm_scale * 1.44269504088896f;
  const int64_t page_bytes = (int64_t)c.num_kv * DH << c.page_shift;

  for (; p < pend && s < n; ++s) {
    const int len = uniform(seq_tokens(c, b, s)), T = (len + kTileTokens - 1) / kTileTokens;
    if (T == 0) continue;
    const int32_t* table = b.table + s * b.table_stride;
    while (p < pend && p < sbase + (int64_t)T * HV) {
      const int hv = (int)((p - sbase) / T), h = hv / parts, part = hv - h * parts;
      const int cols = part_cols(L.gqa, part);
      const int64_t first = sbase + (int64_t)hv * T;
      const int t0 = (int)(p - first), t1 = pend - first < T ? (int)(pend - first) : T;
      const int mycol = TWIN ? (col & 7) : col;

      // a column's query: dims 64 j + 16 g + 0..15 in lane group g
      half8 q[DH / 32];
      int back;
      const int64_t row = (int64_t)s;
      {
        struct __attribute__((packed, aligned(2))) U4 { uintx4 v; };
        const int mine = mycol < cols ? mycol : 0;                           // (columns over: the first again, dropped at the end)
        const uint16_t* src = (const uint16_t*)L.q + row * L.q_row + (int64_t)(h * L.gqa + part * 16 + mine) * L.q_head + 16 * g;
        uintx4 raw[DH / 32];
#pragma unroll
        for (int i = 0; i < DH / 32; ++i) raw[i] = ((const U4*)(src + 64 * (i / 2) + 8 * (i & 1)))->v;
        query_fp16<TYPE, DH / 32>(raw, [](float m) { return rows_max(m); }, q, back);
      }
      const float cq = ldexpf(qscale, back);

      // page of run `run` of tile t, or -1
      auto page_at = [&](int t, int run) {
        const int at = t * kTileTokens + run * 16, blk = at >> c.page_shift, pg = table[min(blk, b.max_blocks - 1)];
        const int has = (at < len) & (blk < b.max_blocks) & (pg < (int)c.num_pages);   // (no branch around the load)
        return pg | (has - 1);
      };
      Tile<DH> A;
      auto load_k = [&](int t, int kpage) {
        const int run = col >> 2, in = (t * kTileTokens + run * 16) & ((1 << c.page_shift) - 1);
        const uint8_t* k = c.k + (kpage < 0 ? 0 : kpage) * page_bytes + ((int64_t)h * DH << c.page_shift) +
                           (in + (col & 3)) * DH + 16 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < DH / 64; ++j) A.k[i][j] = *(const uintx4*)(k + 4 * i * DH + 64 * j);
      };
      auto load_v = [&](int t, int vpage) {
        const int in = (t * kTileTokens + g * 16) & ((1 << c.page_shift) - 1);
        const int64_t pg = vpage < 0 ? 0 : vpage;
        const uint8_t* v = c.v + pg * page_bytes + ((int64_t)h * DH << c.page_shift) + in * DH + 16 * col;
#pragma unroll
        for (int d = 0; d < DT; ++d) A.v[d] = *(const uintx4*)(v + 256 * d);
        const float2 sc = *(const float2*)(c.scales + 2 * (pg * c.num_kv + h));
        A.sk = sc.x;
        A.sv = sc.y;
        A.page = vpage;
      };

      floatx4 acc[DT];
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] = floatx4{0, 0, 0, 0};
      float ref = kNoScore, sum = 0.f;

      int t = t0 + wave;
      int kp1 = 0, vp1 = 0;                           // the pages of the wave's next tile
      if (t < t1) {
        const int kp = page_at(t, col >> 2), vp = page_at(t, g);
        kp1 = page_at(t + 4, col >> 2);
        vp1 = page_at(t + 4, g);
        load_k(t, kp);
        __builtin_amdgcn_sched_barrier(0);            // (in the loop's order, for its waits)
        load_v(t, vp);
      }
      for (; t < t1; t += 4) {
        const int kp2 = page_at(t + 8, col >> 2), vp2 = page_at(t + 8, g);
        // scores
        floatx4 sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[i] = floatx4{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < DH / 64; ++j) {
            sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(A.k[i][j].x, A.k[i][j].y), q[2 * j], sc[i], 0, 0, 0);
            sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(A.k[i][j].z, A.k[i][j].w), q[2 * j + 1], sc[i], 0, 0, 0);
          }
        }
        if (t + 4 < t1) load_k(t + 4, kp1);
        // tokens that are not there: behind the length, or of an absent page
        const int have = A.page < 0 ? 0 : len - t * kTileTokens - 16 * g;     // of this lane's 16
        if (__any(have < 16)) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[e >> 2][e & 3] = e < have ? sc[e >> 2][e & 3] : -INFINITY;
          uint32_t keep[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            keep[k] = low_bytes(have - 4 * k);
          }
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k) A.v[d][k] &= keep[k];
          if (have <= 0) A.sk = A.sv = 1.f;                                   // (an unwritten page's may be anything)
        }
        const float ck = fmaxf(cq * A.sk, 0x1p-126f), lsv = log2_of(fmaxf(A.sv, kLeastScale));   // (never 0: 0 * -inf, -inf)
        float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
#pragma unroll
        for (int i = 1; i < 4; ++i) top = fmaxf(top, fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3])));
        top = fmaf(top, ck, lsv);
        if (__any(moves_to(top, ref))) {                                      // (each column by its own scores)
          top = rows_max(top);
          const float to = moves_to(top, ref) ? reference_at(top) : ref;
          const float f = exp2_of(ref - to);
          ref = to;
          sum *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d] *= f;
        }
        // weights
        float cw = ck, off = lsv - ref;
        if (__any((fabsf(ref) > kPlainScore) & (ref > kNoScore))) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[e >> 2][e & 3] = fmaf(sc[e >> 2][e & 3], ck, lsv) - ref;
          cw = 1.f;
          off = 0.f;
        }
        float wsum = 0.f;
        half8 w[2], rest[2];                                                  // fp16 numbers, and what they leave out
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float x = exp2_of(fmaf(sc[e >> 2][e & 3], cw, off)), y = exp2_of(fmaf(sc[e >> 2][(e & 3) + 1], cw, off));
          wsum += x + y;
          _Float16 hx = (_Float16)x, hy = (_Float16)y;
          const _Float16 rx = (_Float16)(x - (float)hx), ry = (_Float16)(y - (float)hy);
          if (TWIN && col >= 8) {
            hx = rx;
            hy = ry;
          }
          w[e >> 3][e & 7] = hx;
          w[e >> 3][(e & 7) + 1] = hy;
          rest[e >> 3][e & 7] = rx;
          rest[e >> 3][(e & 7) + 1] = ry;
        }
        sum = fmaf(wsum, exp2_of(-lsv), sum);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const half8 lo = codes8<FMT>(A.v[d].x, A.v[d].y), hi = codes8<FMT>(A.v[d].z, A.v[d].w);
          acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, w[0], acc[d], 0, 0, 0);
          acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, w[1], acc[d], 0, 0, 0);
          if constexpr (!TWIN) {
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, rest[0], acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, rest[1], acc[d], 0, 0, 0);
          }
        }
        if (t + 4 < t1) load_v(t + 4, vp1);
        kp1 = kp2;
        vp1 = vp2;
      }

      // the waves' sums, joined: reference, sum, then acc under the common reference
      sum = rows_sum(sum);
      if (g == 0) {
        s_ref[wave][col] = ref;
        s_sum[wave][col] = sum;
      }
      __syncthreads();
      const float R = fmaxf(fmaxf(s_ref[0][col], s_ref[1][col]), fmaxf(s_ref[2][col], s_ref[3][col]));
      const float f = exp2_of(ref - R);
#pragma unroll
      for (int d = 0; d < DT; ++d) *(floatx4*)&s_acc[wave][col][16 * d + 4 * g] = acc[d] * f;
      __syncthreads();
      const bool whole = t0 == 0 && t1 == T;
      float* part_out = partials + (2 * (int64_t)blockIdx.x + (t0 == 0)) * partial8_floats(L.gqa, DH);
      for (int i = threadIdx.x; i < cols * DH; i += 256) {
        const int cc = i / DH, d = i % DH;
        float o = s_acc[0][cc][d] + s_acc[1][cc][d] + s_acc[2][cc][d] + s_acc[3][cc][d];
        if constexpr (TWIN) o += s_acc[0][cc + 8][d] + s_acc[1][cc + 8][d] + s_acc[2][cc + 8][d] + s_acc[3][cc + 8][d];
        const float Rc = fmaxf(fmaxf(s_ref[0][cc], s_ref[1][cc]), fmaxf(s_ref[2][cc], s_ref[3][cc]));
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l = fmaf(s_sum[w][cc], exp2_of(s_ref[w][cc] - Rc), l);
        const int64_t at = row * c.num_kv * L.gqa + h * L.gqa + part * 16 + cc;
        if (whole) {
          store1<TYPE>(L.out, at * DH + d, l == 0.f ? 0.f : o / l);
          if (L.lse && d == 0) L.lse[at] = l == 0.f ? -INFINITY : (Rc + log2_of(l)) * 0.693147180559945f;
        } else {
          part_out[32 + cc * DH + d] = o;
          if (d == 0) {
            part_out[cc] = Rc;
            part_out[16 + cc] = l;
          }
        }
      }
      __syncthreads();
      p = first + t1;
    }
    sbase += (int64_t)T * HV;
  }
}

// Joins the partials of each (sequence, kv head) that several workgroups hold,
// and writes the rows of sequences without a token.  WAVES waves per query head
// share its partials: four where there are few pairs and many partials of each
// (one document of 32K tokens, 8 pairs, 64 of each head: 3.9 us, 7.8 with one wave),
// one where there are many pairs of one or two (64 short contexts, 512 pairs: 4.4 us,
// 7.3 with four).
template <int TYPE, int DH, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void cache8_decode_merge_kernel(Cache8AttendLaunch L, const float* partials,
                                                                  const int64_t* base_of) {
  constexpr int DPL = DH / 64;
  __shared__ float s_r[WAVES], s_l[WAVES], s_a[WAVES][DH];
  const Cache8& c = L.c;
  const int heads = c.num_kv * L.gqa, s = blockIdx.x / heads, hq = blockIdx.x % heads;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int h = hq / L.gqa, part = (hq - h * L.gqa) / 16, cc = (hq - h * L.gqa) % 16, parts = head_parts(L.gqa);
  const int64_t per = base_of[0], a = base_of[1 + s], T = (base_of[2 + s] - a) / (c.num_kv * parts);
  const int64_t at = (int64_t)s * heads + hq;
  if (T == 0) {
    for (int d = threadIdx.x; d < DH; d += 64 * WAVES) store1<TYPE>(L.out, at * DH + d, 0.f);
    if (L.lse && threadIdx.x == 0) L.lse[at] = -INFINITY;
    return;
  }
  const int64_t first = a + (int64_t)(h * parts + part) * T, g0 = first / per, g1 = (first + T - 1) / per;
  if (g0 == g1) return;
  const int64_t floats = partial8_floats(L.gqa, DH);
  float R, l, acc[DPL];
  join<DPL, WAVES == 4 ? 16 : 4>(g0 + wave, g1 + 1, WAVES, 16, [&](int64_t g) {
    const float* p = partials + (2 * g + (g == g0)) * floats;
    return Partial{p + cc, p + 32 + cc * DH};
  }, R, l, acc);
  if constexpr (WAVES == 1) {
#pragma unroll
    for (int d = 0; d < DPL; ++d) store1<TYPE>(L.out, at * DH + lane * DPL + d, l == 0.f ? 0.f : acc[d] / l);
    if (L.lse && lane == 0) L.lse[at] = l == 0.f ? -INFINITY : (R + log2_of(l)) * 0.693147180559945f;
  } else {
    if (lane == 0) {
      s_r[wave] = R;
      s_l[wave] = l;
    }
#pragma unroll
    for (int d = 0; d < DPL; ++d) s_a[wave][lane * DPL + d] = acc[d];
    __syncthreads();
    if (threadIdx.x >= DH) return;
    float M = s_r[0], o = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) M = fmaxf(M, s_r[w]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = exp2_of(s_r[w] - M);
      sum = fmaf(s_l[w], f, sum);
      o = fmaf(s_a[w][threadIdx.x], f, o);
    }
    store1<TYPE>(L.out, at * DH + threadIdx.x, sum == 0.f ? 0.f : o / sum);
    if (L.lse && threadIdx.x == 0) L.lse[at] = sum == 0.f ? -INFINITY : (M + log2_of(sum)) * 0.693147180559945f;
  }
}

// ---- prefill -----------------------------------------------------------------
//
// The same sums for many query rows.  A kv head's rows are its gqa heads of each
// token in turn: a workgroup takes 128 or 256 of them, 32 per wave, and walks the tiles
// of 64 tokens that the last of them sees.  Codes become fp16 once per workgroup,
// on their way into LDS (two buffers: the next tile's bytes are on the way while
// this one is multiplied).  S^T = K Q^T as two 32x32 blocks per wave
// (v_mfma_f32_32x32x16_f16), O^T += V^T P^T.  Token 16 x + 8 h + y of a block is
// score row 16 x + 4 h + y for y < 4 and 16 x + 4 h + y + 4 above, so that lane
// (h, row) holds its part of the second product's B operand, and every group of 8
// scores lies in one 16-token run, whose scales are the same for the wave.
// LDS rows are 16-byte chunks, exclusive-or'ed with the row so that the 16 rows
// that a read touches at once lie in different banks.
//
// A weight meets its value as one fp16 number where outputs are bf16, and as two, the
// second for what the first leaves out, where they are fp16.  One number's 2^-11 is an
// eighth of bf16's own step and not seen beside it: 1.627e-3 from the 64-bit
// definition, the plain form 1.623e-3 (8 prompts of 100 to 500 tokens, relative
// norm).  fp16's step is as fine as the weight's: 2.35e-4 with one, the plain form and
// two 2.03e-4.  The second product is matrix work, half as much again: 4 prompts of 1K
// 64.9 us with one, 76.7 with two; 8K in bf16 would take 720 us for 553.
//
// With few row tiles the keys of each are split over workgroups, whose partials a
// second kernel joins.
//
// A bf16 prompt of 8K tokens, 32 heads on 8 of 128: 0.55 TFLOP in 550 to 580 us over
// cards (1.0 to 0.95 PFLOP/s; a library product of 8192^3 has 1.21), the matrix cores
// 47 % and the vector units 55 % busy, 8 vector instructions for each matrix one.  At
// head dim 64 a score has half the products: 14 vector instructions for each matrix
// one, vector units 70 %, matrix cores 34 %.  A wave of 64 rows would halve the LDS reads, but
// sums, scores, queries and weights alone are 288 registers: one wave per SIMD, with
// nothing beside its products.

// A workgroup's shape.  At DH 128 eight waves fill a CU's registers and share its
// tiles: 256 rows; or, where the sequences have 128 rows or fewer on average, 128
// rows by two groups of four waves that take the tiles in turn (a tile's step is
// then a wave's 600 instructions, whatever the rows: four long documents of 28 to 72
// rows a head 85.7 us with all waves on the same tile, 75.4 in turn; in fp16 98.4 and
// 87.3).  At DH 64 four waves, 128 rows, and three workgroups to a CU.
struct PrefillShape {
  int row_shift, groups, turns;         // log2 of a tile's rows, workgroups at once, wave groups that take turns
};
__host__ __device__ __forceinline__ PrefillShape prefill_shape(int64_t num_rows, int num_seqs, int gqa, int dh) {
  if (dh == 64) return {7, 768, 1};
  return num_rows * gqa <= 128 * (int64_t)num_seqs ? PrefillShape{7, 256, 2} : PrefillShape{8, 256, 1};
}
constexpr int kSplitLeast = 4;          // tiles of a split
constexpr int kSplitMost = 64;

__host__ __device__ __forceinline__ int64_t row_tiles(int64_t num_rows, int num_seqs, int gqa, int row_shift) {
  return ((num_rows * gqa) >> row_shift) + num_seqs;
}
// Splits of each row tile: the workgroups at once over the fewest tiles that the
// rows can make (twice as many at most, whose workgroups then take two rounds of
// half the keys; by the most they can make, eight chunks of 64 tokens on 4K ran on
// half of the CUs).  The lengths, which the host does not know, have no part in it: 16
// tokens on 100K take 66 us alone and 1,940 beside 15 prompts of 500, whose rows
// leave the long one a single workgroup per head.
__host__ __device__ __forceinline__ int prefill_splits(int64_t num_rows, int num_seqs, int num_kv, int gqa, PrefillShape p) {
  const int64_t whole = (num_rows * gqa) >> p.row_shift, s = p.groups / ((whole > num_seqs ? whole : num_seqs) * num_kv);
  return (int)(s < 1 ? 1 : (s > kSplitMost ? kSplitMost : s));
}
// floats of one split's partial: reference and sum per row, then acc[rows][DH]
__host__ __device__ __forceinline__ int64_t split_floats(int dh, int row_shift) { return (int64_t)(dh + 2) << row_shift; }

// tokens that a sequence's row of token `last_token` sees, and the splits that
// so many are worth
__device__ __forceinline__ int tile_seen(const Cache8AttendLaunch& L, int len, int n, int last_token) {
  return L.causal ? clampi((int64_t)len - n + last_token + 1, 0, len) : len;
}
__device__ __forceinline__ int splits_of(int seen, int splits) {
  const int most = (seen + kTileTokens - 1) / kTileTokens / kSplitLeast;
  return most < 1 ? 1 : (most < splits ? most : splits);
}

template <int DH>
__device__ __forceinline__ int k_at(int token, int chunk) {        // fp16 elements
  return token * DH + 8 * (DH == 128 ? (chunk ^ (token & 15)) : (chunk ^ ((token >> 1) & 7)));
}
__device__ __forceinline__ int v_at(int d, int chunk) { return d * kTileTokens + 8 * (chunk ^ ((d >> 1) & 7)); }

// N LDS reads that feed M matrix instructions each: kAhead of them in flight
constexpr int kAhead = 6;
template <int N, int M>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
  for (int i = 0; i < N - kAhead; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, kAhead * M, 0);
}

template <int FMT, int TYPE, int DH, int TURNS>
__global__ __launch_bounds__(DH == 128 ? 512 : 256, 2) void cache8_prefill_kernel(Cache8AttendLaunch L, int splits, float* partials) {
  constexpr int KS = DH / 16, DB = DH / 32;                        // k-steps, value blocks
  constexpr int kRowWaves = (DH == 128 ? 8 : 4) / TURNS, kRowTile = 32 * kRowWaves, RS = kRowTile == 256 ? 8 : 7;
  constexpr int NB = 2 * TURNS, HALF = TURNS;                      // tiles in LDS; half of them between two barriers
  constexpr int NR = 2;                                    // tiles on the way
  constexpr bool kRest = TYPE == kFp16;                            // weights as two fp16 numbers (above)
  __shared__ __align__(16) _Float16 s_k[NB][kTileTokens * DH], s_v[NB][kTileTokens * DH];
  __shared__ float s_sk[NB][4], s_lsv[NB][4], s_inv[NB][4];
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, half = lane >> 5;
  // Neighbours take the splits of one row tile, then different heads (unsplit and
  // eight of them: one per XCD and its L2, which the row tiles of a head share; with
  // splits the heads could as well come first: four long documents 75.1 us, 75.4).
  // The longest rows of a sequence come first.
  const uint32_t pair = blockIdx.x / splits;
  const int h = pair % c.num_kv, z = blockIdx.x % splits, gqa = L.gqa;
  const int64_t slot = (gridDim.x / splits - 1 - pair) / c.num_kv;
  const int s = uniform(seq_of_slot(b, slot, gqa, RS, 1));
  int begin, end;
  rows_of(b, s, begin, end);
  begin = uniform(begin);
  const int n = uniform(end) - begin;
  const int64_t r0 = (slot - first_slot(b, s, gqa, RS, 1)) * kRowTile, rows_all = (int64_t)n * gqa;
  if (r0 < 0 || r0 >= rows_all) return;                             // (r0 < 0: row starts that decrease)
  const int len = uniform(seq_tokens(c, b, s));
  const int last = (int)((r0 + kRowTile < rows_all ? r0 + kRowTile : rows_all) - 1);
  const int seen = tile_seen(L, len, n, last / gqa);
  const int parts = splits_of(seen, splits);
  if (z >= parts) return;
  const int NT = (seen + kTileTokens - 1) / kTileTokens;
  const int tbeg = (int)((int64_t)NT * z / parts), tend = (int)((int64_t)NT * (z + 1) / parts);

  // this lane's row
  const int row_wave = wave % kRowWaves, turn = wave / kRowWaves;
  const int64_t r = r0 + row_wave * 32 + col;
  const bool live = r < rows_all;
  const int tok = live ? (int)(r / gqa) : 0, hd = live ? (int)(r - (int64_t)tok * gqa) : 0;
  const int lim = live ? tile_seen(L, len, n, tok) : 0;
  int lim_min = live ? lim : 0x7FFFFFFF, lim_max = lim;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    lim_min = min(lim_min, __shfl_xor(lim_min, m, kWave));
    lim_max = max(lim_max, __shfl_xor(lim_max, m, kWave));
  }
  lim_min = uniform(lim_min);
  lim_max = uniform(lim_max);

  half8 q[KS];
  int back = 0;
  {
    struct __attribute__((packed, aligned(2))) U4 { uintx4 v; };
    const uint16_t* src = (const uint16_t*)L.q + (int64_t)(begin + tok) * L.q_row + (int64_t)(h * gqa + hd) * L.q_head + 8 * half;
    uintx4 raw[KS];                                                 // (a lane without a row takes the first: dropped at the end)
#pragma unroll
    for (int i = 0; i < KS; ++i) raw[i] = ((const U4*)(src + 16 * i))->v;
    query_fp16<TYPE, KS>(raw, [](float m) { return halves_max(m); }, q, back);
  }
  const float cq = ldexpf(L.sm_scale * 1.44269504088896f, back);

  const int32_t* table = b.table + s * b.table_stride;
  // A thread's part of a tile: 16 codes of a key row and 16 of a value row, of a run
  // that is the same for the wave.
  const int run = DH == 128 ? wave >> 1 : wave, in = DH == 128 ? tid & 127 : lane;
  struct Raw {
    uintx4 k, v;
    float2 sc;
    int page;
  } raws[NR];
  int pages[2];
  const int64_t page_bytes = (int64_t)c.num_kv * DH << c.page_shift;
  const uint8_t* kbase = c.k + ((int64_t)h * DH << c.page_shift);
  const uint8_t* vbase = c.v + ((int64_t)h * DH << c.page_shift);
  const float* scbase = c.scales + 2 * h;
  const int ps_mask = (1 << c.page_shift) - 1, last_blk = b.max_blocks - 1;
  // Every step issues the same loads in the same order, so that its waits are for
  // the ones it needs (loads return in order: a tile's pages are looked up before
  // the tile before it is fetched).  Beyond the last tile, and of absent pages, they
  // read page 0, whose tokens are dropped.
  auto find = [&](int t) { return table[min((t * kTileTokens + run * 16) >> c.page_shift, last_blk)]; };
  auto fetch = [&](int t, int found, Raw& raw) {
    const int at = t * kTileTokens + run * 16;
    asm volatile("" : "+v"(found));                                 // (waited for here and no earlier)
    int pg = uniform(found);
    pg = t < tend && at < len && pg < (int)c.num_pages ? pg : -1;
    raw.page = pg;
    const int64_t p = max(pg, 0), base = p * page_bytes + (at & ps_mask) * DH;
    raw.k = *(const uintx4*)(kbase + base + 16 * in);
    raw.v = *(const uintx4*)(vbase + base + 16 * in);
    raw.sc = *(const float2*)(scbase + p * (2 * c.num_kv));
  };
  auto stage = [&](int t, int bf, Raw raw) {
    const int have = raw.page < 0 ? 0 : len - t * kTileTokens - run * 16;   // tokens of the run that are there
    if (have < 16) {
      if (in / (DH / 16) >= have) raw.k = uintx4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 4; ++k) raw.v[k] &= low_bytes(have - 4 * k);
    }
    if (in == 0) {
      const float lsv = have > 0 ? log2_of(fmaxf(raw.sc.y, kLeastScale)) : -INFINITY;
      s_sk[bf][run] = have > 0 ? raw.sc.x : 1.f;
      s_lsv[bf][run] = lsv;
      s_inv[bf][run] = have > 0 ? exp2_of(-lsv) : 0.f;
    }
    const int token = run * 16 + in / (DH / 16), chunk = 2 * (in % (DH / 16));
    *(half8*)&s_k[bf][k_at<DH>(token, chunk)] = codes8<FMT>(raw.k.x, raw.k.y);
    *(half8*)&s_k[bf][k_at<DH>(token, chunk + 1)] = codes8<FMT>(raw.k.z, raw.k.w);
    *(half8*)&s_v[bf][v_at(in, 2 * run)] = codes8<FMT>(raw.v.x, raw.v.y);
    *(half8*)&s_v[bf][v_at(in, 2 * run + 1)] = codes8<FMT>(raw.v.z, raw.v.w);
  };

  floatx16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  float ref = kNoScore, sum = 0.f;
  const int ktok = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);   // token of score row `col`

  // Tile t from LDS buffer bf (a constant), by the waves whose turn it is; then tile
  // t + HALF, whose loads had NR steps, into its own, and the loads of the tile NR
  // later.
  auto step = [&](int t, auto buffer) {
    constexpr int bf = buffer.value, nx = (bf + HALF) % NR, px = nx & 1;
    const int t0 = t * kTileTokens;
    if (t0 < lim_max && t < tend && (TURNS == 1 || turn == bf % TURNS)) {
      floatx16 sc[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[x][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const half8 a = *(const half8*)&s_k[bf][k_at<DH>(32 * x + ktok, 2 * k + half)];
          sc[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q[k], sc[x], 0, 0, 0);
        }
      }
      reads_ahead<2 * KS, 1>();
      if (t0 + kTileTokens > lim_min) {
        const int left = lim - t0 - 8 * half;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          sc[e >> 4][e & 15] = 16 * (e >> 3) + (e & 7) < left ? sc[e >> 4][e & 15] : -INFINITY;
      }
      float ck[4], lsv[4], top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        ck[u] = fmaxf(cq * s_sk[bf][u], 0x1p-126f);                   // (never 0: 0 * -inf)
        lsv[u] = s_lsv[bf][u];
        float m = sc[u >> 1][8 * (u & 1)];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, sc[u >> 1][8 * (u & 1) + i]);
        top = fmaxf(top, fmaf(m, ck[u], lsv[u]));
      }
      if (__any(moves_to(top, ref))) {                                // (each row by its own scores)
        top = halves_max(top);
        const float to = moves_to(top, ref) ? reference_at(top) : ref;
        const float f = exp2_of(ref - to);
        ref = to;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= f;
      }
      float off[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) off[u] = lsv[u] - ref;
      if (__any((fabsf(ref) > kPlainScore) & (ref > kNoScore))) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
          for (int i = 0; i < 8; ++i) sc[u >> 1][8 * (u & 1) + i] = fmaf(sc[u >> 1][8 * (u & 1) + i], ck[u], lsv[u]) - ref;
          ck[u] = 1.f;
          off[u] = 0.f;
        }
      }
      half8 w[4], rest[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float ws = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float x = exp2_of(fmaf(sc[u >> 1][8 * (u & 1) + i], ck[u], off[u]));
          const float y = exp2_of(fmaf(sc[u >> 1][8 * (u & 1) + i + 1], ck[u], off[u]));
          ws += x;
          ws += y;
          const half2v a = fp16_pair(x, y);
          w[u][i] = a[0];
          w[u][i + 1] = a[1];
          if constexpr (kRest) {
            const half2v r = fp16_pair(x - (float)a[0], y - (float)a[1]);
            rest[u][i] = r[0];
            rest[u][i + 1] = r[1];
          }
        }
        sum = fmaf(ws, s_inv[bf][u], sum);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const half8 a = *(const half8*)&s_v[bf][v_at(32 * d + col, 2 * u + half)];
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, w[u], acc[d], 0, 0, 0);
          if constexpr (kRest) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, rest[u], acc[d], 0, 0, 0);
        }
      reads_ahead<4 * DB, kRest ? 2 : 1>();
    }
    stage(t + HALF, (bf + HALF) % NB, raws[nx]);
    __builtin_amdgcn_sched_barrier(0);
    pages[1 - px] = find(t + HALF + NR + 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch(t + HALF + NR, pages[px], raws[nx]);
    __builtin_amdgcn_sched_barrier(0);
    if (bf % HALF == HALF - 1) __syncthreads();
  };
  if (tbeg < tend) {
    pages[0] = find(tbeg);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      pages[(i + 1) & 1] = find(tbeg + i + 1);
      fetch(tbeg + i, pages[i & 1], raws[i]);
    }
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
      stage(tbeg + i, i, raws[i]);
      pages[(NR + i + 1) & 1] = find(tbeg + NR + i + 1);
      fetch(tbeg + NR + i, pages[(NR + i) & 1], raws[i]);
    }
    // (nothing on the way into the loop: its waits are then for its own loads, not
    // for registers that only the loads before it used)
    __builtin_amdgcn_s_waitcnt(0x0F70);                              // vmcnt(0)
    __syncthreads();
    for (int t = tbeg; t < tend; t += NB) {                          // (one exit: every step knows what is on the way)
      step(t, Int<0>{});
      step(t + 1, Int<1>{});
      if constexpr (NB == 4) {
        step(t + 2, Int<2>{});
        step(t + 3, Int<3>{});
      }
    }
  }

  sum = halves_sum(sum);
  if constexpr (TURNS == 2) {                                         // the second group's sums, through LDS, to the first
    float* o = (float*)s_k;                                           // [DH / 4][kRowTile][4]
    float* rs = (float*)s_v;                                          // references, sums
    const int row = row_wave * 32 + col;
    static_assert(sizeof(s_k) >= sizeof(float) * kRowTile * DH && sizeof(s_v) >= sizeof(float) * 2 * kRowTile, "");
    if (turn == 1) {
      if (half == 0) {
        rs[row] = ref;
        rs[kRowTile + row] = sum;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(floatx4*)&o[((8 * d + 2 * i + half) * kRowTile + row) * 4] =
              floatx4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
    }
    __syncthreads();
    if (turn == 1) return;
    const float other = rs[row], R = fmaxf(ref, other), f = exp2_of(ref - R), g = exp2_of(other - R);
    ref = R;
    sum = fmaf(sum, f, rs[kRowTile + row] * g);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const floatx4 x = *(const floatx4*)&o[((8 * d + 2 * i + half) * kRowTile + row) * 4];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[d][4 * i + e] = fmaf(acc[d][4 * i + e], f, x[e] * g);
      }
  }
  if (!live) return;
  const int64_t at = (int64_t)(begin + tok) * c.num_kv * gqa + h * gqa + hd;
  if (parts == 1) {
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        store1<TYPE>(L.out, at * DH + 32 * d + 8 * (i >> 2) + 4 * half + (i & 3), sum == 0.f ? 0.f : acc[d][i] * inv);
    if (L.lse && half == 0) L.lse[at] = sum == 0.f ? -INFINITY : (ref + log2_of(sum)) * 0.693147180559945f;
  } else {
    float* o = partials + ((slot * c.num_kv + h) * splits + z) * split_floats(DH, RS);
    const int row = row_wave * 32 + col;
    if (half == 0) {
      o[row] = ref;
      o[kRowTile + row] = sum;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(floatx4*)&o[2 * kRowTile + row * DH + 32 * d + 8 * i + 4 * half] =
            floatx4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
  }
}

// Joins the splits of each row; one wave per (row, query head).
template <int TYPE, int DH>
__global__ __launch_bounds__(256) void cache8_prefill_merge_kernel(Cache8AttendLaunch L, int RS, int splits,
                                                                   const float* partials) {
  const int kRowTile = 1 << RS;
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  const int heads = c.num_kv * L.gqa, lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), row = at / heads;
  if (row >= b.num_rows) return;
  const int hq = (int)(at - row * heads), h = hq / L.gqa;
  const int s = seq_of_slot(b, row, 1, 0, 0);
  int begin, end;
  rows_of(b, s, begin, end);
  if (row < begin || row >= end) return;
  const int n = end - begin, len = seq_tokens(c, b, s);
  const int64_t r = (row - begin) * L.gqa + hq - h * L.gqa, rows_all = (int64_t)n * L.gqa, r0 = r & ~(int64_t)(kRowTile - 1);
  const int last = (int)((r0 + kRowTile < rows_all ? r0 + kRowTile : rows_all) - 1);
  const int parts = splits_of(tile_seen(L, len, n, last / L.gqa), splits);
  if (parts == 1) return;
  const int64_t slot = first_slot(b, s, L.gqa, RS, 1) + (r >> RS);
  const int in = (int)(r & (kRowTile - 1));
  const float* x = partials + (slot * c.num_kv + h) * splits * split_floats(DH, RS);
  constexpr int DPL = DH / 64;
  float R, l, acc[DPL];
  join<DPL, 16>(0, parts, 1, kRowTile, [&](int64_t z) {
    const float* p = x + z * split_floats(DH, RS);
    return Partial{p + in, p + 2 * kRowTile + in * DH};
  }, R, l, acc);
#pragma unroll
  for (int i = 0; i < DPL; ++i) store1<TYPE>(L.out, at * DH + lane * DPL + i, l == 0.f ? 0.f : acc[i] / l);
  if (L.lse && lane == 0) L.lse[at] = l == 0.f ? -INFINITY : (R + log2_of(l)) * 0.693147180559945f;
}

template <template <int, int, int> class K, class... A>
int pick(int type, int fmt, int dh, A... a) {
#define SPHKV_PICK(T, F, D) if (type == T && fmt == F && dh == D) return K<T, F, D>::go(a...)
  SPHKV_PICK(kFp16, kCache8Int8, 64); SPHKV_PICK(kFp16, kCache8Int8, 128);
  SPHKV_PICK(kFp16, kCache8E4M3, 64); SPHKV_PICK(kFp16, kCache8E4M3, 128);
  SPHKV_PICK(kBf16, kCache8Int8, 64); SPHKV_PICK(kBf16, kCache8Int8, 128);
  SPHKV_PICK(kBf16, kCache8E4M3, 64); SPHKV_PICK(kBf16, kCache8E4M3, 128);
  SPHKV_PICK(kFp32, kCache8Int8, 64); SPHKV_PICK(kFp32, kCache8Int8, 128);
  SPHKV_PICK(kFp32, kCache8E4M3, 64); SPHKV_PICK(kFp32, kCache8E4M3, 128);
#undef SPHKV_PICK
  return -1;
}

// slots of 2^shift rows that cover the batch's rows wherever they start
int64_t row_slots(const Cache8Batch& b, int shift) {
  return b.cu ? (b.num_rows >> shift) + 2 * (int64_t)b.num_seqs : b.num_seqs;
}

template <int T, int F, int D> struct Write {
  static int go(const Cache8RowsLaunch& L, hipStream_t st) {
    const uint32_t items = (uint32_t)(row_slots(L.b, L.c.page_shift) * L.c.num_kv);
    switch (L.c.page_shift) {
      case 4: cache8_write_kernel<T, F, D, 1><<<(items + 3) / 4, 256, 0, st>>>(L, items); break;
      case 5: cache8_write_kernel<T, F, D, 2><<<(items + 1) / 2, 256, 0, st>>>(L, items); break;
      case 6: cache8_write_kernel<T, F, D, 4><<<items, 256, 0, st>>>(L, items); break;
      default: cache8_write_kernel<T, F, D, 8><<<items, 512, 0, st>>>(L, items);
    }
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
  }
};
template <int T, int F, int D> struct Read {
  static int go(const Cache8RowsLaunch& L, hipStream_t st) {
    const uint32_t items = (uint32_t)(row_slots(L.b, 4) * L.c.num_kv);
    cache8_read_kernel<T, F, D><<<(items + 3) / 4, 256, 0, st>>>(L, items);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
  }
};
template <int T, int F, int D> struct Decode {
  static int go(const Cache8AttendLaunch& L, hipStream_t st) {
    if constexpr (T == kFp32) {
      return -1;
    } else {
      int64_t* plan = (int64_t*)L.ws;
      float* partials = (float*)((uint8_t*)L.ws + plan_bytes(L.b.num_seqs));
      if (L.gqa <= 8) cache8_decode_kernel<F, T, D, true><<<decode_groups(D), 256, 0, st>>>(L, partials, plan);
      else cache8_decode_kernel<F, T, D, false><<<decode_groups(D), 256, 0, st>>>(L, partials, plan);
      const int heads = L.b.num_seqs * L.c.num_kv * L.gqa;
      if (L.b.num_seqs * L.c.num_kv * head_parts(L.gqa) < 128)
        cache8_decode_merge_kernel<T, D, 4><<<heads, 256, 0, st>>>(L, partials, plan);
      else
        cache8_decode_merge_kernel<T, D, 1><<<heads, 64, 0, st>>>(L, partials, plan);
      return hipPeekAtLastError() == hipSuccess ? 0 : -1;
    }
  }
};

template <int T, int F, int D> struct Prefill {
  static int go(const Cache8AttendLaunch& L, hipStream_t st) {
    if constexpr (T == kFp32) {
      return -1;
    } else {
      const PrefillShape shape = prefill_shape(L.b.num_rows, L.b.num_seqs, L.gqa, D);
      const int64_t tiles = row_tiles(L.b.num_rows, L.b.num_seqs, L.gqa, shape.row_shift);
      const int splits = prefill_splits(L.b.num_rows, L.b.num_seqs, L.c.num_kv, L.gqa, shape);
      const unsigned grid = (unsigned)(tiles * L.c.num_kv * splits);
      if constexpr (D == 128) {
        if (shape.turns == 2) cache8_prefill_kernel<F, T, D, 2><<<grid, 512, 0, st>>>(L, splits, (float*)L.ws);
        else cache8_prefill_kernel<F, T, D, 1><<<grid, 512, 0, st>>>(L, splits, (float*)L.ws);
      } else {
        cache8_prefill_kernel<F, T, D, 1><<<grid, 256, 0, st>>>(L, splits, (float*)L.ws);
      }
      if (splits > 1) {
        const int64_t waves = L.b.num_rows * L.c.num_kv * L.gqa;
        cache8_prefill_merge_kernel<T, D><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(L, shape.row_shift, splits, (const float*)L.ws);
      }
      return hipPeekAtLastError() == hipSuccess ? 0 : -1;
    }
  }
};

}  // namespace

int launch_cache8_write(const Cache8RowsLaunch& L, hipStream_t stream) {
  return pick<Write>(L.type, L.c.fmt, L.c.dh, L, stream);
}
int launch_cache8_read(const Cache8RowsLaunch& L, hipStream_t stream) {
  return pick<Read>(L.type, L.c.fmt, L.c.dh, L, stream);
}
int launch_cache8_attend(const Cache8AttendLaunch& L, hipStream_t stream) {
  return L.b.cu ? pick<Prefill>(L.type, L.c.fmt, L.c.dh, L, stream) : pick<Decode>(L.type, L.c.fmt, L.c.dh, L, stream);
}
int64_t cache8_decode_ws_bytes(int32_t num_seqs, int32_t, int32_t gqa, int32_t dh) {
  return plan_bytes(num_seqs) + 2 * decode_groups(dh) * 4 * partial8_floats(gqa, dh);
}
int64_t cache8_prefill_ws_bytes(int64_t num_rows, int32_t num_seqs, int32_t num_kv, int32_t gqa, int32_t dh) {
  if (num_rows == 0 || num_seqs == 0) return 0;
  const PrefillShape p = prefill_shape(num_rows, num_seqs, gqa, dh);
  const int splits = prefill_splits(num_rows, num_seqs, num_kv, gqa, p);
  return splits == 1 ? 0 : row_tiles(num_rows, num_seqs, gqa, p.row_shift) * num_kv * splits * split_floats(dh, p.row_shift) * 4;
}

}  // namespace sphkv
