// The 8-bit KV cache: write, read back and attention (include/sphkv.h, "8-bit
// KV cache").  No reference counterpart: the reference keeps angle codes and
// fp16 values.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include "sphkv_common.h"
#include "sphkv_internal.h"

namespace sphkv {
namespace {

constexpr float kLeastScale = 0x1p-60f, kMostScale = 0x1p60f;

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

// the page of block blk of sequence s, or -1
__device__ __forceinline__ int page_of(const Cache8& c, const Cache8Batch& b, int s, int64_t blk) {
  if (blk < 0 || blk >= b.max_blocks) return -1;
  const int p = b.table[s * b.table_stride + blk];
  return p >= 0 && p < c.num_pages ? p : -1;
}

template <int TYPE>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (TYPE == kFp16) return (float)((const _Float16*)p)[i];
  if constexpr (TYPE == kBf16) return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)p)[i] << 16);
  return ((const float*)p)[i];
}

template <int TYPE>
__device__ __forceinline__ void store1(void* p, int64_t i, float x) {
  if constexpr (TYPE == kFp16) ((_Float16*)p)[i] = (_Float16)x;
  else if constexpr (TYPE == kBf16) ((__bf16*)p)[i] = (__bf16)x;
  else ((float*)p)[i] = x;
}

template <int FMT>
__device__ __forceinline__ float decode1(uint8_t c) {
  if constexpr (FMT == kCache8Int8) return (float)(int8_t)c;
  return __builtin_amdgcn_cvt_f32_fp8(c, 0);
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
__device__ __forceinline__ uint8_t code_of(float x, float s, float inv) {
  if (!(x == x)) return 0;
  if constexpr (FMT == kCache8Int8) {
    float r = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
    const float d = fmaf(-r, s, x), h = 0.5f * s;
    if (fabsf(d) > h || (fabsf(d) == h && ((int)r & 1))) r += d > 0.f ? 1.f : -1.f;
    return (uint8_t)(int)fminf(fmaxf(r, -127.f), 127.f);
  }
  const float y = fminf(fmaxf(x * inv, -448.f), 448.f);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
}

// A code of scale s as a code of scale t > s (both exact in 64 bits).
template <int FMT>
__device__ __forceinline__ uint8_t recode(uint8_t c, float s, float t) {
  const double y = (double)decode1<FMT>(c) * s / t;
  if constexpr (FMT == kCache8Int8) return (uint8_t)(int)fmin(fmax(rint(y), -127.), 127.);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32((float)y, (float)y, 0, false);
}

__device__ __forceinline__ float wave_max(float x) {
  for (int m = 1; m < kWave; m <<= 1) x = fmaxf(x, shfl_xor(x, m));
  return x;
}

// One wave per (touched page, kv head).
template <int TYPE, int FMT, int DH>
__global__ __launch_bounds__(256) void cache8_write_kernel(Cache8RowsLaunch L, int64_t slots) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  if (w >= slots * c.num_kv) return;
  const int64_t j = w / c.num_kv;
  const int h = (int)(w - j * c.num_kv), ps = 1 << c.page_shift;
  int s, begin, end;
  int64_t jj = 0;
  if (b.cu) {
    s = seq_of_slot(b, j, 1, c.page_shift, 2);
    jj = j - first_slot(b, s, 1, c.page_shift, 2);
  } else {
    s = (int)j;
  }
  rows_of(b, s, begin, end);
  const int64_t start = b.at[s];
  if (start < 0) return;
  const int64_t blk = (start >> c.page_shift) + jj, pos0 = blk << c.page_shift;
  const int o = jj ? 0 : (int)(start & (ps - 1));                     // first new slot of the page
  const int64_t left = start + (end - begin) - pos0;
  const int e = left < ps ? (int)left : ps;                           // one past the last
  const int page = page_of(c, b, s, blk);
  if (page < 0 || o >= e) return;
  const int64_t row0 = begin + (pos0 + o - start);                    // row of slot o
  const int64_t ph = (int64_t)page * c.num_kv + h;
  uint8_t* kc = c.k + ph * ps * DH;
  uint8_t* vc = c.v + ph * ps * DH;
  for (int which = 0; which < 2; ++which) {
    const void* x = which ? L.v : L.k;
    const int64_t rs = which ? L.v_row : L.k_row, at = h * (which ? L.v_head : L.k_head);
    float a = 0.f;
    for (int t = o; t < e; ++t)
      for (int d = lane; d < DH; d += 64) {
        const float y = fabsf(load1<TYPE>(x, (row0 + t - o) * rs + at + d));
        if (y < INFINITY) a = fmaxf(a, y);
      }
    a = wave_max(a);
    const float old = c.scales[2 * ph + which];
    float sc = block_scale<FMT>(a);
    if (o > 0 && !(sc > old)) sc = old;
    const float inv = __fdiv_rn(1.0f, sc);
    if (o > 0 && sc > old)
      for (int t = 0; t < o; ++t)
        for (int d = lane; d < DH; d += 64) {
          uint8_t* p = which ? vc + (t >> 4) * 16 * DH + d * 16 + (t & 15) : kc + t * DH + d;
          *p = recode<FMT>(*p, old, sc);
        }
    for (int t = o; t < e; ++t)
      for (int d = lane; d < DH; d += 64) {
        uint8_t* p = which ? vc + (t >> 4) * 16 * DH + d * 16 + (t & 15) : kc + t * DH + d;
        *p = code_of<FMT>(load1<TYPE>(x, (row0 + t - o) * rs + at + d), sc, inv);
      }
    if (lane == 0) c.scales[2 * ph + which] = sc;
  }
}

// One wave per (16-token run, kv head).
template <int TYPE, int FMT, int DH>
__global__ __launch_bounds__(256) void cache8_read_kernel(Cache8RowsLaunch L, int64_t slots) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  if (w >= slots * c.num_kv) return;
  const int64_t j = w / c.num_kv;
  const int h = (int)(w - j * c.num_kv), ps = 1 << c.page_shift;
  int s, begin, end;
  int64_t jj = 0;
  if (b.cu) {
    s = seq_of_slot(b, j, 1, 4, 2);
    jj = j - first_slot(b, s, 1, 4, 2);
  } else {
    s = (int)j;
  }
  rows_of(b, s, begin, end);
  const int64_t start = b.at[s], pos0 = ((start >> 4) + jj) << 4;
  const int o = jj ? 0 : (int)(start & 15);
  const int64_t left = start + (end - begin) - pos0;
  const int e = left < 16 ? (int)left : 16;
  if (o >= e) return;
  const int page = page_of(c, b, s, pos0 >> c.page_shift);
  const int64_t ph = (int64_t)page * c.num_kv + h;
  const int run = (int)(pos0 & (ps - 1)) >> 4;
  const uint8_t* kc = c.k + (ph * ps + run * 16) * DH;
  const uint8_t* vc = c.v + (ph * ps + run * 16) * DH;
  const float sk = page < 0 ? 0.f : c.scales[2 * ph], sv = page < 0 ? 0.f : c.scales[2 * ph + 1];
  for (int t = o; t < e; ++t) {
    const int64_t row = begin + (pos0 + t - start);
    for (int d = lane; d < DH; d += 64) {
      if (L.k) store1<TYPE>(L.k, row * L.k_row + h * L.k_head + d, page < 0 ? 0.f : decode1<FMT>(kc[t * DH + d]) * sk);
      if (L.v) store1<TYPE>(L.v, row * L.v_row + h * L.v_head + d, page < 0 ? 0.f : decode1<FMT>(vc[d * 16 + t]) * sv);
    }
  }
}

// One workgroup per (query row, q head), 256 tokens at a time.
template <int TYPE, int FMT, int DH>
__global__ __launch_bounds__(256) void cache8_attend_kernel(Cache8AttendLaunch L) {
  __shared__ float sq[DH], sw[256], red[8], accs[256];
  const Cache8& c = L.c;
  const Cache8Batch& b = L.b;
  const int hq = blockIdx.x, h = hq / L.gqa, tid = threadIdx.x, ps = 1 << c.page_shift;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * 32768;
  if (row >= b.num_rows) return;
  const int s = b.cu ? seq_of_slot(b, row, 1, 0, 0) : (int)row;
  int begin, end;
  rows_of(b, s, begin, end);
  if (row < begin || row >= end) return;
  int n = clampi(b.at[s], 0, (int64_t)b.max_blocks << c.page_shift);      // tokens attended
  if (L.causal) n = clampi((int64_t)n - (end - begin) + (row - begin) + 1, 0, n);
  for (int d = tid; d < DH; d += 256) sq[d] = load1<TYPE>(L.q, row * L.q_row + hq * L.q_head + d);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc = 0.f;
  const int d = tid % DH, part = tid / DH, parts = 256 / DH;
  for (int t0 = 0; t0 < n; t0 += 256) {
    const int t = t0 + tid;
    float x = -INFINITY, sv = 0.f;
    if (t < n) {
      const int page = page_of(c, b, s, t >> c.page_shift);
      if (page >= 0) {
        const int64_t ph = (int64_t)page * c.num_kv + h;
        const uint8_t* kc = c.k + (ph * ps + (t & (ps - 1))) * DH;
        x = 0.f;
        for (int i = 0; i < DH; ++i) x = fmaf(sq[i], decode1<FMT>(kc[i]), x);
        x *= c.scales[2 * ph] * L.sm_scale;
        sv = c.scales[2 * ph + 1];
      }
    }
    float top = wave_max(x);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float M = fmaxf(m, top);
    const float R = M == -INFINITY ? 0.f : M;                         // (a NaN score stays one)
    const float f = expf(m - R), w = expf(x - R);
    l = l * f + w;                                                    // this thread's tokens
    sw[tid] = w * sv;
    m = M;
    __syncthreads();
    acc *= f;
    const int lim = n - t0 < 256 ? n - t0 : 256;
    for (int i = part; i < lim; i += parts) {
      const int page = page_of(c, b, s, (t0 + i) >> c.page_shift);
      if (page < 0) continue;
      const int r = (t0 + i) & (ps - 1);
      acc = fmaf(sw[i], decode1<FMT>(c.v[((int64_t)page * c.num_kv + h) * ps * DH + (r >> 4) * 16 * DH + d * 16 + (r & 15)]), acc);
    }
    __syncthreads();
  }
  for (int k = 1; k < 64; k <<= 1) l += shfl_xor(l, k);
  if ((tid & 63) == 0) red[tid >> 6] = l;
  accs[tid] = acc;
  __syncthreads();
  l = red[0] + red[1] + red[2] + red[3];
  if (tid < DH) {
    float o = 0.f;
    for (int p = 0; p < parts; ++p) o += accs[p * DH + tid];
    const int64_t at = row * c.num_kv * L.gqa + hq;
    store1<TYPE>(L.out, at * DH + tid, l > 0.f ? o / l : (l == 0.f ? 0.f : NAN));
    if (L.lse && tid == 0) L.lse[at] = l == 0.f ? -INFINITY : m + logf(l);
  }
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
    const int64_t slots = row_slots(L.b, L.c.page_shift), waves = slots * L.c.num_kv;
    cache8_write_kernel<T, F, D><<<dim3((unsigned)((waves + 3) / 4)), 256, 0, st>>>(L, slots);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
  }
};
template <int T, int F, int D> struct Read {
  static int go(const Cache8RowsLaunch& L, hipStream_t st) {
    const int64_t slots = row_slots(L.b, 4), waves = slots * L.c.num_kv;
    cache8_read_kernel<T, F, D><<<dim3((unsigned)((waves + 3) / 4)), 256, 0, st>>>(L, slots);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
  }
};
template <int T, int F, int D> struct Attend {
  static int go(const Cache8AttendLaunch& L, hipStream_t st) {
    const int64_t rows = L.b.num_rows;
    const dim3 grid(L.c.num_kv * L.gqa, (unsigned)(rows < 32768 ? rows : 32768), (unsigned)((rows + 32767) / 32768));
    if constexpr (T == kFp32) return -1;
    else cache8_attend_kernel<T, F, D><<<grid, 256, 0, st>>>(L);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
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
  return pick<Attend>(L.type, L.c.fmt, L.c.dh, L, stream);
}
int64_t cache8_decode_ws_bytes(int32_t, int32_t, int32_t, int32_t) { return 0; }
int64_t cache8_prefill_ws_bytes(int64_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

}  // namespace sphkv
