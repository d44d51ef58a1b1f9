// The 16-bit KV cache: append with rotation, attention and differential
// attention (include/sphkv.h, "16-bit KV cache").  No reference counterpart.
#include <hip/hip_runtime.h>

#include "sphkv_attend.h"

namespace sphkv {
namespace {

typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

// eight 16-bit numbers (four dwords) of a lane as a matrix operand
template <int TYPE>
__device__ __forceinline__ floatx4 mfma16(uintx4 a, uintx4 b, floatx4 c) {
  if constexpr (TYPE == kFp16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int TYPE>
__device__ __forceinline__ floatx16 mfma32(uintx4 a, uintx4 b, floatx16 c) {
  if constexpr (TYPE == kFp16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two numbers, half to even, and the numbers that a pair stands for
template <int TYPE>
__device__ __forceinline__ uint32_t pair_of(float x, float y) {
  if constexpr (TYPE == kFp16) return __builtin_bit_cast(uint32_t, fp16_pair(x, y));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{x, y}, bf16x2));
}
template <int TYPE>
__device__ __forceinline__ float low_of(uint32_t p) {
  if constexpr (TYPE == kFp16) return (float)__builtin_bit_cast(half2v, p)[0];
  else return __builtin_bit_cast(float, p << 16);
}
template <int TYPE>
__device__ __forceinline__ float high_of(uint32_t p) {
  if constexpr (TYPE == kFp16) return (float)__builtin_bit_cast(half2v, p)[1];
  else return __builtin_bit_cast(float, p & 0xFFFF0000u);
}

// the low or the high halves of two dwords
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

__device__ __forceinline__ int seq_tokens(const Cache16& c, const Cache8Batch& b, int s) {
  return clampi(b.at[s], 0, (int64_t)b.max_blocks << c.page_shift);
}

// From this size on a score and the reference are rounded alike before their
// difference is taken (one multiply-add below it), so that the largest weight is
// what the reference says at any magnitude.
constexpr float kPlainScore = 0x1p18f;
__device__ __forceinline__ float score_less(float x, float cq, float ref) {
#pragma clang fp contract(off)                                       // (__fmul_rn and __fsub_rn are contracted)
  const float s = x * cq;
  return s - ref;
}
constexpr float kLog2e = 1.44269504088896f, kLn2 = 0.693147180559945f;

// ---- append --------------------------------------------------------------------
//
// y_j = x_j cos a - x_j' sin a, y_j' = x_j' cos a + x_j sin a, a = p f: HBM-bound (16
// prompts of 500 to 12,000 tokens, 8 kv heads of 4 query heads, dim 128, in fp16: 2.5
// GB in 475 us, 5.3 TB/s), a chain of dependent loads for few tokens (one: 4.5 us).
// A lane owns 16 elements of a head (the two sides of eight pairs, or 16 that
// stay) and keeps them for every head that it takes, so their eight angles are
// formed once per token: the turns p f / 2 pi in 64 bits, less their nearest whole
// number, then sine and cosine in 32.  A wave takes one token; where a call has
// fewer than eight per CU, its heads are spread over waves (one token 4.5 us, by one
// wave 6.9; 256 tokens 6.0 and 8.6).

template <int TYPE>
struct Eight { typename Elem<TYPE>::T x[8]; };

template <int TYPE>
__device__ __forceinline__ Eight<TYPE> load8(const void* p, int64_t at) {
  typedef typename Elem<TYPE>::T E;
  Eight<TYPE> r;
  *(Unaligned<E, 8>*)&r = *(const Unaligned<E, 8>*)((const E*)p + at);
  return r;
}

template <int IN, int OUT, int DH>
__global__ __launch_bounds__(256) void cache16_append_kernel(Cache16AppendLaunch L, uint32_t items, int splits) {
  constexpr int UNITS = DH / 16, HEADS = 64 / UNITS;                  // 16-element units of a head, heads at once
  const Cache16& c = L.c;
  const Cache8Batch& b = L.b;
  const uint32_t item = blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (item >= items) return;
  const int lane = threadIdx.x & 63, unit = lane % UNITS;
  const int64_t row = item / splits;
  const int nq = c.num_kv * L.gqa, heads = nq + 2 * c.num_kv;         // q, k, v heads in a row
  const int first = (item - (uint32_t)row * splits) * HEADS + lane / UNITS, step = splits * HEADS;

  // this lane's elements: o0 .. o0 + 7 and o1 .. o1 + 7, turned (pairs 8 u ..) or not
  const int width = DH / L.parts, per_part = UNITS / L.parts, part = unit / per_part, u = unit - part * per_part;
  const bool turns = u < L.freqs / 8;
  const bool half = turns && !L.interleaved;
  const int o0 = part * width + (half ? 8 * u : 16 * u), o1 = half ? o0 + L.freqs : o0 + 8;

  auto load = [&](int j, Eight<IN>& x, Eight<IN>& y) {
    const bool is_q = j < nq, is_k = j < nq + c.num_kv;
    const void* src = is_q ? L.q : is_k ? L.k : L.v;
    const int64_t at = is_q ? row * L.q_row + j * L.q_head
                     : is_k ? row * L.k_row + (j - nq) * L.k_head : row * L.v_row + (j - nq - c.num_kv) * L.v_head;
    x = load8<IN>(src, at + o0);
    y = load8<IN>(src, at + o1);
  };
  const int s = b.cu ? uniform(seq_of_slot(b, row, 1, 0, 0)) : (int)row;
  int begin, end;
  rows_of(b, s, begin, end);
  if (row < begin || row >= end) return;
  const int64_t start = b.at[s], pos = start + (row - begin), blk = pos >> c.page_shift;
  int page = -1;
  if (start >= 0 && blk < b.max_blocks) {
    page = b.table[s * b.table_stride + blk];
    if (page >= c.num_pages) page = -1;
  }
  const int slot = (int)(pos & ((1 << c.page_shift) - 1));

  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (turns) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double f = L.freq_type == kFp64 ? ((const double*)L.inv_freq)[8 * u + i] : (double)((const float*)L.inv_freq)[8 * u + i];
      double t = (double)pos * (f * 0.15915494309189535);             // 1 / 2 pi
      t -= __builtin_rint(t);
      sincospif(2.0f * (float)t, &sn[i], &cs[i]);
    }
  }
  for (int j = first; j < heads; j += step) {
    Eight<IN> x, y;
    load(j, x, y);
    const bool is_q = j < nq, is_k = j < nq + c.num_kv, turn = turns && is_k;
    uint32_t xo[4], yo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a0 = value_of<IN>(x.x[2 * i]), a1 = value_of<IN>(x.x[2 * i + 1]), b0 = value_of<IN>(y.x[2 * i]), b1 = value_of<IN>(y.x[2 * i + 1]);
      if (turn) {
        if (half) {                                                   // pairs (a0, b0), (a1, b1)
          const float p = a0, q = a1;
          a0 = fmaf(p, cs[2 * i], -(b0 * sn[2 * i]));
          a1 = fmaf(q, cs[2 * i + 1], -(b1 * sn[2 * i + 1]));
          b0 = fmaf(b0, cs[2 * i], p * sn[2 * i]);
          b1 = fmaf(b1, cs[2 * i + 1], q * sn[2 * i + 1]);
        } else {                                                      // pairs (a0, a1), (b0, b1)
          const float p = a0, q = b0;
          a0 = fmaf(p, cs[i], -(a1 * sn[i]));
          a1 = fmaf(a1, cs[i], p * sn[i]);
          b0 = fmaf(q, cs[i + 4], -(b1 * sn[i + 4]));
          b1 = fmaf(b1, cs[i + 4], q * sn[i + 4]);
        }
      }
      xo[i] = pair_of<OUT>(a0, a1);
      yo[i] = pair_of<OUT>(b0, b1);
    }
    if constexpr (IN == OUT) {                                        // numbers that stay keep their bits
      if (!turn) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xo[i] = (uint32_t)x.x[2 * i] | (uint32_t)x.x[2 * i + 1] << 16;
          yo[i] = (uint32_t)y.x[2 * i] | (uint32_t)y.x[2 * i + 1] << 16;
        }
      }
    }
    if (is_q) {
      struct __attribute__((packed, aligned(2))) U4 { uintx4 v; };
      uint16_t* to = (uint16_t*)L.q_out + row * L.o_row + j * L.o_head;
      ((U4*)(to + o0))->v = uintx4{xo[0], xo[1], xo[2], xo[3]};
      ((U4*)(to + o1))->v = uintx4{yo[0], yo[1], yo[2], yo[3]};
    } else if (page >= 0) {
      uint16_t* to = is_k ? c.k + page * c.k_page + (j - nq) * c.k_head + slot * c.k_token
                          : c.v + page * c.v_page + (j - nq - c.num_kv) * c.v_head + slot * c.v_token;
      *(uintx4*)(to + o0) = uintx4{xo[0], xo[1], xo[2], xo[3]};
      *(uintx4*)(to + o1) = uintx4{yo[0], yo[1], yo[2], yo[3]};
    }
  }
}

// ---- an output row ---------------------------------------------------------------
//
// DH / 64 consecutive elements of a lane, of one map (sums x under reference R with
// weights' sum l) or of two.

// The launch's arguments read again, where only the end of a kernel uses them:
// scalar registers are scarce before it.  (They are a kernel's first argument.)
typedef const __attribute__((address_space(4))) Cache16AttendLaunch* LateArgs;
__device__ __forceinline__ LateArgs late_args() {
  LateArgs p = (LateArgs)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

struct RowOut { const float *lambda, *norm_weight; float norm_eps; void* out; float* lse; };
template <class ARGS>
__device__ __forceinline__ RowOut row_out(ARGS p) { return {p->lambda, p->norm_weight, p->norm_eps, p->out, p->lse}; }

template <int DH>
struct RowSum { float x[DH / 64], R, l; };

template <int TYPE, int DH, bool DIFF>
__device__ __forceinline__ void finish_row(const RowOut& L, int64_t at, int head, const RowSum<DH>& a,
                                           const RowSum<DH>& b) {
  constexpr int DPL = DH / 64;
  const int lane = threadIdx.x & 63;
  float y[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) y[i] = a.l == 0.f ? 0.f : a.x[i] / a.l;
  if constexpr (DIFF) {
    const float lam = L.lambda[head];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      y[i] = fmaf(-lam, b.l == 0.f ? 0.f : b.x[i] / b.l, y[i]);
      sq = fmaf(y[i], y[i], sq);
    }
    if (L.norm_weight) {
      const float scale = 1.0f / __builtin_sqrtf(fmaf(wave_sum(sq), 1.0f / DH, L.norm_eps));
#pragma unroll
      for (int i = 0; i < DPL; ++i) y[i] *= scale * L.norm_weight[lane * DPL + i];
      if (a.l == 0.f)                                                 // (no eps: 0 * inf)
#pragma unroll
        for (int i = 0; i < DPL; ++i) y[i] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < DPL; ++i) store1<TYPE>(L.out, at * DH + lane * DPL + i, y[i]);
  if (L.lse && lane == 0) {
    const float e = a.l == 0.f ? -INFINITY : (a.R + log2_of(a.l)) * kLn2;
    if constexpr (DIFF) {
      L.lse[2 * at] = e;
      L.lse[2 * at + 1] = b.l == 0.f ? -INFINITY : (b.R + log2_of(b.l)) * kLn2;
    } else {
      L.lse[at] = e;
    }
  }
}

// ---- decode ------------------------------------------------------------------
//
// out = sum_t w_t v_t / sum_t w_t,  w_t = 2^(s_t - R),  s_t = sm_scale log2(e) <q, k_t>,
// R a reference near the largest s_t.  HBM-bound: every key and value is read once
// (64 contexts of 2K to 32K tokens, 8 kv heads of 8 query heads, dim 128: 4.6 GB in
// 757 us, 6.0 TB/s; below some hundred MB the start, the joins and the merge show:
// 32K tokens of one context, 134 MB, in 30.7 us, 4.4 TB/s, from HBM).
//
// A tile is 32 tokens, one wave's step: S^T = K Q^T as two 16x16 blocks
// (v_mfma_f32_16x16x32), O^T += V^T P^T as DH/16 blocks.  Token 8 g + 4 x + r of a
// tile is row 4 g + r of score block x, so lane (g, column) ends up with the scores
// of tokens 8 g .. 8 g + 7, in order: its part of the second product's B operand
// as they stand.  Its part of the A operand is dim d of the same eight tokens: the
// lane loads DH / 16 consecutive dims of each (16 lanes a whole row), and block j
// takes the j-th of them, paired by v_perm (one per dword), so that row i of block
// j is dim DH / 16 i + j.  Nothing passes through LDS.
//
// A column is a query head, or one of the two maps of a head in differential
// attention, whose scores come from half of the dims each.  A weight meets its value
// as two 16-bit numbers, a product each.  (Up to 8 columns could take the second in
// the idle ones: one product less, and no faster, 116.0 us against 114.7 for 256
// contexts of 100 to 900 tokens, for the products wait for the loads.)
//
// Work: the tiles of all (sequence, kv head) pairs in a row, cut into equal runs,
// one per workgroup; its four waves take the tiles of a pair in turn and join their
// sums in LDS.  A pair that one workgroup holds is written out there; the others
// leave a partial per workgroup (two at most: its first and its last pair) for the
// merge kernel.
constexpr int kDecodeTile = 32, kDecodeWaves = 4;
// Workgroups: as many as run at once by their registers, two per CU at dh 128 and
// three at 64.  (64 contexts of 150 to 2,100 tokens, 8 kv heads of 4 query heads, dh
// 64: 29.8 us with 768, 31.6 with 512, 29.9 with 1,024.  dh 128 in the registers of
// three per CU spills: 32K tokens in 27.7 us, 25.7 with two.)
__host__ __device__ constexpr int decode_groups(int dh) { return dh == 128 ? 512 : 768; }

// columns handled together: a kv head's first 16, next 16, ...
__host__ __device__ __forceinline__ int col_parts(int cols) { return (cols + 15) / 16; }
__host__ __device__ __forceinline__ int part_cols(int cols, int part) { return cols - part * 16 < 16 ? cols - part * 16 : 16; }
// floats of one partial: reference and sum per column, then acc[cols][DH]
__host__ __device__ __forceinline__ int64_t partial_size(int cols, int dh) { return 32 + (int64_t)(cols < 16 ? cols : 16) * dh; }
__host__ __device__ __forceinline__ int64_t plan_size(int num_seqs) { return (16 + 8 * ((int64_t)num_seqs + 1) + 255) / 256 * 256; }

// what a decoding sequence sees: tokens first .. len - 1, in tiles of 32 from tile `tile` on
struct Span { int first, len, tile, tiles; };
__device__ __forceinline__ Span span_of(const Cache16AttendLaunch& L, int len) {
  const int first = L.window > 0 && len > L.window ? len - L.window : 0;
  const int tile = first / kDecodeTile;
  return {first, len, tile, (len + kDecodeTile - 1) / kDecodeTile - tile};
}

// inclusive scan over the wave: within rows of 16, then a row's last to those behind
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t scan32(uint32_t x) {
  x += moved<0x111, 0xF>(x);
  x += moved<0x112, 0xF>(x);
  x += moved<0x114, 0xF>(x);
  x += moved<0x118, 0xF>(x);
  x += moved<0x142, 0xA>(x);
  x += moved<0x143, 0xC>(x);
  return x;
}

template <int TYPE, int DH, bool DIFF>
__global__ __launch_bounds__(256, 2) void cache16_decode_kernel(Cache16AttendLaunch L, float* partials, int64_t* base_of) {
  constexpr int KS = DH / 32, VD = DH / 16, DPL = DH / 64;          // k-steps; dims of a lane's value rows; of its output
  constexpr int MAPS = DIFF ? 2 : 1, KM = KS / MAPS;
  __shared__ float s_ref[4][16], s_sum[4][16];
  __shared__ float s_acc[4][16][DH + 4];
  const Cache16& c = L.c;
  const Cache8Batch& b = L.b;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int columns = L.gqa * MAPS, parts = col_parts(columns), HV = c.num_kv * parts, n = b.num_seqs;

  // This workgroup's tiles.  The first 64 sequences' lengths stay with the lanes (the
  // tiles of 64 are at most 2^31).
  auto tiles_of_lane = [&](int len) { return (uint32_t)span_of(L, len).tiles; };
  const int len0 = lane < n ? seq_tokens(c, b, lane) : 0;
  const uint32_t scan0 = scan32(tiles_of_lane(len0));
  auto last_of = [](uint32_t scan) { return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)scan, 63); };
  int64_t total = last_of(scan0);
  for (int i = kWave + lane; i - lane < n; i += kWave) total += last_of(scan32(i < n ? tiles_of_lane(seq_tokens(c, b, i)) : 0));
  total *= HV;
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
      const uint32_t t = tiles_of_lane(i0 == 0 ? len0 : i < n ? seq_tokens(c, b, i) : 0), scan = i0 == 0 ? scan0 : scan32(t);
      if (writes_plan && i < n) base_of[1 + i] = before + (int64_t)(scan - t) * HV;
      const uint64_t past = __ballot(before + (int64_t)scan * HV > p);
      if (!found && past) {
        const int l = __ffsll((unsigned long long)past) - 1;
        found = true;
        s = i0 + l;
        sbase = before + (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(scan - t), l) * HV;
      }
      before += last_of(scan) * HV;
    }
    if (writes_plan && lane == 0) {
      base_of[0] = per;
      base_of[1 + n] = total;
    }
  }
  const float cq = L.sm_scale * kLog2e;
  const int ps_mask = (1 << c.page_shift) - 1;

  for (; p < pend && s < n; ++s) {
    const Span sp = span_of(L, s < kWave ? __builtin_amdgcn_readlane(len0, s) : seq_tokens(c, b, s));
    const int len = uniform(sp.len), first = uniform(sp.first), tile0 = uniform(sp.tile), T = uniform(sp.tiles);
    if (T == 0) continue;
    const int32_t* table = b.table + s * b.table_stride;
    while (p < pend && p < sbase + (int64_t)T * HV) {
      const int hv = (int)((p - sbase) / T), h = hv / parts, part = hv - h * parts;
      const int cols = part_cols(columns, part);
      const int64_t begin = sbase + (int64_t)hv * T;
      const int t0 = (int)(p - begin), t1 = pend - begin < T ? (int)(pend - begin) : T;

      // page of run `run` (16 tokens) of tile t, or -1
      auto page_at = [&](int t, int run) {
        const int at = (tile0 + t) * kDecodeTile + run * 16, blk = at >> c.page_shift, pg = table[min(blk, b.max_blocks - 1)];
        const int has = (at < len) & (blk < b.max_blocks) & (pg < (int)c.num_pages);   // (no branch around the load)
        return pg | (has - 1);
      };
      // the first tiles' pages, asked for before the queries (a wave without a tile takes
      // the last one's and drops them)
      int t = t0 + wave;
      const int tl = min(t, t1 - 1), kp = page_at(tl, col >> 3), vp = page_at(tl, g >> 1);
      int kp1 = page_at(t + 4, col >> 3), vp1 = page_at(t + 4, g >> 1);        // of the wave's next tile
      // a column's query: dims 32 j + 8 g .. in lane group g
      uintx4 q[KS];
      {
        struct __attribute__((packed, aligned(2))) U4 { uintx4 v; };
        const int mine = part * 16 + (col < cols ? col : 0);                   // (columns over: the first again, dropped at the end)
        const uint16_t* src = (const uint16_t*)L.q + s * L.q_row + (int64_t)(h * L.gqa + mine / MAPS) * L.q_head + 8 * g;
#pragma unroll
        for (int j = 0; j < KS; ++j) q[j] = ((const U4*)(src + 32 * j))->v;
      }

      uintx4 kx[2][KS];                               // block x: token 8 (col >> 2) + 4 x + (col & 3), dims 32 j + 8 g ..
      uint32_t vx[8][VD / 2];                         // token 8 g + e, dims VD col ..
      int vpage;
      const uint16_t* kh = c.k + h * c.k_head + 8 * g;
      const uint16_t* vh = c.v + h * c.v_head + VD * col;
      auto load_k = [&](int t, int page) {
        const int slot = (((tile0 + t) * kDecodeTile + 16 * (col >> 3)) & ps_mask) + 8 * ((col >> 2) & 1) + (col & 3);
        const uint16_t* k = kh + (page < 0 ? 0 : page) * c.k_page + slot * c.k_token;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int j = 0; j < KS; ++j) kx[x][j] = *(const uintx4*)(k + 4 * x * c.k_token + 32 * j);
      };
      auto load_v = [&](int t, int page) {
        const int slot = (((tile0 + t) * kDecodeTile + 16 * (g >> 1)) & ps_mask) + 8 * (g & 1);
        const uint16_t* v = vh + (page < 0 ? 0 : page) * c.v_page + slot * c.v_token;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (VD == 8) {
            const uintx4 x = *(const uintx4*)(v + e * c.v_token);
#pragma unroll
            for (int i = 0; i < 4; ++i) vx[e][i] = x[i];
          } else {
            const uintx2 x = *(const uintx2*)(v + e * c.v_token);
            vx[e][0] = x[0];
            vx[e][1] = x[1];
          }
        }
        vpage = page;
      };

      floatx4 acc[VD];
#pragma unroll
      for (int d = 0; d < VD; ++d) acc[d] = floatx4{0, 0, 0, 0};
      float ref = kNoScore, sum = 0.f;

      load_k(tl, kp);
      __builtin_amdgcn_sched_barrier(0);              // (in the loop's order, for its waits)
      load_v(tl, vp);
      // (used here, so that their wait is here: a wait at the first product, inside
      // the loop, would in every turn be for the loads of the next tile too)
#pragma unroll
      for (int j = 0; j < KS; ++j) asm volatile("" : "+v"(q[j]));
      // One tile.  The next one's loads are on the way meanwhile, issued without a
      // condition: a path past them would make every wait one for all loads.
      auto step = [&](auto more) {
        constexpr bool kMore = decltype(more)::value != 0;
        int kp2 = 0, vp2 = 0;
        if constexpr (kMore) {
          kp2 = page_at(t + 8, col >> 3);
          vp2 = page_at(t + 8, g >> 1);
        }
        // scores
        floatx4 sc[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          floatx4 m[MAPS];
#pragma unroll
          for (int i = 0; i < MAPS; ++i) {
            m[i] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < KM; ++j) m[i] = mfma16<TYPE>(kx[x][i * KM + j], q[i * KM + j], m[i]);
          }
          sc[x] = m[0];
          if constexpr (DIFF)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[x][r] = col & 1 ? m[MAPS - 1][r] : m[0][r];
        }
        if constexpr (kMore) load_k(t + 4, kp1);
        // tokens that are not there: behind the length, before the window, of an absent page
        const int at = (tile0 + t) * kDecodeTile + 8 * g, have = vpage < 0 ? 0 : len - at, cut = first - at;
        if (__any((have < 8) | (cut > 0))) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool there = e < have && e >= cut;
            sc[e >> 2][e & 3] = there ? sc[e >> 2][e & 3] : -INFINITY;
#pragma unroll
            for (int i = 0; i < VD / 2; ++i) vx[e][i] = there ? vx[e][i] : 0u;
          }
        }
        float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
        top = fmaxf(top, fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3]))) * cq;
        if (__any(moves_to(top, ref))) {                                      // (each column by its own scores)
          top = rows_max(top);
          const float to = moves_to(top, ref) ? reference_at(top) : ref;
          const float f = exp2_of(ref - to);
          ref = to;
          sum *= f;
#pragma unroll
          for (int d = 0; d < VD; ++d) acc[d] *= f;
        }
        // weights
        float cw = cq, off = -ref;
        if (__any((fabsf(ref) > kPlainScore) & (ref > kNoScore))) {
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[e >> 2][e & 3] = score_less(sc[e >> 2][e & 3], cq, ref);
          cw = 1.f;
          off = 0.f;
        }
        uintx4 w, rest;                                                       // 16-bit numbers, and what they leave out
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float x = exp2_of(fmaf(sc[e >> 2][e & 3], cw, off)), y = exp2_of(fmaf(sc[e >> 2][(e & 3) + 1], cw, off));
          sum += x + y;
          const uint32_t hi = pair_of<TYPE>(x, y), lo = pair_of<TYPE>(x - low_of<TYPE>(hi), y - high_of<TYPE>(hi));
          w[e / 2] = hi;
          rest[e / 2] = lo;
        }
#pragma unroll
        for (int d = 0; d < VD; ++d) {
          uintx4 a;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            a[i] = d & 1 ? highs(vx[2 * i][d / 2], vx[2 * i + 1][d / 2]) : lows(vx[2 * i][d / 2], vx[2 * i + 1][d / 2]);
          acc[d] = mfma16<TYPE>(a, w, acc[d]);
          acc[d] = mfma16<TYPE>(a, rest, acc[d]);
        }
        if constexpr (kMore) load_v(t + 4, vp1);
        kp1 = kp2;
        vp1 = vp2;
      };
      for (; t + 4 < t1; t += 4) step(Int<1>{});
      if (t < t1) step(Int<0>{});

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
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < VD; d += 4)                                       // dims VD (4 g + r) + d ..
          *(floatx4*)&s_acc[wave][col][VD * (4 * g + r) + d] =
              floatx4{acc[d][r] * f, acc[d + 1][r] * f, acc[d + 2][r] * f, acc[d + 3][r] * f};
      __syncthreads();
      const bool whole = t0 == 0 && t1 == T;
      float* part_out = partials + (2 * (int64_t)blockIdx.x + (t0 == 0)) * partial_size(columns, DH);
      auto column = [&](int cc) {
        RowSum<DH> y;
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
          const int d = lane * DPL + i;
          y.x[i] = s_acc[0][cc][d] + s_acc[1][cc][d] + s_acc[2][cc][d] + s_acc[3][cc][d];
        }
        y.R = fmaxf(fmaxf(s_ref[0][cc], s_ref[1][cc]), fmaxf(s_ref[2][cc], s_ref[3][cc]));
        y.l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) y.l = fmaf(s_sum[w][cc], exp2_of(s_ref[w][cc] - y.R), y.l);
        return y;
      };
      if (whole) {
        const RowOut to = row_out(late_args());
        for (int o = wave; o < cols / MAPS; o += kDecodeWaves) {
          const int head = h * L.gqa + part * (16 / MAPS) + o;
          const RowSum<DH> a = column(o * MAPS), bb = DIFF ? column(o * MAPS + MAPS - 1) : a;
          finish_row<TYPE, DH, DIFF>(to, (int64_t)s * c.num_kv * L.gqa + head, head, a, bb);
        }
      } else {
        for (int cc = wave; cc < cols; cc += kDecodeWaves) {
          const RowSum<DH> a = column(cc);
#pragma unroll
          for (int i = 0; i < DPL; ++i) part_out[32 + cc * DH + lane * DPL + i] = a.x[i];
          if (lane == 0) {
            part_out[cc] = a.R;
            part_out[16 + cc] = a.l;
          }
        }
      }
      __syncthreads();
      p = begin + t1;
    }
    sbase += (int64_t)T * HV;
  }
}

// Joins the partials of each (sequence, kv head) that several workgroups hold,
// and writes the rows of sequences without a token.  WAVES waves per query head
// share its partials: four where there are few pairs and many partials of each (8
// pairs of 32K tokens: 25.9 us in all, 34.0 with one), one where there are many pairs
// of one or two (2,048 of 100 to 900 tokens: 115.7 us, 123.4 with four).
template <int TYPE, int DH, bool DIFF, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void cache16_decode_merge_kernel(Cache16AttendLaunch L, const float* partials,
                                                                  const int64_t* base_of) {
  constexpr int DPL = DH / 64, MAPS = DIFF ? 2 : 1;
  __shared__ float s_r[MAPS][WAVES], s_l[MAPS][WAVES], s_a[MAPS][WAVES][DH];
  const Cache16& c = L.c;
  const int heads = c.num_kv * L.gqa, s = blockIdx.x / heads, hq = blockIdx.x % heads;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int columns = L.gqa * MAPS, h = hq / L.gqa, vh = (hq - h * L.gqa) * MAPS, part = vh / 16, cc = vh % 16, parts = col_parts(columns);
  const int64_t per = base_of[0], a = base_of[1 + s], T = (base_of[2 + s] - a) / (c.num_kv * parts);
  const int64_t at = (int64_t)s * heads + hq;
  RowSum<DH> y[2];
  if (T == 0) {
    if (wave != 0) return;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      y[m].l = y[m].R = 0.f;
#pragma unroll
      for (int i = 0; i < DPL; ++i) y[m].x[i] = 0.f;
    }
    finish_row<TYPE, DH, DIFF>(row_out(&L), at, hq, y[0], y[1]);
    return;
  }
  const int64_t first = a + (int64_t)(h * parts + part) * T, g0 = first / per, g1 = (first + T - 1) / per;
  if (g0 == g1) return;
  const int64_t floats = partial_size(columns, DH);
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
    join<DPL, WAVES == 4 ? 16 : 4>(g0 + wave, g1 + 1, WAVES, 16, [&](int64_t g) {
      const float* p = partials + (2 * g + (g == g0)) * floats;
      return Partial{p + cc + m, p + 32 + (cc + m) * DH};
    }, y[m].R, y[m].l, y[m].x);
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      if (lane == 0) {
        s_r[m][wave] = y[m].R;
        s_l[m][wave] = y[m].l;
      }
#pragma unroll
      for (int i = 0; i < DPL; ++i) s_a[m][wave][lane * DPL + i] = y[m].x[i];
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      float M = s_r[m][0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) M = fmaxf(M, s_r[m][w]);
      y[m].R = M;
      y[m].l = 0.f;
#pragma unroll
      for (int i = 0; i < DPL; ++i) y[m].x[i] = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = exp2_of(s_r[m][w] - M);
        y[m].l = fmaf(s_l[m][w], f, y[m].l);
#pragma unroll
        for (int i = 0; i < DPL; ++i) y[m].x[i] = fmaf(s_a[m][w][lane * DPL + i], f, y[m].x[i]);
      }
    }
  }
  finish_row<TYPE, DH, DIFF>(row_out(&L), at, hq, y[0], y[MAPS - 1]);
}

// ---- prefill -----------------------------------------------------------------
//
// The same sums for many query rows.  A kv head's rows are its gqa heads of each
// token in turn: a workgroup takes them in tiles, 32 per wave, and walks the tiles
// of 64 tokens that any of them sees.  A tile's keys and values go from the pages
// straight into LDS (16 bytes a lane), one to four tiles ahead, row by row, the
// 16-byte chunks of a row exclusive-or'ed with the row so that the rows that a read
// touches at once lie in different banks.  S^T = K Q^T as two 32x32 blocks per wave
// (v_mfma_f32_32x32x16), O^T += V^T P^T: lane (h, row) holds scores 8 a + 4 h + r of
// a block, which is its part of the second product's B operand when its part of the
// A operand is the same tokens: two transposing LDS reads (ds_read_b64_tr_b16) of
// four tokens by 16 dims each.
//
// Bound by the matrix cores' rate under load: a prompt of 8,192 tokens, 8 kv heads of
// 4 query heads, dim 128, bf16, in 638 to 660 us, 1.29 to 1.25 PFLOP/s of the products
// below, where a library product of 8192^3 reaches 1.31.  In eight waves of one step
// the weights would alternate with the products; half a step apart, the one half's
// weights run beside the other half's products (with one product a weight 524 us when
// it came, 570 before).
//
// A weight meets its value as two 16-bit numbers, a product each: outputs show one
// number's rounding.  (In bf16 they were 5 % further from 64 bits with one, 1.73e-3
// relative norm for 1.65e-3, nearly all of that their own rounding, and where values
// cancel by 2^-9 of what cancels.  One number took 478 us for that prompt.)
//
// In differential attention the two maps are two groups of waves over the same
// rows, each with its half of the dims, whose sums meet in LDS at the end.
//
// A masked token's weight is 0, but 0 times an infinity or a NaN is not.  Tokens
// behind the length or of an absent page are read as zeros.  In a tile that some
// rows see in part, values that are not finite count as zeros in the product, and
// are added at the end to the outputs of the rows that see them.
constexpr int kTileTokens = 64;
// The reference moves where a weight has passed 2^kMostWeight and a lane's 32 of a
// tile add up to kMostSum or more: with less each is below kMostSum, which fp16 holds.
constexpr float kMostWeight = 10.0f, kMostSum = 0x1p15f;
constexpr float kNearScore = 64.f;

// A workgroup's shape: row waves of 32 rows, and groups of them: the two maps, or,
// where the rows of a sequence are 128 at most on average, two that take its tiles in
// turn, so that eight waves have work.  (dim 128; 4 times 5 to 24 tokens of 4 heads on
// 20K to 32K, fp16: 94.1 us, 130.7 without turns; 64 times 4 tokens on 2K 94.1 and 113.9;
// at 256 rows, 4 times 64 tokens on 16K, 111.6 in turn, 107.3 without.)
struct PrefillShape {
  int row_waves, groups, at_once;       // at_once: workgroups that run at the same time
  __host__ __device__ constexpr int row_shift() const { return row_waves == 8 ? 8 : 7; }
};
__host__ __device__ __forceinline__ PrefillShape prefill_shape(int64_t num_rows, int num_seqs, int gqa, int dh, bool diff) {
  if (diff) return {4, 2, 256};
  if (dh == 64) return {4, 1, 768};
  return num_rows * gqa <= 128 * (int64_t)num_seqs ? PrefillShape{4, 2, 256} : PrefillShape{8, 1, 256};
}
constexpr int kSplitLeast = 4;          // tiles of a split (2 to 8: no difference)
constexpr int kSplitMost = 64;

__host__ __device__ __forceinline__ int64_t row_tiles(int64_t num_rows, int num_seqs, int gqa, int row_shift) {
  return ((num_rows * gqa) >> row_shift) + num_seqs;
}
// Splits of each row tile: the workgroups at once over the fewest tiles that the
// rows can make (twice as many: 100.1 us for those 94.1, 82.6 for 69.5 with 8 times 64
// tokens on 4K).  The lengths, which the host does not know, have no part in it.
__host__ __device__ __forceinline__ int prefill_splits(int64_t num_rows, int num_seqs, int num_kv, int gqa, PrefillShape p) {
  const int64_t whole = (num_rows * gqa) >> p.row_shift(), s = p.at_once / ((whole > num_seqs ? whole : num_seqs) * num_kv);
  return (int)(s < 1 ? 1 : (s > kSplitMost ? kSplitMost : s));
}
// floats of one split's partial: reference and sum per row, then acc[rows][DH];
// the rows of the second map behind those of the first
__host__ __device__ __forceinline__ int64_t split_floats(int dh, int rows) { return (int64_t)(dh + 2) * rows; }

// the tokens [lo, hi) that the row of a sequence's new token `tok` of n sees
struct Sees { int lo, hi; };
__device__ __forceinline__ Sees row_sees(const Cache16AttendLaunch& L, int len, int n, int tok) {
  if (!L.causal) return {0, len};
  const int end = len - n + tok + 1, hi = end < 0 ? 0 : end;         // (at most len)
  return {L.window > 0 && hi > L.window ? hi - L.window : 0, hi};
}
// the tiles [first, first + count) that the rows of tokens a .. b see, and the
// splits that so many are worth
struct Tiles { int first, count; };
__device__ __forceinline__ Tiles tiles_of(const Cache16AttendLaunch& L, int len, int n, int a, int b) {
  const int lo = row_sees(L, len, n, a).lo / kTileTokens, hi = (row_sees(L, len, n, b).hi + kTileTokens - 1) / kTileTokens;
  return {lo, hi > lo ? hi - lo : 0};
}
__device__ __forceinline__ int splits_of(int tiles, int splits) {
  const int most = tiles / kSplitLeast;
  return most < 1 ? 1 : (most < splits ? most : splits);
}

// The row tile that a batch's workgroups take `turn`-th: its sequence, that one's
// rows, length and first slot (as first_slot, one extra), and the tile's number in
// it (none: -1 or past its rows).  A sequence's tiles come last one first, for they
// see most; `ordered`: those of 2 to 8 sequences by the tokens that they see, so
// that the last workgroups are short ones.  (4 prompts of 1,024 tokens 61.2 us,
// sequence by sequence 68.4.  Where all run at once, or with 16 sequences, finding
// the tile costs more than it gives: 8 times 64 rows on 4,096 tokens 73.2 against
// 69.5, 16 sequences of 750 to 5,000 tokens, a window of 2,000, 171.9 against 168.2.)
struct Turn { int s, first, begin, end, len, tile; };
constexpr int kOrdered = 8;
__device__ __forceinline__ Turn turn_of(const Cache16& c, const Cache8Batch& b, int turn, int turns, int gqa, int shift,
                                        bool ordered) {
  const int lane = threadIdx.x & (kWave - 1), n = b.num_seqs;
  int lo = 0, hi = n;
  while (hi - lo > kWave) {                                           // (as seq_of_slot, down to 64)
    const int step = (hi - lo + kWave - 1) / kWave, p = lo + lane * step;
    const bool le = p < hi && first_slot(b, p < hi ? p : lo, gqa, shift, 1) <= turns - 1 - turn;
    const int cnt = __popcll(__ballot(le));
    lo += (cnt > 0 ? cnt - 1 : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  // the sequences that it may be, a lane each, with all that is wanted of the one it is
  const bool mine = lo + lane < hi;
  const int p = mine ? lo + lane : lo, from = b.cu[p], to = b.cu[p + 1], len = seq_tokens(c, b, p);
  const int begin = clampi(from, 0, b.num_rows), end = clampi(to, begin, b.num_rows), first = (begin * gqa >> shift) + p;
  int l, tile;
  if (!ordered || n == 1 || n > kOrdered) {
    // slot by slot, a sequence's last tile first
    const int cnt = __popcll(__ballot(mine && first <= turns - 1 - turn));
    l = cnt > 0 ? cnt - 1 : 0;
    tile = turns - 1 - turn - __builtin_amdgcn_readlane(first, l);
  } else {
    // By the number of tiles' rows up to their own: A .. E - 1 are a sequence's.  `turn`
    // tiles or fewer lie above the one looked for, K: 64 candidates at a time.
    const int before = len - (end - begin);
    const int A = before > 0 ? (int)((int64_t)before * gqa >> shift) : 0;
    const int E = A + (mine ? ((end - begin) * gqa + (1 << shift) - 1) >> shift : 0);
    int K = 0x7FFFFFFF, top = 0;
    for (int i = 0; i < n; ++i) {
      const int a = __builtin_amdgcn_readlane(A, i), e = __builtin_amdgcn_readlane(E, i);
      if (e > a) {
        K = min(K, a);
        top = max(top, e);
      }
    }
    int above = -1;
    while (K < top) {
      const int step = (top - K + kWave - 1) / kWave, at = K + lane * step;
      int sum = 0;                                                    // tiles at `at` or above
      for (int i = 0; i < n; ++i) {
        const int a = __builtin_amdgcn_readlane(A, i), e = __builtin_amdgcn_readlane(E, i);
        sum += max(e - max(at, a), 0);
      }
      const int cnt = __popcll(__ballot(at < top && sum > turn));
      if (cnt == 0) break;                                            // (fewer tiles than turns)
      K += (cnt - 1) * step;
      if (step == 1) {
        above = __builtin_amdgcn_readlane(sum, cnt - 1);
        break;
      }
      top = min(top, K + step);
    }
    uint64_t has = __ballot(A <= K && K < E);
    for (int i = above - __popcll(has); i < turn; ++i) has &= has - 1;
    l = above < 0 ? 0 : __ffsll((unsigned long long)has) - 1;
    tile = above < 0 ? -1 : K - __builtin_amdgcn_readlane(A, l);
  }
  return {lo + l, __builtin_amdgcn_readlane(first, l), __builtin_amdgcn_readlane(begin, l), __builtin_amdgcn_readlane(end, l),
          __builtin_amdgcn_readlane(len, l), tile};
}

// 16 bytes a lane from global memory (`base` uniform) to LDS: lane i's at to + 16 i.
// As an instruction of its own, so that the compiler does not wait for it at the
// next LDS read, which is of another buffer: whoever reads these bytes waits for
// vmcnt first.  (M0 is read one wait state after it is written.)
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(offset), "s"(base), "s"(uniform((int)to)) : "memory", "m0");
}

typedef short short4v __attribute__((ext_vector_type(4)));
// column i of four rows of 16 numbers, for lane i of 16; lane i points to row i / 4, column 4 (i & 3)
__device__ __forceinline__ uintx2 read_columns(const uint16_t* p) {
  return __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p));
}

// the numbers of a pair that are finite, zeros in the place of others
template <int TYPE>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t p) {
  constexpr uint32_t kExponent = TYPE == kFp16 ? 0x7C00u : 0x7F80u;
  uint32_t keep = 0;
  if ((p & kExponent) != kExponent) keep |= 0xFFFFu;
  if ((p & kExponent << 16) != kExponent << 16) keep |= 0xFFFF0000u;
  return p & keep;
}

// N groups of R LDS reads that feed M matrix instructions each: AHEAD groups in flight
template <int N, int R, int M, int AHEAD>
__device__ __forceinline__ void groups_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * R, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * M, 0);
}

template <int TYPE, int DH, int ROW_WAVES, int GROUPS, bool DIFF>
__global__ __launch_bounds__(64 * ROW_WAVES * GROUPS, 2) void cache16_prefill_kernel(Cache16AttendLaunch L, int turns, int splits,
                                                                                       float* partials) {
  constexpr int KS = DH / 16, DB = DH / 32, KM = DIFF ? KS / 2 : KS;  // k-steps, value blocks, k-steps of a map
  constexpr int WAVES = ROW_WAVES * GROUPS, kRowTile = 32 * ROW_WAVES, RS = ROW_WAVES == 8 ? 8 : 7;
  constexpr bool kTurns = GROUPS == 2 && !DIFF;
  constexpr int STEP = kTurns ? 2 : 1;                                // tiles of a step
  constexpr bool kPing = WAVES == 8 && !kTurns;                       // two halves of the waves, half a step apart
  constexpr int NB = kPing ? 4 : 2;                                   // steps in LDS
  constexpr int CH = DH / 8, RPL = 64 / CH, TOK = kTileTokens / WAVES * STEP, NL = TOK / RPL;   // chunks of a row; rows a copy;
                                                                      // a wave's tokens of a step and copies of each kind
  __shared__ __align__(16) uint16_t s_k[NB][STEP][kTileTokens * DH], s_v[NB][STEP][kTileTokens * DH];
  __shared__ int s_odd;                                               // a value of a cleaned tile was not finite
  const Cache16& c = L.c;
  const Cache8Batch& b = L.b;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, half = lane >> 5;
  // Neighbours take the splits of one row tile, then different heads (unsplit and
  // eight of them: one per XCD and its L2, which the row tiles of a head share).  The
  // rows that see most come first.
  // (The rows of a call times gqa are fewer than 2^30.)
  const uint32_t pair = splits == 1 ? blockIdx.x : blockIdx.x / (uint32_t)splits, z = blockIdx.x - pair * splits;
  const uint32_t turn = pair / (uint32_t)c.num_kv;
  const int h = pair - turn * c.num_kv, gqa = L.gqa;
  if (tid == 0) s_odd = 0;
  const Turn of = turn_of(c, b, turn, turns, gqa, RS, splits == 1 && L.causal);
  const int s = of.s, begin = of.begin, n = of.end - of.begin, len = of.len, slot = of.first + of.tile;
  const int r0 = of.tile * kRowTile, rows_all = n * gqa;
  if (r0 < 0 || r0 >= rows_all) return;
  const int last = (r0 + kRowTile < rows_all ? r0 + kRowTile : rows_all) - 1;
  const int first_tok = (uint32_t)r0 / (uint32_t)gqa, last_tok = (uint32_t)last / (uint32_t)gqa;
  const Tiles tiles = tiles_of(L, len, n, first_tok, last_tok);
  const int parts = splits_of(tiles.count, splits);
  if ((int)z >= parts) return;
  int tbeg = tiles.first, tend = tiles.first + tiles.count;
  if (parts > 1) {                                                  // (a count is at most 2^24, parts 64)
    tend = tiles.first + (uint32_t)(tiles.count * (z + 1)) / (uint32_t)parts;
    tbeg = tiles.first + (uint32_t)(tiles.count * z) / (uint32_t)parts;
  }

  // this lane's row
  const int row_wave = wave % ROW_WAVES, group = wave / ROW_WAVES;
  const int r = r0 + row_wave * 32 + col;
  const bool live = r < rows_all;
  const int tok = live ? (int)((uint32_t)r / (uint32_t)gqa) : 0, hd = live ? r - tok * gqa : 0;
  const Sees sees = row_sees(L, len, n, tok);
  const int lo = live ? sees.lo : 0, lim = live ? sees.hi : 0;
  // Tiles that no row of the wave sees, and tiles that all of them see whole: by its
  // first and last row, for both ends grow with the row.
  const int rows_wave = rows_all - r0 - row_wave * 32, end_row = (rows_wave < 32 ? rows_wave : 32) - 1;
  int lim_min = 0x7FFFFFFF, lim_max = 0, lo_min = 0x7FFFFFFF, lo_max = 0;
  if (end_row >= 0) {
    lim_min = __builtin_amdgcn_readlane(lim, 0);
    lo_min = __builtin_amdgcn_readlane(lo, 0);
    lim_max = __builtin_amdgcn_readlane(lim, end_row);
    lo_max = __builtin_amdgcn_readlane(lo, end_row);
  }

  // The pages of the first 64 tiles are asked for before the queries, and used before
  // the queries are.
  const int32_t* table = b.table + s * b.table_stride;
  const int last_blk = b.max_blocks - 1;
  int ids[4] = {0, 0, 0, 0};
  auto ask = [&](int t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) ids[r] = table[min((t * kTileTokens + 16 * r) >> c.page_shift, last_blk)];
  };
  if (tbeg < tend) ask(tbeg + lane);
  __builtin_amdgcn_sched_barrier(0);

  uintx4 q[KM];
  const int dim0 = DIFF ? group * (DH / 2) : 0;                     // first dim of this wave's map
  {
    struct __attribute__((packed, aligned(2))) U4 { uintx4 v; };
    const uint16_t* src = (const uint16_t*)L.q + (int64_t)(begin + tok) * L.q_row + (int64_t)(h * gqa + hd) * L.q_head + dim0 + 8 * half;
#pragma unroll
    for (int i = 0; i < KM; ++i) q[i] = ((const U4*)(src + 16 * i))->v;   // (a lane without a row takes the first: dropped at the end)
  }
  const float cq = L.sm_scale * kLog2e;

  // A wave's part of a step's tiles: TOK tokens in copies of RPL rows, all of one
  // run of 16 tokens, whose page is the same for the wave.
  const uint16_t* kh = c.k + h * c.k_head;
  const uint16_t* vh = c.v + h * c.v_head;
  const int ps_mask = (1 << c.page_shift) - 1;
  const int ctile = STEP == 2 ? (wave * TOK) / kTileTokens : 0, ctok = (wave * TOK) % kTileTokens;   // of its copies
  // Bytes of this lane from a copy's first token: its token's, and its chunk's, which
  // the first token's number turns too (tokens and chunks are exclusive-or'ed bit by bit).
  const int ltok = lane / CH, lch = lane % CH;
  auto k_swizzle = [](int t) { return DH == 128 ? t & 15 : (t >> 1) & 7; };
  auto v_swizzle = [](int t) { return DH == 128 ? (t & 3) << 2 : (t & 2) << 1; };
  const uint32_t ktok = 2 * ltok * c.k_token, kchunk = 16 * (lch ^ k_swizzle(ltok));
  const uint32_t vtok = 2 * ltok * c.v_token + 16 * (lch ^ v_swizzle(ltok));
  // This wave's copies, of run crun of a tile: offsets of a lane, then of the tile.
  const int crun = ctok / 16;
  uint32_t koff[NL], voff[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    koff[i] = ktok + 2 * i * RPL * c.k_token + (kchunk ^ 16 * k_swizzle((ctok & 15) + i * RPL));
    voff[i] = vtok + 2 * i * RPL * c.v_token;
  }
  constexpr int kTileBytes = 2 * kTileTokens * DH;
  const uint32_t k_lds = lds_address(s_k), v_lds = lds_address(s_v);
  auto copy_one = [&](const uint16_t* from, const uint32_t (&off)[NL], uint32_t tile, int i) {
    copy_to_lds(from, off[i], tile + 2 * (ctok + i * RPL) * DH);
  };
  auto copy = [&](const uint16_t* from, const uint32_t (&off)[NL], uint32_t tile) {
#pragma unroll
    for (int i = 0; i < NL; ++i) copy_one(from, off, tile, i);
  };
  static_assert(RPL % 4 == 0, "the values' chunks turn by a token's low bits");

  floatx16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  float ref = 0.f, sum = 0.f;                                       // the reference in units of <q, k>
  // LDS bytes: key row col, chunk 2 k + half of the map; value row 4 half + (lane & 15) / 4
  // and its 4 columns.  A step forms the others from these by exclusive or.
  int kat = 2 * (col * DH + 8 * ((dim0 / 8 + half) ^ k_swizzle(col)));
  int vat = 2 * ((4 * half + ((lane & 15) >> 2)) * DH + 4 * (lane & 1) +
                 8 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_swizzle((lane & 15) >> 2)));
  auto k_at = [&](const uint16_t* tile, int x, int k) {
    return *(const uintx4*)((const char*)tile + (kat ^ 32 * k) + 64 * x * DH);
  };
  auto v_at = [&](const uint16_t* tile, int u, int d) {
    const char* p = (const char*)tile + (vat ^ 64 * d) + 32 * u * DH;
    const uintx2 x = read_columns((const uint16_t*)p), y = read_columns((const uint16_t*)(p + 16 * DH));
    return uintx4{x[0], x[1], y[0], y[1]};
  };

  // What the steps need to know of the tiles, 64 at a time, a lane each: where this
  // wave's copies come from, and the tile's cases.  Of an absent page the copies read
  // page 0, behind the length what the page holds.  A tile that some rows of the
  // workgroup see in part, or that is not all there, is cleaned by the waves that
  // copied it, before any reads it: values of tokens that are not there and values
  // that are not finite become zeros.
  enum { kVisible = 16, kCut = 32, kUnclean = 64 };                   // low bits: the runs that have a page
  const int all_lim = row_sees(L, len, n, first_tok).hi, all_lo = row_sees(L, len, n, last_tok).lo;
  int64_t kplace = 0, vplace = 0;                                     // elements
  int cases = 0, batch = 0;                                           // the batch's first tile
  auto cases_of = [&](int t, int& own) {                             // (of the pages in ids)
    int f = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = t * kTileTokens + 16 * r, id = ids[r];
      const bool held = at < len && (uint32_t)id < (uint32_t)c.num_pages;
      f |= held ? 1 << r : 0;
      if (r == crun) own = held ? id : 0;
    }
    const int a = t * kTileTokens, b = a + kTileTokens;
    if (t < tend && a < lim_max && b > lo_min) f |= kVisible;
    if (f % 16 != 15 || b > lim_min || a < lo_max) f |= kCut;
    if (t < tend && (f % 16 != 15 || b > all_lim || a < all_lo)) f |= kUnclean;
    return f;
  };
  auto place = [&](int t) {
    int own = 0;
    batch = t;
    cases = cases_of(t + lane, own);
    const int slot = (((t + lane) * kTileTokens + 16 * crun) & ps_mask) + (ctok & 15);
    kplace = own * c.k_page + (int64_t)slot * c.k_token;
    vplace = own * c.v_page + (int64_t)slot * c.v_token;
  };
  auto look_up = [&](int t) {
    ask(t + lane);
    place(t);
  };
  auto of_tile = [&](int64_t x, int t) {                              // a tile's, from its lane
    const int lo = __builtin_amdgcn_readlane((int)x, t - batch), hi = __builtin_amdgcn_readlane((int)(x >> 32), t - batch);
    return ((int64_t)hi << 32) | (uint32_t)lo;
  };
  auto k_from = [&](int t) { return kh + of_tile(kplace, t); };
  auto v_from = [&](int t) { return vh + of_tile(vplace, t); };
  auto cases_at = [&](int t) { return __builtin_amdgcn_readlane(cases, t - batch); };
  auto clean = [&](int t, int what, uint16_t* vt) {
    const int have = what >> crun & 1 ? len - t * kTileTokens - 16 * crun : 0;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      uintx4* at = (uintx4*)(vt + (ctok + i * RPL) * DH + 8 * lane);
      uintx4 x = *at;
      const bool there = (ctok & 15) + i * RPL + ltok < have;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t y = there ? x[k] : 0u;
        x[k] = finite_or_zero<TYPE>(y);
        bad |= x[k] ^ y;
      }
      *at = x;
    }
    if (__any(bad != 0) && lane == 0) s_odd = 1;
  };

  floatx16 sc[2];
  uintx4 w[4], rest[4];

  auto scores = [&](const uint16_t* kt) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[x][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KM; ++k) sc[x] = mfma32<TYPE>(k_at(kt, x, k), q[k], sc[x]);
    }
  };
  // scores of tile t that do not count
  auto mask = [&](int t, int what) {
    const uint32_t first = t * kTileTokens + 4 * half - lo, width = lim - lo;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t n = what >> u & 1 ? width : 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = 8 * (u & 1) + i;
        sc[u >> 1][e] = first + (16 * u + 8 * (i >> 2) + (i & 3)) < n ? sc[u >> 1][e] : -INFINITY;
      }
    }
  };
  // The tile's weights, 2^kTopWeight at the reference.  Their largest is not looked
  // for where a lane's 32 add up to less than kMostSum.  Otherwise, and at a row's first
  // scores, the reference becomes the row's largest score if that one's weight passes
  // 2^kMostWeight (both halves of a row decide alike).  Every score is a sum from zero,
  // less the reference, so that equal ones weigh the same in any tile and at any
  // magnitude.  Up to exponents of kNearScore the difference is part of the exponent's
  // one multiply-add, whose rounding is at most 2^-19 of a weight there (always apart:
  // an 8K prompt 661 us for 638, differential prompts of 1,000 to 2,000 tokens 198 for
  // 193).
  auto weigh = [&]() {
    float ws = 0.f;
    auto pass = [&](auto exponent) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float x = exp2_of(exponent(sc[u >> 1][8 * (u & 1) + i]));
          const float y = exp2_of(exponent(sc[u >> 1][8 * (u & 1) + i + 1]));
          ws += x;
          ws += y;
          w[u][i / 2] = pair_of<TYPE>(x, y);
          rest[u][i / 2] = pair_of<TYPE>(x - low_of<TYPE>(w[u][i / 2]), y - high_of<TYPE>(w[u][i / 2]));
        }
    };
    auto plain = [&](float x) { return fmaf(x - ref, cq, kTopWeight); };
    const float off = fmaf(-ref, cq, kTopWeight);
    if (__any(fabsf(off) > kNearScore)) pass(plain);
    else pass([&](float x) { return fmaf(x, cq, off); });
    if (__any(!(ws < kMostSum) | (sum == 0.f))) {
      float top = sc[0][0];
#pragma unroll
      for (int e = 1; e < 32; ++e) top = fmaxf(top, sc[e >> 4][e & 15]);
      top = halves_max(top);
      const bool fresh = halves_max(sum) == 0.f, moves = top > -INFINITY && (fresh || fmaf(top - ref, cq, kTopWeight) > kMostWeight);
      const float to = moves ? top : ref, f = fresh ? 1.f : exp2_of((ref - to) * cq);
      ref = to;
      sum *= f;
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[d] *= f;
      ws = 0.f;
      pass(plain);
    }
    sum += ws;
  };
  auto values = [&](const uint16_t* vt) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const uintx4 a = v_at(vt, u, d);
        acc[d] = mfma32<TYPE>(a, w[u], acc[d]);
        acc[d] = mfma32<TYPE>(a, rest[u], acc[d]);
      }
  };
  // Both, in this order: each product with the reads of the one kAheadReads later
  // before it (a SIMD's matrix cores have this wave alone then), and between(j) behind
  // it.  The first reads come before, by read_ahead.
  constexpr int NK = 2 * KM, kProducts = NK + 4 * DB, kAheadReads = 6;
  uintx4 part[kAheadReads + 1];
  auto read_ahead = [&](const uint16_t* kt) {
#pragma unroll
    for (int j = 0; j < kAheadReads; ++j) part[j] = j < NK ? k_at(kt, j / KM, j % KM) : uintx4{0, 0, 0, 0};
  };
  auto products = [&](const uint16_t* kt, const uint16_t* vt, auto&& between) {
    auto read = [&](int j) { return j < NK ? k_at(kt, j / KM, j % KM) : v_at(vt, (j - NK) / DB, (j - NK) % DB); };
#pragma unroll
    for (int j = NK; j < kAheadReads; ++j) part[j] = read(j);
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[0][i] = sc[1][i] = 0.f;
#pragma unroll
    for (int j = 0; j < kProducts; ++j) {
      if (j + kAheadReads < kProducts) part[(j + kAheadReads) % (kAheadReads + 1)] = read(j + kAheadReads);
      const uintx4 x = part[j % (kAheadReads + 1)];
      if (j < NK) {
        sc[j / KM] = mfma32<TYPE>(x, q[j % KM], sc[j / KM]);
      } else {
        const int u = (j - NK) / DB, d = (j - NK) % DB;
        acc[d] = mfma32<TYPE>(x, w[u], acc[d]);
        acc[d] = mfma32<TYPE>(x, rest[u], acc[d]);
      }
      between(j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto barrier = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  if (tbeg < tend) place(tbeg);
#pragma unroll
  for (int i = 0; i < KM; ++i) asm volatile("" : "+v"(q[i]));       // (arrived here, before any copy that a wait would be for too)
  __builtin_amdgcn_s_waitcnt(0xC07F);                               // lgkmcnt(0): s_odd is 0 for every wave
  barrier();

  if constexpr (kPing) {
    // The matrix part of a step (scores of the next tile, values of this one) by one
    // half of the waves while the other half, on the same SIMDs, is at its weights:
    // a barrier ends each part.  Step i's matrix part reads K(i + 1) and V(i), one half
    // of the waves a part after the other, and issues the copies of K(i + 4) and
    // V(i + 3), over what every wave has read by then.  The first keys are read before
    // the barrier that the part starts at; so K(i + 1) and V(i) have to arrive a part
    // earlier than the first half reads them: the first half waits behind its products
    // i - 1, for all but the last two steps' copies (each step issues 2 NL, and nothing
    // else), the second behind its weights i - 1, for all but the last step's.  V(i) is
    // cleaned before the barrier that the first half's products i start at.
    static_assert(NL == 1 || NL == 2, "copies of a step");
    constexpr int kOneStep = 0x0F70 | (2 * NL), kTwoSteps = 0x0F70 | (4 * NL), kPrologue = 0x0F70 | (6 * NL);
    const bool late = wave >= 4;
    int what = 0;                                                   // of the next step's tile
    const uint16_t* from = kh;
    // what step i does beside its products, in parts (a copy takes as long to issue as
    // a product, and the scores' part has less time to spare)
    constexpr int kParts = 3 + 2 * NL;
    auto advance = [&](int i, int part) {
      const int t = tbeg + i;
      if (part == 0) {
        what = cases_at(t + 1);
        asm volatile("" : "+s"(what));                              // (here, not where it is used)
      } else if (part == 1) {
        from = v_from(t + 3);
      } else if (part < 2 + NL) {
        copy_one(from, voff, v_lds + ((i + 3) & 3) * kTileBytes, part - 2);
      } else if (part == 2 + NL) {
        from = k_from(t + 4);
      } else {
        copy_one(from, koff, k_lds + (i & 3) * kTileBytes, part - 3 - NL);
      }
    };
    // cleans this wave's part of V(i)
    auto tidy = [&](int i) {
      if (what & kUnclean) {
        clean(tbeg + i, what, s_v[i & 3][0]);
        __builtin_amdgcn_s_waitcnt(0xC07F);                         // lgkmcnt(0)
      }
    };
    const int count = tend - tbeg;
    if (count > 0) {
      copy(k_from(tbeg), koff, k_lds);
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        copy(v_from(tbeg + i - 1), voff, v_lds + (i - 1) * kTileBytes);
        copy(k_from(tbeg + i), koff, k_lds + i * kTileBytes);
      }
      what = cases_at(tbeg);
      __builtin_amdgcn_s_waitcnt(kPrologue);                        // K(0)
      barrier();
      if (late) {
        __builtin_amdgcn_s_waitcnt(kTwoSteps);
        barrier();
      }
      scores(s_k[0][0]);
      if (!late) __builtin_amdgcn_s_waitcnt(kTwoSteps);
      if (late) tidy(0);
      barrier();
      for (int i = 0; i < count; ++i) {
        // weights
        if (what & kVisible) {
          if (what & kCut) mask(tbeg + i, what);
          weigh();
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) w[u] = rest[u] = uintx4{0, 0, 0, 0};
        }
        asm volatile("" : "+v"(kat), "+v"(vat));                    // (formed anew in every step: registers are dearer)
        read_ahead(s_k[(i + 1) & 3][0]);
        if (!late) tidy(i);
        if (late) __builtin_amdgcn_s_waitcnt(kOneStep);
        barrier();
        // products (of a tile that this wave's rows do not see: others see it in part, it is clean)
        __builtin_amdgcn_s_setprio(1);
        products(s_k[(i + 1) & 3][0], s_v[i & 3][0], [&](int j) {
          constexpr int kFirst = kProducts / 2 - 1, kEvery = (kProducts - kFirst) / kParts;
          static_assert(kEvery >= 1, "every part has a product of its own");
          if (j == 0 && tbeg + i + 4 - batch >= kWave) look_up(tbeg + i + 1);   // (its loads wait for the copies, too)
          if (j >= kFirst && (j - kFirst) % kEvery == 0 && (j - kFirst) / kEvery < kParts) advance(i, (j - kFirst) / kEvery);
        });
        __builtin_amdgcn_s_setprio(0);
        if (!late) __builtin_amdgcn_s_waitcnt(kTwoSteps);
        if (late) tidy(i + 1);
        barrier();
      }
      if (!late) barrier();
      __builtin_amdgcn_s_waitcnt(0x0F70);                           // vmcnt(0): no copy outlives the wave
    }
  } else if (tbeg < tend) {
    const int mine = kTurns ? group : 0;
    copy(k_from(tbeg + ctile), koff, k_lds + ctile * kTileBytes);
    copy(v_from(tbeg + ctile), voff, v_lds + ctile * kTileBytes);
    for (int t = tbeg; t < tend; t += 2 * STEP) {
#pragma unroll
      for (int bf = 0; bf < 2; ++bf) {
        const int tt = t + bf * STEP;
        if (tt < tend) {
          const int what = cases_at(tt + mine), copied = cases_at(tt + ctile);
          // this step's bytes have arrived and are clean, for every wave; the other buffer is read no more
          __builtin_amdgcn_s_waitcnt(0x0F70);                       // vmcnt(0)
          if (copied & kUnclean) clean(tt + ctile, copied, s_v[bf][ctile]);
          __syncthreads();
          if (tt + STEP < tend) {
            if (tt + 2 * STEP - 1 - batch >= kWave) look_up(tt + STEP);
            copy(k_from(tt + STEP + ctile), koff, k_lds + ((1 - bf) * STEP + ctile) * kTileBytes);
            copy(v_from(tt + STEP + ctile), voff, v_lds + ((1 - bf) * STEP + ctile) * kTileBytes);
          }
          if (what & kVisible) {
            asm volatile("" : "+v"(kat), "+v"(vat));                // (formed anew in every step: registers are dearer)
            scores(s_k[bf][mine]);
            groups_ahead<2 * KM, 1, 1, KM < 6 ? KM : 6>();
            if (what & kCut) mask(tt + mine, what);
            weigh();
            values(s_v[bf][mine]);
            groups_ahead<4 * DB, 2, 2, DB < 4 ? DB : 4>();
          }
        }
      }
    }
  }
  // values that are not finite, of the tiles where they count as zeros, on the
  // outputs of the rows that see them
  __syncthreads();
  if (s_odd) {
#pragma unroll 1
    for (int t = tbeg; t < tend; ++t) {
      int own = 0;
      ask(t);
      const int what = uniform(cases_of(t, own));
      if (!(what & kUnclean) || (kTurns && ((t - tbeg) & 1) != group)) continue;
#pragma unroll 1
      for (int token = t * kTileTokens; token < (t + 1) * kTileTokens; ++token) {
        if (!(what >> (token >> 4 & 3) & 1) || token < lo || token >= lim) continue;
        const uint16_t* v = vh + (int64_t)table[token >> c.page_shift] * c.v_page + (token & ps_mask) * c.v_token;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = value_of<TYPE>(v[32 * d + 8 * (i >> 2) + 4 * half + (i & 3)]);
            if (!(fabsf(x) < INFINITY)) acc[d][i] += x;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  const LateArgs late = late_args();
  sum = halves_sum(sum);
  if (sum == 0.f) ref = kNoScore;
  float lam = 0.f, ref2 = 0.f, sum2 = 0.f;
  if constexpr (GROUPS == 2) {                                        // the second group's sums, through LDS, to the first
    float* o = (float*)s_k;                                           // [DH / 4][kRowTile][4]
    float* rs = (float*)s_v;                                          // references, sums
    const int row = row_wave * 32 + col;
    static_assert(sizeof(s_k) >= sizeof(float) * kRowTile * DH && sizeof(s_v) >= sizeof(float) * 2 * kRowTile, "");
    const bool whole = DIFF && parts == 1;
    __syncthreads();                                                  // (the last tile is read no more)
    if (group == 1 && (!DIFF || whole)) {
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
    if (group == 0 && (!DIFF || whole)) {
      const float other = rs[row], osum = rs[kRowTile + row];
      float f, g;
      if constexpr (DIFF) {
        lam = late->lambda[h * gqa + hd];
        f = sum == 0.f ? 0.f : 1.0f / sum;
        g = osum == 0.f ? 0.f : -lam / osum;
        ref2 = other;
        sum2 = osum;
      } else {
        const float R = fmaxf(ref, other);
        f = exp2_of((ref - R) * cq);
        g = exp2_of((other - R) * cq);
        ref = R;
        sum = fmaf(sum, f, osum * g);
      }
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const floatx4 x = *(const floatx4*)&o[((8 * d + 2 * i + half) * kRowTile + row) * 4];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[d][4 * i + e] = fmaf(acc[d][4 * i + e], f, x[e] * g);
        }
    }
    if (group == 1 && (!DIFF || whole)) return;
  }
  const int at = (begin + tok) * c.num_kv * gqa + h * gqa + hd;      // (below 2^30: rows * gqa * num_kv is)
  if (parts == 1) {
    if constexpr (DIFF) {
      if (late->norm_weight) {
        float sq = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) sq = fmaf(acc[d][i], acc[d][i], sq);
        const float scale = sum == 0.f ? 0.f : 1.0f / __builtin_sqrtf(fmaf(halves_sum(sq), 1.0f / DH, late->norm_eps));
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= scale * late->norm_weight[32 * d + 8 * (i >> 2) + 4 * half + (i & 3)];
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[d] *= inv;
    }
    const bool none = sum == 0.f;
    // The rows pass through LDS (their chunks exclusive-or'ed with the row), so that a
    // store writes whole rows: it takes as long per row that it touches as for 64 bytes
    // of one.
    char* mine = (char*)s_v + (GROUPS == 2 ? 8 * kRowTile : 0) + 2 * DH * 32 * row_wave;
    static_assert(sizeof(s_v) >= (GROUPS == 2 ? 8 * kRowTile : 0) + 2 * DH * kRowTile, "");
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = pair_of<TYPE>(acc[d][4 * i], acc[d][4 * i + 1]), y = pair_of<TYPE>(acc[d][4 * i + 2], acc[d][4 * i + 3]);
        *(uintx2*)(mine + 2 * DH * col + 16 * ((4 * d + i) ^ (col & (CH - 1))) + 8 * half) = none ? uintx2{0, 0} : uintx2{x, y};
      }
#pragma unroll
    for (int i = 0; i < 32; i += RPL) {
      const int row = i + lane / CH, to = __shfl(at, row, kWave);
      const uintx4 x = *(const uintx4*)(mine + 2 * DH * row + 16 * ((lane % CH) ^ (row & (CH - 1))));
      struct __attribute__((packed, aligned(2))) U4 { uintx4 v; };
      if (row <= end_row) ((U4*)((uint16_t*)late->out + (int64_t)to * DH + 8 * (lane % CH)))->v = x;
    }
    if (late->lse && half == 0 && live) {
      const float e = none ? -INFINITY : (fmaf(ref, cq, -kTopWeight) + log2_of(sum)) * kLn2;
      if constexpr (DIFF) {
        late->lse[2 * (int64_t)at] = e;
        late->lse[2 * (int64_t)at + 1] = sum2 == 0.f ? -INFINITY : (fmaf(ref2, cq, -kTopWeight) + log2_of(sum2)) * kLn2;
      } else {
        late->lse[at] = e;
      }
    }
  } else if (live) {
    constexpr int rows = DIFF ? 2 * kRowTile : kRowTile;
    float* o = partials + (((int64_t)slot * c.num_kv + h) * splits + z) * split_floats(DH, rows);
    const int row = (DIFF ? group * kRowTile : 0) + row_wave * 32 + col;
    if (half == 0) {
      o[row] = ref;
      o[rows + row] = sum;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(floatx4*)&o[2 * rows + row * DH + 32 * d + 8 * i + 4 * half] =
            floatx4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
  }
}

// Joins the splits of each row; one wave per (row, query head).
template <int TYPE, int DH, bool DIFF>
__global__ __launch_bounds__(256) void cache16_prefill_merge_kernel(Cache16AttendLaunch L, int RS, int splits,
                                                                    const float* partials) {
  constexpr int DPL = DH / 64, MAPS = DIFF ? 2 : 1;
  const int kRowTile = 1 << RS, rows = MAPS * kRowTile;
  const Cache16& c = L.c;
  const Cache8Batch& b = L.b;
  const int heads = c.num_kv * L.gqa;
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
  const int parts = splits_of(tiles_of(L, len, n, (int)(r0 / L.gqa), last / L.gqa).count, splits);
  if (parts == 1) return;
  const int64_t slot = first_slot(b, s, L.gqa, RS, 1) + (r >> RS);
  const int in = (int)(r & (kRowTile - 1));
  const float* x = partials + (slot * c.num_kv + h) * splits * split_floats(DH, rows);
  RowSum<DH> y[2];
  const float cq = L.sm_scale * kLog2e;
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    join<DPL, 16>(0, parts, 1, rows, [&](int64_t z) {
      const float* p = x + z * split_floats(DH, rows) + m * kRowTile;
      return Partial{p + in, x + z * split_floats(DH, rows) + 2 * rows + (m * kRowTile + in) * DH};
    }, y[m].R, y[m].l, y[m].x, cq);
    y[m].R = fmaf(y[m].R, cq, -kTopWeight);
  }
  finish_row<TYPE, DH, DIFF>(row_out(&L), at, hq, y[0], y[MAPS - 1]);
}

// ---- launches ------------------------------------------------------------------

int launched() { return hipPeekAtLastError() == hipSuccess ? 0 : -1; }

template <int IN, int OUT, int DH>
int append(const Cache16AppendLaunch& L, hipStream_t st) {
  constexpr int HEADS = 64 / (DH / 16);
  const int heads = L.c.num_kv * (L.gqa + 2), most = (heads + HEADS - 1) / HEADS;
  const int64_t want = (2048 + L.b.num_rows - 1) / L.b.num_rows;     // waves of a row: eight per CU in all, if it has as many
  const int splits = (int)(want < most ? want : most);
  const uint32_t items = (uint32_t)(L.b.num_rows * splits);
  cache16_append_kernel<IN, OUT, DH><<<(items + 3) / 4, 256, 0, st>>>(L, items, splits);
  return launched();
}

template <int TYPE, int DH, bool DIFF>
int decode(const Cache16AttendLaunch& L, hipStream_t st) {
  int64_t* plan = (int64_t*)L.ws;
  float* partials = (float*)((uint8_t*)L.ws + plan_size(L.b.num_seqs));
  const int columns = L.gqa * (DIFF ? 2 : 1);
  cache16_decode_kernel<TYPE, DH, DIFF><<<decode_groups(DH), 256, 0, st>>>(L, partials, plan);
  const int heads = L.b.num_seqs * L.c.num_kv * L.gqa;
  if (L.b.num_seqs * L.c.num_kv * col_parts(columns) < 128)
    cache16_decode_merge_kernel<TYPE, DH, DIFF, 4><<<heads, 256, 0, st>>>(L, partials, plan);
  else
    cache16_decode_merge_kernel<TYPE, DH, DIFF, 1><<<heads, 64, 0, st>>>(L, partials, plan);
  return launched();
}

template <int TYPE, int DH, bool DIFF>
int prefill(const Cache16AttendLaunch& L, hipStream_t st) {
  const PrefillShape shape = prefill_shape(L.b.num_rows, L.b.num_seqs, L.gqa, DH, DIFF);
  const int64_t tiles = row_tiles(L.b.num_rows, L.b.num_seqs, L.gqa, shape.row_shift());
  const int splits = prefill_splits(L.b.num_rows, L.b.num_seqs, L.c.num_kv, L.gqa, shape);
  const unsigned grid = (unsigned)(tiles * L.c.num_kv * splits);
  float* ws = (float*)L.ws;
  if constexpr (DIFF) {
    cache16_prefill_kernel<TYPE, DH, 4, 2, true><<<grid, 512, 0, st>>>(L, (int)tiles, splits, ws);
  } else if constexpr (DH == 128) {
    if (shape.groups == 2) cache16_prefill_kernel<TYPE, DH, 4, 2, false><<<grid, 512, 0, st>>>(L, (int)tiles, splits, ws);
    else cache16_prefill_kernel<TYPE, DH, 8, 1, false><<<grid, 512, 0, st>>>(L, (int)tiles, splits, ws);
  } else {
    cache16_prefill_kernel<TYPE, DH, 4, 1, false><<<grid, 256, 0, st>>>(L, (int)tiles, splits, ws);
  }
  if (splits > 1) {
    const int64_t waves = L.b.num_rows * L.c.num_kv * L.gqa;
    cache16_prefill_merge_kernel<TYPE, DH, DIFF><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(L, shape.row_shift(), splits, ws);
  }
  return launched();
}

template <int TYPE, int DH, bool DIFF>
int attend(const Cache16AttendLaunch& L, hipStream_t st) {
  return L.b.cu ? prefill<TYPE, DH, DIFF>(L, st) : decode<TYPE, DH, DIFF>(L, st);
}

}  // namespace

int launch_cache16_append(const Cache16AppendLaunch& L, hipStream_t stream) {
#define SPHKV_PICK(I, O, D) if (L.type == I && L.c.type == O && L.c.dh == D) return append<I, O, D>(L, stream)
  SPHKV_PICK(kFp16, kFp16, 64); SPHKV_PICK(kFp16, kFp16, 128); SPHKV_PICK(kFp16, kBf16, 64); SPHKV_PICK(kFp16, kBf16, 128);
  SPHKV_PICK(kBf16, kFp16, 64); SPHKV_PICK(kBf16, kFp16, 128); SPHKV_PICK(kBf16, kBf16, 64); SPHKV_PICK(kBf16, kBf16, 128);
  SPHKV_PICK(kFp32, kFp16, 64); SPHKV_PICK(kFp32, kFp16, 128); SPHKV_PICK(kFp32, kBf16, 64); SPHKV_PICK(kFp32, kBf16, 128);
#undef SPHKV_PICK
  return -1;
}
int launch_cache16_attend(const Cache16AttendLaunch& L, hipStream_t stream) {
#define SPHKV_PICK(T, D, X) if (L.c.type == T && L.c.dh == D && (L.lambda != nullptr) == X) return attend<T, D, X>(L, stream)
  SPHKV_PICK(kFp16, 64, false); SPHKV_PICK(kFp16, 128, false); SPHKV_PICK(kBf16, 64, false); SPHKV_PICK(kBf16, 128, false);
  SPHKV_PICK(kFp16, 64, true); SPHKV_PICK(kFp16, 128, true); SPHKV_PICK(kBf16, 64, true); SPHKV_PICK(kBf16, 128, true);
#undef SPHKV_PICK
  return -1;
}
int64_t cache16_decode_ws_bytes(int32_t num_seqs, int32_t, int32_t gqa, int32_t dh, bool diff) {
  return plan_size(num_seqs) + 2 * decode_groups(dh) * 4 * partial_size(gqa * (diff ? 2 : 1), dh);
}
int64_t cache16_prefill_ws_bytes(int64_t num_rows, int32_t num_seqs, int32_t num_kv, int32_t gqa, int32_t dh, bool diff) {
  if (num_rows == 0 || num_seqs == 0) return 0;
  const PrefillShape p = prefill_shape(num_rows, num_seqs, gqa, dh, diff);
  const int splits = prefill_splits(num_rows, num_seqs, num_kv, gqa, p);
  const int rows = (diff ? 2 : 1) << p.row_shift();
  return splits == 1 ? 0 : row_tiles(num_rows, num_seqs, gqa, p.row_shift()) * num_kv * splits * split_floats(dh, rows) * 4;
}

}  // namespace sphkv
