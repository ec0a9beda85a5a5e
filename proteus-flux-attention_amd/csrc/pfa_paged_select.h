// Selection of a paged cache's pages: scores from the bounds of their keys, and
// the best `count` of each sequence and key-value head.
#pragma once

#include "pfa_choose.h"
#include "pfa_paged.h"

namespace pfa {
namespace paged {

// Entries [p0, pe) of a sequence's row hold the positions to attend to.
struct Span {
  int p0, pe;
};
__device__ __forceinline__ Span span_at(const int32_t* lengths, const int32_t* starts, int P, int shift, int b) {
  const int len = length_at(lengths, P, shift, b), start = start_at(starts, b);
  if (start >= len) return Span{0, 0};
  return Span{start >> shift, (len + (1 << shift) - 1) >> shift};
}

constexpr int kScoreHeads = 8;  // query heads in LDS at once
constexpr int kSteps = 4;        // pages of a lane at once
// Query heads at once.  f32 bounds leave three waves a SIMD, whose products wait for
// one another less with two (15.4 -> 14.1 us at 15,000 pages and heads, eight query
// heads); 16-bit bounds leave eight (27.6 -> 29.2 at 196,608, four query heads).
__host__ __device__ constexpr int pair_of(int bt) { return bt == PFA_F32 ? 2 : 1; }

// The value of lane ^ MASK, 64 bits: a quad permute, or a swizzle.
template <int MASK>
__device__ __forceinline__ double across(double x) {
  const int lo = __double2loint(x), hi = __double2hiint(x);
  if constexpr (MASK < 4) {
    constexpr int PERM = MASK == 1 ? 0xB1 : 0x4E;  // [1, 0, 3, 2], [2, 3, 0, 1]
    return __hiloint2double(__builtin_amdgcn_mov_dpp(hi, PERM, 0xf, 0xf, true),
                            __builtin_amdgcn_mov_dpp(lo, PERM, 0xf, 0xf, true));
  } else {
    constexpr int XOR = MASK << 10 | 0x1f;
    return __hiloint2double(__builtin_amdgcn_ds_swizzle(hi, XOR), __builtin_amdgcn_ds_swizzle(lo, XOR));
  }
}

// One exchange of `spread`s: N sums of a lane become N / 2, or, where one is left,
// the sum of both lanes'.
template <int MASK, int N, int LP>
__device__ __forceinline__ void spread(double* sum, int lane) {
  if constexpr (MASK < LP) {
    if constexpr (N > 1) {
      const bool up = lane & MASK;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const double mine = up ? sum[N / 2 + i] : sum[i], other = up ? sum[i] : sum[N / 2 + i];
        sum[i] = mine + across<MASK>(other);
      }
      spread<2 * MASK, N / 2, LP>(sum, lane);
    } else {
      sum[0] += across<MASK>(sum[0]);
      spread<2 * MASK, 1, LP>(sum, lane);
    }
  }
}

// Scores.  D / 8 lanes hold a page's two bounds of a head, eight channels each,
// of kSteps pages at once, and go over the query heads; sums are 64 bits, so
// that the order of the summands decides nothing that is not equal to 2^-53:
// with bf16 or f16 values the sums are as good as always exact.  The bounds are
// read once for all heads of a group; a channel is a select, a widening and a
// fused multiply-add.  Heads of one page are neighbours in the grid, as their
// bounds are in memory.  196,608 pages and heads of 128 bf16 channels (100 MB),
// four query heads each: 28 us, 3.6 TB/s, of which 3 us are three of the four heads'
// arithmetic.  Widening the bounds once and two products of max(q, 0) and min(q, 0) a
// channel: 35 us (160 registers, three waves a SIMD); two pages of a lane at once: 31.
//
// Pages base .. base + WAVES * 64 / (D / 8) * kSteps - 1 of a workgroup's row; put
// gets each page of the span and its key.
template <int QT, int BT, int D, int WAVES, typename Put>
__device__ __forceinline__ void score_pages(const Pages& pg, const int32_t* __restrict__ ids, int P, const Span& sp, int h,
                                            const typename Elem<QT>::T* __restrict__ q, int64_t q_h, int G, int first,
                                            int last, int base, float (&qs)[kScoreHeads][D], Put&& put) {
  constexpr int LP = D / 8;       // lanes of a page
  constexpr int PW = kWave / LP;  // pages of a wave at once
  using BoundT = typename Elem<BT>::T;
  const int tid = threadIdx.x, lane = tid & 63, part = lane % LP;
  constexpr int STEPS = kSteps, PAIR = pair_of(BT);
  const int page0 = base + (tid >> 6) * STEPS * PW + lane / LP;  // of step s: + s * PW
  // the first heads' queries, on their way before the bounds are waited for
  constexpr int QN = kScoreHeads * D / (WAVES * kWave) > 0 ? kScoreHeads * D / (WAVES * kWave) : 1;
  float qr[QN];
  auto load_q = [&](int g0, int heads) {
#pragma unroll
    for (int u = 0; u < QN; ++u) {
      const int i = tid + u * WAVES * kWave;
      qr[u] = i < heads * D ? load_f<QT>(q + (int64_t)(h * G + g0 + i / D) * q_h + i % D) : 0.0f;
    }
  };
  auto store_q = [&](int heads) {
#pragma unroll
    for (int u = 0; u < QN; ++u) {
      const int i = tid + u * WAVES * kWave;
      if (i < heads * D) qs[i / D][i % D] = qr[u];
    }
  };
  const int heads0 = G < kScoreHeads ? G : kScoreHeads;
  const int wave0 = base + __builtin_amdgcn_readfirstlane(tid >> 6) * STEPS * PW;
  const bool busy = wave0 < sp.pe && wave0 + STEPS * PW > sp.p0;  // the wave has pages
  int id[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int page = page0 + s * PW;
    id[s] = page < P ? ids[page] : -1;  // before the span is known: a load less in a row
  }
  load_q(0, heads0);
  float lo[STEPS][8], hi[STEPS][8];
  bool have[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int page = page0 + s * PW;
    have[s] = page >= sp.p0 && page < sp.pe && (uint32_t)id[s] < (uint32_t)pg.n_pages;
    const BoundT* at = (const BoundT*)pg.bounds + ((int64_t)(have[s] ? id[s] : 0) * pg.H + h) * 2 * D + 8 * part;
    load8<BT>(at, lo[s]);
    load8<BT>(at + D, hi[s]);
  }
  // NV sums of a lane, heads first; each exchange leaves a lane half of them, until
  // one is left or the lanes are through: KEEP of them, from value `mine` on
  constexpr int NV = PAIR * STEPS, SPLITS = LP >= NV ? NV : LP, KEEP = NV / SPLITS;
  float best[KEEP];
  bool nan[KEEP];
#pragma unroll
  for (int s = 0; s < KEEP; ++s) best[s] = -INFINITY, nan[s] = false;
  for (int g0 = 0; g0 < G; g0 += kScoreHeads) {
    const int heads = G - g0 < kScoreHeads ? G - g0 : kScoreHeads;
    if (g0 > 0) load_q(g0, heads);
    __syncthreads();
    store_q(heads);
    __syncthreads();
    for (int g = 0; g < (busy ? heads : 0); g += PAIR) {
      double sum[NV] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int u = 0; u < PAIR; ++u) {
          const float x = qs[g + u < heads ? g + u : heads - 1][8 * part + i];  // an odd last head counts twice
          const bool up = x > 0.0f;
          const double xd = x;
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
            sum[u * STEPS + s] = fma(xd, (double)(up ? hi[s][i] : lo[s][i]), sum[u * STEPS + s]);
        }
      spread<1, NV, LP>(sum, lane);
#pragma unroll
      for (int s = 0; s < KEEP; ++s) {
        const float f = (float)sum[s];
        nan[s] = nan[s] || f != f;
        best[s] = fmaxf(best[s], f);
      }
    }
  }
  // value of sum[0]: lane bit 0 chose between halves, bit 1 between quarters, ...
  int mine = 0;
#pragma unroll
  for (int o = 1; o < SPLITS; o <<= 1) mine += part & o ? NV / (2 * o) : 0;
  if constexpr (PAIR == 2) {
#pragma unroll
    for (int s = 0; s < KEEP; ++s) {
      best[s] = fmaxf(best[s], __shfl_xor(best[s], 1));
      nan[s] = nan[s] | (bool)__shfl_xor((int)nan[s], 1);
    }
  }
  if (part >= SPLITS || mine >= STEPS) return;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int s = mine + k;
    const int page = page0 + s * PW;
    if (s >= STEPS || page < sp.p0 || page >= sp.pe) continue;
    bool ok = false;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) ok = i == s ? have[i] : ok;
    uint32_t u = best[k] == 0.0f ? 0u : __float_as_uint(best[k]);  // -0, a sum that underflows, ties with +0
    u = u & 0x80000000u ? ~u : u | 0x80000000u;  // -inf is 0x007fffff, +inf 0xff800000
    if (nan[k]) u = kNan;
    if (page - sp.p0 < first || sp.pe - page <= last) u = kForced;
    put(page, ok ? u : kNone);
  }
}

// Pages of a workgroup of `waves` waves at once.
__host__ __device__ constexpr int score_span(int waves, int D) { return waves * (kWave / (D / 8)) * kSteps; }

template <int QT, int BT, int D>
__global__ void __launch_bounds__(256) score_kernel(Pages pg, const int32_t* __restrict__ table, int64_t table_stride,
                                                    int P, const typename Elem<QT>::T* __restrict__ q, int64_t q_b,
                                                    int64_t q_h, int G, const int32_t* __restrict__ lengths,
                                                    const int32_t* __restrict__ starts, int first, int last,
                                                    int64_t row_keys, uint32_t* __restrict__ keys) {
  const int b = blockIdx.z, h = blockIdx.x;
  const Span sp = span_at(lengths, starts, P, pg.shift, b);
  constexpr int SPAN = score_span(4, D);
  __shared__ float qs[kScoreHeads][D];
  uint32_t* row = keys + ((int64_t)b * pg.H + h) * row_keys;
  for (int base = blockIdx.y * SPAN; base < sp.pe; base += gridDim.y * SPAN) {
    if (base + SPAN <= sp.p0) continue;
    score_pages<QT, BT, D, 4>(pg, table + b * table_stride, P, sp, h, q + b * q_b, q_h, G, first, last, base, qs,
                              [&](int page, uint32_t key) { row[page] = key; });
  }
}

template <int THREADS, int K, bool HELD>
__global__ void __launch_bounds__(THREADS) choose_kernel(int H, int P, int64_t row_keys, int shift, int count,
                                                         const int32_t* __restrict__ lengths,
                                                         const int32_t* __restrict__ starts,
                                                         const uint32_t* __restrict__ keys,
                                                         int32_t* __restrict__ chosen) {
  const uint32_t* key = keys + (int64_t)blockIdx.x * row_keys;
  const Span sp = span_at(lengths, starts, P, shift, blockIdx.x / H);
  const int from0 = HELD ? 0 : sp.p0 & ~3;  // rows of keys are 16-byte aligned
  const int rounds = HELD ? 1 : (sp.pe - from0 + THREADS * K - 1) / (THREADS * K);
  int32_t* out = chosen + (int64_t)blockIdx.x * count;
  auto fetch = [&](int r, uint32_t (&x)[K]) {
    const int p = from0 + (r * THREADS + (int)threadIdx.x) * K;
#pragma unroll
    for (int i = 0; i < K; i += 4) {
      // held rows before the span is known: what lies outside of it is masked
      uint4 a = make_uint4(0, 0, 0, 0);
      if (p + i < (HELD ? P : sp.pe)) a = *reinterpret_cast<const uint4*>(key + p + i);
      x[i] = a.x, x[i + 1] = a.y, x[i + 2] = a.z, x[i + 3] = a.w;
    }
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (p + i < sp.p0 || p + i >= sp.pe) x[i] = kNone;
  };
  choose_best<THREADS, K, HELD>(from0, rounds, count, fetch, [&](int i, int entry) { out[i] = entry; });
}

// Both in one workgroup for rows that four waves score in two rounds, with the keys
// in LDS: a launch (3.6 us of the host) less, and 7.6 us against 4.0 + 5.4 for 8 rows
// of 251 pages of 64 channels.  Longer rows are quicker apart (8 rows of 501 pages of
// 128 channels: 25 us with their attention in one, 22 apart).
constexpr int kFused = 512;
__host__ __device__ constexpr bool few_pages(int P, int D) { return P <= kFused && P <= 2 * score_span(4, D); }

template <int QT, int BT, int D, typename Put>
__device__ __forceinline__ void select_row(const Pages& pg, const int32_t* __restrict__ ids, int P, int b, int h,
                                           const typename Elem<QT>::T* __restrict__ q, int64_t q_h, int G,
                                           const int32_t* lengths, const int32_t* starts, int first, int last, int count,
                                           Put&& put) {
  const int tid = threadIdx.x;
  const Span sp = span_at(lengths, starts, P, pg.shift, b);
  __shared__ float qs[kScoreHeads][D];
  __shared__ uint32_t keys[kFused];
  for (int base = 0; base < P; base += score_span(4, D))
    score_pages<QT, BT, D, 4>(pg, ids, P, sp, h, q, q_h, G, first, last, base, qs,
                              [&](int page, uint32_t key) { keys[page] = key; });
  __syncthreads();
  constexpr int K = kFused / 256;
  auto fetch = [&](int, uint32_t (&x)[K]) {
#pragma unroll
    for (int i = 0; i < K; ++i) x[i] = K * tid + i >= sp.p0 && K * tid + i < sp.pe ? keys[K * tid + i] : kNone;
  };
  choose_best<256, K, true>(0, 1, count, fetch, put);
}

template <int QT, int BT, int D>
__global__ void __launch_bounds__(256) select_kernel(Pages pg, const int32_t* __restrict__ table, int64_t table_stride,
                                                     int P, const typename Elem<QT>::T* __restrict__ q, int64_t q_b,
                                                     int64_t q_h, int G, const int32_t* __restrict__ lengths,
                                                     const int32_t* __restrict__ starts, int first, int last, int count,
                                                     int32_t* __restrict__ chosen) {
  const int b = blockIdx.x / pg.H, h = blockIdx.x % pg.H;
  int32_t* out = chosen + (int64_t)blockIdx.x * count;
  select_row<QT, BT, D>(pg, table + b * table_stride, P, b, h, q + b * q_b, q_h, G, lengths, starts, first, last, count,
                        [&](int i, int entry) { out[i] = entry; });
}

}  // namespace paged
}  // namespace pfa
