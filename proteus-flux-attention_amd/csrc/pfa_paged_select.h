// Selection of a paged cache's pages: scores from the bounds of their keys, and
// the best `count` of each sequence and key-value head.
#pragma once

#include "pfa_paged.h"

namespace pfa {
namespace paged {

// A page's key in the order of choice: 0 for no candidate, 1 for a score that is
// not a number, the score's bits in order above, and the pages that are always
// taken on top.
constexpr uint32_t kNone = 0, kNan = 1, kForced = 0xffffffffu;

// Entries [p0, pe) of a sequence's row hold the positions to attend to.
struct Span {
  int p0, pe;
};
__device__ __forceinline__ Span span_at(const int32_t* lengths, const int32_t* starts, int P, int shift, int b) {
  const int64_t n = lengths[b], most = (int64_t)P << shift;
  const int len = (int)(n < 0 ? 0 : n < most ? n : most);
  const int start = starts && starts[b] > 0 ? starts[b] : 0;
  if (start >= len) return Span{0, 0};
  return Span{start >> shift, (len + (1 << shift) - 1) >> shift};
}

constexpr int kScoreHeads = 32;  // query heads in LDS at once
constexpr int kSteps = 4;        // pages of a lane at once

// Scores.  D / 8 lanes hold a page's two bounds of a head, eight channels each,
// of kSteps pages at once, and go over the query heads; sums are 64 bits, so
// that the order of the summands decides nothing that is not equal to 2^-53:
// with bf16 or f16 values the sums are as good as always exact.  The bounds are
// read once and are the bound: 4 D bytes a page and head for 16-bit cells against
// 3 D G instructions over 64 lanes (select, widen, fused multiply-add; the last
// runs at f32's rate on this chip).
template <int QT, int BT, int D>
__global__ void __launch_bounds__(256) score_kernel(Pages pg, const int32_t* __restrict__ table, int64_t table_stride,
                                                    int P, const typename Elem<QT>::T* __restrict__ q, int64_t q_b,
                                                    int64_t q_h, int G, const int32_t* __restrict__ lengths,
                                                    const int32_t* __restrict__ starts, int first, int last,
                                                    uint32_t* __restrict__ keys) {
  constexpr int LP = D / 8;            // lanes of a page
  constexpr int PW = kWave / LP;       // pages of a wave at once
  constexpr int AT_ONCE = 4 * PW * kSteps;  // pages of a workgroup
  using BoundT = typename Elem<BT>::T;
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const Span sp = span_at(lengths, starts, P, pg.shift, b);
  const int base = blockIdx.x * AT_ONCE;
  if (base >= sp.pe || base + AT_ONCE <= sp.p0) return;
  __shared__ float qs[kScoreHeads][D];
  const int part = lane % LP;
  // page of step s: base + (4 waves x kSteps + s) x PW + lane / LP
  const int page0 = base + (tid >> 6) * kSteps * PW + lane / LP;
  float lo[kSteps][8], hi[kSteps][8];
  bool have[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int page = page0 + s * PW;
    const int id = page >= sp.p0 && page < sp.pe ? table[b * table_stride + page] : -1;
    have[s] = (uint32_t)id < (uint32_t)pg.n_pages;
    const BoundT* at = (const BoundT*)pg.bounds + ((int64_t)(have[s] ? id : 0) * pg.H + h) * 2 * D + 8 * part;
    load8<BT>(at, lo[s]);
    load8<BT>(at + D, hi[s]);
  }
  // after the exchanges a lane holds the sums of KEEP steps
  constexpr int KEEP = LP == 2 ? 2 : 1;
  float best[KEEP];
  bool nan[KEEP];
#pragma unroll
  for (int s = 0; s < KEEP; ++s) best[s] = -INFINITY, nan[s] = false;
  const bool odd = lane & 1, upper = lane & 2;
  for (int g0 = 0; g0 < G; g0 += kScoreHeads) {
    const int heads = G - g0 < kScoreHeads ? G - g0 : kScoreHeads;
    __syncthreads();
    for (int i = tid; i < heads * D; i += 256)
      qs[i / D][i % D] = load_f<QT>(q + b * q_b + (int64_t)(h * G + g0 + i / D) * q_h + i % D);
    __syncthreads();
    for (int g = 0; g < heads; ++g) {
      double sum[kSteps] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = qs[g][8 * part + i];
        const bool up = x > 0.0f;
        const double xd = x;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) sum[s] = fma(xd, (double)(up ? hi[s][i] : lo[s][i]), sum[s]);
      }
      // lanes 2a, 2a + 1 share the steps out, then pairs of pairs
      double r[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const double mine = odd ? sum[2 + s] : sum[s], other = odd ? sum[s] : sum[2 + s];
        r[s] = mine + __shfl_xor(other, 1);
      }
      double t[KEEP];
      if constexpr (LP == 2) {
        t[0] = r[0], t[1] = r[1];
      } else {
        const double mine = upper ? r[1] : r[0], other = upper ? r[0] : r[1];
        t[0] = mine + __shfl_xor(other, 2);
#pragma unroll
        for (int o = 4; o < LP; o <<= 1) t[0] += __shfl_xor(t[0], o);
      }
#pragma unroll
      for (int s = 0; s < KEEP; ++s) {
        const float f = (float)t[s];
        nan[s] = nan[s] || f != f;
        best[s] = fmaxf(best[s], f);
      }
    }
  }
  if (part >= 4) return;
  uint32_t* row = keys + ((int64_t)b * pg.H + h) * P;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int s = LP == 2 ? 2 * odd + k : 2 * odd + upper;
    const int page = page0 + s * PW;
    if (page < sp.p0 || page >= sp.pe) continue;
    bool ok = false;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) ok = i == s ? have[i] : ok;
    uint32_t u = __float_as_uint(best[k]);
    u = u & 0x80000000u ? ~u : u | 0x80000000u;  // -inf is 0x007fffff, +inf 0xff800000
    if (nan[k]) u = kNan;
    if (page - sp.p0 < first || sp.pe - page <= last) u = kForced;
    row[page] = ok ? u : kNone;
  }
}

// The best `count` of a row of keys, ascending.  The keys' range is cut into
// 2,048 bins and the bin that holds the last one to take is cut again, until all
// of a bin or, among equal keys, the lowest entries are taken: mostly two
// rounds.  A workgroup a row; a thread holds four entries in a row of every
// 4 * THREADS, in registers where R rounds of them hold the row (R = 0: read
// again from the L2 each time).
constexpr int kBins = 2048;

template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* sums, int& all) {  // exclusive
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  return before + incl - x;
}

template <int THREADS, int R>
__global__ void __launch_bounds__(THREADS) choose_kernel(int H, int P, int shift, int count,
                                                         const int32_t* __restrict__ lengths,
                                                         const int32_t* __restrict__ starts,
                                                         const uint32_t* __restrict__ keys,
                                                         int32_t* __restrict__ chosen) {
  constexpr int WAVES = THREADS / kWave;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t* key = keys + (int64_t)blockIdx.x * P;
  int32_t* out = chosen + (int64_t)blockIdx.x * count;
  const Span sp = span_at(lengths, starts, P, shift, blockIdx.x / H);
  const int rounds = (sp.pe - sp.p0 + 4 * THREADS - 1) / (4 * THREADS);
  __shared__ int hist[kBins];
  __shared__ int sums[WAVES], sums2[WAVES];
  __shared__ uint32_t range[2][WAVES];
  __shared__ int cut[3];

  uint32_t held[R > 0 ? R : 1][4];
  auto fetch = [&](int r, uint32_t (&x)[4]) {
    const int p = sp.p0 + (r * THREADS + tid) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p + i < sp.pe ? key[p + i] : kNone;
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) fetch(r, held[r]);
  }
  auto each = [&](auto&& f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) f(r, held[r]);
    } else {
      for (int r = 0; r < rounds; ++r) {
        uint32_t x[4];
        fetch(r, x);
        f(r, x);
      }
    }
  };

  uint32_t lo = 0xffffffffu, hi = 0;
  int forced = 0, others = 0;
  each([&](int, const uint32_t (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool normal = x[i] != kNone && x[i] != kForced;
      forced += x[i] == kForced;
      others += normal;
      if (normal) lo = x[i] < lo ? x[i] : lo, hi = x[i] > hi ? x[i] : hi;
    }
  });
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t a = __shfl_xor(lo, o), z = __shfl_xor(hi, o);
    lo = a < lo ? a : lo, hi = z > hi ? z : hi;
    forced += __shfl_xor(forced, o), others += __shfl_xor(others, o);
  }
  if (lane == 0) range[0][wave] = lo, range[1][wave] = hi, sums[wave] = forced, sums2[wave] = others;
  __syncthreads();
  forced = others = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    lo = range[0][w] < lo ? range[0][w] : lo, hi = range[1][w] > hi ? range[1][w] : hi;
    forced += sums[w], others += sums2[w];
  }
  // taken: forced, keys above `over`, and `ties` keys that equal it
  int need = count - forced;
  uint32_t over = 0;
  int ties = 0;
  if (need >= others) {
    over = kNone;
  } else if (need <= 0) {
    over = kForced - 1;
  } else {
    while (true) {
      const int bits = hi == lo ? 0 : 32 - __clz(hi - lo);
      const int cutshift = bits > 11 ? bits - 11 : 0;
      if (hi == lo) {
        over = lo, ties = need;
        break;
      }
      for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
      __syncthreads();
      each([&](int, const uint32_t (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (x[i] >= lo && x[i] <= hi && x[i] != kForced) atomicAdd(&hist[(x[i] - lo) >> cutshift], 1);
      });
      __syncthreads();
      // bins from the top: thread t's are kBins - 1 - PER * t ...
      constexpr int PER = kBins / THREADS;
      int mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) mine += hist[kBins - 1 - PER * tid - i];
      int all;
      int above = block_scan<THREADS>(mine, sums, all);
      if (above < need && above + mine >= need) {
        for (int i = 0; i < PER; ++i) {
          const int bin = kBins - 1 - PER * tid - i, n = hist[bin];
          if (above + n >= need) {
            cut[0] = bin, cut[1] = need - above, cut[2] = n;
            break;
          }
          above += n;
        }
      }
      __syncthreads();
      const int bin = cut[0];
      need = cut[1];
      const uint32_t from = lo + ((uint32_t)bin << cutshift), to = from + ((1u << cutshift) - 1u);
      if (cut[2] == need) {  // all of the bin
        over = from - 1;
        break;
      }
      lo = from, hi = to < hi ? to : hi;
      __syncthreads();
    }
  }
  // ascending: ties count by entry, too
  int base = 0, tied = 0;
  each([&](int r, const uint32_t (&x)[4]) {
    if (R > 0 && r >= rounds) return;
    int eq = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) eq += ties > 0 && x[i] == over;
    int all_eq = 0, before_eq = 0;
    if (ties > 0) before_eq = tied + block_scan<THREADS>(eq, sums, all_eq);
    bool take[4];
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool tie = ties > 0 && x[i] == over;
      take[i] = x[i] > over || (tie && before_eq < ties);
      before_eq += tie;
      n += take[i];
    }
    int all;
    int at = base + block_scan<THREADS>(n, sums2, all);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (take[i]) out[at++] = sp.p0 + (r * THREADS + tid) * 4 + i;
    base += all, tied += all_eq;
  });
  for (int i = base + tid; i < count; i += THREADS) out[i] = -1;
}

}  // namespace paged
}  // namespace pfa
