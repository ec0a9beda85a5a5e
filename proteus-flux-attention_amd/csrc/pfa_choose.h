// The best `count` keys of a row, by one workgroup.  Nothing here but LDS, lane
// exchanges and barriers, so that its steps can be followed on the host in any
// order of the waves.
#pragma once

#include "pfa_common.h"

namespace pfa {
namespace paged {

// A page's key in the order of choice: 0 for no candidate, 1 for a score that is
// not a number, the score's bits in order above, and the pages that are always
// taken on top.
constexpr uint32_t kNone = 0, kNan = 1, kForced = 0xffffffffu;

// The best `count` of a row of keys, ascending.  The keys' range is cut into
// 2,048 bins and the bin that holds the last one to take is cut again, until all
// of a bin or, among equal keys, the lowest entries are taken: mostly two
// rounds.  A workgroup a row, a thread K entries in a row, in registers where
// THREADS * K hold all of them (HELD), else read again from the L2 each time.  32
// rows of 8,192 pages: 8 us, all of it latency.
constexpr int kBins = 2048;

// Exclusive sum over the workgroup; `all`: the whole.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* sums, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(incl, o);
    if (lane >= o) incl += y;
  }
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

// fetch(r, x): the K keys of the thread's entries from + (r * THREADS + thread) * K
// on in round r, kNone where there are none.  put(i, entry): the i-th choice, -1
// behind the last.
template <int THREADS, int K, bool HELD, typename Fetch, typename Put>
__device__ __forceinline__ void choose_best(int from0, int rounds, int count, Fetch&& fetch, Put&& put) {
  constexpr int WAVES = THREADS / kWave;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ int hist[kBins];
  __shared__ int sums[3][WAVES];
  __shared__ uint32_t range[2][WAVES];
  __shared__ int cut[3];

  uint32_t held[K];
  if constexpr (HELD) fetch(0, held);
  auto each = [&](auto&& f) {
    if constexpr (HELD) f(0, held);
    else {
      for (int r = 0; r < rounds; ++r) {
        fetch(r, held);
        f(r, held);
      }
    }
  };

  uint32_t lo = 0xffffffffu, hi = 0;
  int forced = 0, others = 0;
  each([&](int, const uint32_t (&x)[K]) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const bool normal = x[i] != kNone && x[i] != kForced;
      forced += x[i] == kForced;
      others += normal;
      if (normal) lo = x[i] < lo ? x[i] : lo, hi = x[i] > hi ? x[i] : hi;
    }
  });
  for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t a = __shfl_xor(lo, o), z = __shfl_xor(hi, o);
    lo = a < lo ? a : lo, hi = z > hi ? z : hi;
    forced += __shfl_xor(forced, o), others += __shfl_xor(others, o);
  }
  if (lane == 0) range[0][wave] = lo, range[1][wave] = hi, sums[0][wave] = forced, sums[1][wave] = others;
  __syncthreads();
  forced = others = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    lo = range[0][w] < lo ? range[0][w] : lo, hi = range[1][w] > hi ? range[1][w] : hi;
    forced += sums[0][w], others += sums[1][w];
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
      if (hi == lo) {
        over = lo, ties = need;
        break;
      }
      const int bits = 32 - __clz(hi - lo), cutshift = bits > 11 ? bits - 11 : 0;
      each([&](int, const uint32_t (&x)[K]) {
#pragma unroll
        for (int i = 0; i < K; ++i)
          if (x[i] >= lo && x[i] <= hi) atomicAdd(&hist[(x[i] - lo) >> cutshift], 1);
      });
      __syncthreads();
      // bins from the top: thread t's are kBins - 1 - PER * t ...
      constexpr int PER = kBins / THREADS;
      int bin_n[PER], mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        int& bin = hist[kBins - 1 - PER * tid - i];
        mine += bin_n[i] = bin;
        bin = 0;
      }
      int all;
      int above = block_scan<THREADS>(mine, sums[2], all);
      if (above < need && above + mine >= need) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (above < need && above + bin_n[i] >= need)
            cut[0] = kBins - 1 - PER * tid - i, cut[1] = need - above, cut[2] = bin_n[i];
          above += bin_n[i];
        }
      }
      __syncthreads();
      need = cut[1];
      const uint32_t from = lo + ((uint32_t)cut[0] << cutshift), to = from + ((1u << cutshift) - 1u);
      if (cut[2] == need) {  // all of the bin
        over = from - 1;
        break;
      }
      lo = from, hi = to < hi ? to : hi;
    }
  }
  // ascending, ties by entry; counts of the taken above and of the ties, 16 bits
  // each: THREADS * K < 2^16
  int base = 0, tied = 0;
  each([&](int r, const uint32_t (&x)[K]) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) n += x[i] > over ? 1 << 16 : ties > 0 && x[i] == over ? 1 : 0;
    int all;
    if (!HELD) __syncthreads();  // the last round's sums are read
    // sums[2]: its readers in the cuts are behind a barrier.  sums[0] and sums[1] may
    // still have some: rows that need no cut come here without one.
    const int before = block_scan<THREADS>(n, sums[2], all);
    int eq = tied + (before & 0xffff), at = base + (before >> 16) + (eq < ties ? eq - tied : ties > tied ? ties - tied : 0);
    const int p = from0 + (r * THREADS + tid) * K;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const bool tie = ties > 0 && x[i] == over;
      if (x[i] > over || (tie && eq < ties)) put(at++, p + i);
      eq += tie;
    }
    const int eqs = all & 0xffff, left = ties > tied ? ties - tied : 0;
    base += (all >> 16) + (eqs < left ? eqs : left);
    tied += eqs;
  });
  for (int i = base + tid; i < count; i += THREADS) put(i, -1);
}

}  // namespace paged
}  // namespace pfa
