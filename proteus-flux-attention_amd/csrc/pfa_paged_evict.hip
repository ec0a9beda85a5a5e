// Eviction from a paged cache: the keys that were attended to most, and their move into
// fresh pages.
#include "pfa_choose.h"
#include "pfa_paged.h"

namespace pfa {

using namespace paged;

namespace {

// Keys of one sequence and head by the attention they got.
struct Weights {
  const float* p;  // (B, H, T), rows apart by
  int64_t s_b, s_h;
  int T, most;  // positions of a row, and those of them that may be kept
  int vec;      // rows are aligned to four, and T is a multiple of it
};

// ---------------------------------------------------------------------
// Choice: a workgroup a sequence and head.  The weights' bits in their order are keys;
// their range is cut into 2,048 bins and the bin that holds the last one to take is
// cut again, as choose_best does it for pages, mostly twice.  A thread holds four
// neighbours of every 4 * THREADS positions, so that loads are in one piece, and a
// position's place among the kept is counted by ballots: within its wave, then over
// the waves of all pieces.  All is LDS and latency: 48 rows of up to 20,480 positions
// in registers, 8,192 kept: 16 us (choose_best with 32 neighbours a thread: 23).
// Positions without a page (where there is a table) are no candidates.
// ---------------------------------------------------------------------
// What is chosen from, and how.
struct Keep {
  Weights w;
  Table tab;
  int shift, n_pages, H;
  const int32_t* lengths;
  int count, first, last;

  __device__ __forceinline__ int length(int b) const {
    const int n = lengths[b];
    return n < 0 ? 0 : n < w.most ? n : w.most;
  }
  __device__ __forceinline__ const float* row(int b, int h) const { return w.p + b * w.s_b + h * w.s_h; }
  __device__ __forceinline__ const int32_t* pages(int b) const { return tab.ids ? tab.ids + b * tab.stride : nullptr; }
};

// Keys of a thread's positions of a slice [p0, end) of a row of `len` positions: four
// neighbours of every 4 * THREADS, C times.  One CU has a row's arithmetic to itself:
// pieces behind the slice's end are left out, and those without an end of the row or a
// position that is always taken go without the comparisons for them.
template <int THREADS, int C>
struct Keys {
  static constexpr int WAVES = THREADS / kWave, PIECE = 4 * THREADS;
  uint32_t x[C][4];
  int p0, end;

  __device__ __forceinline__ bool any(int c) const { return p0 + c * PIECE < end; }
  __device__ __forceinline__ int position(int c) const { return p0 + c * PIECE + 4 * (int)threadIdx.x; }

  // end: a multiple of four, or the row's
  __device__ __forceinline__ void fetch(const Keep& k, const float* row, const int32_t* ids, int len, int from, int to) {
    p0 = from, end = to;
    float4 v[C];
    int id[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int p = position(c);
      id[c] = ids && p < end ? ids[p >> k.shift] : 0;
      v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k.w.vec) {
        if (p < end) v[c] = *reinterpret_cast<const float4*>(row + p);
      } else {
        if (p < end) v[c].x = row[p];
        if (p + 1 < end) v[c].y = row[p + 1];
        if (p + 2 < end) v[c].z = row[p + 2];
        if (p + 3 < end) v[c].w = row[p + 3];
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!any(c)) continue;
      const bool have = (uint32_t)id[c] < (uint32_t)k.n_pages || !ids;
      const float y[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = __float_as_uint(y[j] + 0.0f);  // -0 ties with +0
        const uint32_t key = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
        x[c][j] = !have ? kNone : y[j] != y[j] ? kNan : key;
      }
      const int at = p0 + c * PIECE;
      if (at < k.first || at + PIECE > end || at + PIECE > len - k.last) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int p = position(c) + j;
          if (have && (p < k.first || len - p <= k.last)) x[c][j] = kForced;
          if (p >= end) x[c][j] = kNone;
        }
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!any(c)) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) f(x[c][j]);
    }
  }
};

// What is known of the last key to take: `need` of the keys in [lo, hi] are; done: those
// above `over` are taken, and the lowest `ties` positions of those that equal it.
struct Cut {
  uint32_t lo, hi, over;
  int need, ties, done;

  __device__ __forceinline__ int shift() const {
    const int bits = 32 - __clz(hi - lo);
    return bits > 11 ? bits - 11 : 0;
  }
  // of the lowest and highest key, how many are always taken and how many are others
  static __device__ __forceinline__ Cut first(uint32_t lo, uint32_t hi, int forced, int others, int count) {
    Cut c{lo, hi, 0, count - forced, 0, 1};
    if (c.need >= others) c.over = kNone;
    else if (c.need <= 0) c.over = kForced - 1;
    else if (lo == hi) c.over = lo, c.ties = c.need;
    else c.done = 0;
    return c;
  }
  // from the bins of the keys in [lo, hi]; bins: the thread's, from the top, PER to each
  template <int THREADS>
  __device__ __forceinline__ void narrow(const int (&bins)[kBins / THREADS], int* sums, int* cut) {
    constexpr int PER = kBins / THREADS;
    int mine = 0, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += bins[i];
    int above = block_scan<THREADS>(mine, sums, all);
    if (above < need && above + mine >= need) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (above < need && above + bins[i] >= need)
          cut[0] = kBins - 1 - PER * threadIdx.x - i, cut[1] = need - above, cut[2] = bins[i];
        above += bins[i];
      }
    }
    __syncthreads();
    const int by = shift();
    const uint32_t from = lo + ((uint32_t)cut[0] << by), to = from + ((1u << by) - 1u);
    need = cut[1];
    if (cut[2] == need) {  // all of the bin
      over = from - 1, done = 1;
      return;
    }
    lo = from, hi = to < hi ? to : hi;
    if (lo == hi) over = lo, ties = need, done = 1;
  }
};

// Range and numbers of a thread's keys, of its wave's, and of the workgroup's in all
// threads.
struct Range {
  uint32_t lo = 0xffffffffu, hi = 0;
  int forced = 0, others = 0;

  __device__ __forceinline__ void add(uint32_t key) {
    const bool normal = key != kNone && key != kForced;
    forced += key == kForced;
    others += normal;
    if (normal) lo = key < lo ? key : lo, hi = key > hi ? key : hi;
  }
  __device__ __forceinline__ void join(const Range& r) {
    lo = r.lo < lo ? r.lo : lo, hi = r.hi > hi ? r.hi : hi;
    forced += r.forced, others += r.others;
  }
  __device__ __forceinline__ void over_wave() {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      Range r;
      r.lo = __shfl_xor(lo, o), r.hi = __shfl_xor(hi, o);
      r.forced = __shfl_xor(forced, o), r.others = __shfl_xor(others, o);
      join(r);
    }
  }
  template <int WAVES>
  __device__ __forceinline__ void over_block(uint4 (&part)[WAVES]) {
    over_wave();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = packed();
    __syncthreads();
    *this = Range{};
#pragma unroll
    for (int i = 0; i < WAVES; ++i) join(of(part[i]));
  }
  __device__ __forceinline__ uint4 packed() const { return make_uint4(lo, hi, (uint32_t)forced, (uint32_t)others); }
  static __device__ __forceinline__ Range of(uint4 p) {
    Range r;
    r.lo = p.x, r.hi = p.y, r.forced = (int)p.z, r.others = (int)p.w;
    return r;
  }
};

// put(i, position) for the kept positions of a slice; `base` keys above and `tied` equal
// ones stand before it, and are counted on.
template <int THREADS, int C, typename Put>
__device__ __forceinline__ void place(const Keys<THREADS, C>& k, uint32_t over, int ties, int& base, int& tied,
                                      int (&taken)[2][C * (THREADS / kWave) + 1], Put&& put) {
  constexpr int WAVES = THREADS / kWave;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // of the lanes before this one, above in the lower half and equal in the upper
  uint32_t before[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    uint32_t mine = 0, whole = 0;
    auto vote = [&](bool yes, int at) {
      const uint64_t m = __ballot(yes);
      mine += __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0)) << at;
      whole += __popcll(m) << at;
    };
    if (k.any(c)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) vote(k.x[c][j] > over, 0);
      if (ties > 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) vote(k.x[c][j] == over, 16);
      }
    }
    before[c] = mine;
    if (lane == 0) taken[0][c * WAVES + wave] = whole & 0xffff, taken[1][c * WAVES + wave] = whole >> 16;
  }
  __syncthreads();
  if (wave < 2) {  // sums of those before, a wave each
    constexpr int N = C * WAVES, PER = (N + kWave - 1) / kWave;
    int v[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = lane * PER + i;
      v[i] = at < N ? taken[wave][at] : 0;
      mine += v[i];
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int y = __shfl_up(incl, o);
      if (lane >= o) incl += y;
    }
    int sum = incl - mine;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = lane * PER + i;
      if (at < N) taken[wave][at] = sum;
      sum += v[i];
    }
    if (lane == 63) taken[wave][N] = incl;
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!k.any(c)) continue;
    int at = base + taken[0][c * WAVES + wave] + (int)(before[c] & 0xffff);
    int eq = tied + taken[1][c * WAVES + wave] + (int)(before[c] >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool above = k.x[c][j] > over, tie = ties > 0 && k.x[c][j] == over;
      if (above || (tie && eq < ties)) put(at + (eq < ties ? eq : ties), k.position(c) + j);
      at += above, eq += tie;
    }
  }
  base += taken[0][C * WAVES], tied += taken[1][C * WAVES];
}

// A row that one workgroup holds.  put(i, position): the i-th kept position, -1 behind
// the last.
template <int THREADS, int C, typename Put>
__device__ __forceinline__ void choose_tokens(const Keep& k, int b, int h, Put&& put) {
  constexpr int WAVES = THREADS / kWave, PER = kBins / THREADS;
  const int tid = threadIdx.x;
  const int len = k.length(b);
  __shared__ int hist[kBins];
  __shared__ int sums[WAVES];
  __shared__ uint4 range[WAVES];
  __shared__ int cuts[3];
  __shared__ int taken[2][C * WAVES + 1];

  Keys<THREADS, C> keys;
  keys.fetch(k, k.row(b, h), k.pages(b), len, 0, len);
  Range r;
  keys.each([&](uint32_t key) { r.add(key); });
  for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
  r.over_block(range);
  Cut cut = Cut::first(r.lo, r.hi, r.forced, r.others, k.count);
  while (!cut.done) {
    const int by = cut.shift();
    keys.each([&](uint32_t key) {
      if (key - cut.lo <= cut.hi - cut.lo) atomicAdd(&hist[(key - cut.lo) >> by], 1);
    });
    __syncthreads();
    int bins[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int& bin = hist[kBins - 1 - PER * tid - i];
      bins[i] = bin;
      bin = 0;
    }
    cut.narrow<THREADS>(bins, sums, cuts);
  }
  int base = 0, tied = 0;
  place<THREADS, C>(keys, cut.over, cut.ties, base, tied, taken, put);
  for (int i = base + (tied < cut.ties ? tied : cut.ties) + tid; i < k.count; i += THREADS) put(i, -1);
}

template <int THREADS, int C>
__global__ void __launch_bounds__(THREADS) choose_tokens_kernel(Keep k, int32_t* __restrict__ kept) {
  int32_t* out = kept + (int64_t)blockIdx.x * k.count;
  choose_tokens<THREADS, C>(k, blockIdx.x / k.H, blockIdx.x % k.H, [&](int i, int position) { out[i] = position; });
}

// Longer rows are cut into slices, a workgroup each, in six launches: the slices'
// ranges; three times their bins, each from what the ones before leave (32 bits less 11
// each time: the third leaves single keys); how many of a slice are taken; their
// places.  A launch adds the slices' bins up in each of its workgroups, a cache's
// reads (8 KB a slice), and has no atomics in memory and nothing to clear.
// 8 rows of 65,536 positions by a workgroup each: 32 us, cut 37 (128 rows: 34 and 58);
// of 131,072, which one workgroup has to read again each time: 87, 46 cut; of 1,048,576:
// 630, 71 cut, eight to twelve a launch, the bins' sum (256 KB of them) half of it.
constexpr int kSlices = 32;    // of a row, at most (1,048,576: 85 us with 16, 106 with 64)
constexpr int kHeld = 65536;   // positions of a row that one workgroup takes
constexpr int kPieces = 2;     // of a thread at once (512 rows of 70,000: 152 us, 164 with 4, 195 with 8)
constexpr int kEnough = 256;   // workgroups of a launch, where rows are fewer (32 rows of 100,000: 44 us, 56 with 512)
struct Split {
  int slices, length;  // of a row, and positions of each
  uint4* ranges;       // (rows, slices)
  int* bins;           // two of (rows, slices, kBins): of one launch and of the one before
  int2* numbers;       // (rows, slices): above, and equal
  Cut* cuts;           // (rows, 4)
};

enum Step { RANGE, BINS1, BINS2, BINS3, COUNT, PLACE };

template <int STEP>
__global__ void __launch_bounds__(1024) split_kernel(Keep k, Split s, int32_t* __restrict__ kept) {
  constexpr int THREADS = 1024, C = kPieces, WAVES = THREADS / kWave, PER = kBins / THREADS;
  static_assert(PER == 2, "a thread's bins are one load");
  using K = Keys<THREADS, C>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x / s.slices, here = blockIdx.x;
  const int slice = blockIdx.x % s.slices, b = (int)(row / k.H), h = (int)(row % k.H);
  const int len = k.length(b);
  const int64_t from = (int64_t)slice * s.length;
  const int begin = from < len ? (int)from : len, end = from + s.length < len ? (int)from + s.length : len;
  const float* weights = k.row(b, h);
  const int32_t* ids = k.pages(b);
  __shared__ int sums[WAVES];
  __shared__ int cuts[3];
  K keys;
  auto rounds = [&](auto&& f) {
    for (int p = begin; p < end; p += C * K::PIECE) {
      keys.fetch(k, weights, ids, len, p, end - p < C * K::PIECE ? end : p + C * K::PIECE);
      f();
    }
  };

  if constexpr (STEP == RANGE) {
    __shared__ uint4 part[WAVES];
    Range r;
    rounds([&] { keys.each([&](uint32_t key) { r.add(key); }); });
    r.over_block(part);
    if (tid == 0) s.ranges[here] = r.packed();
    return;
  }

  Cut cut;
  if constexpr (STEP == BINS1) {
    Range r;
    if (lane < s.slices) r = Range::of(s.ranges[row * s.slices + lane]);
    r.over_wave();
    cut = Cut::first(r.lo, r.hi, r.forced, r.others, k.count);
  } else if constexpr (STEP != RANGE) {
    cut = s.cuts[row * 4 + (STEP == PLACE ? 3 : STEP - 2)];
  }
  if constexpr (STEP == BINS2 || STEP == BINS3 || STEP == COUNT) {
    if (!cut.done) {
      const int2* at = reinterpret_cast<const int2*>(s.bins + (STEP & 1 ? 0 : (int64_t)gridDim.x * kBins) + row * s.slices * kBins) +
                       kBins / 2 - 1 - tid;
      int bins[PER] = {};
#pragma unroll 8
      for (int i = 0; i < s.slices; ++i) {
        const int2 x = at[i * (kBins / 2)];
        bins[0] += x.y, bins[1] += x.x;
      }
      cut.narrow<THREADS>(bins, sums, cuts);
    }
  }
  if constexpr (STEP != PLACE) {
    if (slice == 0 && tid == 0) s.cuts[row * 4 + STEP - 1] = cut;
  }

  if constexpr (STEP == BINS1 || STEP == BINS2 || STEP == BINS3) {
    if (cut.done) return;
    __shared__ int hist[kBins];
    for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
    __syncthreads();
    const int by = cut.shift();
    rounds([&] {
      keys.each([&](uint32_t key) {
        if (key - cut.lo <= cut.hi - cut.lo) atomicAdd(&hist[(key - cut.lo) >> by], 1);
      });
    });
    __syncthreads();
    int* to = s.bins + (STEP & 1 ? (int64_t)gridDim.x * kBins : 0) + here * kBins;
    for (int i = tid; i < kBins; i += THREADS) to[i] = hist[i];
  } else if constexpr (STEP == COUNT) {
    int above = 0, equal = 0;
    rounds([&] { keys.each([&](uint32_t key) { above += key > cut.over, equal += cut.ties > 0 && key == cut.over; }); });
    __syncthreads();  // the cut's sums are read
    int all_above, all_equal;
    block_scan<THREADS>(above, sums, all_above);
    __syncthreads();
    block_scan<THREADS>(equal, sums, all_equal);
    if (tid == 0) s.numbers[here] = make_int2(all_above, all_equal);
  } else if constexpr (STEP == PLACE) {
    __shared__ int taken[2][C * WAVES + 1];
    int32_t* out = kept + row * k.count;
    int base = 0, tied = 0, all = 0, equal = 0;
    for (int i = 0; i < s.slices; ++i) {
      const int2 n = s.numbers[row * s.slices + i];
      if (i < slice) base += n.x, tied += n.y;
      all += n.x, equal += n.y;
    }
    rounds([&] {
      place<THREADS, C>(keys, cut.over, cut.ties, base, tied, taken, [&](int i, int position) { out[i] = position; });
      __syncthreads();  // the places are read
    });
    const int64_t left = all + (equal < cut.ties ? equal : cut.ties);
    for (int64_t i = left + slice * THREADS + tid; i < k.count; i += s.slices * THREADS) out[i] = -1;
  }
}

// ---------------------------------------------------------------------
// Move: a workgroup a fresh page and head, D / 8 lanes a row, four rows of a lane on
// their way at once.  Cells and scales move as they are; the page's bounds are
// those of its new rows.  A copy's bytes bound it.
// ---------------------------------------------------------------------
constexpr int kMoveRows = 4;

template <int CT>
__device__ __forceinline__ void values8(const uint32_t* w, float scale, float (&o)[8]) {
  if constexpr (CT == PFA_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(w[i]);
  } else if constexpr (CT == PFA_BF16 || CT == PFA_F16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t u = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
      o[i] = CT == PFA_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
    }
  } else if constexpr (is4(CT)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2_t y = e2m1_f32(w[0], scale, i);
      o[2 * i] = y[0], o[2 * i + 1] = y[1];
    }
  } else {
    cells8<CT>(reinterpret_cast<const typename Cell<CT>::T*>(w), o);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= scale;
  }
}

template <int BYTES>
__device__ __forceinline__ void copy_in(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (BYTES == 8) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    w[0] = a.x, w[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 a = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
    }
  }
}
template <int BYTES>
__device__ __forceinline__ void copy_out(uint8_t* p, const uint32_t* w) {
  if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

// The lanes' eight channels of kMoveRows rows on their way from slots of one page to
// slots of another.
template <int CT, int D>
struct Moving {
  static constexpr int LANES = D / 8, UB = cells_bytes(CT, 8), ROW = cells_bytes(CT, D);
  static constexpr int NS = scales_of(CT, D), PER = LANES / NS;  // scales of a row, lanes of one
  static constexpr int ES = (int)sizeof(typename Cell<CT>::T);
  int page[kMoveRows];
  uint32_t k[kMoveRows][UB / 4], v[kMoveRows][UB / 4];
  float ks[kMoveRows], vs[kMoveRows];

  // src[u]: the row's position, -1 for none
  __device__ __forceinline__ void load(const Pages& pg, const Table& from, int b, int h, const int (&src)[kMoveRows]) {
    const int lane = threadIdx.x % LANES;
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) page[u] = src[u] >= 0 ? page_at(from, pg, b, src[u] >> pg.shift) : -1;
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      if (page[u] < 0) continue;
      const int64_t slot = (int64_t)h * pg.ps + (src[u] & (pg.ps - 1));
      copy_in<UB>((const uint8_t*)pg.k + page[u] * pg.k_page * ES + slot * ROW + lane * UB, k[u]);
      copy_in<UB>((const uint8_t*)pg.v + page[u] * pg.v_page * ES + slot * ROW + lane * UB, v[u]);
      const int64_t s = (int64_t)page[u] * pg.H * pg.ps + slot;
      if constexpr (is8(CT)) ks[u] = ((const float*)pg.k_scale)[s], vs[u] = ((const float*)pg.v_scale)[s];
      if constexpr (is4(CT)) {
        ks[u] = power_of(((const uint8_t*)pg.k_scale)[s * NS + lane / PER]);
        vs[u] = power_of(((const uint8_t*)pg.v_scale)[s * NS + lane / PER]);
      }
    }
  }
  __device__ __forceinline__ void store(const Pages& pg, int id, int h, int at, int u) const {
    const int lane = threadIdx.x % LANES;
    const int64_t slot = (int64_t)h * pg.ps + at;
    copy_out<UB>((uint8_t*)pg.k + id * pg.k_page * ES + slot * ROW + lane * UB, k[u]);
    copy_out<UB>((uint8_t*)pg.v + id * pg.v_page * ES + slot * ROW + lane * UB, v[u]);
    const int64_t s = (int64_t)id * pg.H * pg.ps + slot;
    if constexpr (is8(CT)) {
      if (lane == 0) ((float*)pg.k_scale)[s] = ks[u], ((float*)pg.v_scale)[s] = vs[u];
    }
    if constexpr (is4(CT)) {
      if (lane % PER == 0) {
        ((uint8_t*)pg.k_scale)[s * NS + lane / PER] = (uint8_t)(__float_as_uint(ks[u]) >> 23);
        ((uint8_t*)pg.v_scale)[s * NS + lane / PER] = (uint8_t)(__float_as_uint(vs[u]) >> 23);
      }
    }
  }
};

template <int CT, int D>
__global__ void __launch_bounds__(256) move_kernel(Pages pg, Table from, Table to, Weights w, const int32_t* __restrict__ kept,
                                                   int count, float* __restrict__ fresh) {
  using M = Moving<CT, D>;
  constexpr int ROWS = 256 / M::LANES;
  const int b = blockIdx.z, h = blockIdx.y;
  const int64_t list = (int64_t)b * pg.H + h;
  // the weights of the kept ones, and zeros behind them
  const float* weights = w.p + b * w.s_b + h * w.s_h;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < w.T; i += (int64_t)gridDim.x * 256) {
    const int src = i < count ? kept[list * count + i] : -1;
    fresh[list * w.T + i] = src >= 0 ? weights[src] : 0.0f;
  }
  __shared__ float part[2][4][D];
  for (int64_t ordinal = blockIdx.x; ordinal << pg.shift < count; ordinal += gridDim.x) {
    const int64_t at = ordinal << pg.shift;
    const int id = page_at(to, pg, b, ordinal);
    if (id < 0 || kept[list * count + at] < 0) continue;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    for (int r0 = threadIdx.x / M::LANES; r0 < pg.ps; r0 += kMoveRows * ROWS) {
      int src[kMoveRows];
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        const int r = r0 + u * ROWS;
        src[u] = r < pg.ps && at + r < count ? kept[list * count + at + r] : -1;
      }
      M m;
      m.load(pg, from, b, h, src);
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        if (m.page[u] < 0) continue;
        m.store(pg, id, h, r0 + u * ROWS, u);
        if (pg.bounds) {
          float x[8];
          values8<CT>(m.k[u], scaled(CT) ? m.ks[u] : 1.0f, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) lo[j] = min_nan(lo[j], x[j]), hi[j] = max_nan(hi[j], x[j]);
        }
      }
    }
    if (pg.bounds) {
      constexpr int BT = bound_dtype(CT);
      auto* out = (typename Elem<BT>::T*)pg.bounds + ((int64_t)id * pg.H + h) * 2 * D;
      join_bounds<D>(lo, hi, part, [&](int d, float a, float z) {
        store_f<BT>(out + d, a);
        store_f<BT>(out + D + d, z);
      });
    }
  }
}

// Both in one workgroup for a few rows without bounds, with the kept positions in LDS: a
// launch less, which is 3.6 us of the host (8 rows of 700 positions, 512 kept, 256 bytes
// each: 15.4 us a call, 11.8 so).  One unit moves 128 KB in 4 us; with more of it than
// kSmallBytes the launch is the cheaper.  It also fills the weights behind the kept ones,
// which may be many more than the table has positions: beyond kSmallFill of them the launch
// is the cheaper where rows leave units free (8 rows, 4,096 positions, weights of 16,384:
// 12.6 us in one launch, 12.9 in two; of 65,536 18.3 and 13.1; of 1,048,576 130 and 18.5;
// 64 rows of 1,048,576: 132 and 70), but not from kSmallRows on (128 rows of 32,768: 15.0
// and 19.2, of 1,048,576 136 and 137; 512 rows: 26.4 and 44.5, 396 and 523).
constexpr int kSmall = 1024;
constexpr int64_t kSmallBytes = 256 << 10;
constexpr int64_t kSmallFill = 16384;
constexpr int kSmallRows = 128;
template <int CT, int D>
__global__ void __launch_bounds__(1024) evict_kernel(Keep k, Pages pg, Table to, int32_t* __restrict__ kept,
                                                     float* __restrict__ fresh) {
  using M = Moving<CT, D>;
  constexpr int ROWS = 1024 / M::LANES;
  const int b = blockIdx.x / pg.H, h = blockIdx.x % pg.H;
  const Weights& w = k.w;
  __shared__ int32_t list[kSmall];
  int32_t* out = kept + (int64_t)blockIdx.x * k.count;
  choose_tokens<1024, 1>(k, b, h, [&](int i, int position) { out[i] = list[i] = position; });
  __syncthreads();
  const float* weights = w.p + b * w.s_b + h * w.s_h;
  for (int i = threadIdx.x; i < w.T; i += 1024) {
    const int src = i < k.count ? list[i] : -1;
    fresh[(int64_t)blockIdx.x * w.T + i] = src >= 0 ? weights[src] : 0.0f;
  }
  for (int i0 = threadIdx.x / M::LANES; i0 < k.count; i0 += kMoveRows * ROWS) {
    int src[kMoveRows], id[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      const int i = i0 + u * ROWS;
      id[u] = i < k.count ? page_at(to, pg, b, i >> pg.shift) : -1;
      src[u] = id[u] >= 0 ? list[i] : -1;
    }
    M m;
    m.load(pg, k.tab, b, h, src);
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
      if (m.page[u] >= 0) m.store(pg, id[u], h, (i0 + u * ROWS) & (pg.ps - 1), u);
  }
}

int tokens_check(const char* what, const float* weights, int64_t n, int B, int H, int count, int first, int last) {
  PFA_CHECK_ARG(B >= 0 && B <= 65535 && H > 0 && H <= 65535, "%s: 0 to 65535 sequences and 1 to 65535 heads", what);
  PFA_CHECK_ARG((int64_t)B * H <= 1 << 21, "%s: up to 2^21 rows (got %d x %d)", what, B, H);
  PFA_CHECK_ARG(n >= 0 && n <= 1 << 30, "%s: weights of up to 2^30 positions", what);
  PFA_CHECK_ARG(count > 0 && count <= 1 << 30 && first >= 0 && last >= 0 && first <= count && last <= count - first,
                "%s: count > 0 tokens, the %d first and %d last among them (got %d)", what, first, last, count);
  PFA_CHECK_ARG((weights || n == 0 || B == 0) && (uintptr_t)weights % 4 == 0, "%s: null or unaligned weights", what);
  return PFA_OK;
}

// Slices of rows of `most` positions; none of those that a workgroup holds.
Split split_of(int64_t rows, int64_t most) {
  Split s{};
  if (most <= kHeld || rows == 0) return s;
  int64_t slices = kEnough / rows;
  slices = slices < 1 ? 1 : slices > kSlices ? kSlices : slices;
  const int64_t length = ((most + slices - 1) / slices + 4095) / 4096 * 4096;
  s.slices = (int)((most + length - 1) / length), s.length = (int)length;
  return s;
}
size_t split_bytes(int64_t rows, const Split& s) {
  return (size_t)rows * (s.slices * (sizeof(uint4) + 2 * kBins * sizeof(int) + sizeof(int2)) +
                         (s.slices ? 4 * sizeof(Cut) : 0));
}

int choose_launch(const char* what, const Keep& k, int rows, int32_t* kept, void* workspace, size_t ws_bytes,
                  hipStream_t stream) {
#define PFA_CHOOSE(THREADS, C) choose_tokens_kernel<THREADS, C><<<rows, THREADS, 0, stream>>>(k, kept)
  Split s = split_of(rows, k.w.most);
  if (s.slices) {
    const size_t need = split_bytes(rows, s);
    if (ws_bytes < need || !workspace || (uintptr_t)workspace % 16 != 0) {
      set_error("%s: workspace of %zu bytes, %zu needed, 16-byte aligned", what, ws_bytes, need);
      return PFA_E_WORKSPACE;
    }
    const int64_t all = (int64_t)rows * s.slices;
    s.bins = (int*)workspace;
    s.ranges = (uint4*)(s.bins + 2 * all * kBins);
    s.numbers = (int2*)(s.ranges + all);
    s.cuts = (Cut*)(s.numbers + all);
    split_kernel<RANGE><<<(unsigned)all, 1024, 0, stream>>>(k, s, kept);
    split_kernel<BINS1><<<(unsigned)all, 1024, 0, stream>>>(k, s, kept);
    split_kernel<BINS2><<<(unsigned)all, 1024, 0, stream>>>(k, s, kept);
    split_kernel<BINS3><<<(unsigned)all, 1024, 0, stream>>>(k, s, kept);
    split_kernel<COUNT><<<(unsigned)all, 1024, 0, stream>>>(k, s, kept);
    split_kernel<PLACE><<<(unsigned)all, 1024, 0, stream>>>(k, s, kept);
  } else if (k.w.most <= 256 * 4) {
    PFA_CHOOSE(256, 1);
  } else if (k.w.most <= 1024 * 4) {
    PFA_CHOOSE(1024, 1);
  } else if (k.w.most <= 1024 * 16) {
    PFA_CHOOSE(1024, 4);
  } else if (k.w.most <= 1024 * 32) {
    PFA_CHOOSE(1024, 8);
  } else {
    PFA_CHOOSE(1024, 16);
  }
#undef PFA_CHOOSE
  return PFA_OK;
}

}  // namespace
}  // namespace pfa

using namespace pfa;

extern "C" int pfa_kv_tokens_workspace_size(int B, int H, int64_t n, size_t* bytes) {
  clear_error();
  PFA_CHECK_ARG(bytes, "kv_tokens: null argument");
  if (int rc = tokens_check("kv_tokens", nullptr, 0, B, H, 1, 0, 0)) return rc;
  PFA_CHECK_ARG(n >= 0 && n <= 1 << 30, "kv_tokens: weights of up to 2^30 positions");
  *bytes = split_bytes((int64_t)B * H, split_of((int64_t)B * H, n));
  return PFA_OK;
}

extern "C" int pfa_kv_tokens_select(const float* weights, int64_t weights_b, int64_t weights_h, int64_t n, int B, int H,
                                    const int32_t* lengths, int count, int first, int last, int32_t* kept, void* workspace,
                                    size_t ws_bytes, void* stream) {
  clear_error();
  if (int rc = tokens_check("kv_tokens_select", weights, n, B, H, count, first, last)) return rc;
  if (B == 0) return PFA_OK;
  PFA_CHECK_ARG(lengths && kept, "kv_tokens_select: null argument");
  const bool vec = (uintptr_t)weights % 16 == 0 && weights_b % 4 == 0 && weights_h % 4 == 0 && n % 4 == 0;
  const Keep keep{Weights{weights, weights_b, weights_h, (int)n, (int)n, vec}, Table{nullptr, 0, 0}, 0, 0, H, lengths, count,
                  first, last};
  if (int rc = choose_launch("kv_tokens_select", keep, B * H, kept, workspace, ws_bytes, as_stream(stream))) return rc;
  PFA_CHECK_LAUNCH("kv_tokens_select");
  return PFA_OK;
}

extern "C" int pfa_kv_tokens_evict(const pfa_kv_evict* c, void* stream) {
  clear_error();
  PFA_CHECK_ARG(c, "kv_tokens_evict: null argument");
  const int B = c->B, count = c->count;
  const float* weights = c->weights;
  const int64_t n = c->n;
  int32_t* kept = c->kept;
  float* fresh = c->fresh;
  Pages p;
  Table from, to;
  if (int rc = paged_check(&c->pages, c->into, c->into_stride, c->into_pages, B, &p, &to)) return rc;
  if (int rc = paged_check(&c->pages, c->table, c->table_stride, c->table_pages, B, &p, &from)) return rc;
  if (int rc = tokens_check("kv_tokens_evict", weights, n, B, p.H, count, c->first, c->last)) return rc;
  if (B == 0) return PFA_OK;
  PFA_CHECK_ARG(c->lengths && kept && (fresh || n == 0), "kv_tokens_evict: null argument");
  const bool vec = (uintptr_t)weights % 16 == 0 && c->weights_b % 4 == 0 && c->weights_h % 4 == 0 && n % 4 == 0;
  hipStream_t s = as_stream(stream);
  const int64_t held = (int64_t)from.P << p.shift;
  const Weights w{weights, c->weights_b, c->weights_h, (int)n, (int)(held < n ? held : n), vec};
  const Keep keep{w, from, p.shift, p.n_pages, p.H, c->lengths, count, c->first, c->last};
  const int64_t bytes = (int64_t)count * 2 * cells_bytes(c->pages.dtype, c->pages.head_dim);
  const bool small = !p.bounds && count <= kSmall && w.most <= 1024 * 4 && bytes <= kSmallBytes &&
                     (n <= kSmallFill || B * p.H >= kSmallRows);
  if (!small)
    if (int rc = choose_launch("kv_tokens_evict", keep, B * p.H, kept, c->workspace, c->ws_bytes, s)) return rc;
  // a workgroup a page, but no more than 4,096 of the weights to each (8 rows of
  // 1,048,576, two pages of 256 kept: the move takes 330 us with two workgroups a row, 49 so)
  const int64_t fresh_pages = ((int64_t)count + p.ps - 1) >> p.shift, fills = (n + 4095) / 4096;
  const int64_t blocks = fresh_pages > fills ? fresh_pages : fills;
  const dim3 grid((unsigned)(blocks < 65535 ? blocks : 65535), p.H, B);
  by_cells(c->pages.dtype, [&](auto ct) {
    by_width(c->pages.head_dim, [&](auto width) {
      constexpr int CT = decltype(ct)::value, D = decltype(width)::value;
      if (small) evict_kernel<CT, D><<<B * p.H, 1024, 0, s>>>(keep, p, to, kept, fresh);
      else move_kernel<CT, D><<<grid, 256, 0, s>>>(p, from, to, w, kept, count, fresh);
    });
  });
  PFA_CHECK_LAUNCH("kv_tokens_evict");
  return PFA_OK;
}
