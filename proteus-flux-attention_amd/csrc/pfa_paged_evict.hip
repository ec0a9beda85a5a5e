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
// Choice: a workgroup a sequence and head, choose_best over its weights' bits in
// order.  Positions without a page (where there is a table) are no candidates.
// ---------------------------------------------------------------------
template <int THREADS, int K, bool HELD>
__global__ void __launch_bounds__(THREADS) choose_tokens_kernel(Weights w, Table tab, int shift, int n_pages, int H,
                                                                const int32_t* __restrict__ lengths, int count, int first,
                                                                int last, int32_t* __restrict__ kept,
                                                                float* __restrict__ fresh) {
  const int b = blockIdx.x / H, h = blockIdx.x % H;
  const float* row = w.p + b * w.s_b + h * w.s_h;
  const int n = lengths[b], len = n < 0 ? 0 : n < w.most ? n : w.most;
  const int32_t* ids = tab.ids ? tab.ids + b * tab.stride : nullptr;
  int32_t* out = kept + (int64_t)blockIdx.x * count;
  float* moved = fresh ? fresh + (int64_t)blockIdx.x * w.T : nullptr;
  const int rounds = HELD ? 1 : (len + THREADS * K - 1) / (THREADS * K);
  auto fetch = [&](int r, uint32_t (&x)[K]) {
    const int p0 = (r * THREADS + (int)threadIdx.x) * K;
    float v[K];
#pragma unroll
    for (int i = 0; i < K; i += 4) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      const int p = p0 + i;
      if (w.vec) {
        if (p < len) a = *reinterpret_cast<const float4*>(row + p);
      } else {
        if (p < len) a.x = row[p];
        if (p + 1 < len) a.y = row[p + 1];
        if (p + 2 < len) a.z = row[p + 2];
        if (p + 3 < len) a.w = row[p + 3];
      }
      v[i] = a.x, v[i + 1] = a.y, v[i + 2] = a.z, v[i + 3] = a.w;
    }
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int p = p0 + i;
      uint32_t u = v[i] == 0.0f ? 0u : __float_as_uint(v[i]);  // -0 ties with +0
      u = u & 0x80000000u ? ~u : u | 0x80000000u;
      if (v[i] != v[i]) u = kNan;
      if (p < first || len - p <= last) u = kForced;
      x[i] = p < len ? u : kNone;
    }
    if (ids) {  // pages hold 16 tokens or more
#pragma unroll
      for (int i = 0; i < K; i += K < 16 ? K : 16) {
        const bool gone = p0 + i < len && (uint32_t)ids[(p0 + i) >> shift] >= (uint32_t)n_pages;
#pragma unroll
        for (int j = 0; j < (K < 16 ? K : 16); ++j) x[i + j] = gone ? kNone : x[i + j];
      }
    }
  };
  choose_best<THREADS, K, HELD>(0, rounds, count, fetch, [&](int i, int entry) {
    out[i] = entry;
    if (moved && i < w.T) moved[i] = entry >= 0 ? row[entry] : 0.0f;
  });
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

template <int CT, int D>
__global__ void __launch_bounds__(256) move_kernel(Pages pg, Table from, Table to, const int32_t* __restrict__ kept, int count,
                                                   float* __restrict__ fresh, int T) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES, UB = cells_bytes(CT, 8), ROW = cells_bytes(CT, D);
  constexpr int NS = scales_of(CT, D), PER = LANES / NS;  // scales of a row, lanes of one
  constexpr int ES = (int)sizeof(typename Cell<CT>::T);
  const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x % LANES;
  const int64_t list = (int64_t)b * pg.H + h;
  // the weights behind the kept ones
  for (int64_t i = count + (int64_t)blockIdx.x * 256 + threadIdx.x; i < T; i += (int64_t)gridDim.x * 256)
    fresh[list * T + i] = 0.0f;
  __shared__ float part[2][4][D];
  for (int64_t ordinal = blockIdx.x; ordinal << pg.shift < count; ordinal += gridDim.x) {
    const int64_t at = ordinal << pg.shift;
    const int id = page_at(to, pg, b, ordinal);
    if (id < 0 || kept[list * count + at] < 0) continue;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    for (int r0 = threadIdx.x / LANES; r0 < pg.ps; r0 += kMoveRows * ROWS) {
      int src[kMoveRows];
      int page[kMoveRows];
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        const int r = r0 + u * ROWS;
        src[u] = r < pg.ps && at + r < count ? kept[list * count + at + r] : -1;
      }
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) page[u] = src[u] >= 0 ? page_at(from, pg, b, src[u] >> pg.shift) : -1;
      uint32_t k[kMoveRows][UB / 4], v[kMoveRows][UB / 4];
      [[maybe_unused]] float ks[kMoveRows], vs[kMoveRows];
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
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        if (page[u] < 0) continue;
        const int64_t slot = (int64_t)h * pg.ps + r0 + u * ROWS;
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
        if (pg.bounds) {
          float x[8];
          values8<CT>(k[u], scaled(CT) ? ks[u] : 1.0f, x);
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

int tokens_check(const char* what, const float* weights, int64_t n, int B, int H, int count, int first, int last) {
  PFA_CHECK_ARG(B >= 0 && B <= 65535 && H > 0 && H <= 65535, "%s: 0 to 65535 sequences and 1 to 65535 heads", what);
  PFA_CHECK_ARG((int64_t)B * H <= 1 << 21, "%s: up to 2^21 rows (got %d x %d)", what, B, H);
  PFA_CHECK_ARG(n >= 0 && n <= 1 << 30, "%s: weights of up to 2^30 positions", what);
  PFA_CHECK_ARG(count > 0 && count <= 1 << 30 && first >= 0 && last >= 0 && first <= count && last <= count - first,
                "%s: count > 0 tokens, the %d first and %d last among them (got %d)", what, first, last, count);
  PFA_CHECK_ARG((weights || n == 0 || B == 0) && (uintptr_t)weights % 4 == 0, "%s: null or unaligned weights", what);
  return PFA_OK;
}

void choose_tokens(const Weights& w, const Table& t, int shift, int n_pages, int B, int H, const int32_t* lengths, int count,
                   int first, int last, int32_t* kept, float* fresh, hipStream_t stream) {
#define PFA_CHOOSE(THREADS, K, HELD)                                                                                    \
  choose_tokens_kernel<THREADS, K, HELD><<<B * H, THREADS, 0, stream>>>(w, t, shift, n_pages, H, lengths, count, first, \
                                                                        last, kept, fresh)
  if (w.most <= 256 * 4) PFA_CHOOSE(256, 4, true);
  else if (w.most <= 1024 * 4) PFA_CHOOSE(1024, 4, true);
  else if (w.most <= 1024 * 16) PFA_CHOOSE(1024, 16, true);
  else PFA_CHOOSE(1024, 16, false);
#undef PFA_CHOOSE
}

}  // namespace
}  // namespace pfa

using namespace pfa;

extern "C" int pfa_kv_tokens_select(const float* weights, int64_t weights_b, int64_t weights_h, int64_t n, int B, int H,
                                    const int32_t* lengths, int count, int first, int last, int32_t* kept, void* stream) {
  clear_error();
  if (int rc = tokens_check("kv_tokens_select", weights, n, B, H, count, first, last)) return rc;
  if (B == 0) return PFA_OK;
  PFA_CHECK_ARG(lengths && kept, "kv_tokens_select: null argument");
  const bool vec = (uintptr_t)weights % 16 == 0 && weights_b % 4 == 0 && weights_h % 4 == 0 && n % 4 == 0;
  choose_tokens(Weights{weights, weights_b, weights_h, (int)n, (int)n, vec}, Table{nullptr, 0, 0}, 0, 0, B, H, lengths, count, first,
                last, kept, nullptr, as_stream(stream));
  PFA_CHECK_LAUNCH("kv_tokens_select");
  return PFA_OK;
}

extern "C" int pfa_kv_tokens_evict(const pfa_kv_pages* pages, const float* weights, int64_t weights_b, int64_t weights_h,
                                   int64_t n, int B, const int32_t* table, int64_t table_stride, int table_pages,
                                   const int32_t* lengths, int count, int first, int last, const int32_t* into,
                                   int64_t into_stride, int into_pages, int32_t* kept, float* fresh, void* stream) {
  clear_error();
  Pages p;
  Table from, to;
  if (int rc = paged_check(pages, into, into_stride, into_pages, B, &p, &to)) return rc;
  if (int rc = paged_check(pages, table, table_stride, table_pages, B, &p, &from)) return rc;
  if (int rc = tokens_check("kv_tokens_evict", weights, n, B, p.H, count, first, last)) return rc;
  PFA_CHECK_ARG((int64_t)into_pages << p.shift >= count, "kv_tokens_evict: %d tokens into %d pages of %d", count, into_pages,
                p.ps);
  if (B == 0) return PFA_OK;
  PFA_CHECK_ARG(lengths && kept && (fresh || n == 0), "kv_tokens_evict: null argument");
  const bool vec = (uintptr_t)weights % 16 == 0 && weights_b % 4 == 0 && weights_h % 4 == 0 && n % 4 == 0;
  hipStream_t s = as_stream(stream);
  const int64_t held = (int64_t)table_pages << p.shift;
  const Weights w{weights, weights_b, weights_h, (int)n, (int)(held < n ? held : n), vec};
  choose_tokens(w, from, p.shift, p.n_pages, B, p.H, lengths, count, first, last, kept, fresh, s);
  const int64_t fresh_pages = ((int64_t)count + p.ps - 1) >> p.shift;
  const dim3 grid((unsigned)(fresh_pages < 65535 ? fresh_pages : 65535), p.H, B);
  by_cells(pages->dtype, [&](auto ct) {
    by_width(pages->head_dim, [&](auto width) {
      move_kernel<decltype(ct)::value, decltype(width)::value>
          <<<grid, 256, 0, s>>>(p, from, to, kept, count, fresh, (int)n);
    });
  });
  PFA_CHECK_LAUNCH("kv_tokens_evict");
  return PFA_OK;
}
