// Paged key-value cache: write, read, page selection and the attention of one
// new token over it.
#include "pfa_paged.h"
#include "pfa_paged_attn.h"
#include "pfa_paged_select.h"

namespace pfa {

using namespace paged;

static int shift_of(int page_size) {
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  return shift;
}

static int sizes_check(int kv_heads, int page_size, int head_dim, int dtype, int table_pages, int B) {
  PFA_CHECK_ARG(dtype == PFA_F32 || dtype == PFA_BF16 || dtype == PFA_F16 || scaled(dtype), "pages: unknown cell type %d",
                dtype);
  PFA_CHECK_ARG(head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128,
                "pages: head_dim must be 16, 32, 64 or 128 (got %d)", head_dim);
  PFA_CHECK_ARG(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
                "pages: page_size must be 16, 32, 64, 128 or 256 (got %d)", page_size);
  PFA_CHECK_ARG(kv_heads > 0 && kv_heads <= 65535, "pages: 1 to 65535 heads (got %d)", kv_heads);
  PFA_CHECK_ARG(B >= 0 && B <= 65535, "pages: 0 <= B <= 65535 sequences (got %d)", B);
  PFA_CHECK_ARG(table_pages >= 0 && (int64_t)table_pages * page_size <= (1ll << 30),
                "pages: a block table of up to 2^30 positions (got %d pages)", table_pages);
  return PFA_OK;
}

int paged_check(const pfa_kv_pages* pg, const int32_t* table, int64_t table_stride, int table_pages, int B, Pages* p,
                Table* t) {
  PFA_CHECK_ARG(pg, "pages: null argument");
  if (int rc = sizes_check(pg->kv_heads, pg->page_size, pg->head_dim, pg->dtype, table_pages, B)) return rc;
  PFA_CHECK_ARG(pg->n_pages > 0 && pg->k && pg->v, "pages: an empty pool");
  PFA_CHECK_ARG(!scaled(pg->dtype) || (pg->k_scale && pg->v_scale), "pages: cells of 8 or 4 bits need k_scale and v_scale");
  const int64_t cells = (int64_t)pg->kv_heads * pg->page_size * cells_at(pg->dtype, pg->head_dim);
  const int e = is4(pg->dtype) ? 1 : cells_bytes(pg->dtype, 1);
  PFA_CHECK_ARG(pg->n_pages == 1 || (pg->k_page >= cells && pg->v_page >= cells), "pages: pages overlap");
  PFA_CHECK_ARG((uintptr_t)pg->k % 16 == 0 && (uintptr_t)pg->v % 16 == 0 && pg->k_page * e % 16 == 0 &&
                    pg->v_page * e % 16 == 0 && (uintptr_t)pg->k_scale % 16 == 0 && (uintptr_t)pg->v_scale % 16 == 0 &&
                    (uintptr_t)pg->k_bounds % 16 == 0,
                "pages: rows must be 16-byte aligned");
  PFA_CHECK_ARG(table || table_pages == 0 || B == 0, "pages: null argument");
  *p = Pages{pg->k, pg->v, pg->k_scale, pg->v_scale, pg->k_bounds, pg->k_page, pg->v_page,
             pg->n_pages, pg->kv_heads, pg->page_size, shift_of(pg->page_size)};
  *t = Table{table, table_stride, table_pages};
  return PFA_OK;
}

namespace {

// ---------------------------------------------------------------------
// Write.  A workgroup takes the tokens of one page and head.  D / 8 lanes
// hold a row, eight values each: absmax by lane exchanges, the cells in one
// store, the page's bounds in registers over the rows and joined over the
// lanes and waves at the end, so no atomics and the same bits in any split of
// the tokens over calls.
//
// A copy's bytes bound it, if the arithmetic stays out of the way: quotients by
// the row's scale come from its one reciprocal with two corrections by fused
// multiply-adds (Markstein 1990), the same bits as a division in 5 instructions
// for 11, and int8 from the sum with 1.5 * 2^23, whose low bits are the rounded
// quotient.  25,600 rows of 8 heads of 128 bf16 values into int8 pages with bounds:
// 41 to 52 us, 162 MB (58 with divisions and selects for NaN).
// ---------------------------------------------------------------------
// The largest over 2, 4, 8 or 16 lanes that lie together.
template <int LANES>
__device__ __forceinline__ float max_lanes(float x) {
  auto step = [&](auto ctrl) {
    x = max_nan(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  step(std::integral_constant<int, 0xB1>{});                             // the neighbour
  if constexpr (LANES > 2) step(std::integral_constant<int, 0x4E>{});   // the other pair
  if constexpr (LANES > 4) step(std::integral_constant<int, 0x141>{});  // mirrored in eight
  if constexpr (LANES > 8) step(std::integral_constant<int, 0x140>{});  // mirrored in sixteen
  return x;
}

struct NewRows {
  const void* p;
  int64_t s_b, s_h, s_t;
  int vec;  // rows aligned to eight elements
};

template <int DT>
__device__ __forceinline__ void row8(const NewRows& r, int64_t at, float (&o)[8]) {
  using T = typename Elem<DT>::T;
  const T* p = (const T*)r.p + at;
  if (r.vec) load8<DT>(p, o);
  else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = load_f<DT>(p + i);
  }
}

// Eight values, from channel 8 * lane on of a row of LANES lanes, into its cells; with
// `back`, x comes back as the values that the cells stand for.
template <int CT, int LANES>
__device__ __forceinline__ void put8(typename Cell<CT>::T* dst, void* scales, int64_t slot, int lane, bool back,
                                     float (&x)[8]) {
  if constexpr (!scaled(CT)) {
    store8<CT>(dst, x);
  } else if constexpr (is4(CT)) {
    // a group's scale is a power of two, so that the quotients are exact and the
    // hardware's rounding to nearest even, saturating at 6, is the only one
    constexpr int GROUP = LANES < 4 ? LANES : 4;
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(x[i]));
    m = max_lanes<GROUP>(m);
    const bool ok = m < INFINITY;
    const uint32_t p = ok ? power_for(m) : kNanPower;
    if (lane % GROUP == 0) ((uint8_t*)scales)[slot * (LANES / GROUP) + lane / GROUP] = (uint8_t)p;
    const float s = power_of(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ok ? x[i] : 0.0f;
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
    if (!ok) w = 0;  // whatever a scale that is NaN makes of it
    if (back) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2_t y = e2m1_f32(w, s, i);
        x[2 * i] = y[0], x[2 * i + 1] = y[1];
      }
    }
    *reinterpret_cast<uint32_t*>(dst) = w;
  } else {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(x[i]));
    m = max_lanes<LANES>(m);
    const bool ok = m < INFINITY;
    const float s = ok ? fmaxf(m / top_of(CT), kLeastScale) : __builtin_nanf("");
    if (lane == 0) ((float*)scales)[slot] = s;
    // x / s to nearest: s >= 1e-6 and at most 448 in size, so that nothing that
    // decides a cell underflows
    const float y = 1.0f / s;
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = x[i] * y;
      q = fmaf(fmaf(-q, s, x[i]), y, q);
      q = fmaf(fmaf(-q, s, x[i]), y, q);
      if constexpr (CT == PFA_E4M3) q = copysignf(q, x[i]);  // -0 loses its sign in the corrections
      c[i] = ok ? q : 0.0f;
    }
    uint32_t w[2];
    if constexpr (CT == PFA_I8) {
      constexpr float kRound = 12582912.0f;  // 1.5 * 2^23
      uint32_t u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float r = c[i] + kRound;
        u[i] = __float_as_uint(r);
        if (back) x[i] = (r - kRound) * s;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t a = __builtin_amdgcn_perm(u[4 * i + 1], u[4 * i], 0x0c0c0400);
        const uint32_t b = __builtin_amdgcn_perm(u[4 * i + 3], u[4 * i + 2], 0x0c0c0400);
        w[i] = a | b << 16;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * i], c[4 * i + 1], 0, false);
        p = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * i + 2], c[4 * i + 3], p, true);
        w[i] = (uint32_t)p;
        if (back) {
          x[4 * i] = __builtin_amdgcn_cvt_f32_fp8(p, 0) * s;
          x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(p, 1) * s;
          x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(p, 2) * s;
          x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(p, 3) * s;
        }
      }
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  }
}

template <int DT, int CT, int D>
__global__ void __launch_bounds__(1024) write_kernel(Pages pg, Table tab, NewRows k, NewRows v, int64_t n,
                                                    int64_t units,
                                                    const int32_t* __restrict__ starts,
                                                    const int32_t* __restrict__ counts) {
  using CellT = typename Cell<CT>::T;
  constexpr int LANES = D / 8;
  const int64_t b = blockIdx.y;
  const int64_t start = starts[b];
  int64_t count = counts ? (int64_t)counts[b] : n;
  count = count < 0 ? 0 : count < n ? count : n;
  const int64_t first = start < 0 ? 0 : start;  // positions written: [first, end)
  const int64_t end = start + count;
  const int lane = threadIdx.x % LANES, rows = blockDim.x / LANES;
  const bool back = pg.bounds != nullptr;
  __shared__ float part[2][16][D];
  // heads of one page are neighbours, as their new rows are in memory
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int64_t touched = quotient(unit, pg.H);
    const int h = (int)(unit - touched * pg.H);
    const int64_t ordinal = (first >> pg.shift) + touched, base = ordinal << pg.shift;
    const int64_t from = first > base ? first : base, to = end < base + pg.ps ? end : base + pg.ps;
    if (from >= to) continue;
    const int id = page_at(tab, pg, b, ordinal);
    if (id < 0) continue;

    constexpr int ROW = cells_at(CT, D), UNIT = cells_at(CT, 8);
    const int64_t kpage = id * pg.k_page + (int64_t)h * pg.ps * ROW, vpage = id * pg.v_page + (int64_t)h * pg.ps * ROW;
    const int64_t spage = ((int64_t)id * pg.H + h) * pg.ps;
    const int64_t k_at = b * k.s_b + h * k.s_h + 8 * lane, v_at = b * v.s_b + h * v.s_h + 8 * lane;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    for (int64_t pos = from + threadIdx.x / LANES; pos < to; pos += rows) {
      const int slot = (int)(pos - base);
      const int64_t i = pos - start;
      float x[8], y[8];
      row8<DT>(k, k_at + i * k.s_t, x);
      row8<DT>(v, v_at + i * v.s_t, y);
      put8<CT, LANES>((CellT*)pg.k + kpage + slot * ROW + UNIT * lane, pg.k_scale, spage + slot, lane, back, x);
      put8<CT, LANES>((CellT*)pg.v + vpage + slot * ROW + UNIT * lane, pg.v_scale, spage + slot, lane, false, y);
      if (back) {
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = min_nan(lo[j], x[j]), hi[j] = max_nan(hi[j], x[j]);
      }
    }
    if (!back) continue;
    constexpr int BT = bound_dtype(CT);
    using BoundT = typename Elem<BT>::T;
    BoundT* out = (BoundT*)pg.bounds + ((int64_t)id * pg.H + h) * 2 * D;
    join_bounds<D>(lo, hi, part, [&](int d, float a, float z) {
      if (from > base) a = min_nan(a, load_f<BT>(out + d)), z = max_nan(z, load_f<BT>(out + D + d));
      store_f<BT>(out + d, a);
      store_f<BT>(out + D + d, z);
    });
  }
}

// ---------------------------------------------------------------------
// Read: eight values a thread and row, one row or two of each of k and v at
// once, rows in the output's order.  A copy's bytes bound it.  The place of a workgroup's
// first row is divided out once for all its threads.
// ---------------------------------------------------------------------
// 262,144 rows of 8 heads of 128 e4m3 cells into bf16: two rows 305 us, one 320;
// 25,600 of int8 into f32: 67 and 59; 3,000 of 8 heads of 32 bf16: 5.0 and 4.2.
__host__ __device__ constexpr int read_rows(int ct, int ot) { return scaled(ct) && ot != PFA_F32 ? 2 : 1; }

template <int CT, int OT, int D>
__global__ void __launch_bounds__(256) read_kernel(Pages pg, Table tab, int64_t n, int64_t blocks,
                                                   const int32_t* __restrict__ starts,
                                                   const int32_t* __restrict__ counts, void* __restrict__ k_out,
                                                   void* __restrict__ v_out) {
  using CellT = typename Cell<CT>::T;
  using OutT = typename Elem<OT>::T;
  constexpr int LANES = D / 8, ROWS = 256 / LANES, kReadRows = read_rows(CT, OT);
  const int64_t b = blockIdx.y, rows = n * pg.H;
  const int64_t start = starts[b];
  int64_t count = counts ? (int64_t)counts[b] : n;
  const int lane = threadIdx.x % LANES;
  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const int64_t r0 = block * (ROWS * kReadRows), i0 = quotient(r0, pg.H);
    const uint32_t h0 = (uint32_t)(r0 - i0 * pg.H);
    float x[kReadRows][8], y[kReadRows][8];
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
      const uint32_t at = threadIdx.x / LANES + u * ROWS;
      const uint32_t skip = (h0 + at) / (uint32_t)pg.H;
      const int h = (int)(h0 + at - skip * pg.H);
      const int64_t i = i0 + skip, pos = start + i;
      const int id = i < n && i < count && pos >= 0 ? page_at(tab, pg, b, pos >> pg.shift) : -1;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[u][j] = y[u][j] = 0.0f;
      if (id >= 0) {
        const int64_t slot = (int64_t)h * pg.ps + (pos & (pg.ps - 1));
        constexpr int ROW = cells_at(CT, D), UNIT = cells_at(CT, 8);
        const CellT* kp = (const CellT*)pg.k + id * pg.k_page + slot * ROW + UNIT * lane;
        const CellT* vp = (const CellT*)pg.v + id * pg.v_page + slot * ROW + UNIT * lane;
        const int64_t s = (int64_t)id * pg.H * pg.ps + slot;
        if constexpr (is4(CT)) {
          constexpr int NS = scales_of(CT, D);
          const float a = power_of(((const uint8_t*)pg.k_scale)[s * NS + lane / (LANES / NS)]);
          const float c = power_of(((const uint8_t*)pg.v_scale)[s * NS + lane / (LANES / NS)]);
          const uint32_t kw = *reinterpret_cast<const uint32_t*>(kp), vw = *reinterpret_cast<const uint32_t*>(vp);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x2_t p = e2m1_f32(kw, a, j), q = e2m1_f32(vw, c, j);
            x[u][2 * j] = p[0], x[u][2 * j + 1] = p[1], y[u][2 * j] = q[0], y[u][2 * j + 1] = q[1];
          }
        } else {
          cells8<CT>(kp, x[u]);
          cells8<CT>(vp, y[u]);
        }
        if constexpr (is8(CT)) {
          const float a = ((const float*)pg.k_scale)[s], c = ((const float*)pg.v_scale)[s];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[u][j] *= a, y[u][j] *= c;
            // f16: the product is rounded to f32 before its rounding to 16 bits, as
            // with the other types (v_fma_mixlo_f16 would do with one)
            if constexpr (OT == PFA_F16) asm("" : "+v"(x[u][j]), "+v"(y[u][j]));
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
      const int64_t r = r0 + threadIdx.x / LANES + u * ROWS;
      if (r >= rows) continue;
      const int64_t to = (b * rows + r) * D + 8 * lane;
      store8<OT>((OutT*)k_out + to, x[u]);
      store8<OT>((OutT*)v_out + to, y[u]);
    }
  }
}

// Calls f with the (values, cells) types as template arguments: the cells' own
// float type, or any of the three with cells of 8 or 4 bits.
template <typename F>
void by_types(int dt, int ct, F&& f) {
#define PFA_PAIR(A, C) \
  if (dt == A && ct == C) return f(std::integral_constant<int, A>{}, std::integral_constant<int, C>{});
  PFA_PAIR(PFA_F32, PFA_F32) PFA_PAIR(PFA_BF16, PFA_BF16) PFA_PAIR(PFA_F16, PFA_F16)
  PFA_PAIR(PFA_F32, PFA_I8) PFA_PAIR(PFA_BF16, PFA_I8) PFA_PAIR(PFA_F16, PFA_I8)
  PFA_PAIR(PFA_F32, PFA_E4M3) PFA_PAIR(PFA_BF16, PFA_E4M3) PFA_PAIR(PFA_F16, PFA_E4M3)
  PFA_PAIR(PFA_F32, PFA_E2M1) PFA_PAIR(PFA_BF16, PFA_E2M1) PFA_PAIR(PFA_F16, PFA_E2M1)
#undef PFA_PAIR
}

int types_check(int dt, int ct) {
  PFA_CHECK_ARG(dt == PFA_F32 || dt == PFA_BF16 || dt == PFA_F16, "pages: unknown value type %d", dt);
  PFA_CHECK_ARG(scaled(ct) || dt == ct, "pages: values of type %d for cells of type %d", dt, ct);
  return PFA_OK;
}

}  // namespace
}  // namespace pfa

using namespace pfa;

extern "C" int pfa_kv_pages_write(const pfa_kv_pages* pages, const pfa_tensor4* k, const pfa_tensor4* v, int dtype, int B, int64_t n,
                                  const int32_t* table, int64_t table_stride, int table_pages, const int32_t* starts,
                                  const int32_t* counts, void* stream) {
  clear_error();
  Pages p;
  Table t;
  if (int rc = paged_check(pages, table, table_stride, table_pages, B, &p, &t)) return rc;
  if (int rc = types_check(dtype, pages->dtype)) return rc;
  PFA_CHECK_ARG(n >= 0 && n <= (1 << 26), "kv_pages_write: 0 <= n <= 2^26 tokens");
  if (B == 0 || n == 0 || table_pages == 0) return PFA_OK;
  PFA_CHECK_ARG(k && v && k->ptr && v->ptr && starts, "kv_pages_write: null argument");
  const int D = pages->head_dim;
  const int e = cells_bytes(dtype, 1);
  auto rows = [&](const pfa_tensor4& x) {
    const bool vec = (uintptr_t)x.ptr % 16 == 0 && x.s_b * e % 16 == 0 && x.s_h * e % 16 == 0 && x.s_t * e % 16 == 0;
    return NewRows{x.ptr, x.s_b, x.s_h, x.s_t, vec};
  };
  const int64_t touched = (n + p.ps - 2) / p.ps + 1;
  const int64_t at_once = (n < p.ps ? n : p.ps) * (D / 8);
  // a page's rows at once where there are few pages, else four waves each (99 pages and
  // heads of 256 rows of 128 channels: 11 us with 16 waves, 21 with four; 4,200 of 64
  // rows: 84 and 50)
  const int most = touched * p.H * B < 2048 ? 1024 : 256;
  int threads = 64;
  while (threads < at_once && threads < most) threads *= 2;
  const int64_t units = touched * p.H;
  const dim3 grid((unsigned)(units < (1 << 22) ? units : 1 << 22), B);
  by_types(dtype, pages->dtype, [&](auto dt, auto ct) {
    by_width(D, [&](auto width) {
      write_kernel<decltype(dt)::value, decltype(ct)::value, decltype(width)::value>
          <<<grid, threads, 0, as_stream(stream)>>>(p, t, rows(*k), rows(*v), n, units, starts, counts);
    });
  });
  PFA_CHECK_LAUNCH("kv_pages_write");
  return PFA_OK;
}

extern "C" int pfa_kv_pages_read(const pfa_kv_pages* pages, int B, int64_t n, const int32_t* table, int64_t table_stride,
                                 int table_pages, const int32_t* starts, const int32_t* counts, void* k_out,
                                 void* v_out, int out_dtype, void* stream) {
  clear_error();
  Pages p;
  Table t;
  if (int rc = paged_check(pages, table, table_stride, table_pages, B, &p, &t)) return rc;
  PFA_CHECK_ARG(out_dtype == PFA_F32 || out_dtype == PFA_BF16 || out_dtype == PFA_F16,
                "kv_pages_read: unknown value type %d", out_dtype);
  PFA_CHECK_ARG(n >= 0 && n <= (1 << 30), "kv_pages_read: 0 <= n <= 2^30 tokens");
  if (B == 0 || n == 0) return PFA_OK;
  PFA_CHECK_ARG(k_out && v_out && starts && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0,
                "kv_pages_read: null or unaligned argument");
  const int D = pages->head_dim;
  auto launch = [&](auto ct, auto ot) {
    const int at_once = 256 / (D / 8) * read_rows(decltype(ct)::value, decltype(ot)::value);
    const int64_t blocks = (n * p.H + at_once - 1) / at_once;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20), B);
    by_width(D, [&](auto width) {
      read_kernel<decltype(ct)::value, decltype(ot)::value, decltype(width)::value>
          <<<grid, 256, 0, as_stream(stream)>>>(p, t, n, blocks, starts, counts, k_out, v_out);
    });
  };
  auto by_out = [&](auto ct) {
    if (out_dtype == PFA_F32) launch(ct, std::integral_constant<int, PFA_F32>{});
    else if (out_dtype == PFA_BF16) launch(ct, std::integral_constant<int, PFA_BF16>{});
    else launch(ct, std::integral_constant<int, PFA_F16>{});
  };
  by_cells(pages->dtype, by_out);
  PFA_CHECK_LAUNCH("kv_pages_read");
  return PFA_OK;
}

namespace {

int query_check(const char* what, const pfa_paged_query* a, Pages* p, Table* t) {
  PFA_CHECK_ARG(a, "%s: null argument", what);
  if (int rc = paged_check(&a->pages, a->table, a->table_stride, a->table_pages, a->B, p, t)) return rc;
  if (int rc = types_check(a->dtype, a->pages.dtype)) return rc;
  PFA_CHECK_ARG(a->H > 0 && a->H <= 65535 && a->H % p->H == 0, "%s: %d query heads over %d key-value heads", what, a->H,
                p->H);
  PFA_CHECK_ARG((int64_t)a->B * a->H <= 1 << 21, "%s: up to 2^21 rows (got %d x %d)", what, a->B, a->H);
  PFA_CHECK_ARG(a->B == 0 || (a->q.ptr && a->lengths), "%s: null argument", what);
  return PFA_OK;
}

}  // namespace

// Keys of a row, 16-byte aligned.
static int64_t row_keys(int table_pages) { return ((int64_t)table_pages + 3) & ~3ll; }

extern "C" int pfa_kv_pages_select_workspace_size(int B, int kv_heads, int head_dim, int table_pages, size_t* bytes) {
  clear_error();
  PFA_CHECK_ARG(bytes && B >= 0 && kv_heads > 0 && head_dim > 0 && head_dim <= 128 && table_pages >= 0,
                "kv_pages_select: bad sizes");
  *bytes = few_pages(table_pages, head_dim) ? 0 : (size_t)B * kv_heads * row_keys(table_pages) * 4;
  return PFA_OK;
}

static int choice_check(const char* what, const Pages& p, int count, int first, int last) {
  PFA_CHECK_ARG(p.bounds, "%s: the pool has no key bounds", what);
  PFA_CHECK_ARG(count > 0 && first >= 0 && last >= 0 && first <= count && last <= count - first,
                "%s: count > 0 pages, the %d first and %d last among them (got %d)", what, first, last, count);
  return PFA_OK;
}

extern "C" int pfa_kv_pages_select(const pfa_paged_query* query, int count, int first, int last, int32_t* chosen,
                                   void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  Pages p;
  Table t;
  if (int rc = query_check("kv_pages_select", query, &p, &t)) return rc;
  if (int rc = choice_check("kv_pages_select", p, count, first, last)) return rc;
  const int B = query->B, H = query->H, D = query->pages.head_dim, P = query->table_pages;
  if (B == 0) return PFA_OK;
  PFA_CHECK_ARG(chosen, "kv_pages_select: null argument");
  size_t need = 0;
  pfa_kv_pages_select_workspace_size(B, p.H, D, P, &need);
  if (ws_bytes < need || (need && (!workspace || (uintptr_t)workspace % 16 != 0))) {
    set_error("kv_pages_select: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return PFA_E_WORKSPACE;
  }
  uint32_t* keys = (uint32_t*)workspace;
  const int rows = B * p.H;
  const pfa_tensor4* q = &query->q;
  const int32_t *lengths = query->lengths, *starts = query->starts;
  by_types(query->dtype, query->pages.dtype, [&](auto dt, auto ct) {
    constexpr int QT = decltype(dt)::value, BT = bound_dtype(decltype(ct)::value);
    const auto* qp = (const typename Elem<QT>::T*)q->ptr;
    by_width(D, [&](auto width) {
      constexpr int W = decltype(width)::value;
      const int spans = (P + score_span(4, W) - 1) / score_span(4, W);
      if (few_pages(P, W))
        select_kernel<QT, BT, W><<<rows, 256, 0, as_stream(stream)>>>(p, t.ids, t.stride, P, qp, q->s_b, q->s_h, H / p.H,
                                                                     lengths, starts, first, last, count, chosen);
      else
        score_kernel<QT, BT, W><<<dim3(p.H, spans < 65535 ? spans : 65535, B), 256, 0, as_stream(stream)>>>(
            p, t.ids, t.stride, P, qp, q->s_b, q->s_h, H / p.H, lengths, starts, first, last, row_keys(P), keys);
    });
  });
#define PFA_CHOOSE(THREADS, K, HELD)                                                                          \
  choose_kernel<THREADS, K, HELD><<<rows, THREADS, 0, as_stream(stream)>>>(p.H, P, row_keys(P), p.shift, count, \
                                                                           lengths, starts, keys, chosen)
  if (few_pages(P, D)) {
  } else if (P <= 256 * 4) PFA_CHOOSE(256, 4, true);
  else if (P <= 1024 * 4) PFA_CHOOSE(1024, 4, true);
  else if (P <= 1024 * 8) PFA_CHOOSE(1024, 8, true);
  else if (P <= 1024 * 16) PFA_CHOOSE(1024, 16, true);
  else PFA_CHOOSE(1024, 16, false);
#undef PFA_CHOOSE
  PFA_CHECK_LAUNCH("kv_pages_select");
  return PFA_OK;
}

extern "C" int pfa_paged_attn_workspace_size(int B, int H, int kv_heads, int page_size, int head_dim, int cell_dtype,
                                             int table_pages, int n_selected, size_t* bytes) {
  clear_error();
  if (int rc = sizes_check(kv_heads, page_size, head_dim, cell_dtype, table_pages, B)) return rc;
  PFA_CHECK_ARG(bytes && H > 0 && H % kv_heads == 0, "paged_attn: bad sizes");
  *bytes = attend_plan(B, H, kv_heads, head_dim, shift_of(page_size), table_pages, n_selected < 0 ? -1 : n_selected,
                       attend_tile(cell_dtype, head_dim), false)
               .bytes;
  return PFA_OK;
}

// The workgroups that attend select their pages themselves: a workgroup a pair,
// 16 query heads at most, and few pages.
static bool selects_itself(const Plan& plan, int P, int D) {
  return plan.bytes == 0 && plan.deal.RT == 1 && few_pages(P, D);
}

// Behind a call's own workspace, where it weighs its keys: the scores and the rows'
// statistics.
static int score_rows(int G) { return G < 16 ? G : 16; }
static size_t score_count(int B, int H, int kv_heads, int P, int shift) {
  const int G = H / kv_heads;
  return (size_t)B * kv_heads * ((G + 15) / 16) * score_rows(G) * ((size_t)P << shift);
}
static size_t weigh_bytes(int B, int H, int kv_heads, int P, int shift) {
  return score_count(B, H, kv_heads, P, shift) * sizeof(float) + (size_t)B * H * sizeof(float2);
}
static size_t aligned16(size_t bytes) { return (bytes + 15) & ~(size_t)15; }

static int attend(const char* what, const pfa_paged_query* query, const Pages& p, const Table& t, const int32_t* selected,
                  int64_t selected_stride, int S, const Choice& choice, Weigh weigh, float scale, void* out,
                  void* workspace, size_t ws_bytes, void* stream) {
  const float c = scale * 1.44269504088896340736f;
  PFA_CHECK_ARG(c > 0.0f && c < INFINITY, "%s: scale must be positive and finite", what);
  const int B = query->B, H = query->H, D = query->pages.head_dim, ct = query->pages.dtype;
  if (B == 0) return PFA_OK;
  PFA_CHECK_ARG(out && (uintptr_t)out % 16 == 0, "%s: null or unaligned argument", what);
  const Plan plan = attend_plan(B, H, p.H, D, p.shift, t.P, S, attend_tile(ct, D), choice.count > 0);
  const size_t need = weigh.weights ? aligned16(plan.bytes) + weigh_bytes(B, H, p.H, t.P, p.shift) : plan.bytes;
  if (ws_bytes < need || (need && (!workspace || (uintptr_t)workspace % 16 != 0))) {
    set_error("%s: workspace of %zu bytes, %zu needed, 16-byte aligned", what, ws_bytes, need);
    return PFA_E_WORKSPACE;
  }
  if (weigh.weights) {
    weigh.cap = (int64_t)t.P << p.shift;
    weigh.scores = (float*)((char*)workspace + aligned16(plan.bytes));
    weigh.rows = score_rows(H / p.H);
    weigh.stats = (float2*)(weigh.scores + score_count(B, H, p.H, t.P, p.shift));
  }
  const AttendCall a{p, t.ids, t.stride, t.P, B, H, D, query->q, query->lengths, query->starts, selected,
                     selected_stride, S, c, choice, weigh, out, (float*)workspace, as_stream(stream)};
  if (ct == PFA_I8) attend_i8(query->dtype, a);
  else if (ct == PFA_E4M3) attend_e4m3(query->dtype, a);
  else if (ct == PFA_E2M1) attend_e2m1(query->dtype, a);
  else attend_float(query->dtype, a);
  PFA_CHECK_LAUNCH(what);
  return PFA_OK;
}

extern "C" int pfa_paged_attn_fwd(const pfa_paged_query* query, const int32_t* selected, int64_t selected_stride,
                                  int n_selected, float scale, void* out, void* workspace, size_t ws_bytes,
                                  void* stream) {
  clear_error();
  Pages p;
  Table t;
  if (int rc = query_check("paged_attn", query, &p, &t)) return rc;
  PFA_CHECK_ARG(n_selected <= 0 || (selected && selected_stride >= n_selected),
                "paged_attn: lists that are null or overlap");
  PFA_CHECK_ARG((int64_t)n_selected << p.shift <= (1ll << 30), "paged_attn: lists of up to 2^30 positions");
  return attend("paged_attn", query, p, t, selected, selected_stride, n_selected < 0 ? -1 : n_selected, Choice{}, Weigh{}, scale,
                out, workspace, ws_bytes, stream);
}

extern "C" int pfa_paged_weigh_attn_workspace_size(int B, int H, int kv_heads, int page_size, int head_dim, int cell_dtype,
                                                   int table_pages, size_t* bytes) {
  if (int rc = pfa_paged_attn_workspace_size(B, H, kv_heads, page_size, head_dim, cell_dtype, table_pages, -1, bytes))
    return rc;
  *bytes = aligned16(*bytes) + weigh_bytes(B, H, kv_heads, table_pages, shift_of(page_size));
  return PFA_OK;
}

extern "C" int pfa_paged_weigh_attn_fwd(const pfa_paged_query* query, float* weights, int64_t weights_b, int64_t weights_h,
                                        int64_t weights_n, float scale, void* out, void* workspace, size_t ws_bytes,
                                        void* stream) {
  clear_error();
  Pages p;
  Table t;
  if (int rc = query_check("paged_weigh_attn", query, &p, &t)) return rc;
  PFA_CHECK_ARG(weights || query->B == 0 || t.P == 0, "paged_weigh_attn: null argument");
  PFA_CHECK_ARG((uintptr_t)weights % 4 == 0 && weights_n >= (int64_t)t.P << p.shift,
                "paged_weigh_attn: weights of %lld positions for a table of %lld", (long long)weights_n,
                (long long)((int64_t)t.P << p.shift));
  if (t.P == 0) weights = nullptr;  // no keys to weigh
  const bool vec = (uintptr_t)weights % 16 == 0 && weights_b % 4 == 0 && weights_h % 4 == 0;
  const Weigh weigh{weights, weights_b, weights_h, vec, nullptr, 0, 0, nullptr};
  return attend("paged_weigh_attn", query, p, t, nullptr, 0, -1, Choice{}, weigh, scale, out, workspace, ws_bytes, stream);
}

extern "C" int pfa_paged_sparse_attn_workspace_size(int B, int H, int kv_heads, int page_size, int head_dim,
                                                    int cell_dtype, int table_pages, int count, size_t* bytes) {
  size_t select = 0;
  if (int rc = pfa_paged_attn_workspace_size(B, H, kv_heads, page_size, head_dim, cell_dtype, table_pages,
                                             count < table_pages ? count : table_pages, bytes))
    return rc;
  PFA_CHECK_ARG(count > 0, "paged_sparse_attn: count > 0 pages (got %d)", count);
  if (int rc = pfa_kv_pages_select_workspace_size(B, kv_heads, head_dim, table_pages, &select)) return rc;
  if (select > *bytes) *bytes = select;  // one after the other
  return PFA_OK;
}

extern "C" int pfa_paged_sparse_attn_fwd(const pfa_paged_query* query, int count, int first, int last, float scale,
                                         int32_t* chosen, void* out, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  Pages p;
  Table t;
  if (int rc = query_check("paged_sparse_attn", query, &p, &t)) return rc;
  if (int rc = choice_check("paged_sparse_attn", p, count, first, last)) return rc;
  const int B = query->B, H = query->H, D = query->pages.head_dim;
  PFA_CHECK_ARG(scale > 0.0f && scale < INFINITY, "paged_sparse_attn: scale must be positive and finite");
  PFA_CHECK_ARG(B == 0 || (chosen && out && (uintptr_t)out % 16 == 0), "paged_sparse_attn: null or unaligned argument");
  size_t need = 0;
  if (int rc = pfa_paged_sparse_attn_workspace_size(B, H, p.H, p.ps, D, query->pages.dtype, t.P, count, &need)) return rc;
  if (ws_bytes < need || (need && (!workspace || (uintptr_t)workspace % 16 != 0))) {
    set_error("paged_sparse_attn: workspace of %zu bytes, %zu needed, 16-byte aligned", ws_bytes, need);
    return PFA_E_WORKSPACE;
  }
  const int S = count < t.P ? count : t.P;  // no row holds more than its table does
  Choice choice{};
  if (selects_itself(attend_plan(B, H, p.H, D, p.shift, t.P, S, attend_tile(query->pages.dtype, D), true), t.P, D))
    choice = Choice{count, first, last, chosen};
  else if (int rc = pfa_kv_pages_select(query, count, first, last, chosen, workspace, ws_bytes, stream))
    return rc;
  return attend("paged_sparse_attn", query, p, t, chosen, count, S, choice, Weigh{}, scale, out, workspace, ws_bytes, stream);
}
