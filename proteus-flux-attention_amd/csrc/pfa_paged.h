// Pages of a key-value cache: shared by the kernels that write, read, select
// and attend to them.
#pragma once

#include "pfa_common.h"

namespace pfa {
namespace paged {

// Scales of 8-bit rows are at least this (the floor of the library's other
// int8 scales): a row of zeros divides by it.
constexpr float kLeastScale = 1e-6f;

template <int DT> struct Cell { using T = typename Elem<DT>::T; };
template <> struct Cell<PFA_E4M3> { using T = uint8_t; };

__host__ __device__ constexpr bool is8(int dt) { return dt == PFA_I8 || dt == PFA_E4M3; }
__host__ __device__ constexpr float top_of(int dt) { return dt == PFA_I8 ? 127.0f : 448.0f; }
__host__ __device__ constexpr int cell_bytes(int dt) { return dt == PFA_F32 ? 4 : is8(dt) ? 1 : 2; }
// Type of the key bounds: the cells' own (a bound is one of the stored keys),
// f32 for 8-bit cells, whose keys are products with f32 scales.
__host__ __device__ constexpr int bound_dtype(int dt) { return is8(dt) ? PFA_F32 : dt; }

// What a kernel needs of pfa_kv_pages and of a block table.
struct Pages {
  void *k, *v;
  float *k_scale, *v_scale;
  void* bounds;
  int64_t k_page, v_page;  // cells between pages
  int n_pages, H, ps, shift;  // page size 1 << shift
};
struct Table {
  const int32_t* ids;
  int64_t stride;
  int P;  // entries of a row
};

// Page of a row's entry, or -1 where the row has none: entries that name no
// page of the pool hold no keys.
__device__ __forceinline__ int page_at(const Table& t, const Pages& p, int64_t b, int64_t ordinal) {
  if ((uint64_t)ordinal >= (uint64_t)t.P) return -1;
  const int id = t.ids[b * t.stride + ordinal];
  return (uint32_t)id < (uint32_t)p.n_pages ? id : -1;
}

// Tokens that a sequence holds: no more than its row has pages for, 2^30 at most.
__device__ __forceinline__ int length_at(const int32_t* lengths, int P, int shift, int b) {
  const int n = lengths[b], most = P << shift;
  return n < 0 ? 0 : n < most ? n : most;
}
// The first position that it looks at.
__device__ __forceinline__ int start_at(const int32_t* starts, int b) {
  return starts && starts[b] > 0 ? starts[b] : 0;
}

// a / b of positive numbers, in 32 bits where they are enough.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// Eight consecutive cells as f32 (e4m3: v_cvt_f32_fp8, the OCP form on gfx950); the
// address aligned to eight of them.
template <int DT>
__device__ __forceinline__ void cells8(const typename Cell<DT>::T* p, float (&o)[8]) {
  if constexpr (DT == PFA_E4M3) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int w = (int)(i ? a.y : a.x);
      o[4 * i] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
      o[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
      o[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
      o[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
    }
  } else {
    load8<DT>(p, o);
  }
}

}  // namespace paged

// Host: checks of a pool and a block table, shared by the entry points.
int paged_check(const pfa_kv_pages* pages, const int32_t* table, int64_t table_stride, int table_pages, int B,
                paged::Pages* p, paged::Table* t);

}  // namespace pfa
