// Pages of a key-value cache: shared by the kernels that write, read, select
// and attend to them.
#pragma once

#include <type_traits>

#include "pfa_common.h"

namespace pfa {
namespace paged {

// Scales of 8-bit rows are at least this (the floor of the library's other
// int8 scales): a row of zeros divides by it.
constexpr float kLeastScale = 1e-6f;

template <int DT> struct Cell { using T = typename Elem<DT>::T; };
template <> struct Cell<PFA_E4M3> { using T = uint8_t; };
template <> struct Cell<PFA_E2M1> { using T = uint8_t; };  // two cells

__host__ __device__ constexpr bool is8(int dt) { return dt == PFA_I8 || dt == PFA_E4M3; }
__host__ __device__ constexpr bool is4(int dt) { return dt == PFA_E2M1; }
__host__ __device__ constexpr bool scaled(int dt) { return is8(dt) || is4(dt); }
__host__ __device__ constexpr float top_of(int dt) { return dt == PFA_I8 ? 127.0f : 448.0f; }
__host__ __device__ constexpr int cell_bits(int dt) { return dt == PFA_F32 ? 32 : is8(dt) ? 8 : is4(dt) ? 4 : 16; }
// What `cells` cells take: bytes, and elements of Cell<DT>::T.
__host__ __device__ constexpr int cells_bytes(int dt, int cells) { return cells * cell_bits(dt) / 8; }
__host__ __device__ constexpr int cells_at(int dt, int cells) { return is4(dt) ? cells / 2 : cells; }
// Channels that share a scale of 4-bit cells, and scales of a row.
__host__ __device__ constexpr int scale_group(int D) { return D < 32 ? D : 32; }
__host__ __device__ constexpr int scales_of(int dt, int D) { return is4(dt) ? D / scale_group(D) : 1; }
// Type of the key bounds: the cells' own (a bound is one of the stored keys),
// f32 for 8-bit cells, whose keys are products with f32 scales, bf16 for 4-bit
// cells, whose keys have two bits and a power of two.
__host__ __device__ constexpr int bound_dtype(int dt) { return is8(dt) ? PFA_F32 : is4(dt) ? PFA_BF16 : dt; }

// Powers of two that scale 4-bit cells: a byte, the exponent of an f32, as the
// conversions take it (v_cvt_scalef32_*: the exponent's bits alone; 255 gives NaN,
// 0 the 2^-127 that it stands for).
constexpr int kLeastPower = 127 - 20, kMostPower = 127 + 125, kNanPower = 255;
__device__ __forceinline__ float power_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// The least power of two that is a seventh of `most` or above, in that range: the
// mantissa of 7 is 1.75.  With a sixth, where nothing saturates, groups of 32 normal
// values are off by 6 % more in the mean square.
__device__ __forceinline__ uint32_t power_for(float most) {
  const int p = (int)((__float_as_uint(most) + 0x1fffffu) >> 23) - 2;
  return p < kLeastPower ? kLeastPower : p > kMostPower ? kMostPower : p;
}

// Cells 2i and 2i + 1 of a dword of 4-bit cells, scaled, as two bf16 in a dword or two
// f32; i is known when this is compiled.
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2_t;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2_t;
__device__ __forceinline__ uint32_t e2m1_bf16(uint32_t w, float scale, int i) {
  const bf16x2_t x = i == 0   ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)
                     : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)
                     : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)
                              : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return __builtin_bit_cast(uint32_t, x);
}
__device__ __forceinline__ f32x2_t e2m1_f32(uint32_t w, float scale, int i) {
  return i == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0)
         : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1)
         : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2)
                  : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
}

// What a kernel needs of pfa_kv_pages and of a block table.
struct Pages {
  void *k, *v;
  void *k_scale, *v_scale;  // f32, or bytes of 4-bit cells
  void* bounds;
  int64_t k_page, v_page;  // elements of Cell::T between pages
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

__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The bounds of a page's rows over a workgroup, whose threads hold eight channels of
// some rows each, D / 8 neighbours a row: put(d, least, largest) for every channel.
template <int D, int WAVES, typename Put>
__device__ __forceinline__ void join_bounds(float (&lo)[8], float (&hi)[8], float (&part)[2][WAVES][D], Put&& put) {
  constexpr int LANES = D / 8;
  const int lane = threadIdx.x % LANES, wave = threadIdx.x / kWave;
#pragma unroll
  for (int o = LANES; o < kWave; o <<= 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = min_nan(lo[j], __shfl_xor(lo[j], o));
      hi[j] = max_nan(hi[j], __shfl_xor(hi[j], o));
    }
  }
  if (threadIdx.x % kWave < LANES) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[0][wave][8 * lane + j] = lo[j], part[1][wave][8 * lane + j] = hi[j];
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float a = part[0][0][d], z = part[1][0][d];
    for (int w = 1; w < (int)blockDim.x / kWave; ++w) a = min_nan(a, part[0][w][d]), z = max_nan(z, part[1][w][d]);
    put(d, a, z);
  }
  __syncthreads();
}

// Calls f with the head's width as a template argument.
template <typename F>
void by_width(int D, F&& f) {
  if (D == 16) f(std::integral_constant<int, 16>{});
  else if (D == 32) f(std::integral_constant<int, 32>{});
  else if (D == 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 128>{});
}

// Calls f with the cells' type as a template argument.
template <typename F>
void by_cells(int ct, F&& f) {
  switch (ct) {
    case PFA_F32: return f(std::integral_constant<int, PFA_F32>{});
    case PFA_BF16: return f(std::integral_constant<int, PFA_BF16>{});
    case PFA_F16: return f(std::integral_constant<int, PFA_F16>{});
    case PFA_I8: return f(std::integral_constant<int, PFA_I8>{});
    case PFA_E4M3: return f(std::integral_constant<int, PFA_E4M3>{});
    default: return f(std::integral_constant<int, PFA_E2M1>{});
  }
}

}  // namespace paged

// Host: checks of a pool and a block table, shared by the entry points.
int paged_check(const pfa_kv_pages* pages, const int32_t* table, int64_t table_stride, int table_pages, int B,
                paged::Pages* p, paged::Table* t);

}  // namespace pfa
