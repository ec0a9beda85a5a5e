// Attention of one new token over a paged cache, on the matrix cores.
//
// For a key-value head h and the G query heads that share it:
//   S = K Q^T (keys x heads),  m = max S,  P = exp(S - m),  O = V^T P / sum P.
//
// Every key and value is read once, so the cache's bytes are the bound (G is
// small: 4 D G operations for 2 D cells).  The kernel is built around loads
// that need no shuffle behind them:
//
// - A wave takes 32 keys at a time.  S^T = K Q^T puts keys in the rows of the
//   product: lane (n, g), n = lane % 16, g = lane / 16, loads 16-byte units of
//   key n's row, 16 keys x 64 bytes a load, which is the operand as it stands
//   (the order of the channels is free as long as Q's is the same).
// - S comes back with head n in lane (n, g) and keys 4g .. 4g + 3 of each 16 in
//   its registers.  The second product contracts over keys, whose order is free
//   too: O^T = V^T P^T with lane group g holding keys 4g .. 4g + 3 of both 16s is
//   P as it stands.
// - V's operand needs eight keys of one channel in a lane.  Lane (n, g) loads
//   D / 16 neighbouring channels of each of its eight keys (a row is 16 lanes,
//   in one piece), and byte permutes between registers of the same lane turn
//   keys and channels around: one for every two cells.
// - O^T has head n in lane (n, g) again, so the running maximum's correction is
//   one factor a lane, and lane (n, g) ends with D / 4 neighbouring channels.
//
// Keys, values, scores and P pass through no LDS and no lane exchange but the
// maximum over g, two row swaps, until a workgroup's four waves are joined.  A tile's
// pages are read from LDS, where the workgroup looks up those of a run of tiles at
// once, between two barriers (kEntries).
//
// Precision: f32 stays on v_mfma_f32_16x16x4f32.  8-bit cells are whole in
// bf16; their scales multiply S and P in f32.  4-bit cells with their scales, which are
// powers of two, are whole in bf16, too: the conversion multiplies them.  Queries of f16
// or f32 on cells of 8 or 4 bits are split into two or three bf16 parts, which hold all
// their bits.  P goes
// in three parts, each cut off from what the ones before leave: all of its 24
// bits.  f16 parts are of 2^15 P, which has its 24 bits down to 2^-16 of the row's
// largest and 2^-39 absolutely below.  Two bf16 parts hold 16 bits and put 7 to 19
// times as many results of bf16 queries, or of f16 queries on 8-bit cells, on the
// other side of their rounding, and take the same time (1,000,003 int8 tokens: 201
// us a call with two, 202 with three): the loads are what is waited for.  4-bit cells
// are near what the arithmetic takes (1,000,003 tokens: 115 us a call with two, 117.5 with
// three; 64 ragged sequences: 39.8 and 41.2).  Sums, maxima and O are f32 throughout.
//
// Measured (one MI355X, a large copy at 4.7 to 5.1 TB/s; this kernel alone, averages of 20
// launches): 1,000,003 tokens of 4 heads of 128, 8 query heads each: int8 191 us, 5.5
// TB/s, 4 bits 108 us, 5.0 TB/s; 64 ragged sequences of up to 16,384 4-bit tokens of 8
// heads of 128, 4 query heads each: 37 us, 3.3 TB/s; 24 windows of up to 6,000 f32 tokens
// of 8 heads of 64: 75 us, 5.0 TB/s; 64 ragged sequences of up to 8,192 bf16 tokens of
// 8 heads of 128, 4 query heads each: 59 us, 4.2 TB/s; 8 heads of 64 over 173 tokens:
// 7 to 8 us, of which the launch and four loads one behind the other (length, table, key,
// value) are nearly all.  A key at a time with a lane exchange for its score, as these
// kernels began, a million int8 tokens, the windows and the ragged bf16: 1,150,000, 7,400
// and 13,700 us.
#pragma once

#include "pfa_paged.h"
#include "pfa_paged_select.h"

namespace pfa {
namespace paged {

constexpr int kWaves = 4;  // of a workgroup

typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4_t;
typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8_t;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// BYTES (1, 2, 4, 8, 16 or 32) at p, into dwords.
template <int BYTES>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* o) {
  if constexpr (BYTES == 1) o[0] = *p;
  else if constexpr (BYTES == 2) o[0] = *reinterpret_cast<const uint16_t*>(p);
  else if constexpr (BYTES == 4) o[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (BYTES == 8) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    o[0] = a.x, o[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 a = reinterpret_cast<const uint4*>(p)[i];
      o[4 * i] = a.x, o[4 * i + 1] = a.y, o[4 * i + 2] = a.z, o[4 * i + 3] = a.w;
    }
  }
}

// Two f32 cut off to bf16 or f16 in one dword.
__device__ __forceinline__ uint32_t cut_bf16(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);  // the upper halves
}
__device__ __forceinline__ uint32_t cut_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}

// Cells 2i and 2i + 1 of a dword of 8-bit cells as bf16, exactly.
template <int CT>
__device__ __forceinline__ uint32_t cells2_bf16(uint32_t w, int i) {
  if constexpr (CT == PFA_I8) {
    const float a = (float)(int8_t)(w >> (16 * i)), b = (float)(int8_t)(w >> (16 * i + 8));
    return cut_bf16(a, b);
  } else {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2_;
    const f32x2_ f = i ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    return cut_bf16(f[0], f[1]);
  }
}

// 32-key groups of a tile: 4 KB of keys for rows of 128 bytes and more.  Two groups of
// such rows leave no registers: 1,000,003 int8 tokens of 128 channels 195 -> 226 us.
__host__ __device__ constexpr int tile_groups(int ct, int D) { return cells_bytes(ct, D) >= 128 ? 1 : 2; }

// Cells of a call's kernel, by the types of queries and cells and the head's width.
template <int QT_, int CT_, int D_>
struct Form {
  static constexpr int QT = QT_, CT = CT_, D = D_;
  static constexpr int BITS = cell_bits(CT), ROW = cells_bytes(CT, D);
  static constexpr bool F32 = CT == PFA_F32, F16 = CT == PFA_F16;
  static constexpr int NS = scales_of(CT, D);  // scales of a row
  static constexpr int NQ = !scaled(CT) || QT == PFA_BF16 ? 1 : QT == PFA_F16 ? 2 : 3;  // parts of Q
  static constexpr int NP = 3;                                                        // parts of P
  static constexpr int EL = D / 4;                     // channels of a lane in S
  static constexpr int U = EL < 128 / BITS ? EL : 128 / BITS;  // of one load
  static constexpr int UB = U * BITS / 8;                      // their bytes
  static constexpr int KW = EL * BITS < 32 ? 1 : EL * BITS / 32;  // dwords of a lane's share of 16 keys
  static constexpr int NC = F32 ? EL : EL < 8 ? 1 : EL / 8;  // products over it
  static constexpr int VD = D / 16;                    // channels of a lane in O
  static constexpr int VB = VD * BITS < 8 ? 1 : VD * BITS / 8;  // their bytes of a key
  static constexpr int VW = VB < 4 ? 1 : VB / 4;
  static constexpr int NG = tile_groups(CT, D);  // 32-key groups that a wave loads at once
  static constexpr int TILE = 32 * NG;
  // Waves of a SIMD, at least: three, but two where three would spill what a tile reads
  // (f16 queries on 1,000,003 4-bit tokens of 128 channels: 135 us a call with three, 126
  // with two).  bf16 queries on 4-bit cells of 128 channels spill 8 bytes a lane at three,
  // 32 where scores are kept, none at two: 1,000,003 tokens 118.5 us with three, 121.5 with
  // two, 64 ragged sequences 41.5 and 42.0; with weights 192 and 188, 32 ragged sequences
  // 54.4 and 54.0.  f16 cells of 128 channels spill 8 where scores are kept: 32 ragged
  // sequences with weights 133 with three, 140 with two, 400,003 tokens 207 and 221.
  static constexpr int AT_LEAST = D == 128 && (QT == PFA_F32 || (is4(CT) && QT == PFA_F16)) ? 2 : 3;
  // Whether a wave that keeps scores holds those of some tiles back in LDS: a wait for
  // loads waits for the stores before them, too.  32 ragged sequences of up to 16,384
  // tokens, int8 of 128 channels: 82.3 -> 80.1 us, bf16 of 64 76.6 -> 73.9.  Elsewhere
  // it takes registers that are not there (4 bits of 128: 64.9 -> 68.1, bf16 of 128:
  // 121.4 -> 126.8) or a wave of a SIMD.
  static constexpr bool HOLDS = NG == 1 && (D < 128 || is8(CT));
  static constexpr float PSCALE = F16 ? 32768.0f : 1.0f;
};

// 16 keys in a row of a page: the position of the first, far behind every
// length where there are none.
struct Block {
  int id, slot, pos;
};
constexpr int kNowhere = 0x7ffff000;  // positions are below 2^30; no sum with a tile's keys overflows

// Pages of a run of tiles, in LDS: looked up by all of the workgroup's threads at
// once, so that a tile's lookup, two loads one behind the other, is not in front
// of every tile's keys (48 sequences with 48 listed pages each: 22 -> 19 us).
constexpr int kEntries = 512;
struct Entry {
  int id, pos;  // the page, and the position of its first slot or kNowhere
};

// One sequence and key-value head.
struct Row {
  const Entry* entries;  // the run's
  int first;             // entry of the run's first
  int shift, start, len;

  // `key` counts positions, or the slots of the listed pages
  __device__ __forceinline__ Block block(int key) const {
    const Entry e = entries[(key >> shift) - first];
    const int slot = key & ((1 << shift) - 1);
    return Block{__builtin_amdgcn_readfirstlane(e.id), slot, __builtin_amdgcn_readfirstlane(e.pos) + slot};
  }
};

template <typename F>
struct Tile {
  Block b[2 * F::NG];
  __device__ __forceinline__ void find(const Row& r, int tile) {
#pragma unroll
    for (int i = 0; i < F::NG; ++i) {
      const int key = tile * F::TILE + 32 * i;
      b[2 * i] = r.block(key);
      if (r.shift > 4) b[2 * i + 1] = Block{b[2 * i].id, b[2 * i].slot + 16, b[2 * i].pos + 16};
      else b[2 * i + 1] = r.block(key + 16);
    }
  }
  // the first of tiles t, t + kWaves, ... before `end` that has a key to see
  __device__ __forceinline__ int find_seen(const Row& r, int t, int end) {
    for (; t < end; t += kWaves) {
      find(r, t);
      bool any = false;
#pragma unroll
      for (int i = 0; i < 2 * F::NG; ++i) any = any || (b[i].pos < r.len && b[i].pos + 16 > r.start);
      if (any) break;
    }
    return t;
  }
  // whether all its keys are seen
  __device__ __forceinline__ bool whole(const Row& r) const {
    bool w = true;
#pragma unroll
    for (int i = 0; i < 2 * F::NG; ++i) w = w && b[i].pos >= r.start && b[i].pos + 16 <= r.len;
    return w;
  }
};

// A wave's running state: O^T of head n in lane (n, g), channels
// VD * (4g + i) + j, the row's maximum (of the products as they are: the scale is
// multiplied on when the maximum is off) and sum (of the lane's own keys).
template <typename F>
struct State {
  f32x4_t o[F::VD];
  float m, l;
};

template <typename F>
struct Wave {
  int n, g;
  u32x4_t q[F::F32 ? 1 : F::NQ][F::F32 ? 1 : F::NC];
  float qf[F::F32 ? F::EL : 1];
  uint32_t k[2 * F::NG][F::KW];
  uint32_t ks[is4(F::CT) ? 2 * F::NG : 1];  // scales of 4-bit cells: of the lane's channels, which are of one group

  // Channel of a lane's element x: unit x / U of 4U channels, one U a lane group.
  __device__ __forceinline__ int channel(int x) const { return x / F::U * 4 * F::U + g * F::U + x % F::U; }

  // `vec`: the row is 16-byte aligned
  __device__ __forceinline__ void load_q(const typename Elem<F::QT>::T* p, bool row, bool vec) {
    if constexpr (F::F32) {
#pragma unroll
      for (int x = 0; x < F::EL; x += 4) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        const float* at = p + channel(x);
        if (row) {
          if (vec) a = *reinterpret_cast<const float4*>(at);
          else a = make_float4(at[0], at[1], at[2], at[3]);
        }
        qf[x] = a.x, qf[x + 1] = a.y, qf[x + 2] = a.z, qf[x + 3] = a.w;
      }
    } else {
#pragma unroll
      for (int c = 0; c < F::NC; ++c) {
        float x[8] = {};
        const typename Elem<F::QT>::T* at = p + channel(8 * c);
        if (row) {
          if (vec && F::EL >= 8) load8<F::QT>(at, x);
          else {
#pragma unroll
            for (int e = 0; e < (F::EL < 8 ? F::EL : 8); ++e) x[e] = load_f<F::QT>(at + e);
          }
        }
        parts<F::NQ, F::F16, true>(x, [&](int part, u32x4_t w) { q[part][c] = w; });
      }
    }
  }

  // Eight f32 as N 16-bit operands, each cut off from what the ones before leave; with
  // INF an infinity leaves nothing.
  template <int N, bool HALF, bool INF, typename Put>
  static __device__ __forceinline__ void parts(float (&x)[8], Put&& put) {
    auto leave = [](float a, float part) { return INF && fabsf(a) == INFINITY ? 0.0f : a - part; };
#pragma unroll
    for (int part = 0; part < N; ++part) {
      u32x4_t w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = HALF ? cut_f16(x[2 * i], x[2 * i + 1]) : cut_bf16(x[2 * i], x[2 * i + 1]);
        w[i] = u;
        if (part + 1 < N) {
          const float a = HALF ? f16_to_f32((uint16_t)u) : __uint_as_float(u << 16);
          const float b = HALF ? f16_to_f32((uint16_t)(u >> 16)) : __uint_as_float(u & 0xffff0000u);
          x[2 * i] = leave(x[2 * i], a), x[2 * i + 1] = leave(x[2 * i + 1], b);
        }
      }
      put(part, w);
    }
  }

  static __device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
    if constexpr (F::F16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                    0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                     0, 0, 0);
  }

  static __device__ __forceinline__ const uint8_t* page_of(const void* cells, int64_t page, int id) {
    return (const uint8_t*)cells + (int64_t)id * page * (int64_t)sizeof(typename Cell<F::CT>::T);
  }

  __device__ __forceinline__ void load_k(const Pages& pg, int h, const Tile<F>& t) {
    const int lane_at = n * F::ROW + g * F::UB;
#pragma unroll
    for (int i = 0; i < 2 * F::NG; ++i) {
      const uint8_t* base = page_of(pg.k, pg.k_page, t.b[i].id) + (int64_t)(h * pg.ps + t.b[i].slot) * F::ROW;
#pragma unroll
      for (int u = 0; u < F::EL / F::U; ++u) load_bytes<F::UB>(base + lane_at + u * 4 * F::UB, &k[i][u * F::UB / 4]);
      if constexpr (is4(F::CT)) {
        const int64_t row = ((int64_t)t.b[i].id * pg.H + h) * pg.ps + t.b[i].slot;
        ks[i] = ((const uint8_t*)pg.k_scale)[row * F::NS + n * F::NS + g * F::EL / 32];
      }
    }
  }

  // S of the 16 keys of block i.
  __device__ __forceinline__ f32x4_t scores(int i) const {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
    if constexpr (F::F32) {
      f32x4_t s2 = s;
#pragma unroll
      for (int x = 0; x < F::EL; x += 2) {
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i][x]), qf[x], s, 0, 0, 0);
        s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i][x + 1]), qf[x + 1], s2, 0, 0, 0);
      }
      s += s2;
    } else {
#pragma unroll
      for (int c = 0; c < F::NC; ++c) {
        u32x4_t a = {0, 0, 0, 0};
        if constexpr (is4(F::CT)) {
#pragma unroll
          for (int w = 0; w < (F::EL < 8 ? 2 : 4); ++w) a[w] = e2m1_bf16(k[i][c], power_of(ks[i]), w);
        } else if constexpr (is8(F::CT)) {
#pragma unroll
          for (int w = 0; w < (F::EL < 8 ? 2 : 4); ++w) a[w] = cells2_bf16<F::CT>(k[i][2 * c + w / 2], w & 1);
        } else {
#pragma unroll
          for (int w = 0; w < (F::EL < 8 ? 2 : 4); ++w) a[w] = k[i][4 * c + w];
        }
#pragma unroll
        for (int part = F::NQ - 1; part >= 0; --part) s = mma(a, q[part][c], s);
      }
    }
    return s;
  }

  // One tile: V loads, S from the keys that are in registers, the next tile's
  // keys, P, and O.  The next keys are loaded whether or not there is a next tile
  // (`next` is this one then): a load under a condition would have the wait for V
  // wait for them, too.
  // With KEEP it leaves the scores of `score_rows` rows, 16 keys of all rows together:
  // HOLDS in `kept`, LDS, and those keys' positions in `kept_at`, else in the workspace,
  // of whose rows `kept` is the lane's place, if it has one.
  template <bool KEEP>
  __device__ __forceinline__ void step(const Pages& pg, const Row& r, int h, float c, const Tile<F>& t,
                                       const Tile<F>& next, State<F>& st, float* kept, int* kept_at, int score_rows) {
    uint32_t v[2 * F::NG][4][F::VW];
    f32x4_t s[2 * F::NG], vs[2 * F::NG];
    [[maybe_unused]] uint32_t raw[2 * F::NG][F::NS];  // V's scales of 4-bit cells: four keys'
    const int lane_at = 4 * g * F::ROW + n * F::VD * F::BITS / 8;
#pragma unroll
    for (int i = 0; i < 2 * F::NG; ++i) {
      const int64_t slot = (int64_t)(h * pg.ps + t.b[i].slot);
      const uint8_t* base = page_of(pg.v, pg.v_page, t.b[i].id) + slot * F::ROW;
#pragma unroll
      for (int y = 0; y < 4; ++y) load_bytes<F::VB>(base + lane_at + y * F::ROW, v[i][y]);
      const int64_t at = ((int64_t)t.b[i].id * pg.H) * pg.ps + slot + 4 * g;
      if constexpr (is8(F::CT)) {
        s[i] = *reinterpret_cast<const f32x4_t*>((const float*)pg.k_scale + at);
        vs[i] = *reinterpret_cast<const f32x4_t*>((const float*)pg.v_scale + at);
      }
      if constexpr (is4(F::CT)) load_bytes<4 * F::NS>((const uint8_t*)pg.v_scale + at * F::NS, raw[i]);
    }
    __builtin_amdgcn_sched_barrier(0);  // V is on its way before K is waited for
#pragma unroll
    for (int i = 0; i < 2 * F::NG; ++i) {
      if constexpr (is8(F::CT)) s[i] = scores(i) * s[i];
      else s[i] = scores(i);
    }
    load_k(pg, h, next);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (KEEP) {
#pragma unroll
      for (int i = 0; i < 2 * F::NG; ++i) {
        if constexpr (F::HOLDS) {
          if (n < score_rows) *reinterpret_cast<f32x4_t*>(kept + (i * score_rows + n) * 16 + 4 * g) = s[i];
          if (n == 0 && g == 0) kept_at[i] = t.b[i].pos;
        } else {
          if (kept && t.b[i].pos < kNowhere)
            *reinterpret_cast<f32x4_t*>(kept + (int64_t)t.b[i].pos * score_rows) = s[i];
        }
      }
    }
    if constexpr (is4(F::CT)) {
      // byte y * NS + (the lane's group) of the four keys', turned to where an f32 has its
      // exponent: what else comes with it is no part of that
      const int turn = 8 * (n * F::VD / 32) + 9;
#pragma unroll
      for (int i = 0; i < 2 * F::NG; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t w = raw[i][y * F::NS / 4];
          vs[i][y] = __uint_as_float(__builtin_amdgcn_alignbit(w, w, 8 * (y * F::NS % 4) + turn));
          if constexpr (F::VD == 1) v[i][y][0] = v[i][y][0] >> 4 * (n & 1) & 15u;
        }
    }
    if (!t.whole(r)) {
      // keys that are not seen: no weight, and nothing of what stands there
#pragma unroll
      for (int i = 0; i < 2 * F::NG; ++i) {
        const int pos = t.b[i].pos + 4 * g;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const bool seen = pos + y >= r.start && pos + y < r.len;
          s[i][y] = seen ? s[i][y] : -INFINITY;
          if constexpr (scaled(F::CT)) vs[i][y] = seen ? vs[i][y] : 0.0f;
#pragma unroll
          for (int w = 0; w < F::VW; ++w) v[i][y][w] = seen ? v[i][y][w] : 0u;
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2 * F::NG; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) top = fmaxf(top, s[i][y]);
    top = max_over_rows4(top);
    if (__any(top > st.m)) {
      const float m = fmaxf(st.m, top);
      const float alpha = m == -INFINITY ? 1.0f : exp2_((st.m - m) * c);
      st.m = m;
      st.l *= alpha;
#pragma unroll
      for (int j = 0; j < F::VD; ++j) st.o[j] *= alpha;
    }
    const float m = st.m == -INFINITY ? 0.0f : st.m;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * F::NG; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        // off the maximum first: no exponent is above zero, however large the scores
        // (s * c - m * c in one rounding can be, by a rounding of m * c)
        const float p = exp2_((s[i][y] - m) * c);
        sum += p;
        s[i][y] = is8(F::CT) ? p * vs[i][y] : p * F::PSCALE;
      }
    st.l += sum;
    if constexpr (F::F32) {
#pragma unroll
      for (int i = 0; i < 2 * F::NG; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int j = 0; j < F::VD; ++j)
            st.o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[i][y][j]), s[i][y], st.o[j], 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * F::NG; i += 2) {
        float x[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) x[y] = s[i + y / 4][y & 3];
        u32x4_t p[F::NP];
        parts<F::NP, F::F16, false>(x, [&](int part, u32x4_t w) { p[part] = w; });
        // channels 2jj, 2jj + 1 of the eight keys, as pairs of 16-bit cells
        constexpr int PAIRS = F::VD < 2 ? 1 : F::VD / 2;
#pragma unroll
        for (int jj = 0; jj < PAIRS; ++jj) {
          uint32_t w[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            if constexpr (is4(F::CT)) w[y] = e2m1_bf16(v[i + y / 4][y & 3][jj / 4], vs[i + y / 4][y & 3], jj & 3);
            else if constexpr (is8(F::CT)) w[y] = cells2_bf16<F::CT>(v[i + y / 4][y & 3][jj / 2], jj & 1);
            else w[y] = v[i + y / 4][y & 3][jj];
          }
#pragma unroll
          for (int e = 0; e < (F::VD < 2 ? 1 : 2); ++e) {
            u32x4_t a;
#pragma unroll
            for (int x2 = 0; x2 < 4; ++x2)
              a[x2] = __builtin_amdgcn_perm(w[2 * x2 + 1], w[2 * x2], e ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int part = F::NP - 1; part >= 0; --part) st.o[2 * jj + e] = mma(a, p[part], st.o[2 * jj + e]);
          }
        }
      }
    }
  }
};

// What a workgroup's waves, and then a row's workgroups, are joined by: the
// weight of a part with maximum m and sum l under the common maximum.  A part
// without a score above -inf weighs nothing, unless a NaN is in it.  A part that
// weighs nothing is still added: zero, but for values and sums that are not finite,
// which are the row's wherever in it they lie.
__device__ __forceinline__ float part_weight(float m, float l, float top, float c) {
  return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2_((m - top) * c);
}

// How the tiles of all rows are dealt out: a pair is a sequence and 16 heads
// at most of one key-value head, R pairs a sequence.  All pairs lie in one line,
// sequence by sequence, kStart places and one for each of its tiles long, and the
// line is cut in `chunk`s, one a workgroup.  The kStart places stand for what a
// pair costs before its first key arrives and after its last: without them a
// workgroup with a dozen one-tile pairs was the last to end.
// (64 ragged sequences: 70 us with 2, 61 with 4, 57 to 58 with 5, 8 or 12; 48
// sequences with 48 pages each: 21 us with 5, 17 with 8 or 12.)
constexpr int kStart = 8;

struct Deal {
  int B, R, RT;      // sequences; pairs of one; pairs of one of its heads
  int S, shift, P;   // listed entries or -1; the pages
  int tile;          // keys of a tile
  int least;         // places of a chunk, at least
  int groups;        // workgroups

  __device__ __forceinline__ int first_tile(int start) const { return S >= 0 || start <= 0 ? 0 : start / tile; }
  __device__ __forceinline__ int tiles(int start, int len) const {
    if (S >= 0) return (int)((((int64_t)S << shift) + tile - 1) / tile);
    return start >= len ? 0 : (len + tile - 1) / tile - first_tile(start);
  }
  __device__ __forceinline__ int length(const int32_t* lengths, int b) const { return length_at(lengths, P, shift, b); }
  // places of a pair
  __device__ __forceinline__ int places(int start, int len) const {
    const int n = tiles(start, len);
    return n > 0 ? n + kStart : 0;
  }
  __device__ __forceinline__ int64_t chunk(int64_t total) const {
    const int64_t c = quotient(total + groups - 1, groups);
    return c < least ? least : c;
  }
};

// A value that all lanes share, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}

__device__ __forceinline__ int64_t wave_sum(int64_t x) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) x += __shfl_xor(x, o);
  return x;
}

// What a pair's first workgroup leaves for the join.
struct Shared {
  int first, n;  // workgroups first .. first + n - 1 have parts of the pair
};

// Parts of pairs that several workgroups share: slot 2w, the pair that
// workgroup w continues, 2w + 1, the one that it starts and does not end.
// O (rows, D), then the maxima and the sums.
__device__ __forceinline__ float* part_slot(float* parts, int64_t slot, int rows, int D) {
  return parts + slot * rows * (D + 2);
}

// Attention that every key got, summed over the query heads of its head: what a call
// adds to.  The weight of a key is exp2((s - m) c) / l, and m and l are known when
// all keys are through: the scores are kept, G of them for a key, and read again
// behind the join.  K again instead would be 64 to 512 bytes for 4 G.
struct Weigh {
  float* weights;  // (B, H, T), rows apart by
  int64_t s_b, s_h;
  int vec;         // rows are aligned to four
  // (pairs, cap / 16, rows, 16): the products, before the scale.  16 keys of all rows lie
  // together, which is what a wave stores at once: 1,000,003 int8 tokens of four heads,
  // eight query heads each, 310 us with a row in one piece, 295 so (200 without weights).
  float* scores;
  int64_t cap;
  int rows;        // of a pair
  float2* stats;   // (B * query heads): the maximum, and one over the sum
};

// A row's statistics, as the weights of its keys need them: a row without a score
// above -inf has none.
__device__ __forceinline__ float2 row_stats(float m, float l) {
  return make_float2(m == -INFINITY ? 0.0f : m, l == 0.0f ? 0.0f : 1.0f / l);
}

// Adds the weights of the positions [start, len), of the G rows of a key-value head in
// their order: the same bits every time.  A thread takes four neighbours of every
// 4 * step, the first of them `unit` fours behind the four that hold the start.  A start
// may be any number of 32 bits: at or behind the length there is nothing to add, and 4 *
// unit more than it is a number of 64.
template <typename Stats>
__device__ __forceinline__ void add_weights(const Weigh& w, const Pages& pg, const int32_t* __restrict__ ids, int b, int h,
                                            int G, float c, int start, int len, int64_t unit, int step, Stats&& stats) {
  if (start >= len) return;
  float* to = w.weights + b * w.s_b + h * w.s_h;
  const int pairs = (G + 15) / 16;
  for (int64_t p = (start & ~3) + 4 * unit; p < len; p += 4 * (int64_t)step) {
    if ((uint32_t)ids[p >> pg.shift] >= (uint32_t)pg.n_pages) continue;
    float sum[4] = {};
    for (int g0 = 0; g0 < G; g0 += 16) {
      const int64_t pair = ((int64_t)b * pg.H + h) * pairs + g0 / 16;
      const float* at = w.scores + (pair * w.cap + (p & ~15ll)) * w.rows + (p & 15);
      const int here = G - g0 < 16 ? G - g0 : 16;
#pragma unroll 4
      for (int g = 0; g < here; ++g) {
        const f32x4_t s = *reinterpret_cast<const f32x4_t*>(at + 16 * g);
        const float2 st = stats(g0 + g);
#pragma unroll
        for (int y = 0; y < 4; ++y) sum[y] += exp2_((s[y] - st.x) * c) * st.y;
      }
    }
    if (w.vec && p >= start && p + 4 <= len) {
      f32x4_t x = *reinterpret_cast<const f32x4_t*>(to + p);
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] += sum[y];
      *reinterpret_cast<f32x4_t*>(to + p) = x;
    } else {
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (p + y >= start && p + y < len) to[p + y] += sum[y];
    }
  }
}

// Rows of more heads than a tile has, behind the join: a workgroup four times its
// threads' positions of a sequence and key-value head.
static __global__ void __launch_bounds__(256) weigh_kernel(Weigh w, Pages pg, const int32_t* __restrict__ table,
                                                           int64_t table_stride, int P, int G, float c,
                                                           const int32_t* __restrict__ lengths,
                                                           const int32_t* __restrict__ starts) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int len = length_at(lengths, P, pg.shift, b), start = start_at(starts, b);
  const int64_t row = ((int64_t)b * pg.H + h) * G;
  add_weights(w, pg, table + b * table_stride, b, h, G, c, start, len, (int64_t)blockIdx.x * blockDim.x + threadIdx.x,
              (int)(gridDim.x * blockDim.x), [&](int g) { return w.stats[row + g]; });
}

// What paged_sparse_attention chooses before it attends.
struct Choice {
  int count, first, last;
  int32_t* chosen;
};

// A barrier for what passes through LDS: stores to memory stay on their way.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Between what lanes of a wave leave in LDS and what others of it read: an order, no wait.
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// What a call does beside attending.  SELECT: the workgroup first selects its pair's
// pages itself, for a launch and several dependent loads less.  WEIGH: it keeps the
// scores, and where a workgroup has all of a key's rows it adds their weights itself.
enum class Also { NOTHING, SELECT, WEIGH };

constexpr int kKept = 8;  // tiles whose scores a wave holds back, at most

template <typename F, Also ALSO>
__global__ void __launch_bounds__(64 * kWaves, F::AT_LEAST) attend_kernel(
    Pages pg, Deal deal, const int32_t* __restrict__ table, int64_t table_stride,
    const typename Elem<F::QT>::T* __restrict__ q, int64_t q_b, int64_t q_h, int q_vec, int G,
    const int32_t* __restrict__ lengths, const int32_t* __restrict__ starts, const int32_t* __restrict__ selected,
    int64_t selected_stride, float c, typename Elem<F::QT>::T* __restrict__ out, float* __restrict__ parts_ws, Shared* __restrict__ shared,
    Choice choice, Weigh weigh) {
  constexpr int D = F::D;
  constexpr bool SELECT = ALSO == Also::SELECT, WEIGH = ALSO == Also::WEIGH;
  constexpr bool HOLDS = WEIGH && F::HOLDS;
  // a wave's O, and before that the scores of some of its tiles
  __shared__ __attribute__((aligned(16))) float so[kWaves][16][D + 4];
  static_assert(!HOLDS || D + 4 >= F::TILE, "a tile's scores of 16 rows");
  __shared__ int kept_at[HOLDS ? kWaves : 1][HOLDS ? kKept * 2 * F::NG : 1];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ Entry entries[kEntries + 1];
  __shared__ int64_t sums[kWaves];
  __shared__ int64_t found[2];
  __shared__ int found_at[2];
  __shared__ float2 stats[WEIGH ? 16 : 1];
  deal.tile = F::TILE;  // as it is, and known
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Wave<F> w;
  w.n = lane & 15, w.g = lane >> 4;
  const int rows = G < 16 ? G : 16;

  // the workgroup's chunk: [f, f1) of the line, f in a pair of sequence b, whose
  // first pair begins at `at`
  int64_t f, f1, at, chunk = 1;
  int b;
  // of the sequence at hand, and below the tiles whose pages are in LDS: the next pair of
  // a short sequence, which has the same, goes on without waiting for either
  int at_hand = -1, start = 0, len = 0, nt = 0, np = 0;
  if (parts_ws && deal.S >= 0) {  // all sequences alike
    const int np = deal.places(0, 1);
    const int64_t total = (int64_t)deal.B * deal.R * np;
    chunk = deal.chunk(total);
    f = blockIdx.x * chunk;
    if (f >= total) return;
    f1 = f + chunk < total ? f + chunk : total;
    b = (int)quotient(f, (int64_t)deal.R * np);
    at = (int64_t)b * deal.R * np;
  } else if (parts_ws) {
    // places of the sequences up to this thread's, of 256 at a time
    int its_start = 0, its_len = 0;
    auto places = [&](int i) {
      its_start = i < deal.B ? start_at(starts, i) : 0, its_len = i < deal.B ? deal.length(lengths, i) : 0;
      return deal.places(its_start, its_len) * (int64_t)deal.R;
    };
    int64_t incl, all, mine;
    auto scan = [&](int i) {
      incl = mine = places(i);
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int64_t x = __shfl_up(incl, o);
        if (lane >= o) incl += x;
      }
      if (lane == 63) sums[wave] = incl;
      lds_barrier();
      all = 0;
#pragma unroll
      for (int j = 0; j < kWaves; ++j) {
        if (j < wave) incl += sums[j];
        all += sums[j];
      }
    };
    scan(tid);
    int64_t total = all;
    if (deal.B > 64 * kWaves) {
      const int start0 = its_start, len0 = its_len;
      int64_t rest = 0;
      for (int i = tid + 64 * kWaves; i < deal.B; i += 64 * kWaves) rest += places(i);
      rest = wave_sum(rest);
      lds_barrier();
      if (lane == 0) sums[wave] = rest;
      lds_barrier();
#pragma unroll
      for (int i = 0; i < kWaves; ++i) total += sums[i];
      its_start = start0, its_len = len0;
    }
    total = uniform(total);
    chunk = deal.chunk(total);
    f = blockIdx.x * chunk;
    if (f >= total) return;
    f1 = f + chunk < total ? f + chunk : total;
    int64_t before = 0;
    for (int base = 0;;) {
      if (mine > 0 && before + incl - mine <= f && f < before + incl) {
        found[0] = base + tid, found[1] = before + incl - mine;
        found_at[0] = its_start, found_at[1] = its_len;
      }
      before += all;
      if (f < before) break;
      base += 64 * kWaves;
      lds_barrier();
      scan(base + tid);
    }
    lds_barrier();
    b = (int)uniform(found[0]);
    at = uniform(found[1]);
    at_hand = b;
    start = __builtin_amdgcn_readfirstlane(found_at[0]), len = __builtin_amdgcn_readfirstlane(found_at[1]);
    nt = deal.tiles(start, len), np = deal.places(start, len);
  } else {  // a workgroup a pair
    b = blockIdx.x / deal.R;
    f = (int64_t)(blockIdx.x % deal.R) * deal.tiles(start_at(starts, b), deal.length(lengths, b));
    f1 = f + 1;
    at = 0;
  }
  const bool lone = !parts_ws;
  __shared__ int32_t own[SELECT ? kFused : 1];  // the list of an own selection
  if constexpr (SELECT) {
    const int h = blockIdx.x % deal.R;
    int32_t* chosen = choice.chosen + (int64_t)blockIdx.x * choice.count;
    static_assert(kWaves == 4, "select_row has four waves");
    select_row<F::QT, bound_dtype(F::CT), D>(
        pg, table + b * table_stride, deal.P, b, h, q + b * q_b, q_h, G, lengths, starts, choice.first, choice.last,
        choice.count, [&](int i, int entry) {
          chosen[i] = entry;
          if (i < deal.S) own[i] = entry;
        });
    lds_barrier();
  }

  // The chip gives a unit's oldest wave its turn first, so that of three workgroups with
  // the same work the first is through in 60 % of the last one's time, which then has
  // the unit for itself and does not fill it.  A wave's priority falls with each quarter
  // of its chunk: they go on side by side (1,000,003 4-bit tokens: 124 -> 119 us; 64
  // ragged sequences: 44.9 -> 44.0).  f32 cells keep the units' order: a workgroup's
  // loads fill a unit (24 windows of 6,000 tokens: 77 us, 78 side by side).
  const int64_t f0 = f;
  const int quarter = (int)((f1 - f + 3) >> 2);
  int looked_up = -1, first_up = 0, end_up = 0;
  while (f < f1) {
    if (b != at_hand) {
      at_hand = b;
      start = start_at(starts, b), len = deal.length(lengths, b);
      nt = deal.tiles(start, len), np = deal.places(start, len);
    }
    if (!lone && nt == 0) {
      ++b;
      continue;
    }
    const int pair = lone ? blockIdx.x % deal.R : (int)uniform(quotient(f - at, np));
    // the pair's first tile on the line, and its tiles [ta, tb) in the chunk
    const int64_t pair_at = at + (int64_t)pair * np + kStart;
    const int ta = lone || f < pair_at ? 0 : (int)(f - pair_at);
    const int tb = lone || f1 - pair_at > nt ? nt : f1 < pair_at ? 0 : (int)(f1 - pair_at);
    if (!lone) {
      if (tb == 0) return;  // the chunk ends before the pair's first tile
      f = pair_at + tb;
      if (tb == nt && pair + 1 == deal.R) at = f;
    }
    const int h = pair / deal.RT, row0 = h * G + 16 * (pair % deal.RT);
    const int here = (h + 1) * G - row0 < 16 ? (h + 1) * G - row0 : 16;

    w.load_q(q + b * q_b + (row0 + w.n) * q_h, w.n < here, q_vec);
    float* scores = nullptr;
    if constexpr (WEIGH) {
      scores = weigh.scores + ((int64_t)b * deal.R + pair) * weigh.cap * rows;
      if (!HOLDS) scores = w.n < here ? scores + 16 * w.n + 4 * w.g : nullptr;
    }
    int kept = 0;  // tiles that are held back
    const int tile_kept = F::TILE * rows, room = 16 * (D + 4) / tile_kept;
    auto put_out = [&]() {
      wave_fence();
      const float* from = &so[wave][0][0];
      const int each = 4 * rows, inverse = ((1 << 20) + each - 1) / each;  // quotients of up to 2,048
      for (int u = lane; u < kept * 2 * F::NG * each; u += kWave) {
        const int block = u * inverse >> 20, pos = kept_at[wave][block];
        if (pos < kNowhere)
          *reinterpret_cast<f32x4_t*>(scores + (int64_t)pos * rows + 4 * (u - block * each)) =
              *reinterpret_cast<const f32x4_t*>(from + 4 * u);
      }
      wave_fence();
      kept = 0;
    };
    State<F> st;
#pragma unroll
    for (int j = 0; j < F::VD; ++j) st.o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    st.m = -INFINITY, st.l = 0.0f;
    const int32_t* ids = table + b * table_stride;
    const int32_t* list = selected + ((int64_t)b * pg.H + h) * selected_stride;
    const int t0 = deal.first_tile(start), te = t0 + tb;
    const int run = (kEntries << deal.shift) / F::TILE;  // tiles whose pages fit
    for (int r0 = t0 + ta; r0 < te; r0 += run) {
      const int re = te - r0 < run ? te : r0 + run;
      const Row r{entries, r0 * F::TILE >> deal.shift, deal.shift, start, len};
      const bool there = !SELECT && deal.S < 0 && looked_up == b && first_up == r0 && end_up >= re;
      const int n = there ? 0 : ((re * F::TILE - 1) >> deal.shift) - r.first + 1;
      if (r0 > t0 + ta) lds_barrier();  // the last run's are read
      for (int i = tid; i < n; i += 64 * kWaves) {
        int ordinal = r.first + i;
        if constexpr (SELECT) ordinal = ordinal < deal.S ? own[ordinal] : -1;
        else if (deal.S >= 0) ordinal = ordinal < deal.S ? list[ordinal] : -1;
        const int id = (uint32_t)ordinal < (uint32_t)deal.P ? ids[ordinal] : -1;
        const bool ok = (uint32_t)id < (uint32_t)pg.n_pages;
        entries[i] = Entry{ok ? id : 0, ok ? ordinal << deal.shift : kNowhere};
      }
      if (!there) lds_barrier();
      looked_up = b, first_up = r0, end_up = there ? end_up : re;
      Tile<F> cur, next;
      int t = cur.find_seen(r, r0 + wave, re);
      if (t < re) {
        w.load_k(pg, h, cur);
        while (t < re) {
          if (!lone && !F::F32) {
            const int done = (int)(pair_at - f0) + t - t0;
            if (done < quarter) __builtin_amdgcn_s_setprio(3);
            else if (done < 2 * quarter) __builtin_amdgcn_s_setprio(2);
            else if (done < 3 * quarter) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
          }
          next = cur;
          Tile<F> found;
          t = found.find_seen(r, t + kWaves, re);
          if (t < re) next = found;
          if constexpr (HOLDS) {
            w.template step<true>(pg, r, h, c, cur, next, st, &so[wave][0][0] + kept * tile_kept,
                                  &kept_at[wave][kept * 2 * F::NG], rows);
            if (++kept == kKept || kept == room) put_out();
          } else {
            w.template step<WEIGH>(pg, r, h, c, cur, next, st, scores, nullptr, rows);
          }
          cur = next;
        }
        if (HOLDS && kept) put_out();
      }
    }

    // join the waves
    float l = st.l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (w.n < here) {
      if (w.g == 0) sm[wave][w.n] = st.m, sl[wave][w.n] = l;
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int j = 0; j < F::VD; ++j) so[wave][w.n][F::VD * (4 * w.g + y) + j] = st.o[j][y];
    }
    lds_barrier();
    const bool ends = tb == nt, whole = ta == 0 && ends;
    if (!lone && ta == 0 && tid == 0)
      shared[(int64_t)b * deal.R + pair] =
          Shared{(int)blockIdx.x, ends ? 1 : (int)quotient(pair_at + nt - 1, chunk) - (int)blockIdx.x + 1};
    float* slot = whole ? nullptr : part_slot(parts_ws, 2 * (int64_t)blockIdx.x + (ta == 0), rows, D);
    for (int i = tid; i < here * D; i += 64 * kWaves) {
      const int row = i / D, d = i % D;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < kWaves; ++j) top = fmaxf(top, sm[j][row]);
      float o = 0.0f, sum = 0.0f;
#pragma unroll
      for (int j = 0; j < kWaves; ++j) {
        const float a = part_weight(sm[j][row], sl[j][row], top, c);
        o += a * so[j][row][d];
        sum += a * sl[j][row];
      }
      if (whole) {
        const int64_t out_row = (int64_t)b * (deal.R / deal.RT) * G + row0 + row;
        store_f<F::QT>(out + out_row * D + d, sum == 0.0f ? 0.0f : o / (sum * F::PSCALE));
        if (WEIGH && d == 0) {
          if (lone && deal.RT == 1) stats[row] = row_stats(top, sum);
          else weigh.stats[out_row] = row_stats(top, sum);
        }
      } else {
        slot[i] = o;
        if (d == 0) slot[rows * D + row] = top, slot[rows * (D + 1) + row] = sum;
      }
    }
    if (lone) {
      if (WEIGH && deal.RT == 1) {
        __syncthreads();  // the scores are in memory
        add_weights(weigh, pg, ids, b, h, G, c, start, len, tid, 64 * kWaves, [&](int g) { return stats[g]; });
      }
      return;
    }
    if (ends && pair + 1 == deal.R) ++b;
    lds_barrier();
  }
}

// Joins the parts of a pair's rows, a workgroup a row, or a pair where there are
// many; writes the rows of sequences that see nothing.  Up to 16 parts are a team
// of min(D, 64) lanes' for each row; of more, every team takes some of a row's, and
// the teams are joined in LDS.  Eight parts' loads go out at once.  Its time is its
// chain of loads, 4 to 10 us.
template <int QT, int THREADS>
__device__ __forceinline__ void join_rows(const Deal& deal, int G, int D, float c, float pscale,
                                          const int32_t* __restrict__ lengths, const int32_t* __restrict__ starts,
                                          const float* __restrict__ parts, const Shared* __restrict__ shared,
                                          typename Elem<QT>::T* __restrict__ out, float2* __restrict__ stats, int block,
                                          int first, int step) {
  const int tid = threadIdx.x;
  const int b = block / deal.R, pair = block % deal.R;
  const int h = pair / deal.RT, head0 = h * G + 16 * (pair % deal.RT);
  const int rows = G < 16 ? G : 16, here = (h + 1) * G - head0 < 16 ? (h + 1) * G - head0 : 16;
  const Shared who = shared[block];  // nobody's where the sequence has no tiles
  const int64_t row0 = (int64_t)b * (deal.R / deal.RT) * G + head0;
  typename Elem<QT>::T* to = out + row0 * D;
  if (deal.tiles(start_at(starts, b), deal.length(lengths, b)) == 0) {
    for (int i = first * D + tid; i < here * D; i += THREADS * step) store_f<QT>(to + i, 0.0f);
    return;
  }
  if (who.n == 1) return;  // written by its one workgroup
  const int lanes = D < kWave ? D : kWave, d = tid % lanes, team = tid / lanes, teams = THREADS / lanes;
  const bool two = D > kWave;
  struct Sum {
    float m, l, o0, o1;
  };
  // parts i0, i0 + stride, ... of a row, this lane's channels
  auto gather = [&](int row, int i0, int stride) {
    Sum a{-INFINITY, 0.0f, 0.0f, 0.0f};
    for (; i0 < who.n; i0 += 8 * stride) {
      float m[8], l[8], x[8], y[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * stride;
        const bool in = i < who.n;
        // part i is workgroup first + i's
        const float* s = parts + (2 * (int64_t)(who.first + (in ? i : 0)) + (!in || i == 0)) * rows * (D + 2);
        m[u] = in ? s[rows * D + row] : -INFINITY, l[u] = in ? s[rows * (D + 1) + row] : 0.0f;
        // where there is none, part 0's, which weigh nothing here
        x[u] = s[row * D + d], y[u] = two ? s[row * D + 64 + d] : 0.0f;
      }
      float t = a.m;
#pragma unroll
      for (int u = 0; u < 8; ++u) t = fmaxf(t, m[u]);
      const float w = part_weight(a.m, a.l, t, c);
      a.o0 *= w, a.o1 *= w, a.l *= w;
      a.m = t;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float p = part_weight(m[u], l[u], t, c);
        a.o0 += p * x[u], a.o1 += p * y[u], a.l += p * l[u];
      }
    }
    return a;
  };
  // a team a row (43 x 8 pairs of 5 rows in three parts: 4.5 us, 12 with a row at a time)
  if (who.n <= 16) {
    for (int row = first * teams + team; row < here; row += step * teams) {
      const Sum a = gather(row, 0, 1);
      const bool none = a.l == 0.0f;  // no score above -inf, whatever the values are
      const float inv = 1.0f / (a.l * pscale);
      store_f<QT>(to + row * D + d, none ? 0.0f : a.o0 * inv);
      if (stats && d == 0) stats[row0 + row] = row_stats(a.m, a.l);
      if (two) store_f<QT>(to + row * D + 64 + d, none ? 0.0f : a.o1 * inv);
    }
    return;
  }
  constexpr int TEAMS = THREADS / 16;  // at most
  __shared__ float acc[THREADS * 2], tops[TEAMS], suml[TEAMS];
  for (int row = first; row < here; row += step) {
    const Sum a = gather(row, team, teams);
    acc[team * D + d] = a.o0;
    if (two) acc[team * D + 64 + d] = a.o1;
    if (d == 0) tops[team] = a.m, suml[team] = a.l;
    __syncthreads();
    const int used = who.n < teams ? who.n : teams;
    for (int x = tid; x < D; x += THREADS) {
      float t = -INFINITY, o = 0.0f, l = 0.0f;
      for (int w = 0; w < used; ++w) t = fmaxf(t, tops[w]);
      for (int w = 0; w < used; ++w) {
        const float p = part_weight(tops[w], suml[w], t, c);
        o += p * acc[w * D + x], l += p * suml[w];
      }
      store_f<QT>(to + row * D + x, l == 0.0f ? 0.0f : o / (l * pscale));
      if (stats && x == 0) stats[row0 + row] = row_stats(t, l);
    }
    __syncthreads();
  }
}

template <int QT, int THREADS>
__global__ void __launch_bounds__(THREADS) join_kernel(Deal deal, int G, int D, float c, float pscale,
                                                       const int32_t* __restrict__ lengths,
                                                       const int32_t* __restrict__ starts,
                                                       const float* __restrict__ parts,
                                                       const Shared* __restrict__ shared,
                                                       typename Elem<QT>::T* __restrict__ out,
                                                       float2* __restrict__ stats) {
  join_rows<QT, THREADS>(deal, G, D, c, pscale, lengths, starts, parts, shared, out, stats, blockIdx.x, blockIdx.y,
                         gridDim.y);
}

// The join and the weights beside it: `joins` workgroups join, as join_kernel's do, the
// others take four positions a thread and work their rows' statistics out of the parts
// themselves, which costs less than to wait for the join (32 ragged sequences of up to
// 16,384 int8 tokens: 85 -> 83 us; 700 tokens of 8 heads: 19 -> 16).  16 rows of a
// key-value head at most.
template <int QT, int THREADS>
__global__ void __launch_bounds__(THREADS) join_weigh_kernel(Deal deal, int G, int D, float c, float pscale,
                                                             const int32_t* __restrict__ lengths,
                                                             const int32_t* __restrict__ starts,
                                                             const float* __restrict__ parts,
                                                             const Shared* __restrict__ shared,
                                                             typename Elem<QT>::T* __restrict__ out, int joins,
                                                             int rows_at_once, Weigh w, Pages pg,
                                                             const int32_t* __restrict__ table, int64_t table_stride,
                                                             int pieces) {
  if ((int)blockIdx.x < joins) {
    join_rows<QT, THREADS>(deal, G, D, c, pscale, lengths, starts, parts, shared, out, nullptr, blockIdx.x / rows_at_once,
                           blockIdx.x % rows_at_once, rows_at_once);
    return;
  }
  const int block = (int)blockIdx.x - joins, pair = block / pieces, b = pair / pg.H, h = pair % pg.H;
  const int len = deal.length(lengths, b), start = start_at(starts, b);
  const int64_t first = (int64_t)(block % pieces) * THREADS;  // of the workgroup, in units of four positions
  if (start >= len || (start & ~3) + 4 * first >= len) return;  // a row without tiles has no parts
  const int64_t row0 = (int64_t)pair * G;
  __shared__ float2 stats[16];
  const Shared who = shared[pair];
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < G; g += THREADS / kWave) {
    if (who.n == 1) {  // left by the one workgroup that had the row
      if (lane == 0) stats[g] = w.stats[row0 + g];
      continue;
    }
    float m = -INFINITY, l = 0.0f;
    auto with = [&](float m2, float l2) {
      const float t = fmaxf(m, m2);
      l = l * part_weight(m, l, t, c) + l2 * part_weight(m2, l2, t, c);
      m = t;
    };
    for (int i = lane; i < who.n; i += kWave) {
      const float* s = parts + (2 * (int64_t)(who.first + i) + (i == 0)) * G * (D + 2) + G * D + g;
      with(s[0], s[G]);
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) with(__shfl_xor(m, o), __shfl_xor(l, o));
    if (lane == 0) stats[g] = row_stats(m, l);
  }
  __syncthreads();
  add_weights(w, pg, table + b * table_stride, b, h, G, c, start, len, first + threadIdx.x, pieces * THREADS,
              [&](int g) { return stats[g]; });
}

// A call's arguments behind its checks.
struct AttendCall {
  Pages pg;
  const int32_t* table;
  int64_t table_stride;
  int P, B, H, D;
  pfa_tensor4 q;
  const int32_t *lengths, *starts, *selected;
  int64_t selected_stride;
  int S;
  float c;  // scale * log2(e)
  Choice choice;  // count 0: none
  Weigh weigh;    // weights null: none
  void* out;
  float* parts;
  hipStream_t stream;
};

// Workgroups of a call that shares its rows out: as many as the chip holds at
// once, at most kGroups (twice as many: 64 ragged sequences 69 us for 63).
constexpr int kGroups = 1024;
// Places of a chunk, at least (32 pairs of 4,096 listed keys: 22 us, 25 with 16).
constexpr int kLeast = 8;
constexpr int kMany = 256;

// Tiles of a pair that one workgroup takes, rather than workgroups that share the
// rows out and a join behind them.  Few pairs leave the chip idle soon; two pairs a
// unit, of lengths near one another, go through it better whole (512 pairs of 1,800
// keys of 128 bf16 channels: 101 us shared out, 86 whole; 320 of 3,750 keys of 64
// int8: 50 and 70), and rows that select their pages themselves save two launches
// (8 pairs of 14 pages of 64 keys: 18 us and 14).
inline int lone_tiles(int64_t pairs, bool select) { return pairs >= 512 ? 64 : pairs >= kMany || select ? 32 : 16; }

struct Plan {
  Deal deal;
  size_t parts, bytes;  // of the parts, and of the workspace; 0: a workgroup a pair
};

// select: the call selects its pages first
inline Plan attend_plan(int B, int H, int kv_heads, int D, int shift, int P, int S, int tile, bool select) {
  Plan p{};
  const int G = H / kv_heads, RT = (G + 15) / 16;
  const int64_t keys = (int64_t)(S >= 0 ? S : P) << shift, most = (keys + tile - 1) / tile;
  p.deal = Deal{B, kv_heads * RT, RT, S, shift, P, tile, kLeast, 0};
  if (most > lone_tiles((int64_t)B * p.deal.R, select && RT == 1 && few_pages(P, D))) {
    const int64_t chunks = ((most + kStart) * B * p.deal.R + kLeast - 1) / kLeast;
    p.deal.groups = (int)(chunks < kGroups ? chunks : kGroups);
    p.parts = (size_t)p.deal.groups * 2 * (G < 16 ? G : 16) * (D + 2) * 4;
    p.bytes = p.parts + (size_t)B * p.deal.R * sizeof(Shared);
  }
  return p;
}

inline int attend_tile(int ct, int D) { return 32 * tile_groups(ct, D); }

// Workgroups of a kernel that the chip holds at once.
inline int resident(const void* kernel, int threads) {
  int device = 0, units = 0, each = 0;
  if (hipGetDevice(&device) != hipSuccess ||
      hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess ||
      hipOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, threads, 0) != hipSuccess || units * each <= 0)
    return kGroups;
  return units * each;
}

inline void weigh_launch(const AttendCall& a, int G) {
  const int64_t blocks = (a.weigh.cap + 1023) / 1024;
  weigh_kernel<<<dim3((unsigned)(blocks < 65535 ? blocks : 65535), a.pg.H, a.B), 256, 0, a.stream>>>(
      a.weigh, a.pg, a.table, a.table_stride, a.P, G, a.c, a.lengths, a.starts);
}

template <int QT, int CT, int D>
void attend_launch(const AttendCall& a) {
  using F = Form<QT, CT, D>;
  using T = typename Elem<QT>::T;
  Plan p = attend_plan(a.B, a.H, a.pg.H, D, a.pg.shift, a.P, a.S, F::TILE, a.choice.count > 0);
  Deal& deal = p.deal;
  static const int at_once =
      resident(reinterpret_cast<const void*>(&attend_kernel<F, Also::NOTHING>), 64 * kWaves);
  if (deal.groups > at_once) deal.groups = at_once;
  const int G = a.H / a.pg.H;
  const unsigned pairs = (unsigned)(a.B * deal.R);
  Shared* shared = reinterpret_cast<Shared*>(reinterpret_cast<char*>(a.parts) + p.parts);
  const bool q_vec = ((uintptr_t)a.q.ptr | (uintptr_t)(a.q.s_b * sizeof(T)) | (uintptr_t)(a.q.s_h * sizeof(T))) % 16 == 0;
  const bool weighs = a.weigh.weights != nullptr;
  auto launch = [&](auto also) {
    attend_kernel<F, decltype(also)::value><<<p.bytes ? deal.groups : pairs, 64 * kWaves, 0, a.stream>>>(
        a.pg, deal, a.table, a.table_stride, (const T*)a.q.ptr, a.q.s_b, a.q.s_h, q_vec, G, a.lengths, a.starts,
        a.selected, a.selected_stride, a.c, (T*)a.out, p.bytes ? a.parts : nullptr, shared, a.choice, a.weigh);
  };
  if (a.choice.count > 0) launch(std::integral_constant<Also, Also::SELECT>{});
  else if (weighs) launch(std::integral_constant<Also, Also::WEIGH>{});
  else launch(std::integral_constant<Also, Also::NOTHING>{});
  if (!p.bytes) {
    if (weighs && deal.RT > 1) weigh_launch(a, G);
    return;
  }
  const int rows = pairs >= kMany ? 1 : G < 16 ? G : 16;
  auto join = [&](auto threads) {
    constexpr int THREADS = decltype(threads)::value;
    if (weighs && deal.RT == 1) {
      // pieces of a row: all of it at once, but no more workgroups than go through soon
      const int64_t all = (a.weigh.cap + 4 * THREADS - 1) / (4 * THREADS), most = 8192 / pairs;
      const int pieces = (int)(all < most ? all : most > 0 ? most : 1);
      const int joins = (int)pairs * rows;
      join_weigh_kernel<QT, THREADS><<<joins + (int)pairs * pieces, THREADS, 0, a.stream>>>(
          deal, G, D, a.c, F::PSCALE, a.lengths, a.starts, a.parts, shared, (T*)a.out, joins, rows, a.weigh, a.pg, a.table,
          a.table_stride, pieces);
    } else {
      join_kernel<QT, THREADS><<<dim3(pairs, rows), THREADS, 0, a.stream>>>(deal, G, D, a.c, F::PSCALE, a.lengths, a.starts,
                                                                           a.parts, shared, (T*)a.out, a.weigh.stats);
      if (weighs) weigh_launch(a, G);
    }
  };
  // the rows of a few pairs have parts by the hundred (8 pairs of 60,000 keys: 36.6 us
  // with 16 waves a row, 37.4 with four; 32 of 25,000: 88.6 and 85.8)
  if (pairs >= 32) join(std::integral_constant<int, 256>{});
  else join(std::integral_constant<int, 1024>{});
}

template <int QT, int CT>
void attend_by_width(const AttendCall& a) {
  switch (a.D) {
    case 16: return attend_launch<QT, CT, 16>(a);
    case 32: return attend_launch<QT, CT, 32>(a);
    case 64: return attend_launch<QT, CT, 64>(a);
    default: return attend_launch<QT, CT, 128>(a);
  }
}

// One translation unit each, by the cells' type.
void attend_float(int qt, const AttendCall& a);
void attend_i8(int qt, const AttendCall& a);
void attend_e4m3(int qt, const AttendCall& a);
void attend_e2m1(int qt, const AttendCall& a);

}  // namespace paged
}  // namespace pfa
