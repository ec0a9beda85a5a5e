// Rotary positions of queries and keys.
//
// A pair of channels (a, b) of a token at position p turns by the angle p w, w the
// pair's frequency:  (a cos - b sin, b cos + a sin) * magnitude.  Pairs are (2j, 2j + 1)
// where they are interleaved, (j, j + width / 2) in halves; channels from `width` on
// stay.
//
// Angles.  A frequency comes as turns a position, w / 2 pi, in units of 2^-64: the
// product with the position, modulo 2^64, is the angle's fraction of a turn, exactly,
// at any position of 32 bits.  No table of positions is read, and none limits them.
// The fraction's first three bits give the octant; what is left, at most pi / 4, is
// rounded to f32 once, and its sine and cosine are their Taylor series, cut off where
// the next term is below 2^-25 of the value (x^11 / 11! and x^12 / 12! at pi / 4: 2^-29
// and 2^-33).
//
// Bytes bound it: every value is read and written once.  A workgroup takes some tokens
// of a sequence and computes their sines and cosines into LDS once for all heads, with
// its first rows already on their way.
#include "pfa_common.h"

namespace pfa {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 1024;  // of a workgroup: four a thread
constexpr int kAtOnce = 4;    // rows of a thread on their way at once
constexpr int kPairs = 2048;  // sines and cosines of a workgroup, at most (16 KB)
constexpr int kWidest = 256;  // channels of a head

struct Call {
  pfa_tensor4 in[2], out[2];  // queries and keys
  const uint64_t* turns;
  const int32_t* positions;
  int64_t pos_b, pos_t, n;
  int per_token;
  int H[2];
  int width, D;
  float magnitude;
  int turning, units, shift;  // units of a row that turn, all of them, and log2 of the lanes of a row
  int tile, heads;            // tokens and heads of a workgroup
  uint32_t inverse;           // ceil(2^20 / heads)
};

// The angle of a position in turns of 2^-64: its cosine and sine.
__device__ __forceinline__ float2 cos_sin(int64_t position, uint64_t turns, float magnitude) {
  const uint64_t angle = (uint64_t)position * turns;
  const uint32_t quarter = (uint32_t)((angle + (1ull << 61)) >> 62);  // the nearest
  const float x = (float)(int64_t)(angle - ((uint64_t)quarter << 62)) * 3.40612158e-19f;  // 2 pi / 2^64
  const float y = x * x;
  float s = fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = fmaf(y, s, 1.0f / 120.0f);
  s = fmaf(y, s, -1.0f / 6.0f);
  s = fmaf(y * x, s, x);
  float c = fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = fmaf(y, c, -1.0f / 720.0f);
  c = fmaf(y, c, 1.0f / 24.0f);
  c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.0f);
  const bool swap = quarter & 1;
  const float a = swap ? s : c, b = swap ? c : s;
  return make_float2(((quarter + 1) & 2 ? -a : a) * magnitude, (quarter & 2 ? -b : b) * magnitude);
}

// N elements (8 of them aligned to 16 bytes, or one) as f32.
template <int DT, int N>
__device__ __forceinline__ void get(const void* p, int64_t at, float* x) {
  const auto* q = (const typename Elem<DT>::T*)p + at;
  if constexpr (N == 8) {
    float y[8];
    load8<DT>(q, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
  } else {
    x[0] = load_f<DT>(q);
  }
}

template <int DT, int N>
__device__ __forceinline__ void put(void* p, int64_t at, const float* x) {
  auto* q = (typename Elem<DT>::T*)p + at;
  if constexpr (N == 8 && DT == PFA_BF16) {
    typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
    bf16x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (__bf16)x[i];
    *reinterpret_cast<bf16x8*>(q) = y;
  } else if constexpr (N == 8) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
    store8<DT>(q, y);
  } else {
    store_f<DT>(q, x[0]);
  }
}

// VEC: rows of all four tensors are aligned to 16 bytes and fall into units of eight
// elements; else a unit is a pair, or one of the channels that stay.
template <int DT, bool HALVES, bool VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(Call a) {
  extern __shared__ float2 table[];
  constexpr int N = VEC ? 8 : 1;                      // elements of a load
  constexpr int PAIRS = HALVES ? N : VEC ? 4 : 1;     // of a unit
  constexpr int LOADS = HALVES || !VEC ? 2 : 1;       // of a unit that turns
  const int b = blockIdx.y, h0 = blockIdx.z * a.heads;
  const int64_t t0 = (int64_t)blockIdx.x * a.tile;
  const int tokens = a.n - t0 < a.tile ? (int)(a.n - t0) : a.tile;
  const int heads = a.H[0] + a.H[1] - h0 < a.heads ? a.H[0] + a.H[1] - h0 : a.heads;
  const int rows = tokens * heads, step = blockDim.x >> a.shift;
  const int unit = threadIdx.x & ((1 << a.shift) - 1);
  const bool turn = unit < a.turning;
  const int half = a.width / 2;
  const int at0 = !turn ? a.width + (unit - a.turning) * N : unit * (HALVES ? N : VEC ? 8 : 2);
  const int at1 = HALVES ? at0 + half : at0 + 1;  // of the second load
  int row = unit < a.units ? threadIdx.x >> a.shift : rows;

  struct Place {
    int64_t in, out;
    int token, which;
  };
  auto place = [&](int r) {
    const int token = (int)((uint32_t)r * a.inverse >> 20);
    const int head = h0 + r - token * heads;
    const int which = head >= a.H[0];
    const int h = head - (which ? a.H[0] : 0);
    const pfa_tensor4 &x = a.in[which], &y = a.out[which];
    return Place{b * x.s_b + h * x.s_h + (t0 + token) * x.s_t, b * y.s_b + h * y.s_h + (t0 + token) * y.s_t, token,
                 which};
  };
  float x[kAtOnce][LOADS * N];
  auto fetch = [&](int first) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int r = first + i * step;
      if (r >= rows) continue;
      const Place p = place(r);
      get<DT, N>(a.in[p.which].ptr, p.in + at0, x[i]);
      if (LOADS == 2 && turn) get<DT, N>(a.in[p.which].ptr, p.in + at1, x[i] + N);
    }
  };
  fetch(row);
  for (int i = threadIdx.x; i < tokens * half; i += blockDim.x) {
    const int token = i / half, pair = i - token * half;
    const int32_t* at = a.positions + b * a.pos_b;
    const int64_t position = a.per_token ? (int64_t)at[(t0 + token) * a.pos_t] : *at + t0 + token;
    table[i] = cos_sin(position, a.turns[pair], a.magnitude);
  }
  __syncthreads();
  while (row < rows) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int r = row + i * step;
      if (r >= rows) continue;
      const Place p = place(r);
      void* to = a.out[p.which].ptr;
      if (!turn) {
        put<DT, N>(to, p.out + at0, x[i]);
        continue;
      }
      const float2* cs = table + p.token * half + unit * PAIRS;
      float y[LOADS * N];
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const int u = HALVES ? j : 2 * j, v = HALVES ? j + N : 2 * j + 1;
        const float2 z = cs[j];
        y[u] = fmaf(x[i][u], z.x, -(x[i][v] * z.y));
        y[v] = fmaf(x[i][v], z.x, x[i][u] * z.y);
      }
      put<DT, N>(to, p.out + at0, y);
      if (LOADS == 2) put<DT, N>(to, p.out + at1, y + N);
    }
    row += kAtOnce * step;
    if (row < rows) fetch(row);
  }
}

template <int DT>
void launch(Call a, int B, bool halves, bool vec, hipStream_t stream) {
  const int heads = a.H[0] + a.H[1], half = a.width / 2, pairs = halves ? 8 : 4;
  a.turning = vec ? half / pairs : half;
  a.units = a.turning + (a.D - a.width) / (vec ? 8 : 1);
  while ((1 << a.shift) < a.units) ++a.shift;
  // heads of a workgroup, then tokens
  const int most = kUnits >> a.shift;
  a.heads = heads < most ? heads : most;
  int64_t tile = most / a.heads;
  if (tile > kPairs / half) tile = kPairs / half;
  if (tile > a.n) tile = a.n;
  a.tile = (int)tile;
  a.inverse = ((1u << 20) + a.heads - 1) / a.heads;
  const int64_t lanes = (tile * a.heads) << a.shift;
  const int threads = lanes >= kThreads ? kThreads : (int)((lanes + kWave - 1) / kWave * kWave);
  const dim3 grid((unsigned)((a.n + tile - 1) / tile), B, (heads + a.heads - 1) / a.heads);
  const size_t lds = (size_t)tile * half * sizeof(float2);
#define PFA_ROTARY(HALVES, VEC) rotary_kernel<DT, HALVES, VEC><<<grid, threads, lds, stream>>>(a)
  if (halves && vec) PFA_ROTARY(true, true);
  else if (halves) PFA_ROTARY(true, false);
  else if (vec) PFA_ROTARY(false, true);
  else PFA_ROTARY(false, false);
#undef PFA_ROTARY
}

}  // namespace
}  // namespace pfa

using namespace pfa;

extern "C" int pfa_rotary(const pfa_rotary_call* c, void* stream) {
  clear_error();
  PFA_CHECK_ARG(c, "rotary: null argument");
  PFA_CHECK_ARG(c->dtype == PFA_F32 || c->dtype == PFA_BF16 || c->dtype == PFA_F16, "rotary: unknown value type %d",
                c->dtype);
  PFA_CHECK_ARG(c->head_dim > 0 && c->head_dim <= kWidest, "rotary: 1 to %d channels a head (got %d)", kWidest,
                c->head_dim);
  PFA_CHECK_ARG(c->width > 0 && c->width % 2 == 0 && c->width <= c->head_dim,
                "rotary: an even width of up to the head's %d channels (got %d)", c->head_dim, c->width);
  PFA_CHECK_ARG(c->H > 0 && c->H <= 65535 && c->Hk >= 0 && c->Hk <= 65535, "rotary: 1 to 65535 heads (got %d, %d)",
                c->H, c->Hk);
  PFA_CHECK_ARG(c->B >= 0 && c->B <= 65535 && c->n >= 0 && c->n < (1ll << 31),
                "rotary: up to 65535 sequences and 2^31 - 1 tokens (got %d, %lld)", c->B, (long long)c->n);
  PFA_CHECK_ARG(c->magnitude > 0.0f && c->magnitude < INFINITY, "rotary: magnitude must be positive and finite");
  if (c->B == 0 || c->n == 0) return PFA_OK;
  PFA_CHECK_ARG(c->q.ptr && c->q_out.ptr && c->turns && c->positions && (c->Hk == 0 || (c->k.ptr && c->k_out.ptr)),
                "rotary: null argument");
  Call a{};
  a.in[0] = c->q, a.in[1] = c->k, a.out[0] = c->q_out, a.out[1] = c->k_out;
  a.turns = c->turns, a.positions = c->positions, a.pos_b = c->pos_b, a.pos_t = c->pos_t, a.n = c->n;
  a.per_token = c->per_token, a.H[0] = c->H, a.H[1] = c->Hk, a.width = c->width, a.D = c->head_dim;
  a.magnitude = c->magnitude;
  const int e = c->dtype == PFA_F32 ? 4 : 2;
  bool vec = c->width % (c->interleaved ? 8 : 16) == 0 && c->head_dim % 8 == 0;
  for (int i = 0; i < (c->Hk ? 2 : 1); ++i)
    for (const pfa_tensor4* x : {&a.in[i], &a.out[i]})
      vec = vec && (uintptr_t)x->ptr % 16 == 0 && x->s_b * e % 16 == 0 && x->s_h * e % 16 == 0 && x->s_t * e % 16 == 0;
  auto* s = as_stream(stream);
  if (c->dtype == PFA_F32) launch<PFA_F32>(a, c->B, !c->interleaved, vec, s);
  else if (c->dtype == PFA_BF16) launch<PFA_BF16>(a, c->B, !c->interleaved, vec, s);
  else launch<PFA_F16>(a, c->B, !c->interleaved, vec, s);
  PFA_CHECK_LAUNCH("rotary");
  return PFA_OK;
}
