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
// The nearest quarter turn is taken off exactly; what is left, pi / 4 at most to either
// side, is rounded to f32 as a fraction and once more as an angle, and its sine and cosine
// are their Taylor series, cut off where the next term is below 2^-25 of the value (x^11 /
// 11! and x^12 / 12! at pi / 4: 2^-29 and 2^-33).
//
// Bytes bound it: every value is read and written once.  A workgroup takes some tokens
// of a sequence and computes their sines and cosines into LDS once for all heads, with
// its first rows already on their way.  65,536 f16 tokens of 16 heads of 64, a fused
// projection's slices (268 MB): 43 to 44 us on two sets in turn, of which the last-level
// cache holds a part (6.1 TB/s, where a copy of them takes 55 us); lanes that hold both
// units of a pair, and channels that stay in lanes with half the work: 117.  128 tokens
// of 40 heads of 128: 4.2 us, one of 16 heads of 64: 2.5, both the chain of position,
// sine, LDS and store.
#include <type_traits>

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
  int64_t from;  // a launch's first token
  int per_token;
  int H[2];
  int width, D;
  float magnitude;
  int units, shift;   // of a row, and log2 of its lanes
  int tile, heads;    // tokens and heads of a workgroup: several tokens only with all heads
  uint32_t inverse;   // ceil(2^20 / heads): quotients of up to 1,024 rows
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

// A workgroup's share: some tokens of a sequence, and heads.
struct Share {
  int b, h0, tokens, heads, rows;
  int64_t t0;

  __device__ __forceinline__ explicit Share(const Call& a) {
    b = blockIdx.y, h0 = blockIdx.z * a.heads;
    t0 = a.from + (int64_t)blockIdx.x * a.tile;
    tokens = a.n - t0 < a.tile ? (int)(a.n - t0) : a.tile;
    heads = a.H[0] + a.H[1] - h0 < a.heads ? a.H[0] + a.H[1] - h0 : a.heads;
    rows = tokens * heads;
  }
  // Cosines and sines of its tokens' pairs.  Loads come back in order: those for a
  // thread's first are sent before the rows, so that the rows are not waited for.
  struct Angle {
    int64_t position;
    uint64_t turns;
  };
  __device__ __forceinline__ Angle angle(const Call& a, int i) const {
    const int half = a.width / 2, token = i / half;
    const int32_t* at = a.positions + b * a.pos_b;
    if (i >= tokens * half) return Angle{0, 0};
    return Angle{a.per_token ? (int64_t)at[(t0 + token) * a.pos_t] : *at + t0 + token, a.turns[i - token * half]};
  }
  __device__ __forceinline__ void angles(const Call& a, Angle x, float2* table) const {
    for (int i = threadIdx.x; i < tokens * (a.width / 2); i += blockDim.x) {
      if (i > (int)threadIdx.x) x = angle(a, i);
      table[i] = cos_sin(x.position, x.turns, a.magnitude);
    }
  }
};

// Where a row of it is.
struct Place {
  const void* in;
  void* out;
  int token;

  __device__ __forceinline__ Place(const Call& a, const Share& s, int r, int bytes) {
    token = (int)((uint32_t)r * a.inverse >> 20);
    const int head = s.h0 + r - token * s.heads;
    const bool keys = head >= a.H[0];
    const int h = keys ? head - a.H[0] : head;
    // Field by field: a choice between tensors has every lane read them from memory
    // (65,536 f16 tokens of 16 heads of 64: 66 us, 47 so).
    auto at = [&](const pfa_tensor4& x, const pfa_tensor4& y) {
      const int64_t s_h = keys ? y.s_h : x.s_h, s_t = keys ? y.s_t : x.s_t;
      char* const p0 = (char*)x.ptr + (s.b * x.s_b + s.t0 * x.s_t) * bytes;
      char* const p1 = (char*)y.ptr + (s.b * y.s_b + s.t0 * y.s_t) * bytes;
      return (keys ? p1 : p0) + (h * s_h + token * s_t) * bytes;
    };
    in = at(a.in[0], a.in[1]);
    out = at(a.out[0], a.out[1]);
  }
};

// Eight elements as they are in memory, and as f32.
template <int DT>
struct Eight {
  uint4 w[DT == PFA_F32 ? 2 : 1];

  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const uint4* q = reinterpret_cast<const uint4*>((const typename Elem<DT>::T*)p + at);
    w[0] = q[0];
    if constexpr (DT == PFA_F32) w[1] = q[1];
  }
  __device__ __forceinline__ void store(void* p, int64_t at) const {
    uint4* q = reinterpret_cast<uint4*>((typename Elem<DT>::T*)p + at);
    q[0] = w[0];
    if constexpr (DT == PFA_F32) q[1] = w[1];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    load8<DT>(reinterpret_cast<const typename Elem<DT>::T*>(w), x);
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    if constexpr (DT == PFA_F32) {
      store8<DT>(reinterpret_cast<float*>(w), x);
    } else {
      using T = std::conditional_t<DT == PFA_BF16, __bf16, _Float16>;
      typedef __attribute__((__vector_size__(8 * sizeof(T)))) T V;
      V y;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = (T)x[i];
      w[0] = __builtin_bit_cast(uint4, y);
    }
  }
};

// Rows of all four tensors aligned to 16 bytes, in units of eight channels that lie
// together and turn alike: a lane a unit.  In halves its partner's unit is read, too
// (from the L1: another lane of the wave reads it), so that all lanes have the same
// work, whatever part of the head turns.  A row's lanes are of one wave, and their
// loads are through before the first of its stores: it may turn in place.
template <int DT, bool HALVES>
__global__ void __launch_bounds__(kThreads) rows_kernel(Call a) {
  extern __shared__ float2 table[];
  const Share s(a);
  const int step = blockDim.x >> a.shift, unit = threadIdx.x & ((1 << a.shift) - 1), half = a.width / 2;
  const bool turn = 8 * unit < a.width, upper = HALVES && 8 * unit >= half;
  const int partner = upper ? 8 * unit - half : 8 * unit + half;
  const float2* mine = table + (HALVES ? (upper ? partner : 8 * unit) : 4 * unit);
  int row = unit < a.units ? (int)threadIdx.x >> a.shift : s.rows;
  Eight<DT> x[kAtOnce], y[HALVES ? kAtOnce : 1];
  auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (row + i * step >= s.rows) continue;
      const Place p(a, s, row + i * step, sizeof(typename Elem<DT>::T));
      x[i].load(p.in, 8 * unit);
      if (HALVES && turn) y[i].load(p.in, partner);
    }
  };
  const Share::Angle first = s.angle(a, threadIdx.x);
  fetch();
  s.angles(a, first, table);
  __syncthreads();
  while (row < s.rows) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (row + i * step >= s.rows) continue;
      const Place p(a, s, row + i * step, sizeof(typename Elem<DT>::T));
      if (turn) {
        const float2* cs = mine + p.token * half;
        float u[8], o[8];
        x[i].get(u);
        if constexpr (HALVES) {
          float v[8];
          y[i].get(v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float vs = v[j] * cs[j].y;
            o[j] = fmaf(u[j], cs[j].x, upper ? vs : -vs);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            o[j] = fmaf(u[j], cs[j / 2].x, -(u[j + 1] * cs[j / 2].y));
            o[j + 1] = fmaf(u[j + 1], cs[j / 2].x, u[j] * cs[j / 2].y);
          }
        }
        x[i].set(o);
      }
      x[i].store(p.out, 8 * unit);
    }
    row += kAtOnce * step;
    if (row < s.rows) fetch();
  }
}

// Any other rows: a lane a pair, or one of the channels that stay.
template <int DT>
__global__ void __launch_bounds__(kThreads) pairs_kernel(Call a, int halves) {
  extern __shared__ float2 table[];
  using T = typename Elem<DT>::T;
  const Share s(a);
  s.angles(a, s.angle(a, threadIdx.x), table);
  __syncthreads();
  const int step = blockDim.x >> a.shift, unit = threadIdx.x & ((1 << a.shift) - 1), half = a.width / 2;
  const int at = unit >= half ? unit + half : halves ? unit : 2 * unit, other = halves ? at + half : at + 1;
  for (int row = unit < a.units ? (int)threadIdx.x >> a.shift : s.rows; row < s.rows; row += step) {
    const Place p(a, s, row, sizeof(T));
    const T* in = (const T*)p.in;
    T* out = (T*)p.out;
    if (unit >= half) {
      out[at] = in[at];
      continue;
    }
    const float u = load_f<DT>(in + at), v = load_f<DT>(in + other);
    const float2 cs = table[p.token * half + unit];
    store_f<DT>(out + at, fmaf(u, cs.x, -(v * cs.y)));
    store_f<DT>(out + other, fmaf(v, cs.x, u * cs.y));
  }
}

template <int DT>
void launch(Call a, int B, bool halves, bool vec, hipStream_t stream) {
  const int heads = a.H[0] + a.H[1], half = a.width / 2;
  a.units = vec ? a.D / 8 : half + a.D - a.width;
  while ((1 << a.shift) < a.units) ++a.shift;
  // heads of a workgroup, then tokens
  const int most = kUnits >> a.shift;
  a.heads = heads < most ? heads : most;
  int64_t tile = a.heads < heads ? 1 : most / a.heads;
  if (tile > kPairs / half) tile = kPairs / half;
  if (tile > a.n) tile = a.n;
  a.tile = (int)tile;
  a.inverse = ((1u << 20) + a.heads - 1) / a.heads;
  const int64_t lanes = (tile * a.heads) << a.shift;
  const int threads = lanes >= kThreads ? kThreads : (int)((lanes + kWave - 1) / kWave * kWave);
  const size_t lds = (size_t)tile * half * sizeof(float2);
  // a grid has fewer than 2^32 threads along x: from 2^24 workgroups on, several launches
  const int64_t all = (a.n + tile - 1) / tile, once = (1ll << 32) / threads - 1;
  for (int64_t at = 0; at < all; at += once) {
    a.from = at * tile;
    const dim3 grid((unsigned)(all - at < once ? all - at : once), B, (heads + a.heads - 1) / a.heads);
    if (!vec) pairs_kernel<DT><<<grid, threads, lds, stream>>>(a, halves);
    else if (halves) rows_kernel<DT, true><<<grid, threads, lds, stream>>>(a);
    else rows_kernel<DT, false><<<grid, threads, lds, stream>>>(a);
  }
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
