// wp_heads.hip -- rows of heads between a projection and a paged cache (gfx950):
// norms of queries and keys, rotation by position, rows into the cache's pages
// (in the tensors' type or e4m3) and back.
//
// For a row x of a head at position p, with norm weights w:
//   n = x * w / sqrt(mean x^2 + eps)                      (x itself without)
//   y_a = n_a cos(p f_i) - n_b sin(p f_i),  y_b = n_b cos(p f_i) + n_a sin(p f_i)
// for the pair i of elements (a, b), all in fp32, rounded once: to the tensors'
// type, or, into an 8-bit cache, to e4m3 of y / s, s the smallest power of two
// that brings the row's largest magnitude to at most 448.  (A power of two costs
// e4m3 nothing of its 4 significant bits and makes y / s and its way back exact.)
//
// Angles are 64-bit fractions of a turn: p * f modulo 2^64 is exact, its top 32
// bits are the angle within 2^-32 turns, and an eighth of a turn either way is left to
// polynomials (the Taylor series of sine to t^9 and of cosine to t^10: off by
// at most 2e-9 there).
//
// What bounds it.  Prompts: HBM, each element read and written once; 8192 tokens, 32
// and 8 heads of 128 in bf16 take 37.4 us with norms (4.5 TB/s; 32.5 without, 5.2),
// 43.0 into a cache with their values, 44.2 into one of 8 bits (there the vector unit, in
// part); 32 heads from pages 37.3, from 8-bit ones 27.4 (7.2 and 7.4 TB/s, half of it in the
// last cache).  Few tokens: launch and the chain position, angle, row, store: 5.5 us
// for one, 6.3 for 64.
//
// Layout.  A lane holds both 16-byte vectors of eight pairs, so each angle is computed
// once for all of a token's heads and each element loaded once (55 us where a lane held
// one vector and loaded its partner's beside it).  With eight waves' worth of tokens for
// each compute unit a wave takes all heads of a token, its loads a batch ahead of its
// stores, the first ones before the angles (39.8 us without); with fewer, as many waves
// share a token's heads.  A row stays within a wave, which has read all of it before it
// writes: results may replace their inputs.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "wp_apply.h"
#include "wp_device.h"
#include "wp_paged.h"

namespace wp {
namespace {

constexpr int kWaves = 4;
constexpr int kBatch = 4;  // rows of loads of a wave that are on their way together

// Sum (or maximum) over the L lanes of a row, in every one of them.
template <int L, typename F>
__device__ __forceinline__ float over_row(float v, F f) {
  auto moved = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = f(v, moved(v, std::integral_constant<int, 0xB1>{}));   // its neighbour's
  v = f(v, moved(v, std::integral_constant<int, 0x4E>{}));   // the other two of four
  if constexpr (L >= 8) v = f(v, moved(v, std::integral_constant<int, 0x141>{}));  // the other four of eight, reversed
  if constexpr (L >= 16) v = f(v, moved(v, std::integral_constant<int, 0x140>{}));
  if constexpr (L >= 32) v = f(v, __shfl_xor(v, 16));
  return v;
}

// Cosine and sine of p * turns, times `factor`.
__device__ __forceinline__ void turn(uint64_t p, uint64_t turns, float factor, float& c, float& s) {
  const int32_t phase = static_cast<int32_t>(static_cast<uint32_t>((p * turns) >> 32));
  const uint32_t quarter = (static_cast<uint32_t>(phase) + 0x20000000u) >> 30;
  const int32_t rest = static_cast<int32_t>(static_cast<uint32_t>(phase) - (quarter << 30));  // an eighth either way
  const float t = static_cast<float>(rest) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float u = t * t;
  const float sn = fmaf(t * u, fmaf(u, fmaf(u, fmaf(u, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), t);
  const float cs =
      fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
  const float x = quarter & 1u ? sn : cs, y = quarter & 1u ? cs : sn;
  c = (quarter + 1u) & 2u ? -factor * x : factor * x;  // quarters 1 and 2
  s = quarter & 2u ? -factor * y : factor * y;
}

template <typename T>
__device__ __forceinline__ void unpack8(u32x4 q, float (&v)[8]) {
  const auto h = __builtin_bit_cast(typename VecOf<T>::v8, q);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(h[e]);
}
template <typename T>
__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
  typename VecOf<T>::v8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = static_cast<T>(v[e]);
  return __builtin_bit_cast(u32x4, h);
}

// A lane's N elements of a row in e4m3: its bytes, and the row's scale code in
// every lane.  The scale goes by the finite elements; infinities and NaN become NaN,
// as e4m3 has no infinity.  Magnitudes past the tensors' type's range count as its
// largest, so the scale ends where that one's does (fp16's 65504: 2^8), and where a
// magnitude would come back beyond the range (65504 is 256 * 2^8 in 4 significant
// bits), it becomes the value below.  Such rows are told by their largest
// magnitude, NaN if there is one, and looked at element by element.
template <typename T, int L, int N>
__device__ __forceinline__ void quantise(const float (&y)[N], uint32_t (&q)[N / 4], uint32_t& code) {
  constexpr bool kHalf = __is_same(T, _Float16);
  constexpr int kTopScale = kHalf ? 8 : 120;  // of the type's largest; 2^this * 256 is past its range
  auto most = [](float a, float b) { return __builtin_elementwise_maximum(a, b); };
  // 448 = 1.75 * 2^8.
  auto scale_of = [](float top) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, top);
    return std::clamp(static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126, 127);
  };
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) top = most(top, fabsf(y[e]));
  top = over_row<L>(top, most);
  int x = scale_of(top);
  const bool plain = x < kTopScale;  // (an infinity's and NaN's is past it)
  float z[N];
  if (__all(plain)) {
#pragma unroll
    for (int e = 0; e < N; ++e) z[e] = __builtin_ldexpf(y[e], -x);
  } else {
    top = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) top = fabsf(y[e]) < INFINITY ? fmaxf(top, fabsf(y[e])) : top;
    top = over_row<L>(top, most);
    x = std::min(scale_of(top), kTopScale);
    const float limit = x == kTopScale ? 240.f : 448.f;
#pragma unroll
    for (int e = 0; e < N; ++e)
      z[e] = fabsf(y[e]) < INFINITY ? std::clamp(__builtin_ldexpf(y[e], -x), -limit, limit) : __builtin_nanf("");
  }
  code = static_cast<uint32_t>(x + 127);
#pragma unroll
  for (int h = 0; h < N / 4; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * h], z[4 * h + 1], 0, false);
    q[h] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(z[4 * h + 2], z[4 * h + 3], w, true));
  }
}

// The unit of this wave: heads of a kind from head0 on, or (p.all) all of a token's.
struct Unit {
  int64_t tok;
  int kind, head0;
};
template <int kRows>
__device__ __forceinline__ bool unit_of(const HeadArgs& p, Unit& u) {
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const uint32_t id = blockIdx.x * kWaves + wave;
  if (id >= p.n_units) return false;
  const int tok = over(static_cast<int>(id), p.by_units);
  int at = static_cast<int>(id) - tok * p.units_tok;
  u.tok = tok;
  u.kind = at < p.units[0] ? 0 : at < p.units[0] + p.units[1] ? 1 : 2;
  at -= u.kind == 0 ? 0 : u.kind == 1 ? p.units[0] : p.units[0] + p.units[1];
  u.head0 = at * p.steps * kRows;
  return true;
}

// Entry i of int64 or int32 numbers.
__device__ __forceinline__ int64_t number(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// Moves y, and scales with it, to where the token's rows of a kind go (mine: reads a
// field of it).  False: its slot keeps none.
template <typename F>
__device__ __forceinline__ bool find_results(const HeadArgs& p, const Unit& u, int lane, F mine, bool cached, int64_t y_tok, char*& y,
                                             uint8_t*& scales) {
  if (!cached) {
    y += u.tok * y_tok * 2;
    return true;
  }
  const int64_t slot = number(p.slots, p.slots64, u.tok);
  if (slot < 0) return false;
  if (slot >= p.n_slots) {
    if (lane == 0 && u.head0 == 0) flag_error(p.header, kErrIdRange);
    return false;
  }
  const int64_t page = slot >> p.page_shift, at = slot & ((1ll << p.page_shift) - 1);
  y += (page * mine([](const HeadPart& h) { return h.y_page; }) + at * y_tok) * (p.e4m3 != 0 ? 1 : 2);
  if (p.e4m3 != 0) scales += page * mine([](const HeadPart& h) { return h.s_page; }) + at * mine([](const HeadPart& h) { return h.s_tok; });
  return true;
}

// Rows whose halves lie in whole 16-byte vectors (and what does not rotate, too):
// a lane holds both vectors of eight pairs, so that each element is loaded once
// and each pair's angle computed once a row group.  kAdjacent: the pairs of 16 elements in a row;
// else elements 8 i .. of the first half and of the second, and past them two vectors that pass.
//   y1 = r (x1 w1 c - x2 w2 s),  y2 = r (x2 w2 c + x1 w1 s),  r = 1 / sqrt(mean x^2 + eps)
// with the products of weights and sines computed once for a kind's heads.
template <typename T, int L, bool kAdjacent>
__global__ __launch_bounds__(64 * kWaves) void head_pairs_kernel(HeadArgs p) {
  constexpr int kRows = 64 / L;
  touch_kernel_args<static_cast<int>(sizeof(HeadArgs))>();
  Unit u;
  if (!unit_of<kRows>(p, u)) return;
  const int lane = static_cast<int>(threadIdx.x) & 63, col = lane % L, row = lane / L;
  const int dim = p.dim, rot = p.positions != nullptr ? p.rot : 0, half = rot >> 1;
  const bool holds = col * 16 < dim, turns = col * 16 < rot;
  // The lane's two vectors.
  const int past = 2 * (col - half / 8) * 8 + rot;
  const int d1 = kAdjacent ? col * 16 : turns ? col * 8 : past, d2 = kAdjacent ? d1 + 8 : turns ? d1 + half : past + 8;
  float c[8], s[8];
  bool known = rot == 0;  // the angles
  auto angles = [&] {
    const uint64_t pos = static_cast<uint64_t>(number(p.positions, p.positions64, u.tok));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = 1.f;
      s[e] = 0.f;
    }
    if (turns) {
#pragma unroll
      for (int e = 0; e < 8; ++e) turn(pos, static_cast<uint64_t>(p.turns[col * 8 + e]), p.factor, c[e], s[e]);
    }
    known = true;
  };
  // A vector's elements as the pairs' first and second ones.
  auto pairs_of = [&](u32x4 a, u32x4 b, float (&x1)[8], float (&x2)[8]) {
    float v[8], w[8];
    unpack8<T>(a, v);
    unpack8<T>(b, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x1[e] = !kAdjacent ? v[e] : e < 4 ? v[2 * e] : w[2 * e - 8];
      x2[e] = !kAdjacent ? w[e] : e < 4 ? v[2 * e + 1] : w[2 * e - 7];
    }
  };
  const float inv_dim = 1.f / static_cast<float>(dim);
  const u32x4 zero{0u, 0u, 0u, 0u};
  for (int kind = p.all ? 0 : u.kind; kind < (p.all ? 3 : u.kind + 1); ++kind) {
    // (Selected field by field: a pointer to an argument would move them all to memory.)
    auto mine = [&](auto f) { return kind == 0 ? f(p.part[0]) : kind == 1 ? f(p.part[1]) : f(p.part[2]); };
    const int heads = mine([](const HeadPart& h) { return h.heads; });
    if (heads == 0) continue;
    const T* x = static_cast<const T*>(mine([](const HeadPart& h) { return h.x; })) +
                 u.tok * mine([](const HeadPart& h) { return h.x_tok; });
    const int64_t x_head = mine([](const HeadPart& h) { return h.x_head; });
    const T* w = static_cast<const T*>(mine([](const HeadPart& h) { return h.norm; }));
    const bool cached = mine([](const HeadPart& h) { return h.cached; }) != 0;
    const bool rotates = rot > 0 && mine([](const HeadPart& h) { return h.rotate; }) != 0;
    char* y = static_cast<char*>(mine([](const HeadPart& h) { return h.y; }));
    uint8_t* scales = mine([](const HeadPart& h) { return h.scales; });
    const int64_t y_tok = mine([](const HeadPart& h) { return h.y_tok; }), y_head = mine([](const HeadPart& h) { return h.y_head; });
    const int64_t s_head = mine([](const HeadPart& h) { return h.s_head; });
    const bool small = cached && p.e4m3 != 0;
    if (!find_results(p, u, lane, mine, cached, y_tok, y, scales)) continue;
    const int head0 = p.all ? 0 : u.head0, end = p.all ? heads : std::min(heads, head0 + p.steps * kRows);
    // Loads go a batch ahead, the first ones before the angles are worked out.
    constexpr int kAtOnce = 2;
    u32x4 in1[kAtOnce], in2[kAtOnce];
    auto load = [&](int h0) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int h = h0 + i * kRows + row;
        const bool live = holds && h < end;
        in1[i] = live ? load16_global(x + h * x_head + d1) : zero;
        in2[i] = live ? load16_global(x + h * x_head + d2) : zero;
      }
    };
    load(head0);
    if (!known) angles();
    // Weights times sines.
    float k11[8], k12[8], k21[8], k22[8];
    {
      float w1[8], w2[8];
      if (w != nullptr) pairs_of(holds ? load16_global(w + d1) : zero, holds ? load16_global(w + d2) : zero, w1, w2);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = w != nullptr ? w1[e] : 1.f, b = w != nullptr ? w2[e] : 1.f;
        k11[e] = rotates ? a * c[e] : a;
        k22[e] = rotates ? b * c[e] : b;
        k12[e] = rotates ? -b * s[e] : 0.f;
        k21[e] = rotates ? a * s[e] : 0.f;
      }
    }
    // A row of nothing but copies keeps every bit.
    const bool copies = w == nullptr && !rotates && !small;
    for (int h0 = head0; h0 < end; h0 += kAtOnce * kRows) {
      u32x4 now1[kAtOnce], now2[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        now1[i] = in1[i];
        now2[i] = in2[i];
      }
      if (h0 + kAtOnce * kRows < end) load(h0 + kAtOnce * kRows);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int h = h0 + i * kRows + row;
        const bool live = holds && h < end;
        if (copies) {
          if (live) {
            *reinterpret_cast<u32x4*>(y + (h * y_head + d1) * 2) = now1[i];
            *reinterpret_cast<u32x4*>(y + (h * y_head + d2) * 2) = now2[i];
          }
          continue;
        }
        float x1[8], x2[8], z[16];
        pairs_of(now1[i], now2[i], x1, x2);
        float r = 1.f;
        if (w != nullptr) {
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], sum));
          sum = over_row<L>(sum, [](float a, float b) { return a + b; });
          r = 1.f / sqrtf(fmaf(sum, inv_dim, p.eps));
        }
        if (rotates) {
          // (What passes beside rotating elements must not see its neighbour's infinities.)
          const bool mixes = rot == dim || turns;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = mixes ? x2[e] : 0.f, b = mixes ? x1[e] : 0.f;
            z[kAdjacent ? 2 * e : e] = fmaf(x1[e], k11[e], a * k12[e]) * r;
            z[kAdjacent ? 2 * e + 1 : 8 + e] = fmaf(x2[e], k22[e], b * k21[e]) * r;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            z[kAdjacent ? 2 * e : e] = x1[e] * k11[e] * r;
            z[kAdjacent ? 2 * e + 1 : 8 + e] = x2[e] * k22[e] * r;
          }
        }
        if (small) {
          uint32_t code, q[4];
          quantise<T, L>(z, q, code);
          if (live) {
            *reinterpret_cast<u32x2*>(y + h * y_head + d1) = u32x2{q[0], q[1]};
            *reinterpret_cast<u32x2*>(y + h * y_head + d2) = u32x2{q[2], q[3]};
            if (col == 0) scales[h * s_head] = static_cast<uint8_t>(code);
          }
        } else if (live) {
          float a[8], b[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            a[e] = z[e];
            b[e] = z[8 + e];
          }
          *reinterpret_cast<u32x4*>(y + (h * y_head + d1) * 2) = pack8<T>(a);
          *reinterpret_cast<u32x4*>(y + (h * y_head + d2) * 2) = pack8<T>(b);
        }
      }
    }
  }
}

// Any other rows: the lane's eight columns, and their partners' loaded beside them.
template <typename T, int L>
__global__ __launch_bounds__(64 * kWaves) void head_rows_kernel(HeadArgs p) {
  constexpr int kRows = 64 / L;
  touch_kernel_args<static_cast<int>(sizeof(HeadArgs))>();
  Unit u;
  if (!unit_of<kRows>(p, u)) return;
  // (Selected field by field: a pointer to an argument would move them all to memory.)
  auto mine = [&](auto f) { return u.kind == 0 ? f(p.part[0]) : u.kind == 1 ? f(p.part[1]) : f(p.part[2]); };
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int d0 = lane % L * 8, dim = p.dim, heads = mine([](const HeadPart& h) { return h.heads; });
  const bool holds = d0 < dim;
  const T* x = static_cast<const T*>(mine([](const HeadPart& h) { return h.x; })) +
               u.tok * mine([](const HeadPart& h) { return h.x_tok; });
  const int64_t x_head = mine([](const HeadPart& h) { return h.x_head; });
  const T* w = static_cast<const T*>(mine([](const HeadPart& h) { return h.norm; }));
  const bool cached = mine([](const HeadPart& h) { return h.cached; }) != 0;
  const bool rotates = mine([](const HeadPart& h) { return h.rotate; }) != 0;

  // Where results go.
  char* y = static_cast<char*>(mine([](const HeadPart& h) { return h.y; }));
  uint8_t* scales = mine([](const HeadPart& h) { return h.scales; });
  const int64_t y_tok = mine([](const HeadPart& h) { return h.y_tok; }), y_head = mine([](const HeadPart& h) { return h.y_head; });
  const int64_t s_head = mine([](const HeadPart& h) { return h.s_head; });
  const bool small = cached && p.e4m3 != 0;
  if (!find_results(p, u, lane, mine, cached, y_tok, y, scales)) return;

  // The lane's columns: sines, and where each one's partner is.
  const int rot = rotates ? p.rot : 0, half = rot >> 1;
  const bool apart = rot > 0 && p.interleaved == 0;  // the partner is half a rotation away
  const bool vectors = (half & 7) == 0;              // ... in one 16-byte vector
  const int partner = d0 < half ? d0 + half : d0 - half;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  if (rot > 0 && d0 < rot) {
    const uint64_t pos = static_cast<uint64_t>(number(p.positions, p.positions64, u.tok));
    if (apart) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        if (d >= rot) continue;
        float c, s;
        turn(pos, static_cast<uint64_t>(p.turns[d < half ? d : d - half]), p.factor, c, s);
        cs[e] = c;
        sn[e] = d < half ? -s : s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if (d0 + e >= rot) continue;
        float c, s;
        turn(pos, static_cast<uint64_t>(p.turns[(d0 + e) >> 1]), p.factor, c, s);
        cs[e] = cs[e + 1] = c;
        sn[e] = -s;
        sn[e + 1] = s;
      }
    }
  }
  // The partners of eight columns, zero where there are none.
  auto partners = [&](const T* row, float (&v)[8]) {
    if (vectors) {
      unpack8<T>(d0 < rot ? load16_global(row + partner) : u32x4{0u, 0u, 0u, 0u}, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        v[e] = d < rot ? static_cast<float>(row[d < half ? d + half : d - half]) : 0.f;
      }
    }
  };
  float wn[8], wo[8];
  if (w != nullptr) {
    unpack8<T>(holds ? load16_global(w + d0) : u32x4{0u, 0u, 0u, 0u}, wn);
    if (apart) partners(w, wo);
  }

  const int row = lane / L;
  const float inv_dim = 1.f / static_cast<float>(dim);
  for (int step = 0; step < p.steps && u.head0 + step * kRows < heads; step += kBatch) {
    u32x4 in[kBatch];
    float other[kBatch][8];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = u.head0 + (step + i) * kRows + row;
      const bool live = holds && h < heads && step + i < p.steps;
      in[i] = live ? load16_global(x + h * x_head + d0) : u32x4{0u, 0u, 0u, 0u};
    }
    if (apart) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int h = u.head0 + (step + i) * kRows + row;
        const bool live = holds && h < heads && step + i < p.steps;
        if (live) {
          partners(x + h * x_head, other[i]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) other[i][e] = 0.f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = u.head0 + (step + i) * kRows + row;
      const bool live = holds && h < heads && step + i < p.steps;
      float v[8];
      unpack8<T>(in[i], v);
      if (w != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
        sum = over_row<L>(sum, [](float a, float b) { return a + b; });
        const float r = 1.f / sqrtf(fmaf(sum, inv_dim, p.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * r * wn[e];
        if (apart) {
#pragma unroll
          for (int e = 0; e < 8; ++e) other[i][e] = other[i][e] * r * wo[e];
        }
      }
      if (rot > 0) {
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float o = apart ? other[i][e] : d0 + e < rot ? v[e ^ 1] : 0.f;
          z[e] = fmaf(v[e], cs[e], o * sn[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z[e];
      }
      if (small) {
        uint32_t code, q[2];
        quantise<T, L>(v, q, code);
        if (live) {
          *reinterpret_cast<u32x2*>(y + h * y_head + d0) = u32x2{q[0], q[1]};
          if (d0 == 0) scales[h * s_head] = static_cast<uint8_t>(code);
        }
      } else if (live) {
        *reinterpret_cast<u32x4*>(y + (h * y_head + d0) * 2) = pack8<T>(v);
      }
    }
  }
}

// Rows of the cache, as the tensors' type.  (Codes 0 and 255, which nothing here
// writes, are no factors of fp32's normal numbers: what such rows give is not defined.)
template <typename T, int L, bool kSmall>
__global__ __launch_bounds__(64 * kWaves) void read_rows_kernel(HeadArgs p) {
  constexpr int kRows = 64 / L;
  touch_kernel_args<static_cast<int>(sizeof(HeadArgs))>();
  Unit u;
  if (!unit_of<kRows>(p, u)) return;
  auto mine = [&](auto f) { return u.kind == 0 ? f(p.part[0]) : u.kind == 1 ? f(p.part[1]) : f(p.part[2]); };
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int d0 = lane % L * 8, heads = mine([](const HeadPart& h) { return h.heads; });
  const bool holds = d0 < p.dim;
  const int64_t slot = number(p.slots, p.slots64, u.tok);
  const bool there = slot >= 0 && slot < p.n_slots;
  if (slot >= p.n_slots && lane == 0 && u.head0 == 0) flag_error(p.header, kErrIdRange);
  const int64_t page = there ? slot >> p.page_shift : 0, at = there ? slot & ((1ll << p.page_shift) - 1) : 0;
  constexpr int kSize = kSmall ? 1 : 2;
  const char* x = static_cast<const char*>(mine([](const HeadPart& h) { return h.x; })) +
                  (page * mine([](const HeadPart& h) { return h.y_page; }) + at * mine([](const HeadPart& h) { return h.x_tok; })) * kSize;
  const uint8_t* scales = mine([](const HeadPart& h) { return h.scales; });
  if (kSmall) scales += page * mine([](const HeadPart& h) { return h.s_page; }) + at * mine([](const HeadPart& h) { return h.s_tok; });
  const int64_t x_head = mine([](const HeadPart& h) { return h.x_head; }), s_head = mine([](const HeadPart& h) { return h.s_head; });
  T* y = static_cast<T*>(mine([](const HeadPart& h) { return h.y; })) + u.tok * mine([](const HeadPart& h) { return h.y_tok; });
  const int64_t y_head = mine([](const HeadPart& h) { return h.y_head; });
  const int row = lane / L;
  for (int step = 0; step < p.steps && u.head0 + step * kRows < heads; step += kBatch) {
    u32x4 in[kBatch];
    uint32_t code[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = u.head0 + (step + i) * kRows + row;
      const bool live = there && holds && h < heads && step + i < p.steps;
      in[i] = u32x4{0u, 0u, 0u, 0u};
      code[i] = 1u;
      if (live) {
        if constexpr (kSmall) {
          const u32x2 q = *reinterpret_cast<const u32x2*>(x + h * x_head + d0);
          in[i][0] = q[0];
          in[i][1] = q[1];
          code[i] = scales[h * s_head];
        } else {
          in[i] = load16_global(x + (h * x_head + d0) * 2);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = u.head0 + (step + i) * kRows + row;
      if (!(holds && h < heads && step + i < p.steps)) continue;
      if constexpr (kSmall) {
        const float s = __builtin_bit_cast(float, code[i] << 23);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(in[i][e / 4]), false);
          const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(in[i][e / 4]), true);
          v[e] = a[0] * s;
          v[e + 1] = a[1] * s;
          v[e + 2] = b[0] * s;
          v[e + 3] = b[1] * s;
        }
        *reinterpret_cast<u32x4*>(y + h * y_head + d0) = pack8<T>(v);
      } else {
        *reinterpret_cast<u32x4*>(y + h * y_head + d0) = in[i];
      }
    }
  }
}

// Splits each token's heads of each kind into units of `steps` wave-wide rows:
// one unit if there are tokens enough, else as many as keep the device's
// waves busy.
bool plan_units(HeadArgs& a, int lanes, int n_cu, bool may_join) {
  const int rows = 64 / lanes;
  // Tokens enough for eight waves a compute unit each take a wave for all of
  // their heads, whose angles it computes once.
  a.all = may_join && a.tokens >= 8ll * n_cu ? 1 : 0;
  if (a.all) {
    a.units_tok = 1;
    a.units[0] = 1;
    a.units[1] = a.units[2] = 0;
    a.steps = 0;
    a.n_units = static_cast<uint32_t>(a.tokens);
    a.by_units = divisor_of(1);
    return true;
  }
  int most = 1;
  for (const HeadPart& h : a.part) most = std::max(most, (h.heads + rows - 1) / rows);
  int64_t steps = most;
  // At least eight waves a compute unit, in units of one batch or more.
  while (steps > kBatch && a.tokens * ((most + steps - 1) / steps) < 8ll * n_cu) steps = std::max<int64_t>(kBatch, steps / 2);
  a.steps = static_cast<int32_t>(steps);
  a.units_tok = 0;
  for (int i = 0; i < 3; ++i) {
    a.units[i] = static_cast<int32_t>((a.part[i].heads + steps * rows - 1) / (steps * rows));
    a.units_tok += a.units[i];
  }
  const int64_t n = a.tokens * a.units_tok;
  if (n > 0x7FFFFFFF) return false;
  a.n_units = static_cast<uint32_t>(n);
  a.by_units = divisor_of(a.units_tok);
  return true;
}

}  // namespace

namespace {
template <typename T>
hipError_t head_rows(HeadArgs& a, int n_cu, hipStream_t stream) {
  const bool pairs = a.dim % 16 == 0 && (a.positions == nullptr || a.rot % 16 == 0);
  const int lanes = pairs ? (a.dim <= 64 ? 4 : a.dim <= 128 ? 8 : 16) : a.dim <= 64 ? 8 : a.dim <= 128 ? 16 : 32;
  if (!plan_units(a, lanes, n_cu, pairs)) return hipErrorInvalidValue;
  const dim3 grid((a.n_units + kWaves - 1) / kWaves), block(64 * kWaves);
  auto go = [&](auto* kernel) {
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, a);
    return hipGetLastError();
  };
  if (!pairs)
    return lanes == 8 ? go(head_rows_kernel<T, 8>) : lanes == 16 ? go(head_rows_kernel<T, 16>) : go(head_rows_kernel<T, 32>);
  if (a.interleaved)
    return lanes == 4 ? go(head_pairs_kernel<T, 4, true>) : lanes == 8 ? go(head_pairs_kernel<T, 8, true>) : go(head_pairs_kernel<T, 16, true>);
  return lanes == 4 ? go(head_pairs_kernel<T, 4, false>) : lanes == 8 ? go(head_pairs_kernel<T, 8, false>) : go(head_pairs_kernel<T, 16, false>);
}
}  // namespace

hipError_t launch_head_rows(int dtype_bf16, HeadArgs& a, int n_cu, hipStream_t stream) {
  return dtype_bf16 ? head_rows<__bf16>(a, n_cu, stream) : head_rows<_Float16>(a, n_cu, stream);
}

namespace {
template <typename T, bool kSmall>
hipError_t read_rows(const HeadArgs& a, int lanes, hipStream_t stream) {
  const dim3 grid((a.n_units + kWaves - 1) / kWaves), block(64 * kWaves);
  if (lanes == 8)
    hipLaunchKernelGGL((read_rows_kernel<T, 8, kSmall>), grid, block, 0, stream, a);
  else if (lanes == 16)
    hipLaunchKernelGGL((read_rows_kernel<T, 16, kSmall>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((read_rows_kernel<T, 32, kSmall>), grid, block, 0, stream, a);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_read_rows(int dtype_bf16, HeadArgs& a, int n_cu, hipStream_t stream) {
  const int lanes = a.dim <= 64 ? 8 : a.dim <= 128 ? 16 : 32;
  if (!plan_units(a, lanes, n_cu, false)) return hipErrorInvalidValue;
  if (dtype_bf16) return a.e4m3 ? read_rows<__bf16, true>(a, lanes, stream) : read_rows<__bf16, false>(a, lanes, stream);
  return a.e4m3 ? read_rows<_Float16, true>(a, lanes, stream) : read_rows<_Float16, false>(a, lanes, stream);
}

}  // namespace wp
