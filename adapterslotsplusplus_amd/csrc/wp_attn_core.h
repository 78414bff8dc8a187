// wp_attn_core.h -- what the attention kernels share (gfx950): a wave's 32 query
// rows and their running softmax, fragments of staged keys and values, and the work of
// one staged tile.  Everything sits in an anonymous namespace, as in wp_device.h.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "wp_device.h"
#include "wp_model.h"

namespace wp {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr int kWaveRows = 32;
constexpr int kTileKeys = 64;                  // keys staged at a time for a row tile
// A running bound is raised (and O and l scaled) only once a score exceeds it
// by 2^8: exponentials then stay within 2^8, far inside fp16, and most tiles
// scale nothing.
constexpr float kSlack = 8.f;

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

template <typename T>
__device__ __forceinline__ typename VecOf<T>::v8 negate8(typename VecOf<T>::v8 v) {
  const u32x4 u = __builtin_bit_cast(u32x4, v);
  return __builtin_bit_cast(typename VecOf<T>::v8, u ^ 0x80008000u);
}

// Which of two 16-bit values are infinite or NaN are cleared.
template <typename T>
__device__ __forceinline__ bool finite16(uint32_t half) {
  constexpr uint32_t e = sizeof(T) == 2 && __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;
  return (half & e) != e;
}
template <typename T>
__device__ __forceinline__ i16x4 finite_only(i16x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = finite16<T>(static_cast<uint16_t>(v[i])) ? v[i] : static_cast<short>(0);
  return v;
}

// Head columns computed (DP, a multiple of 32) and how a row of K or V lies in
// LDS: 128 or 256 bytes in 16-byte chunks, columns past the head zero.
//   K row r keeps chunk c at c ^ key_swizzle(r): the rows that a fragment load touches at one c
//   fall on different banks.
//   V row r keeps chunk c at c ^ value_swizzle(r): the transposing read takes 64
//   bytes of each of eight rows, which so fall on different banks too.
template <int DP>
struct Head {
  static constexpr int kRow = DP <= 64 ? 128 : 256;
  static constexpr int kChunks = kRow / 16;
  static constexpr int kRowsPerLoad = 1024 / kRow;  // rows a wave's 16-byte-per-lane load fills
  static constexpr int kSteps = DP / 16;            // contraction steps of S
  static constexpr int kCols = DP / 32;             // 32-column tiles of O
  static __device__ __forceinline__ int key_swizzle(int r) { return kRow == 256 ? r & 15 : (r >> 1) & 7; }
  static __device__ __forceinline__ int value_swizzle(int r) { return kRow == 256 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }
};

// The first key that a query at key position `pos` sees: with the windows the
// host takes, up to 2^31 - 1, pos - window + 1 need not fit 32 bits.
__device__ __forceinline__ int window_start(int pos, int window) {
  return window > 0 ? std::max(0, std::max(0, pos + 1) - window) : 0;
}

// The sum of v over the lanes up to this one, by lane moves within the vector
// unit (a shuffle goes through LDS and takes some ten times as long).
__device__ __forceinline__ int sum_up(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // from 1 lane down, in rows of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);  // 2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);  // 4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);  // 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);  // the row before's last lane
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);  // the first half's last lane
  return v;
}
__device__ __forceinline__ int total_of(int v) { return __builtin_amdgcn_readlane(sum_up(v), 63); }

// K fragment of step `step`: keys row0 .. row0 + 31 of a staged tile.  (The lane by its
// own number here, not handed down: the compiler schedules that better, 58.5 and 60.0 us
// for 16 packed prompts of 512, 32 heads over 8 of 64.)
template <typename T, int DP>
__device__ __forceinline__ typename VecOf<T>::v8 key_fragment(const char* keys, int row0, int step) {
  using H = Head<DP>;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int r = lane & 31, c = step * 2 + (lane >> 5);
  return *reinterpret_cast<const typename VecOf<T>::v8*>(keys + (row0 + r) * H::kRow + ((c ^ H::key_swizzle(r)) << 4));
}

// Four keys of a column at `at`, and the four that are eight rows on.
template <typename T, int DP, bool kCareful>
__device__ __forceinline__ typename VecOf<T>::v8 value_at(const char* values, int at) {
  using H = Head<DP>;
  using L = __attribute__((address_space(3))) i16x4;
  i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(values + at));
  i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(values + (at + 8 * H::kRow)));
  if (kCareful) {
    lo = finite_only<T>(lo);
    hi = finite_only<T>(hi);
  }
  union {
    i16x4 h[2];
    typename VecOf<T>::v8 v;
  } u;
  u.h[0] = lo;
  u.h[1] = hi;
  return u.v;
}

// V^T fragment of columns col * 32 .. + 31 and the 16 keys from key0, in the
// order of the packed exponentials: lane half h has keys 4h .. 4h + 3 and
// 8 + 4h .. 8 + 4h + 3.
template <typename T, int DP, bool kCareful>
__device__ __forceinline__ typename VecOf<T>::v8 value_fragment(const char* values, int key0, int col) {
  using H = Head<DP>;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int i = lane & 15, g = lane >> 4;
  const int r = 4 * (g >> 1) + (i >> 2);
  const int c = col * 4 + (g & 1) * 2 + ((i & 3) >> 1);
  return value_at<T, DP, kCareful>(values, (key0 + r) * H::kRow + ((c ^ H::value_swizzle(r)) << 4) + (i & 1) * 8);
}

// The lane that a wave's work goes by, and its fragments: the thread's own number
// (kOwn) or one that a kernel keeps (kHeld), in a form that the compiler takes for
// a number of that moment alone.  Then one address of either kind is kept, too: a
// step or a column on changes bits of it that no row touches.  kRenewed: those changes are
// made anew for each tile and not kept in registers from tile to tile.
enum LaneKind { kOwn, kHeld, kRenewed };
template <LaneKind kKind>
struct KeptLane;
template <LaneKind kKind>
struct Lane : KeptLane<kKind> {};
template <>
struct Lane<kOwn> {
  __device__ __forceinline__ int lane() const { return static_cast<int>(threadIdx.x) & 63; }
  __device__ __forceinline__ void renew() {}
  template <typename T, int DP>
  __device__ __forceinline__ typename VecOf<T>::v8 key(const char* keys, int row0, int step) const {
    return key_fragment<T, DP>(keys, row0, step);
  }
  template <typename T, int DP, bool kCareful>
  __device__ __forceinline__ typename VecOf<T>::v8 value(const char* values, int key0, int col) const {
    return value_fragment<T, DP, kCareful>(values, key0, col);
  }
};
template <LaneKind kKind>
struct KeptLane {
  int held, key_place, value_place;
  __device__ __forceinline__ int lane() const { return held; }
  template <int DP>
  __device__ __forceinline__ void hold(int lane) {
    using H = Head<DP>;
    held = lane;
    const int k = lane & 31, i = lane & 15, g = lane >> 4, v = 4 * (g >> 1) + (i >> 2);
    key_place = k * H::kRow + (((lane >> 5) ^ H::key_swizzle(k)) << 4);
    value_place = v * H::kRow + ((((g & 1) * 2 + ((i & 3) >> 1)) ^ H::value_swizzle(v)) << 4) + (i & 1) * 8;
  }
  __device__ __forceinline__ void renew() {
    if (kKind == kRenewed) asm volatile("" : "+v"(key_place), "+v"(value_place));
  }
  template <typename T, int DP>
  __device__ __forceinline__ typename VecOf<T>::v8 key(const char* keys, int row0, int step) const {
    return *reinterpret_cast<const typename VecOf<T>::v8*>(keys + (key_place ^ (step << 5)) + row0 * Head<DP>::kRow);
  }
  template <typename T, int DP, bool kCareful>
  __device__ __forceinline__ typename VecOf<T>::v8 value(const char* values, int key0, int col) const {
    return value_at<T, DP, kCareful>(values, (value_place ^ (col << 6)) + key0 * Head<DP>::kRow);
  }
};

// A wave's 32 query rows and their running state.
template <typename T, int DP, LaneKind kKind = kOwn>
struct Rows : Lane<kKind> {
  using H = Head<DP>;
  using V8 = typename VecOf<T>::v8;
  V8 q[H::kSteps];
  f32x16 o[H::kCols];
  float m;      // running bound, in units of c * s
  float l;      // this lane's keys' sum
  int pos;      // key position of the lane's query (causal), else the last key
  int low;      // first key it sees

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < H::kCols; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  // Raises the bound where a score exceeds it by the slack (tops: the lane's
  // largest score of the tile).
  __device__ __forceinline__ void raise(float tops, float c) {
    const float t = tops * c;
    if (__any(t > m + kSlack)) {
      const float top = fmaxf(fmaxf(t, __shfl_xor(t, 32)), m);
      const float fade = top == -INFINITY ? 1.f : exp2_fast(m - top);
      m = top;
      l *= fade;
#pragma unroll
      for (int i = 0; i < H::kCols; ++i) o[i] *= fade;
    }
  }

  // Scores of keys [at, at + 32) that the lane's query does not see become -inf.
  __device__ __forceinline__ void mask(f32x16& s, int at) {
    const int first = at + (this->lane() >> 5) * 4;
    const int up = pos - first, down = low - first;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int key = (e >> 2) * 8 + (e & 3);
      s[e] = key <= up && key >= down ? s[e] : -INFINITY;
    }
  }
};

__device__ __forceinline__ float top_of(const f32x16& s) {
  float t = fmaxf(s[0], s[1]);
#pragma unroll
  for (int e = 2; e < 16; e += 2) t = fmaxf(fmaxf(t, s[e]), s[e + 1]);
  return t;
}

// Adds the infinite and NaN values of n staged keys that a query sees (sees(r):
// the lane's of key r), which value_fragment<careful> left out.
template <typename T, int DP, LaneKind kKind, typename Sees>
__device__ __forceinline__ void add_nonfinite(Rows<T, DP, kKind>& w, const char* values, int n, Sees sees_key) {
  using H = Head<DP>;
  const int lane = w.lane(), half = lane >> 5;
  for (int r = 0; r < n; ++r) {
    const char* row = values + r * H::kRow;
    bool odd = false;
    if (lane < H::kRow / 4) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(row + lane * 4);
      odd = !finite16<T>(u & 0xFFFFu) || !finite16<T>(u >> 16);
    }
    if (!__any(odd)) continue;
    const bool sees = sees_key(r);
#pragma unroll
    for (int i = 0; i < H::kCols; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = i * 32 + (e >> 2) * 8 + half * 4 + (e & 3);
        const int c = (d >> 3) ^ H::value_swizzle(r);
        const uint16_t u = *reinterpret_cast<const uint16_t*>(row + c * 16 + (d & 7) * 2);
        if (sees && !finite16<T>(u)) w.o[i][e] += static_cast<float>(__builtin_bit_cast(T, u));
      }
  }
}

template <typename T>
__device__ __forceinline__ const T* head_row(const void* base, int64_t tok, int64_t tok_stride, int64_t head_offset) {
  return static_cast<const T*>(base) + tok * tok_stride + head_offset;
}

// Exponentials of a 32-key tile, added to the lane's sum in fp32 and packed: the
// two right operands of its two 16-key steps.  The matrix cores take 16-bit
// operands: each weight is rounded to the tensors' type, once, so that O is off
// by at most half a unit of that type of sum p |v| -- what rounding the values
// themselves did.
template <typename T, int DP, LaneKind kKind>
__device__ __forceinline__ void weigh(Rows<T, DP, kKind>& w, const f32x16& s, float c, typename VecOf<T>::v8 (&out)[2]) {
  const float base = w.m == -INFINITY ? 0.f : w.m;
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = exp2_fast(fmaf(s[b * 8 + e], c, -base));
      w.l += x;
      out[b][e] = static_cast<T>(x);
    }
}

// Scores of 32 staged keys from row0 on; LDS reads go four products ahead.
template <typename T, int DP, LaneKind kKind>
__device__ __forceinline__ f32x16 scores(const Rows<T, DP, kKind>& w, const char* keys, int row0) {
  constexpr int kSteps = Head<DP>::kSteps;
  typename VecOf<T>::v8 kf[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) kf[x] = w.template key<T, DP>(keys, row0, x);
  __builtin_amdgcn_sched_barrier(0);
  f32x16 s{};
#pragma unroll
  for (int x = 0; x < kSteps; ++x) {
    s = mfma32(kf[x % 4], w.q[x], s);
    if (x + 4 < kSteps) kf[x % 4] = w.template key<T, DP>(keys, row0, x + 4);
    __builtin_amdgcn_sched_barrier(0);
  }
  return s;
}

// Adds 32 staged keys' weighted values to O.
template <typename T, int DP, bool kCareful, LaneKind kKind>
__device__ __forceinline__ void accumulate(Rows<T, DP, kKind>& w, const char* values, int row0,
                                           const typename VecOf<T>::v8 (&e)[2]) {
  constexpr int kCols = Head<DP>::kCols, kAhead = kCols < 4 ? kCols : 4;
  auto value = [&](int i) { return w.template value<T, DP, kCareful>(values, row0 + i / kCols * 16, i % kCols); };
  typename VecOf<T>::v8 vf[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) vf[i] = value(i);
  if (!kCareful) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 2 * kCols; ++i) {
    w.o[i % kCols] = mfma32(vf[i % kAhead], e[i / kCols], w.o[i % kCols]);
    if (i + kAhead < 2 * kCols) vf[i % kAhead] = value(i + kAhead);
    if (!kCareful) __builtin_amdgcn_sched_barrier(0);
  }
}

// The order of a tile's work is pinned so that products and vector work run
// side by side throughout (two waves a SIMD in the same phase would else wait
// for the one unit together and leave the other idle):
//   the first half's exponentials between three quarters of the next tile's scores,
//   the second half's between the rest of them and the first half's products with V,
//   the next scores' maximum between the second half's products with V.
// LDS reads go two products ahead.
//
// Weighs and adds the 64 staged keys whose masked scores are s0 and s1 (tops: the
// lane's largest of them) and, with `more`, computes the next tile's into their place.
template <typename T, int DP, LaneKind kKind, typename More>
__device__ __forceinline__ void tile_body(Rows<T, DP, kKind>& w, f32x16& s0, f32x16& s1, float& tops, float c, More more,
                                          const char* knext, const char* vnow) {
  using H = Head<DP>;
  using V8 = typename VecOf<T>::v8;
  w.renew();
  constexpr int kScores = 2 * H::kSteps, kFirst = kScores * 3 / 4, kValues = 2 * H::kCols;
  w.raise(tops, c);
  const float base = w.m == -INFINITY ? 0.f : w.m;
  auto weigh = [&](f32x16& s, int from, int to) {
#pragma unroll
    for (int i = from; i < to; ++i) {
      s[i] = exp2_fast(fmaf(s[i], c, -base));
      w.l += s[i];
    }
  };
  auto key = [&](int i) { return w.template key<T, DP>(knext, i / H::kSteps * 32, i % H::kSteps); };
  auto value = [&](int i) { return w.template value<T, DP, false>(vnow, i / H::kCols * 16, i % H::kCols); };
  f32x16 n[2] = {};
  V8 kf[3], vf[3], e[4];
  if (more) {
    kf[0] = key(0);
    kf[1] = key(1);
  }
  auto score = [&](int i) {
    n[i / H::kSteps] = mfma32(kf[i % 3], w.q[i % H::kSteps], n[i / H::kSteps]);
    if (i + 2 < kScores) kf[(i + 2) % 3] = key(i + 2);
  };
  auto add = [&](int i) {
    f32x16& o = w.o[i % H::kCols];
    o = mfma32(vf[i % 3], e[i / H::kCols], o);
    if (i + 2 < 2 * kValues) vf[(i + 2) % 3] = value(i + 2);
  };
  auto pack = [&](const f32x16& s, int to) {
#pragma unroll
    for (int i = 0; i < 16; ++i) e[to + i / 8][i % 8] = static_cast<T>(s[i]);
  };
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    if (more) score(i);
    weigh(s0, i * 16 / kFirst, (i + 1) * 16 / kFirst);
    __builtin_amdgcn_sched_barrier(0);
  }
  pack(s0, 0);
  vf[0] = value(0);
  vf[1] = value(1);
  constexpr int kSecond = kScores - kFirst + kValues;
#pragma unroll
  for (int i = 0; i < kSecond; ++i) {
    if (i < kScores - kFirst) {
      if (more) score(kFirst + i);
    } else {
      add(i - (kScores - kFirst));
    }
    weigh(s1, i * 16 / kSecond, (i + 1) * 16 / kSecond);
    __builtin_amdgcn_sched_barrier(0);
  }
  pack(s1, 2);
#pragma unroll
  for (int i = 0; i < kValues; ++i) {
    add(kValues + i);
    if (more) {
#pragma unroll
      for (int x = i * 16 / kValues; x < (i + 1) * 16 / kValues; ++x)
        tops = x == 0 ? fmaxf(n[0][0], n[1][0]) : fmaxf(fmaxf(tops, n[0][x]), n[1][x]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (more) {
    s0 = n[0];
    s1 = n[1];
  }
}

// LDS of a workgroup.  Each buffer is an array of its own: the compiler then
// sees that a load into one leaves reads of the others alone, and does not wait
// for it.
template <int DP>
struct Staged {
  static constexpr int kBytes = kTileKeys * Head<DP>::kRow;
};
#define WP_STAGED char (&sk0)[Staged<DP>::kBytes], char (&sk1)[Staged<DP>::kBytes], char (&sv0)[Staged<DP>::kBytes], \
                  char (&sv1)[Staged<DP>::kBytes]

template <typename T, int DP, LaneKind kKind>
__device__ __forceinline__ bool has_nonfinite(const Rows<T, DP, kKind>& w) {
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < Head<DP>::kCols; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) z = fmaf(w.o[i][e], 0.f, z);
  return z != 0.f;  // NaN: an infinity or NaN times zero
}

}  // namespace
}  // namespace wp
