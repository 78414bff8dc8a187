// wp_logprobs.hip -- log probabilities of given tokens, the entropy of the
// distribution and its largest alternatives (gfx950).
//
// One pass over the logits.  A thread keeps its largest logit m so far and,
// with y = (x - m) log2(e), s = sum 2^y and w = sum 2^y y; threads and
// workgroups join theirs to a common m, and then
//   log softmax(x) = (x - m) - ln s,   entropy = ln s - (w / s) ln 2.
// The alternatives are kept beside it: a list in LDS of the elements that beat
// a threshold which at least `top` elements are known to reach.  The
// threshold starts as the top-th largest of 64 groups' maxima over the first
// chunk (about top elements reach it) and rises when the list is cut down, so
// nearly every 16-byte vector is dismissed by one comparison of its maximum.
//
// What bounds it: 2 to 4 bytes an element from HBM against some eleven vector
// instructions (one of them an exponential), and six more for the alternatives.
// 4096 rows of 128000, bf16: 210 to 230 us without alternatives (up to 5.0 TB/s),
// 250 with 20, where the vector unit is never idle.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "wp_device.h"
#include "wp_model.h"

namespace wp {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWaves = kRowThreads / 64;
// Elements of a chunk per thread: 16, of any type.  (4096 rows of 128000, top 20:
// 16-bit 251 us, with 32 elements 279, whose registers leave two workgroups a
// compute unit for four; fp32 326 us, with eight 350, for twice the barriers.)
constexpr int kThreadElements = 16;
constexpr int kListCap = 4096;      // candidates held; at least kMaxParts * kMaxTop
// The list is cut down past this many beyond `top`: the threshold then rises
// with nearly every chunk, and fewer vectors hold a candidate (4096 rows of
// 128000 logits, top 20, in chunks twice as long: 306 us at 128, 282 at 48, 279 at 16).
constexpr int kListTrim = 16;
constexpr int kMaxParts = 64;       // workgroups that share a row
constexpr int kPartBytes = 16 + 8 * kMaxTop;
static_assert(kMaxTop + kListTrim <= kRowThreads, "a thread each for the candidates kept");
static_assert(kMaxParts * kMaxTop <= kListCap, "the joined parts' candidates fit the list");

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

// Orders a logit and its id: greater values first, equal ones by the lower
// id, NaN above every number.  Never 0.
__device__ __forceinline__ uint64_t order_key(float v, int id) {
  uint32_t u = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);
  u = v != v ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<uint64_t>(u) << 32) | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __builtin_bit_cast(float, (u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int key_id(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
};
template <typename T>
__device__ __forceinline__ float element(const u32x4& v, int i) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t u = v[i];
    return __builtin_bit_cast(float, u);
  } else {
    const uint16_t h = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
    return static_cast<float>(__builtin_bit_cast(T, h));
  }
}
// The same for an index known only at run time.
template <typename T>
__device__ __forceinline__ float element_at(const u32x4& v, int i) {
  constexpr int kShift = sizeof(T) == 4 ? 0 : 1;
  const int word = i >> kShift;
  const uint32_t u0 = v[0], u1 = v[1], u2 = v[2], u3 = v[3];
  const uint32_t u = word == 0 ? u0 : word == 1 ? u1 : word == 2 ? u2 : u3;
  return element<T>(u32x4{u >> (16 * (i & kShift)), 0u, 0u, 0u}, 0);
}
template <typename T>
__device__ __forceinline__ u32x4 lowest() {
  const uint32_t u = sizeof(T) == 4 ? 0xFF800000u : __is_same(T, __bf16) ? 0xFF80FF80u : 0xFC00FC00u;
  return u32x4{u, u, u, u};
}
// A share of a row: its largest logit (-inf for none), s and w.
struct Stats {
  float m, s, w;
};
// How far b lies under a in units of log2: a share without numbers (m = -inf)
// has s and w zero, or NaN where it saw one, and is taken as it is.
__device__ __forceinline__ float distance(float b, float a) { return b == -INFINITY ? 0.f : (b - a) * kLog2e; }
// A share brought under the maximum d higher.  One 2^200 times smaller adds
// nothing; its distance, which may be infinite, is cut there.
__device__ __forceinline__ void lower(Stats& a, float d) {
  const float f = exp2f(d);
  a.w = f * fmaf(a.s, fmaxf(d, -200.f), a.w);
  a.s *= f;
}
__device__ __forceinline__ Stats join(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  lower(a, distance(a.m, m));
  lower(b, distance(b.m, m));
  return Stats{m, a.s + b.s, a.w + b.w};
}
__device__ __forceinline__ Stats shuffle(const Stats& a, int x) {
  return Stats{__shfl_xor(a.m, x), __shfl_xor(a.s, x), __shfl_xor(a.w, x)};
}

__device__ __forceinline__ float log_prob(float v, float m, float ln_s) { return (v - m) - ln_s; }

struct Shared {
  uint64_t list[kListCap];
  uint64_t best[kMaxTop];
  uint64_t kept[kMaxTop + kListTrim];
  uint64_t group[64];
  uint64_t tau;
  Stats stats[kRowWaves];
  int above[kRowWaves];
  int count;
  int last;
};

// Cuts the list of n candidates down to the `top` largest, in order, and
// raises the threshold to the last of them.  A candidate's place is the number
// of candidates above it.  Every thread calls it; n <= kListCap.
__device__ __forceinline__ int cut_list(Shared& sh, int n, int top, int tid) {
#pragma unroll 1
  for (int at = tid; at < n; at += kRowThreads) {
    const uint64_t key = sh.list[at];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += sh.list[j] > key ? 1 : 0;
    if (rank < top) sh.best[rank] = key;
    if (rank == top - 1) sh.tau = key;
  }
  __syncthreads();
  const int left = std::min(n, top);
  if (tid < left) sh.list[tid] = sh.best[tid];
  if (tid == 0) sh.count = left;
  __syncthreads();
  return left;
}

template <typename T, bool kTop>
__global__ __launch_bounds__(kRowThreads, 4) void logprobs_kernel(LogprobArgs p) {
  constexpr int kN = Vec<T>::kN;
  constexpr int kVecs = kThreadElements / kN;
  constexpr int kChunk = kRowThreads * kVecs;  // vectors
  __shared__ Shared sh;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x % p.parts);
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  // The row's aligned 16-byte vectors, shared out over its workgroups; the
  // elements before and after them go first, one a lane.
  const int head = std::min(p.vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const u32x4* vecs = reinterpret_cast<const u32x4*>(x + head);
  const int n_vecs = (p.vocab - head) / kN;
  const int tail = p.vocab - head - n_vecs * kN;
  const int per = (n_vecs + p.parts - 1) / p.parts;
  const int v0 = std::min(n_vecs, part * per), v1 = std::min(n_vecs, v0 + per);
  const int edge = tid < head ? tid : tid - head < tail ? head + n_vecs * kN + tid - head : -1;

  int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[row] : static_cast<const int32_t*>(p.ids)[row];
  if (id >= p.vocab) {
    if (tid == 0 && part == 0) flag_error(p.header, kErrIdRange);
    id = -1;
  }
  const float given = id >= 0 ? static_cast<float>(x[id]) : INFINITY;

  auto load = [&](int at, u32x4 (&to)[kVecs]) {
    if (at + kChunk <= v1) {  // a whole chunk: no bounds, no filling in
      const u32x4* from = vecs + at;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) to[i] = __builtin_nontemporal_load(from + i * kRowThreads + static_cast<uint32_t>(tid));
      return;
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = at + i * kRowThreads + tid;
      to[i] = v < v1 ? __builtin_nontemporal_load(vecs + v) : lowest<T>();
    }
  };

  if (kTop && tid == 0) {
    sh.count = 0;
    sh.tau = 0;
  }
  Stats st{-INFINITY, 0.f, 0.f};
  int above = 0;  // of the wave
  u32x4 cur[kVecs], nxt[kVecs];
  int held = 0;  // candidates
  int at = v0;
  if (part == 0 && head + tail > 0) {
    at -= kChunk;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) nxt[i] = lowest<T>();
    if (edge >= 0) {
      if constexpr (sizeof(T) == 4)
        nxt[0][0] = __builtin_bit_cast(uint32_t, x[edge]);
      else
        nxt[0][0] = (nxt[0][0] & 0xFFFF0000u) | __builtin_bit_cast(uint16_t, x[edge]);
    }
  } else {
    load(v0, nxt);
  }
  if (kTop) __syncthreads();
  for (; at < v1; at += kChunk) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) cur[i] = nxt[i];
    if (at + kChunk < v1) load(at + kChunk, nxt);

    float tops[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      tops[i] = element<T>(cur[i], 0);
#pragma unroll
      for (int e = 1; e < kN; ++e) tops[i] = fmaxf(tops[i], element<T>(cur[i], e));
    }
    float most = tops[0];
#pragma unroll
    for (int i = 1; i < kVecs; ++i) most = fmaxf(most, tops[i]);
    {
      const float m = fmaxf(st.m, most);
      lower(st, distance(st.m, m));
      st.m = m;
    }
    const float base = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float v = element<T>(cur[i], e);
        const float y = (v - base) * kLog2e, z = __builtin_amdgcn_exp2f(y);
        st.s += z;
        st.w = fmaf(z, fmaxf(y, -200.f), st.w);  // 0 times -inf is not taken
        above += __builtin_popcountll(__ballot(v > given));
      }
    // The sums as finished here: left open, they were taken further down,
    // with every term held in a register until then.
    above = __builtin_amdgcn_readfirstlane(above);
    asm volatile("" : "+v"(st.s), "+v"(st.w), "+s"(above));

    if (kTop) {
      if (at == v0) {
        // The first threshold: the top-th largest of 64 groups' best keys.
        // A thread's key has the value of its largest element and an id no
        // lower than that element's (its vector's last), so it is no larger
        // than the element's key.
        uint64_t best = 0;
#pragma unroll
        for (int i = kVecs - 1; i >= 0; --i) {
          const int v = at + i * kRowThreads + tid;
          if (v < v1 && tops[i] == most) best = order_key(most, head + v * kN + kN - 1);
        }
#pragma unroll
        for (int s = 1; s < kRowWaves; s <<= 1) {
          const uint64_t o = __shfl_xor(static_cast<unsigned long long>(best), s);
          best = o > best ? o : best;
        }
        if (tid % kRowWaves == 0) sh.group[tid / kRowWaves] = best;
        __syncthreads();
        if (wave == 0) {
          const uint64_t mine = sh.group[lane];
          int rank = 0;
#pragma unroll 4
          for (int j = 0; j < 64; ++j) rank += sh.group[j] > mine || (sh.group[j] == mine && j < lane) ? 1 : 0;
          if (rank == p.top - 1 && mine > sh.tau) sh.tau = mine;
        }
        __syncthreads();
      }
      const bool odd = st.s != st.s;  // NaN among them: no comparison dismisses a vector
      for (;;) {
        const uint64_t tau = sh.tau;
        const float floor = tau == 0 ? -INFINITY : key_value(tau);
        if (__any(!(most < floor) || odd)) {
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            if (!__any(!(tops[i] < floor) || odd)) continue;
            // The vector as new values, so that nothing of what follows is
            // computed ahead of the test (and held in registers) for all.
            int v = at + i * kRowThreads + tid;
            asm volatile("" : "+v"(cur[i]), "+v"(v));
            // A lane's elements that reach the threshold: none or one, mostly.
            uint32_t left = 0;
#pragma unroll
            for (int e = 0; e < kN; ++e) left |= element<T>(cur[i], e) < floor ? 0u : 1u << e;
            if (at < v0) left &= edge >= 0 && i == 0 ? 1u : 0u;
            else if (v >= v1) left = 0;
            while (left != 0) {
              const int e = __builtin_ctz(left);
              left &= left - 1;
              const uint64_t key = order_key(element_at<T>(cur[i], e), at >= v0 ? head + v * kN + e : edge);
              if (key < tau) continue;
              const int to = atomicAdd(&sh.count, 1);
              if (to < kListCap) sh.list[to] = key;
            }
          }
        }
        __syncthreads();
        const int n = __builtin_amdgcn_readfirstlane(sh.count);
        __syncthreads();
        if (n <= kListCap) {
          held = n;
          break;
        }
        // More than the list holds: what it holds gives a higher threshold
        // (every candidate below it falls away), and the chunk is gone
        // through again.  The candidates of the chunks before stay: none of
        // them is lost, as the list only grew behind them.
        if (tid < held) sh.kept[tid] = sh.list[tid];
        __syncthreads();
        cut_list(sh, kListCap, p.top, tid);
        if (tid < held) sh.list[tid] = sh.kept[tid];
        if (tid == 0) sh.count = held;
        __syncthreads();
      }
      if (held > p.top + kListTrim) held = cut_list(sh, held, p.top, tid);
    }
  }

  // The workgroup's share.
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) st = join(st, shuffle(st, s));
  if (lane == 0) {
    sh.stats[wave] = st;
    sh.above[wave] = above;
  }
  if (kTop) {
    __syncthreads();
    held = cut_list(sh, held, p.top, tid);
  }
  __syncthreads();
  st = sh.stats[0];
  above = sh.above[0];
#pragma unroll
  for (int i = 1; i < kRowWaves; ++i) {
    st = join(st, sh.stats[i]);
    above += sh.above[i];
  }

  if (p.parts > 1) {
    // Shares of a row joined by its last workgroup, in order.
    char* mine = p.part + static_cast<uint64_t>(blockIdx.x) * kPartBytes;
    if (tid == 0) {
      coherent_store8(mine, __builtin_bit_cast(unsigned long long, f32x2{st.m, st.s}));
      coherent_store8(mine + 8, __builtin_bit_cast(unsigned long long, u32x2{__builtin_bit_cast(uint32_t, st.w),
                                                                            static_cast<uint32_t>(above)}));
    }
    if (kTop && tid < p.top) coherent_store8(mine + 16 + 8 * tid, tid < held ? sh.list[tid] : 0);
    wait_vm();
    __syncthreads();
    if (tid == 0) {
      const bool last = atomic_add_u(&p.counters[row], 1u) == static_cast<unsigned>(p.parts - 1);
      if (last) atomic_store_u(&p.counters[row], 0u);
      sh.last = last ? 1 : 0;
      sh.count = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    const char* first = p.part + static_cast<uint64_t>(row) * p.parts * kPartBytes;
    st = Stats{-INFINITY, 0.f, 0.f};
    above = 0;
    uint64_t least = 0;  // a part's last candidate: the best of them is a threshold
    if (lane < p.parts) {
      const char* at = first + lane * kPartBytes;
      const f32x2 rs = __builtin_bit_cast(f32x2, coherent_load8(at));
      const u32x2 wa = __builtin_bit_cast(u32x2, coherent_load8(at + 8));
      st = Stats{rs[0], rs[1], __builtin_bit_cast(float, wa[0])};
      above = static_cast<int>(wa[1]);
      if (kTop) least = coherent_load8(at + 16 + 8 * (p.top - 1));
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      st = join(st, shuffle(st, s));
      above += __shfl_xor(above, s);
      const uint64_t o = __shfl_xor(static_cast<unsigned long long>(least), s);
      least = o > least ? o : least;
    }
    if (kTop) {
      for (int i = tid; i < p.parts * p.top; i += kRowThreads) {
        const uint64_t key = coherent_load8(first + i / p.top * kPartBytes + 16 + 8 * (i % p.top));
        if (key != 0 && key >= least) sh.list[atomicAdd(&sh.count, 1)] = key;
      }
      __syncthreads();
      held = __builtin_amdgcn_readfirstlane(sh.count);
      __syncthreads();
      held = cut_list(sh, held, p.top, tid);
    }
  }

  const float ln_s = logf(st.s);
  if (tid == 0) {
    p.logprobs[row] = id >= 0 ? log_prob(given, st.m, ln_s) : 0.f;
    p.entropy[row] = fmaf(-st.w / st.s, kLn2, ln_s);
    p.ranks[row] = id >= 0 ? 1 + above : 0;
  }
  if (kTop && tid < p.top) {
    const uint64_t key = sh.list[tid];
    p.top_ids[row * p.top + tid] = key_id(key);
    p.top_lp[row * p.top + tid] = log_prob(key_value(key), st.m, ln_s);
  }
}

template <typename T>
hipError_t launch(const LogprobArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(a.rows * a.parts));
  if (a.top > 0)
    hipLaunchKernelGGL((logprobs_kernel<T, true>), grid, dim3(kRowThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((logprobs_kernel<T, false>), grid, dim3(kRowThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_logprobs(LogprobArgs& a, int n_cu, hipStream_t stream) {
  static_assert(kMostLogprobRows * kRowThreads <= 0xFFFFFFFFll, "a grid has room for a workgroup each");
  // Rows enough for four workgroups a compute unit take one each; fewer are
  // shared by workgroups of at least one whole chunk.
  const int64_t n = a.dtype == 2 ? 4 : 8;
  const int64_t vecs = kRowThreads * kThreadElements / n;  // of a chunk
  const int64_t chunks = ((a.vocab + 2 * n - 2) / n + vecs - 1) / vecs;
  a.parts = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>({chunks, (4 * n_cu + a.rows - 1) / a.rows, kMaxParts})));
  if (a.rows > a.n_counters || static_cast<uint64_t>(a.rows) * a.parts * kPartBytes > a.part_bytes) a.parts = 1;
  if (!grid_fits(a.rows * a.parts, kRowThreads)) return hipErrorInvalidValue;
  return a.dtype == 0 ? launch<_Float16>(a, stream) : a.dtype == 1 ? launch<__bf16>(a, stream) : launch<float>(a, stream);
}

}  // namespace wp
