// wp_logprobs.hip -- log probabilities of given tokens, the entropy of the
// distribution and its largest alternatives (gfx950).
#include <hip/hip_runtime.h>

#include "wp_device.h"
#include "wp_model.h"

namespace wp {
namespace {

constexpr int kRowThreads = 512;

// Orders a logit and its id: greater values first, equal ones by the lower
// id, NaN above every number.
__device__ __forceinline__ uint64_t order_key(float v, int id) {
  uint32_t u = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);
  u = v != v ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<uint64_t>(u) << 32) | static_cast<uint32_t>(~id);
}

template <typename V, typename F>
__device__ __forceinline__ V block_fold(V v, V* s, F f) {
  for (int x = 32; x > 0; x >>= 1) v = f(v, __shfl_xor(v, x));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < kRowThreads / 64; ++i) v = f(v, s[i]);
  return v;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void row_kernel(LogprobArgs p) {
  __shared__ float sf[8];
  __shared__ unsigned long long sk[8];
  const int64_t row = blockIdx.x;
  const int tid = static_cast<int>(threadIdx.x);
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[row] : static_cast<const int32_t*>(p.ids)[row];
  if (id >= p.vocab) {
    if (tid == 0) flag_error(p.header, kErrIdRange);
    id = -1;
  }
  const float given = id >= 0 ? static_cast<float>(x[id]) : 0.f;
  float m = -INFINITY;
  for (int i = tid; i < p.vocab; i += kRowThreads) m = fmaxf(m, static_cast<float>(x[i]));
  m = block_fold(m, sf, [](float a, float b) { return fmaxf(a, b); });
  float s = 0.f, w = 0.f, above = 0.f;
  for (int i = tid; i < p.vocab; i += kRowThreads) {
    const float v = static_cast<float>(x[i]);
    const float d = v - m, e = expf(d);
    s += e;
    w += e == 0.f ? 0.f : e * d;
    above += v > given ? 1.f : 0.f;
  }
  const auto add = [](float a, float b) { return a + b; };
  s = block_fold(s, sf, add);
  w = block_fold(w, sf, add);
  above = block_fold(above, sf, add);
  const float lse = m + logf(s);
  if (tid == 0) {
    p.logprobs[row] = id >= 0 ? given - lse : 0.f;
    p.entropy[row] = logf(s) - w / s;
    p.ranks[row] = id >= 0 ? 1 + static_cast<int32_t>(above) : 0;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < p.vocab; i += kRowThreads) {
      const unsigned long long key = order_key(static_cast<float>(x[i]), i);
      if ((k == 0 || key < last) && key > best) best = key;
    }
    last = block_fold(best, sk, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
    if (tid == 0) {
      const int at = static_cast<int>(~static_cast<uint32_t>(last));
      p.top_ids[row * p.top + k] = at;
      p.top_lp[row * p.top + k] = static_cast<float>(x[at]) - lse;
    }
  }
}

}  // namespace

hipError_t launch_logprobs(const LogprobArgs& a, int n_cu, hipStream_t stream) {
  (void)n_cu;
  const dim3 grid(static_cast<uint32_t>(a.rows));
  if (a.dtype == 0)
    hipLaunchKernelGGL(row_kernel<_Float16>, grid, dim3(kRowThreads), 0, stream, a);
  else if (a.dtype == 1)
    hipLaunchKernelGGL(row_kernel<__bf16>, grid, dim3(kRowThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(row_kernel<float>, grid, dim3(kRowThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace wp
