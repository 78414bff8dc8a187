// wp_attn.hip -- attention over packed sequences of different lengths
// (gfx950): causal, grouped heads, optional window, fp32 softmax statistics.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "wp_device.h"
#include "wp_model.h"

namespace wp {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The sequence of packed row t by its bounds cu[0..n]: b with cu[b] <= t <
// cu[b + 1], or -1.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int n, int64_t t) {
  int lo = 0, hi = n;  // the first bound past t is in (lo, hi + 1]
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo < n && cu[lo] <= t && t < cu[lo + 1] ? lo : -1;
}

// One wave per query row and head: a lane scores one key of 64, then the
// lanes share out the head's columns for the weighted sum.
template <typename T>
__global__ __launch_bounds__(64) void row_kernel(AttnArgs p) {
  __shared__ float sq[256];
  __shared__ float sp[64];
  const int lane = static_cast<int>(threadIdx.x);
  const int64_t t = blockIdx.x;
  const int h = static_cast<int>(blockIdx.y);
  const int hk = h / (p.heads / p.kv_heads);
  const int b = sequence_of(p.cu_q, p.n_seq, t);
  int64_t first = 0, k0 = 0, end = 0;
  if (b >= 0) {
    k0 = std::clamp<int64_t>(p.cu_k[b], 0, p.keys);
    const int64_t n_k = std::clamp<int64_t>(p.cu_k[b + 1], k0, p.keys) - k0;
    const int64_t pos = t - p.cu_q[b] + n_k - (p.cu_q[b + 1] - p.cu_q[b]);
    end = p.causal ? std::clamp<int64_t>(pos + 1, 0, n_k) : n_k;
    first = p.causal && p.window > 0 ? std::max<int64_t>(0, pos - p.window + 1) : 0;
  }
  const T* q = static_cast<const T*>(p.q) + t * p.q_tok + h * p.q_head;
  for (int d = lane; d < p.dim; d += 64) sq[d] = static_cast<float>(q[d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[4] = {};
  for (int64_t at = first; at < end; at += 64) {
    const int64_t j = at + lane;
    float s = -INFINITY;
    if (j < end) {
      const T* k = static_cast<const T*>(p.k) + (k0 + j) * p.k_tok + hk * p.k_head;
      s = 0.f;
      for (int d = 0; d < p.dim; ++d) s += sq[d] * static_cast<float>(k[d]);
      s *= p.scale;
    }
    float top = s;
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    top = fmaxf(top, m);
    const float base = top == -INFINITY ? 0.f : top;
    const float e = exp2f((s - base) * kLog2e);
    const float fade = exp2f((m - base) * kLog2e);
    float sum = e;
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x);
    l = l * fade + sum;
    m = top;
    __syncthreads();
    sp[lane] = e;
    __syncthreads();
    const int n = static_cast<int>(std::min<int64_t>(64, end - at));
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d >= p.dim) break;
      float w = o[i] * fade;
      for (int x = 0; x < n; ++x)
        w += sp[x] * static_cast<float>(static_cast<const T*>(p.v)[(k0 + at + x) * p.v_tok + hk * p.v_head + d]);
      o[i] = w;
    }
  }
  T* out = static_cast<T*>(p.out) + t * p.o_tok + h * p.o_head;
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < p.dim) out[lane + 64 * i] = static_cast<T>(end > first ? o[i] / l : 0.f);
  if (p.lse && lane == 0) p.lse[t * p.heads + h] = end > first ? m + logf(l) : -INFINITY;
}

}  // namespace

hipError_t launch_attention(int dtype_bf16, AttnArgs& a, int n_cu, hipStream_t stream) {
  (void)n_cu;
  const dim3 grid(static_cast<uint32_t>(a.tokens), static_cast<uint32_t>(a.heads));
  if (dtype_bf16)
    hipLaunchKernelGGL(row_kernel<__bf16>, grid, dim3(64), 0, stream, a);
  else
    hipLaunchKernelGGL(row_kernel<_Float16>, grid, dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace wp
