// wp_proj.hip -- projections with a fused epilogue (gfx950):
//   y = rn(act(x . W^T + bias) + residual), or gated
//   y = rn(act(x . Wg^T + bg) * (x . Wu^T + bu) + residual),
// fp32 accumulation, one rounding.
//
// The product is computed as W . X^T: a matrix instruction's rows are output
// features and its columns tokens, so a lane ends with four consecutive
// features of one token and the epilogue reads bias and residual and writes y
// in 8-byte words.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "wp_device.h"
#include "wp_model.h"

namespace wp {
namespace {

constexpr int kStepK = 64;  // columns of x and W staged per K-step: 128 bytes of a row

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case kActRelu:
      return v < 0.f ? 0.f : v;  // NaN stays
    case kActGelu:
      return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    case kActGeluTanh:
      return 0.5f * v * (1.f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
    case kActSilu:
      return v / (1.f + __expf(-v));
    default:
      return v;
  }
}

// 16 bytes of a row that need not be 16-byte aligned, `n` elements of it
// inside the row (n <= 0: none); the rest are zero.
template <typename T>
__device__ __forceinline__ u32x4 load_ragged(const T* p, int n) {
  struct __attribute__((packed, aligned(2))) Loose {
    u32x4 v;
  };
  if (n >= 8) return reinterpret_cast<const Loose*>(p)->v;
  u32x4 r{0u, 0u, 0u, 0u};
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) r[i / 2] |= static_cast<uint32_t>(q[i]) << (16 * (i & 1));
  return r;
}

// Tile of BT tokens x BN weight rows, WT x WN waves.  A gated tile's weight rows
// are, per wave, half gate rows and half the up rows of the same outputs, so
// that both factors of an output end in the same lane.
//
// LDS: a staged row is 64 columns, eight 16-byte chunks; row r keeps its
// chunk c at place c ^ ((r >> 1) & 7), so the 16 rows a fragment load touches
// at one c fall into all banks once.
template <typename T, int BT, int BN, int WT, int WN>
struct Tile {
  static constexpr int kWaves = WT * WN;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kT = BT / WT;       // tokens per wave
  static constexpr int kN = BN / WN;       // weight rows per wave
  static constexpr int kFT = kT / 16;      // token fragments
  static constexpr int kFN = kN / 16;      // weight fragments
  static constexpr int kLoadsX = BT * 8 / kThreads;  // 16-byte chunks per thread and K-step
  static constexpr int kLoadsW = BN * 8 / kThreads;
};

template <typename T, int BT, int BN, int WT, int WN>
__global__ __launch_bounds__(64 * WT * WN) void proj_kernel(ProjArgs p) {
  using C = Tile<T, BT, BN, WT, WN>;
  using V8 = typename VecOf<T>::v8;
  __shared__ u32x4 sx[BT * 8];
  __shared__ u32x4 sw[BN * 8];
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wt = wave % WT, wn = wave / WT;
  const int tile = static_cast<int>(blockIdx.x);
  const int tile_t = tile % p.tiles_t;
  const int tile_n = tile / p.tiles_t;
  const int64_t t0 = static_cast<int64_t>(tile_t) * BT;
  const int gated = p.gated;
  const int outs = gated ? BN / 2 : BN;  // outputs of the tile
  const int n0 = tile_n * outs;

  // Weight row of the tile's row r, or -1 past the weight.
  auto weight_row = [&](int r) -> int64_t {
    if (!gated) return n0 + r < p.n_out ? n0 + r : -1;
    const int w = r / C::kN, i = r % C::kN;
    const int n = n0 + w * (C::kN / 2) + i % (C::kN / 2);
    return n < p.n_out ? n + (i < C::kN / 2 ? 0 : static_cast<int64_t>(p.n_out)) : -1;
  };

  f32x4 acc[C::kFN][C::kFT] = {};
  const T* x = static_cast<const T*>(p.x);
  const T* w = static_cast<const T*>(p.w);
  for (int k0 = 0; k0 < p.d_in; k0 += kStepK) {
    __syncthreads();
    for (int i = 0; i < C::kLoadsX; ++i) {
      const int at = i * C::kThreads + tid, r = at >> 3, c = at & 7;
      const int64_t t = t0 + r;
      const int n = t < p.tokens ? p.d_in - k0 - c * 8 : 0;
      sx[r * 8 + (c ^ ((r >> 1) & 7))] = load_ragged(x + t * p.ldx + k0 + c * 8, n);
    }
    for (int i = 0; i < C::kLoadsW; ++i) {
      const int at = i * C::kThreads + tid, r = at >> 3, c = at & 7;
      const int64_t row = weight_row(r);
      const int n = row >= 0 ? p.d_in - k0 - c * 8 : 0;
      sw[r * 8 + (c ^ ((r >> 1) & 7))] = load_ragged(w + row * p.ldw + k0 + c * 8, n);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      V8 fw[C::kFN], fx[C::kFT];
      const int c = h * 4 + (lane >> 4);
#pragma unroll
      for (int i = 0; i < C::kFN; ++i) {
        const int r = wn * C::kN + i * 16 + (lane & 15);
        fw[i] = __builtin_bit_cast(V8, sw[r * 8 + (c ^ ((r >> 1) & 7))]);
      }
#pragma unroll
      for (int i = 0; i < C::kFT; ++i) {
        const int r = wt * C::kT + i * 16 + (lane & 15);
        fx[i] = __builtin_bit_cast(V8, sx[r * 8 + (c ^ ((r >> 1) & 7))]);
      }
#pragma unroll
      for (int i = 0; i < C::kFN; ++i)
#pragma unroll
        for (int j = 0; j < C::kFT; ++j) acc[i][j] = mfma16(fw[i], fx[j], acc[i][j]);
    }
  }

  // Lane: token lane & 15 of a fragment, features (lane >> 4) * 4 + e.
  const T* bias = static_cast<const T*>(p.bias);
  const T* res = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  const int n_frags = gated ? C::kFN / 2 : C::kFN;
  const int wave_n = n0 + wn * (gated ? C::kN / 2 : C::kN);
#pragma unroll
  for (int i = 0; i < C::kFN; ++i) {
    if (i >= n_frags) break;
    const int n = wave_n + i * 16 + (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < C::kFT; ++j) {
      const int64_t t = t0 + wt * C::kT + j * 16 + (lane & 15);
      if (t >= p.tokens) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n + e >= p.n_out) break;
        float v = acc[i][j][e] + (bias ? static_cast<float>(bias[n + e]) : 0.f);
        v = activate(v, p.act);
        if (gated)
          v *= acc[(i + C::kFN / 2) % C::kFN][j][e] + (bias ? static_cast<float>(bias[p.n_out + n + e]) : 0.f);
        if (res) v += static_cast<float>(res[t * p.ldr + n + e]);
        y[t * p.ldy + n + e] = static_cast<T>(v);
      }
    }
  }
}

template <typename T, int BT, int BN, int WT, int WN>
hipError_t launch_tile(ProjArgs& a, hipStream_t stream) {
  const int outs = a.gated ? BN / 2 : BN;
  a.tiles_t = static_cast<int32_t>((a.tokens + BT - 1) / BT);
  a.tiles_n = (a.n_out + outs - 1) / outs;
  hipLaunchKernelGGL((proj_kernel<T, BT, BN, WT, WN>), dim3(static_cast<uint32_t>(a.tiles_t) * a.tiles_n),
                     dim3(64 * WT * WN), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_proj(int dtype_bf16, ProjArgs& a, int n_cu, hipStream_t stream) {
  (void)n_cu;
  return dtype_bf16 ? launch_tile<__bf16, 128, 128, 2, 2>(a, stream) : launch_tile<_Float16, 128, 128, 2, 2>(a, stream);
}

}  // namespace wp
