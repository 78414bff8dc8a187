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
#include <type_traits>

#include "wp_device.h"
#include "wp_model.h"

namespace wp {
namespace {

constexpr int kStepK = 64;  // columns of x and W staged per K-step: 128 bytes of a row

// 1 / (1 + exp(-v)) by the hardware's exponential and reciprocal (an ulp each;
// an IEEE division would take as long as the rest of an epilogue).
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}

template <int kAct>
__device__ __forceinline__ float activate(float v) {
  switch (kAct) {
    case kActRelu:
      return v < 0.f ? 0.f : v;  // NaN stays
    case kActGelu: {
      // 0.5 v (1 + erf u), u = v / sqrt 2, with 1 - erf |u| = t P(t) exp(-u^2),
      // t = 1 / (1 + 0.36 |u|): a polynomial fitted here for the least error of
      // both sides, within 4e-6 of the tail itself up to |u| = 9.3 (fp32 ends
      // there) and 5e-8 of one.  For negative v the result is the tail, whose
      // relative error is that and the exponent's rounding (4e-5 at v = -13).
      const float u = fabsf(v) * 0.70710678118654752f;
      const float t = __builtin_amdgcn_rcpf(fmaf(0.36f, u, 1.f));
      float q = fmaf(t, -0.162926913f, 0.561451978f);
      q = fmaf(t, q, -0.351465345f);
      q = fmaf(t, q, 0.425491667f);
      q = fmaf(t, q, 0.108845922f);
      q = fmaf(t, q, 0.216382673f);
      q = t * fmaf(t, q, 0.202220065f);
      // (Past 64 the tail is zero, and an infinity must not meet it.)
      const float tail = 0.5f * fminf(v, 64.f) * q * __builtin_amdgcn_exp2f(-1.4426950408889634f * u * u);
      return v < 0.f ? tail : v - tail;
    }
    case kActGeluTanh:
      // 0.5 v (1 + tanh u) = v sigmoid(2 u)
      return v * sigmoid(1.5957691216057308f * (v + 0.044715f * v * v * v));
    case kActSilu:
      return v * sigmoid(v);
    default:
      return v;
  }
}

// How a product's rows lie: each is whole 16-byte vectors, starts on a 4-byte
// word, or on any element.
enum RowKind { kVectors, kWords, kElements };

// 16 bytes from any element on.
template <typename T>
__device__ __forceinline__ u32x4 load_any(const T* p) {
  struct __attribute__((packed, aligned(2))) Loose {
    u32x4 v;
  };
  return reinterpret_cast<const Loose*>(p)->v;
}
// The same as the words that hold them.  Where a wave's neighbouring lanes read
// different rows, the memory pipeline takes some four cycles a lane for 16
// bytes that start inside a word (128 x 8191 -> 1000: 59 us, and as words 32).
struct Words {
  u32x4 v;
  uint32_t next;  // the word after them, if the first starts before p
};
template <typename T>
__device__ __forceinline__ uint32_t inside_word(const T* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 2);
}
template <typename T>
__device__ __forceinline__ Words load_words(const T* p) {
  struct __attribute__((packed, aligned(4))) Loose {
    u32x4 v;
  };
  const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
  return Words{reinterpret_cast<const Loose*>(q)->v, q[3 + inside_word(p) / 2]};
}
__device__ __forceinline__ u32x4 settle(const Words& w, uint32_t inside) {
  const uint32_t w0 = w.v[0], w1 = w.v[1], w2 = w.v[2], w3 = w.v[3];
  return u32x4{__builtin_amdgcn_alignbyte(w1, w0, inside), __builtin_amdgcn_alignbyte(w2, w1, inside),
               __builtin_amdgcn_alignbyte(w3, w2, inside), __builtin_amdgcn_alignbyte(w.next, w3, inside)};
}
// The first `n` elements from p on, 8 at most (n <= 0: none); the rest are zero.
template <typename T>
__device__ __forceinline__ u32x4 load_first(const T* p, int n) {
  if (n >= 8) return load_any(p);
  u32x4 r{0u, 0u, 0u, 0u};
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) r[i / 2] |= static_cast<uint32_t>(q[i]) << (16 * (i & 1));
  return r;
}

constexpr int kRowsPerLoad = 8;       // staged rows that a wave's 16-byte-per-lane load fills
constexpr int64_t kFarRows = 1 << 27; // elements between rows: seven of them and the columns stay under 2 GiB

// Tile of BT tokens x BN weight rows, WT x WN waves.  A gated tile's weight rows
// are, per wave, half gate rows and half the up rows of the same outputs, so
// that both factors of an output end in the same lane.
//
// LDS is a ring of R slots, one K-step's 64 columns of the tile's rows each;
// a step is two halves of 32 columns.  A half's fragments are read from LDS
// while the half before is multiplied, so that the matrix cores need not wait
// for LDS after the step's one barrier.  Past that barrier every wave has read
// the slot that is refilled then, and every wave's loads of the slot that
// is read next have landed: they had R - 1 steps for it.
//
// A staged row is eight 16-byte chunks; row r keeps its chunk c at place
// c ^ ((r >> 1) & 7), so the 16 rows a fragment read touches at one c fall into
// all banks once.
template <int BT, int BN, int WT, int WN, int R>
struct Tile {
  static constexpr int kWaves = WT * WN;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kT = BT / WT;   // tokens per wave
  static constexpr int kN = BN / WN;   // weight rows per wave
  static constexpr int kFT = kT / 16;  // token fragments
  static constexpr int kFN = kN / 16;  // weight fragments
  static constexpr int kLoadsX = BT / kRowsPerLoad / kWaves;  // loads per wave and K-step
  static constexpr int kLoadsW = BN / kRowsPerLoad / kWaves;
  static constexpr int kLoads = kLoadsX + kLoadsW;
  static constexpr int kXBytes = BT * kStepK * 2;  // of a slot
  static constexpr int kWBytes = BN * kStepK * 2;
  static_assert(kLoadsX >= 1 && kLoadsW >= 1, "every wave stages rows of both");
  static_assert(kFN % 2 == 0, "a wave holds both factors of a gate");
  static_assert(R == 2 || R == 4, "the steps of a round are written out");
};

// Weight row of row r of the tile that starts at output n0; past the weight
// where `ok` is false.
template <int kN>
__device__ __forceinline__ int64_t weight_row(const ProjArgs& p, int n0, int r, bool* ok) {
  if (!p.gated) {
    *ok = n0 + r < p.n_out;
    return n0 + r;
  }
  const int n = n0 + r / kN * (kN / 2) + r % (kN / 2);
  *ok = n < p.n_out;
  return n + (r % kN < kN / 2 ? 0 : static_cast<int64_t>(p.n_out));
}

// The biases of four consecutive outputs and, gated, of their up rows.
struct Biases {
  f32x4 gate, up;
};
template <typename T>
__device__ __forceinline__ Biases biases(const ProjArgs& p, int n) {
  Biases b{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  const T* bias = static_cast<const T*>(p.bias);
  if (bias == nullptr) return b;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= p.n_out) break;
    b.gate[e] = static_cast<float>(bias[n + e]);
    if (p.gated) b.up[e] = static_cast<float>(bias[p.n_out + n + e]);
  }
  return b;
}

// Four consecutive outputs of one token: bias, activation, gate, residual, one
// rounding.  kWhole: all four exist, and y and the residual take 8-byte
// accesses; else the first `count` of them are written one by one.
template <typename T, int kAct, bool kWhole>
__device__ __forceinline__ void finish(const ProjArgs& p, int64_t t, int n, int count, f32x4 a, f32x4 up, const Biases& b) {
  const T* res = static_cast<const T*>(p.residual) + t * p.ldr + n;
  T* y = static_cast<T*>(p.y) + t * p.ldy + n;
  f32x4 r{0.f, 0.f, 0.f, 0.f};
  if (p.residual) {
    if constexpr (kWhole) {
      r = unpack4f<T>(*reinterpret_cast<const u32x2*>(res));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < count) r[e] = static_cast<float>(res[e]);
    }
  }
  a += b.gate;
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] = activate<kAct>(a[e]);
  if (p.gated) a *= up + b.up;
  a += r;
  if constexpr (kWhole) {
    store4(y, a);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < count) y[e] = static_cast<T>(a[e]);
  }
}

// Calls f with the activation as a constant: one test for a whole epilogue.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
  switch (act) {
    case kActRelu: return f(std::integral_constant<int, kActRelu>{});
    case kActGelu: return f(std::integral_constant<int, kActGelu>{});
    case kActGeluTanh: return f(std::integral_constant<int, kActGeluTanh>{});
    case kActSilu: return f(std::integral_constant<int, kActSilu>{});
    default: return f(std::integral_constant<int, kActNone>{});
  }
}

// Waits until at most kLeft of this wave's loads are on their way and its LDS
// reads are done, then for the workgroup.  By the builtins, whose counts the
// compiler sees: it then adds no wait of its own to the reads behind them.
template <int kLeft>
__device__ __forceinline__ void staged_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((kLeft & 15) | (kLeft >> 4) << 14 | 7 << 4);  // vmcnt(kLeft) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Four bytes a lane from anywhere to LDS, for the line they bring into L2.
__device__ __forceinline__ void touch_line(const void* src, char* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}

// The last of a tile's K-ranges to arrive: true in all of its threads, with the
// counter cleared for the next call.  Every partial stored before is then visible.
__device__ __forceinline__ bool last_split(uint32_t* cnt, int splits, uint32_t* flag) {
  wait_vm();
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = atomic_add_u(cnt, 1u) == static_cast<unsigned>(splits - 1);
    if (last) atomic_store_u(cnt, 0u);
    *flag = last ? 1u : 0u;
  }
  __syncthreads();
  return *flag != 0u;
}

// kAligned: rows of x and w are 16-byte aligned and whole 16-byte vectors;
// they go to LDS directly.  Else they pass through registers, read as their
// alignment allows.
template <typename T, int BT, int BN, int WT, int WN, int R, bool kAligned>
__global__ __launch_bounds__(64 * WT * WN, 2) void proj_kernel(ProjArgs p) {
  using C = Tile<BT, BN, WT, WN, R>;
  using V8 = typename VecOf<T>::v8;
  // An array per slot, or for two slots one for its x and one for its w rows:
  // the compiler then knows that a load into one leaves reads of the others alone.
  constexpr int kArray = R == 2 ? std::max(C::kXBytes, C::kWBytes) : C::kXBytes + C::kWBytes;
  __shared__ __align__(1024) char mem0[kArray];
  __shared__ __align__(1024) char mem1[kArray];
  __shared__ __align__(1024) char mem2[kArray];
  __shared__ __align__(1024) char mem3[kArray];
  struct Slot {
    char* x;
    char* w;
  };
  const Slot slot0{mem0, R == 2 ? mem2 : mem0 + C::kXBytes}, slot1{mem1, R == 2 ? mem3 : mem1 + C::kXBytes};
  const Slot slot2{mem2, mem2 + C::kXBytes}, slot3{mem3, mem3 + C::kXBytes};  // R == 4
  // The largest tile leaves a compute unit to one workgroup, whose loads have
  // one K-step (about 1 us) to arrive: enough from L2, not always from behind
  // it.  So each step also touches lines of a step four further on.  The rows of
  // x are shared by the tiles beside this one that the XCD's 32 compute units hold at the same
  // time, those of w by the band's: each tile touches its share.
  // (8192 x 5120 x 27648: 1785 us without, 1719 with.)
  constexpr bool kTouch = kAligned && BT * BN >= 256 * 256;
  __shared__ char s_touch[kTouch ? 256 : 4];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wt = wave % WT, wn = wave / WT;
  int tile = static_cast<int>(blockIdx.x);
  const int n_tiles = p.tiles_t * p.tiles_n;
  // Workgroups go to the eight XCDs in turn, and each XCD has an L2 of its
  // own: an XCD takes a contiguous eighth of the tiles, which run through
  // bands of eight token tiles, so that the tiles its compute units hold
  // at a time share their rows of x and of w.
  tile = tile % 8 * (n_tiles / 8) + std::min(tile % 8, n_tiles % 8) + tile / 8;
  constexpr int kBand = 8;
  const int band = tile / (kBand * p.tiles_n);
  const int band_rows = std::min(kBand, p.tiles_t - band * kBand);
  const int in_band = tile - band * kBand * p.tiles_n;
  const int tile_t = band * kBand + in_band % band_rows, tile_n = in_band / band_rows;
  const int64_t t0 = static_cast<int64_t>(tile_t) * BT;
  const int n0 = tile_n * (p.gated ? BN / 2 : BN);
  const int k_end = p.d_in;

  // Fragment reads: lane's row and chunk; a second half's chunk is 4 further,
  // which the swizzle turns into a flipped bit.
  const int frag_row = lane & 15;
  const int frag_off = frag_row * 128 + (((lane >> 4) ^ ((frag_row >> 1) & 7)) << 4);
  auto fragment = [&](const char* rows, int row0, int half) {
    return *reinterpret_cast<const V8*>(rows + row0 * 128 + (frag_off ^ (half * 64)));
  };
  f32x4 acc[C::kFN][C::kFT];
#pragma unroll
  for (int i = 0; i < C::kFN; ++i)
#pragma unroll
    for (int j = 0; j < C::kFT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  V8 aw[C::kFN], ax[C::kFT], bw[C::kFN], bx[C::kFT];
  auto read = [&](const Slot& slot, int half, V8 (&fw)[C::kFN], V8 (&fx)[C::kFT]) {
#pragma unroll
    for (int i = 0; i < C::kFN; ++i) fw[i] = fragment(slot.w, wn * C::kN + i * 16, half);
#pragma unroll
    for (int j = 0; j < C::kFT; ++j) fx[j] = fragment(slot.x, wt * C::kT + j * 16, half);
  };
  auto multiply = [&](V8 (&fw)[C::kFN], V8 (&fx)[C::kFT]) {
#pragma unroll
    for (int j = 0; j < C::kFT; ++j)
#pragma unroll
      for (int i = 0; i < C::kFN; ++i) acc[i][j] = mfma16(fw[i], fx[j], acc[i][j]);
  };

  // Staging: lane l of load i fills chunk l % 8 of row (wave * loads + i) * 8
  // + l / 8, and so takes the row's column chunk (l % 8) ^ ((row >> 1) & 7).
  const int sub = lane >> 3;
  if constexpr (kAligned) {
    int col[2];  // by the parity of the row's group of eight
#pragma unroll
    for (int i = 0; i < 2; ++i) col[i] = ((lane & 7) ^ (i * 4 + (sub >> 1))) * 8;
    int off_x[C::kLoadsX], off_w[C::kLoadsW];
    const T* src_x[C::kLoadsX];
    const T* src_w[C::kLoadsW];
#pragma unroll
    for (int i = 0; i < C::kLoadsX; ++i) {
      const int g = wave * C::kLoadsX + i;
      const int64_t t = t0 + g * kRowsPerLoad;
      src_x[i] = static_cast<const T*>(p.x) + t * p.ldx;
      off_x[i] = t + sub < p.tokens ? (sub * static_cast<int>(p.ldx) + col[g & 1]) * 2 : kOutside;
    }
#pragma unroll
    for (int i = 0; i < C::kLoadsW; ++i) {
      const int g = wave * C::kLoadsW + i;
      bool ok, first_ok;
      const int64_t row = weight_row<C::kN>(p, n0, g * kRowsPerLoad, &first_ok);
      (void)weight_row<C::kN>(p, n0, g * kRowsPerLoad + sub, &ok);
      src_w[i] = static_cast<const T*>(p.w) + row * p.ldw;
      off_w[i] = ok ? (sub * static_cast<int>(p.ldw) + col[g & 1]) * 2 : kOutside;
    }
    auto stage = [&](int k, const Slot& slot) {
      const bool in[2] = {k + col[0] < k_end, k + col[1] < k_end};
#pragma unroll
      for (int i = 0; i < C::kLoadsX; ++i) {
        const int g = wave * C::kLoadsX + i;
        load_to_lds(src_x[i], slot.x + g * 1024, in[(C::kLoadsX % 2 ? g : i) & 1] ? off_x[i] : kOutside, k * 2);
      }
#pragma unroll
      for (int i = 0; i < C::kLoadsW; ++i) {
        const int g = wave * C::kLoadsW + i;
        load_to_lds(src_w[i], slot.w + g * 1024, in[(C::kLoadsW % 2 ? g : i) & 1] ? off_w[i] : kOutside, k * 2);
      }
    };
    const T* line = nullptr;
    if constexpr (kTouch) {
      const int beside = std::max(1, 32 / band_rows);
      const int n_x = (BT + beside - 1) / beside, n_w = (BN + band_rows - 1) / band_rows;
      int at = lane * C::kWaves + wave;  // of the tile's n_x + n_w lines; lanes past them repeat the first
      if (at >= n_x + n_w) at = 0;
      bool ok;
      const int r = at < n_x ? tile_n % beside * n_x + at : tile_t % band_rows * n_w + at - n_x;
      if (at < n_x) {
        const int64_t t = std::min(t0 + r, p.tokens - 1);
        line = static_cast<const T*>(p.x) + t * p.ldx;
      } else {
        const int64_t row = weight_row<C::kN>(p, n0, std::min(r, BN - 1), &ok);
        line = static_cast<const T*>(p.w) + (ok ? row : 0) * p.ldw;
      }
    }
    constexpr int kAhead = 6 * kStepK;  // from the step that is multiplied
    constexpr int kTouches = kTouch ? 1 : 0;
    // One K-step.  Past k_end stage() loads zeros (without memory traffic) and
    // read() what nobody uses, so that a step is free of branches and its
    // reads, loads and products can be put in order: each read or load between two products, so
    // that issuing them leaves no gap in the matrix cores' work.
    constexpr int kReads = C::kFN + C::kFT, kProducts = C::kFN * C::kFT;
    auto step = [&](int k, const Slot& now, const Slot& next) {
      read(now, 1, bw, bx);
      multiply(aw, ax);
#pragma unroll
      for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // product
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kProducts > kReads ? kProducts - kReads : 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      staged_barrier<C::kLoads*(R - 2) + kTouches>();
      stage(k + R * kStepK, now);
      if constexpr (kTouch) touch_line(line + std::min(k + kAhead, k_end - 8), s_touch);
      read(next, 0, aw, ax);
      multiply(bw, bx);
#pragma unroll
      for (int i = 0; i < C::kLoads + kTouches; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);  // load
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
#pragma unroll
      for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    if (k_end > 0) {
      stage(0, slot0);
      stage(kStepK, slot1);
      if constexpr (R == 4) {
        stage(2 * kStepK, slot2);
        stage(3 * kStepK, slot3);
      }
      if constexpr (kTouch) touch_line(line + std::min(2 * kStepK, k_end - 8), s_touch);
      staged_barrier<C::kLoads*(R - 1) + kTouches>();
      read(slot0, 0, aw, ax);
      // Whole rounds of the ring, then the steps left (with a way out of a
      // round the compiler would wait for every load at its top).
      const int round_end = k_end / (R * kStepK) * (R * kStepK);
      int k = 0;
      for (; k < round_end; k += R * kStepK) {
        step(k, slot0, slot1);
        step(k + kStepK, slot1, R == 2 ? slot0 : slot2);
        if constexpr (R == 4) {
          step(k + 2 * kStepK, slot2, slot3);
          step(k + 3 * kStepK, slot3, slot0);
        }
      }
      if (k < k_end) step(k, slot0, slot1);
      if constexpr (R == 4) {
        if (k + kStepK < k_end) step(k + kStepK, slot1, slot2);
        if (k + 2 * kStepK < k_end) step(k + 2 * kStepK, slot2, slot3);
        if (k + 3 * kStepK < k_end) step(k + 3 * kStepK, slot3, slot0);
      } else {
        if (k + kStepK < k_end) step(k + kStepK, slot1, slot0);
      }
    }
  } else {
    // Rows of any alignment: whole K-steps go through registers, kAhead of them
    // on their way, to two slots in turn; the columns left then to a third.
    // (100 x 8191 -> 8000, one step ahead: 112 us, four: 55.)
    constexpr int kAhead = 4;
    static_assert(R == 4, "three slots");
    // Rows past the last read another one: their sums are written nowhere.
    const T* src_x[C::kLoadsX];
    const T* src_w[C::kLoadsW];
    int col_x[C::kLoadsX], col_w[C::kLoadsW];
    auto column = [&](int r) { return ((lane & 7) ^ ((r >> 1) & 7)) * 8; };
#pragma unroll
    for (int i = 0; i < C::kLoadsX; ++i) {
      const int r = (wave * C::kLoadsX + i) * kRowsPerLoad + sub;
      col_x[i] = column(r);
      src_x[i] = static_cast<const T*>(p.x) + (t0 + r < p.tokens ? t0 + r : t0) * p.ldx + col_x[i];
    }
#pragma unroll
    for (int i = 0; i < C::kLoadsW; ++i) {
      const int r = (wave * C::kLoadsW + i) * kRowsPerLoad + sub;
      bool ok;
      const int64_t row = weight_row<C::kN>(p, n0, r, &ok);
      col_w[i] = column(r);
      src_w[i] = static_cast<const T*>(p.w) + (ok ? row : 0) * p.ldw + col_w[i];
    }
    u32x4 rx[kAhead][C::kLoadsX], rw[kAhead][C::kLoadsW];
    auto place = [&](char* rows, int load, const u32x4& v) {
      *reinterpret_cast<u32x4*>(rows + load * 1024 + lane * 16) = v;
    };
    auto products = [&](const Slot& slot) {
      read(slot, 0, aw, ax);
      read(slot, 1, bw, bx);
      multiply(aw, ax);
      multiply(bw, bx);
    };
    const int full = k_end / kStepK * kStepK;
    auto gather = [&](int b, int k) {  // past the last whole step: that one again
      k = std::min(k, full - kStepK);
#pragma unroll
      for (int i = 0; i < C::kLoadsX; ++i) rx[b][i] = load_any(src_x[i] + k);
#pragma unroll
      for (int i = 0; i < C::kLoadsW; ++i) rw[b][i] = load_any(src_w[i] + k);
    };
    if (full > 0) {
#pragma unroll
      for (int b = 0; b < kAhead; ++b) gather(b, b * kStepK);
      auto step = [&](int k, int b) {
        const Slot& slot = b & 1 ? slot1 : slot0;
#pragma unroll
        for (int i = 0; i < C::kLoadsX; ++i) place(slot.x, wave * C::kLoadsX + i, rx[b][i]);
#pragma unroll
        for (int i = 0; i < C::kLoadsW; ++i) place(slot.w, wave * C::kLoadsW + i, rw[b][i]);
        staged_barrier<63>();
        gather(b, k + kAhead * kStepK);
        products(slot);
      };
      // Whole rounds, then the steps left (as above).
      const int round_end = full / (kAhead * kStepK) * (kAhead * kStepK);
      int k = 0;
      for (; k < round_end; k += kAhead * kStepK)
#pragma unroll
        for (int b = 0; b < kAhead; ++b) step(k + b * kStepK, b);
      if (k < full) step(k, 0);
      if (k + kStepK < full) step(k + kStepK, 1);
      if (k + 2 * kStepK < full) step(k + 2 * kStepK, 2);
    }
    if (full < k_end) {
#pragma unroll
      for (int i = 0; i < C::kLoadsX; ++i)
        place(slot2.x, wave * C::kLoadsX + i, load_first(src_x[i] + full, k_end - full - col_x[i]));
#pragma unroll
      for (int i = 0; i < C::kLoadsW; ++i)
        place(slot2.w, wave * C::kLoadsW + i, load_first(src_w[i] + full, k_end - full - col_w[i]));
      staged_barrier<63>();
      products(slot2);
    }
  }

  // Epilogue, through LDS: a wave writes its sums as rows of kN features of a
  // token (16-byte chunk c of token t's row at c ^ (t % chunks), so that
  // neither side's 16 lanes share a bank) and takes them back with the lanes
  // along a row, which makes residual reads and stores whole lines.  A lane
  // holds token lane & 15 of a fragment, four features from (lane >> 4) * 4.
  constexpr int kChunks = C::kN / 4;
  constexpr int kPassFrags = std::min(C::kFT, 4);
  constexpr int kWaveBytes = kPassFrags * 16 * C::kN * 4;
  constexpr int kPerArray = (C::kWaves + 3) / 4;
  static_assert(kPerArray * kWaveBytes <= kArray && C::kFT % kPassFrags == 0, "a wave's rows of a pass fit its share of an array");
  const int array = wave / kPerArray;
  char* rows = (array == 0 ? mem0 : array == 1 ? mem1 : array == 2 ? mem2 : mem3) + wave % kPerArray * kWaveBytes;
  const int outs = p.gated ? C::kN / 2 : C::kN;  // a row's outputs
  const int wave_n = n0 + wn * outs;
  const int64_t wave_t = t0 + wt * C::kT;
  const int lanes = outs / 4;  // along a row
  const int c = lane % lanes, row0 = lane / lanes, row_step = 64 / lanes;
  const int n = wave_n + c * 4;
  const bool whole = p.rows_vec && wave_t + C::kT <= p.tokens && wave_n + outs <= p.n_out;
  const Biases bias = biases<T>(p, n);
  wait_vm();  // loads past the last column write LDS too
  __syncthreads();
#pragma unroll
  for (int pass = 0; pass < C::kFT / kPassFrags; ++pass) {
#pragma unroll
    for (int j = 0; j < kPassFrags; ++j)
#pragma unroll
      for (int i = 0; i < C::kFN; ++i) {
        const int t = j * 16 + (lane & 15), q = i * 4 + (lane >> 4);
        *reinterpret_cast<f32x4*>(rows + t * (C::kN * 4) + ((q ^ (t & (kChunks - 1))) << 4)) =
            acc[i][pass * kPassFrags + j];
      }
    auto sum_of = [&](int r, int chunk) {
      return *reinterpret_cast<const f32x4*>(rows + r * (C::kN * 4) + ((chunk ^ (r & (kChunks - 1))) << 4));
    };
    const int64_t pass_t = wave_t + pass * kPassFrags * 16;
    with_activation(p.act, [&](auto act) {
      constexpr int kAct = decltype(act)::value;
      if (whole) {
#pragma unroll 4
        for (int r = row0; r < kPassFrags * 16; r += row_step)
          finish<T, kAct, true>(p, pass_t + r, n, 4, sum_of(r, c), sum_of(r, c + (p.gated ? kChunks / 2 : 0)), bias);
      } else {
#pragma unroll 2
        for (int r = row0; r < kPassFrags * 16; r += row_step)
          finish<T, kAct, false>(p, pass_t + r, n, pass_t + r < p.tokens ? p.n_out - n : 0, sum_of(r, c),
                                 sum_of(r, c + (p.gated ? kChunks / 2 : 0)), bias);
      }
    });
  }
}

// Small products: a workgroup's eight waves share out the columns of one tile,
// 64 (128 bytes of a row) at a time, and fragments go from memory to registers
// and into the product there: no LDS, no barrier until the waves' sums are
// joined, and the loads of several blocks in flight per wave.  What bounds it is the first loads'
// latency and the tile's bytes, or (few tokens) the weight's bytes.
// kFT x kFN fragments; gated: half of the kFN are gate rows, half the same
// outputs' up rows.
constexpr int kColWaves = 8;
constexpr int kColThreads = 64 * kColWaves;
constexpr int kColBlock = 64;

template <int kFT, int kFN>
struct ColTile {
  static constexpr int kFrags = kFT * kFN;
  // Blocks in flight: about 128 registers of fragments where the sums leave
  // them, 96 beside the largest tile's.
  static constexpr int kDepth = kFrags >= 16 ? 2 : kFrags >= 4 ? 4 : 16 / (2 * (kFT + kFN));
};

template <typename T, int kFT, int kFN, bool kGated, RowKind kRows>
__global__ __launch_bounds__(kColThreads) void proj_cols_kernel(ProjArgs p) {
  using V8 = typename VecOf<T>::v8;
  constexpr bool kAligned = kRows == kVectors;
  constexpr int kFrags = kFT * kFN, kDepth = ColTile<kFT, kFN>::kDepth;
  constexpr int kOutFrags = kGated ? kFN / 2 : kFN;  // fragments of outputs per token fragment
  static_assert(!kGated || kFN % 2 == 0, "both factors of a gate");
  __shared__ f32x4 s_acc[kColWaves][kFrags][64];
  __shared__ uint32_t s_last;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = static_cast<int>(blockIdx.x) / p.splits, split = static_cast<int>(blockIdx.x) % p.splits;
  const int tile_t = tile % p.tiles_t, tile_n = tile / p.tiles_t;
  const int64_t t0 = static_cast<int64_t>(tile_t) * (kFT * 16);
  const int n0 = tile_n * (kOutFrags * 16);
  const int k_begin = split * p.k_range, k_end = std::min(p.d_in, k_begin + p.k_range);
  const int kc = (lane >> 4) * 8;
  const T* w[kFN];
  const T* x[kFT];
  bool w_ok[kFN], x_ok[kFT];
  // (Rows past the last read another one where their loads are not held back:
  // their sums are written nowhere.)
#pragma unroll
  for (int i = 0; i < kFN; ++i) {
    const int n = n0 + i % kOutFrags * 16 + (lane & 15);
    w_ok[i] = n < p.n_out;
    w[i] = static_cast<const T*>(p.w) + ((w_ok[i] ? n : 0) + (i < kOutFrags ? 0 : static_cast<int64_t>(p.n_out))) * p.ldw + kc;
  }
#pragma unroll
  for (int j = 0; j < kFT; ++j) {
    const int64_t t = t0 + j * 16 + (lane & 15);
    x_ok[j] = t < p.tokens;
    x[j] = static_cast<const T*>(p.x) + (x_ok[j] ? t : t0) * p.ldx + kc;
  }
  f32x4 acc[kFN][kFT];
#pragma unroll
  for (int i = 0; i < kFN; ++i)
#pragma unroll
    for (int j = 0; j < kFT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  using Held = std::conditional_t<kRows == kElements, Words, V8>;  // eight elements on their way
  auto get = [&](const T* row, bool ok, int k) -> Held {
    if constexpr (kRows == kVectors)
      return ok && k + kc < k_end ? load8(row + k) : zero8<T>();
    else if constexpr (kRows == kWords)
      return __builtin_bit_cast(V8, load_any(row + k));
    else
      return load_words(row + k);
  };
  auto fragment = [&](const Held& v, const T* row) -> V8 {
    if constexpr (kRows == kElements)
      return __builtin_bit_cast(V8, settle(v, inside_word(row)));
    else
      return v;
  };
  Held fw[kDepth][2][kFN], fx[kDepth][2][kFT];
  auto load = [&](int b, int k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < kFN; ++i) fw[b][h][i] = get(w[i], w_ok[i], k + h * 32);
#pragma unroll
      for (int j = 0; j < kFT; ++j) fx[b][h][j] = get(x[j], x_ok[j], k + h * 32);
    }
  };
  auto multiply = [&](const V8 (&vw)[kFN], const V8 (&vx)[kFT]) {
#pragma unroll
    for (int i = 0; i < kFN; ++i)
#pragma unroll
      for (int j = 0; j < kFT; ++j) acc[i][j] = mfma16(vw[i], vx[j], acc[i][j]);
  };
  constexpr int kStride = kColWaves * kColBlock;
  const int k0 = k_begin + wave * kColBlock;
  // Rows that are not whole vectors: the whole blocks, whose loads need no tests,
  // then the columns left, which are one wave's.
  const int blocks_end = kAligned ? k_end : k_begin + (k_end - k_begin) / kColBlock * kColBlock;
#pragma unroll
  for (int b = 0; b < kDepth; ++b)
    if (kAligned || k0 + b * kStride < blocks_end) load(b, k0 + b * kStride);
  for (int k = k0; k < blocks_end; k += kDepth * kStride) {
#pragma unroll
    for (int b = 0; b < kDepth; ++b) {
      if (k + b * kStride >= blocks_end) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        V8 vw[kFN], vx[kFT];
#pragma unroll
        for (int i = 0; i < kFN; ++i) vw[i] = fragment(fw[b][h][i], w[i]);
#pragma unroll
        for (int j = 0; j < kFT; ++j) vx[j] = fragment(fx[b][h][j], x[j]);
        multiply(vw, vx);
      }
      if (k + (kDepth + b) * kStride < blocks_end) load(b, k + (kDepth + b) * kStride);
    }
  }
  if (blocks_end < k_end && (blocks_end - k_begin) / kColBlock % kColWaves == wave) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = blocks_end + h * 32;
      V8 vw[kFN], vx[kFT];
#pragma unroll
      for (int i = 0; i < kFN; ++i) vw[i] = __builtin_bit_cast(V8, load_first(w[i] + k, k_end - k - kc));
#pragma unroll
      for (int j = 0; j < kFT; ++j) vx[j] = __builtin_bit_cast(V8, load_first(x[j] + k, k_end - k - kc));
      multiply(vw, vx);
    }
  }

#pragma unroll
  for (int i = 0; i < kFN; ++i)
#pragma unroll
    for (int j = 0; j < kFT; ++j) s_acc[wave][i * kFT + j][lane] = acc[i][j];
  __syncthreads();
  // Each wave joins, and finishes, output fragments wave, wave + 8, ...
  constexpr int kOuts = kOutFrags * kFT;
  constexpr int kMine = (kOuts + kColWaves - 1) / kColWaves;
  constexpr uint32_t kTileBytes = kFrags * 1024;
  char* parts = reinterpret_cast<char*>(p.part) + static_cast<uint64_t>(tile) * p.splits * kTileBytes;
  f32x4 sum[kMine][2];
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    const int o = wave + m * kColWaves;
    sum[m][0] = sum[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (o < kOuts)
#pragma unroll
      for (int i = 0; i < kColWaves; ++i) {
        sum[m][0] += s_acc[i][o][lane];
        if constexpr (kGated) sum[m][1] += s_acc[i][kOuts + o][lane];
      }
  }
  if (p.splits > 1) {
    const __amdgpu_buffer_rsrc_t mine = coherent_buffer(parts + static_cast<uint64_t>(split) * kTileBytes, kTileBytes);
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int o = wave + m * kColWaves;
      if (o >= kOuts) break;
      coherent_store16(mine, static_cast<uint32_t>(o * 64 + lane) * 16, sum[m][0]);
      if constexpr (kGated) coherent_store16(mine, static_cast<uint32_t>((kOuts + o) * 64 + lane) * 16, sum[m][1]);
    }
    if (!last_split(p.tile_cnt + tile, p.splits, &s_last)) return;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int o = wave + m * kColWaves;
      if (o >= kOuts) break;
      sum[m][0] = sum[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int s = 0; s < p.splits; ++s) {
        const __amdgpu_buffer_rsrc_t one = coherent_buffer(parts + static_cast<uint64_t>(s) * kTileBytes, kTileBytes);
        sum[m][0] += coherent_load16(one, static_cast<uint32_t>(o * 64 + lane) * 16);
        if constexpr (kGated) sum[m][1] += coherent_load16(one, static_cast<uint32_t>((kOuts + o) * 64 + lane) * 16);
      }
    }
  }
  with_activation(p.act, [&](auto act) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int o = wave + m * kColWaves;
      const int64_t t = t0 + o % kFT * 16 + (lane & 15);
      const int n = n0 + o / kFT * 16 + (lane >> 4) * 4;
      if (o >= kOuts || t >= p.tokens || n >= p.n_out) continue;
      const Biases bias = biases<T>(p, n);
      if (p.rows_vec && n + 4 <= p.n_out)
        finish<T, decltype(act)::value, true>(p, t, n, 4, sum[m][0], sum[m][1], bias);
      else
        finish<T, decltype(act)::value, false>(p, t, n, p.n_out - n, sum[m][0], sum[m][1], bias);
    }
  });
}

// K-ranges of a launch of `tiles` workgroups: as many as bring it to `want`
// of them, each of at least `least` columns, within the scratch.
void split_columns(ProjArgs& a, int64_t tiles, int64_t want, int least, uint64_t tile_bytes) {
  int64_t splits = tiles >= want ? 1 : want / tiles;
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, a.d_in / least));
  while (splits > 1 && static_cast<uint64_t>(tiles * splits) * tile_bytes > a.part_bytes) --splits;
  if (tiles > a.n_cnt) splits = 1;
  const int64_t steps = std::max<int64_t>(1, (a.d_in + kStepK - 1) / kStepK);
  a.k_range = static_cast<int32_t>((steps + splits - 1) / splits * kStepK);
  a.splits = static_cast<int32_t>(std::max<int64_t>(1, (static_cast<int64_t>(a.d_in) + a.k_range - 1) / a.k_range));
}

template <typename T, int BT, int BN, int WT, int WN, int R, bool kAligned>
hipError_t launch_tiles(ProjArgs& a, hipStream_t stream) {
  const int outs = a.gated ? BN / 2 : BN;
  a.tiles_t = static_cast<int32_t>((a.tokens + BT - 1) / BT);
  a.tiles_n = (a.n_out + outs - 1) / outs;
  const int64_t tiles = static_cast<int64_t>(a.tiles_t) * a.tiles_n;
  if (!grid_fits(tiles, 64 * WT * WN)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((proj_kernel<T, BT, BN, WT, WN, R, kAligned>), dim3(static_cast<uint32_t>(tiles)), dim3(64 * WT * WN), 0,
                     stream, a);
  return hipGetLastError();
}

template <typename T, int kFT, int kFN, RowKind kRows>
hipError_t launch_cols(ProjArgs& a, int n_cu, hipStream_t stream) {
  const int outs = kFN * 16 / (a.gated ? 2 : 1);
  a.tiles_t = static_cast<int32_t>((a.tokens + kFT * 16 - 1) / (kFT * 16));
  a.tiles_n = (a.n_out + outs - 1) / outs;
  const int64_t tiles = static_cast<int64_t>(a.tiles_t) * a.tiles_n;
  // A tile's columns are split over workgroups only where tiles leave half of
  // the device idle: joining costs about 5 us.
  split_columns(a, tiles, n_cu, 4 * kColWaves * kColBlock, kFT * kFN * 1024);
  if (!grid_fits(tiles * a.splits, kColThreads)) return hipErrorInvalidValue;
  const dim3 grid(static_cast<uint32_t>(tiles * a.splits));
  if (a.gated) {
    if constexpr (kFN % 2 == 0)
      hipLaunchKernelGGL((proj_cols_kernel<T, kFT, kFN, true, kRows>), grid, dim3(kColThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL((proj_cols_kernel<T, kFT, kFN, false, kRows>), grid, dim3(kColThreads), 0, stream, a);
  }
  return hipGetLastError();
}

template <typename T, RowKind kRows>
hipError_t launch(ProjArgs& a, int n_cu, hipStream_t stream) {
  constexpr bool kAligned = kRows == kVectors;
  if (a.tokens <= 16) {
    if (a.gated) return launch_cols<T, 1, 2, kRows>(a, n_cu, stream);
    return launch_cols<T, 1, 1, kRows>(a, n_cu, stream);
  }
  const int64_t rows = static_cast<int64_t>(a.n_out) * (a.gated ? 2 : 1);
  auto tiles = [&](int64_t b) { return (a.tokens + b - 1) / b * ((rows + b - 1) / b); };
  // (32 x 4096 x 4096: 11.8 us, 14.2 on 64-row tiles; 128 x 8192 x 1024, 32 of
  // those tiles: 19.9 and 24.6; 128 x 2048 x 2048, 64 of them: 9.9 and 8.9.)
  if (a.tokens <= 32 || tiles(64) < n_cu / 4) return launch_cols<T, 2, 2, kRows>(a, n_cu, stream);
  // The tile whose rounds over the device cost least.  A K-step of a round
  // takes 1.5 us with the 256-row tile (one workgroup a compute unit), 0.72
  // with the 128-row one, 0.4 with two 64-row ones a compute unit and 0.22
  // with one.  (512 x 5120 x 27648: 130, 202 and 279 us; 2048 x 2048 x 2048: 49,
  // 20.2 and 26.3; 1000 x 2048 x 2048: 52, 17.5 and 14.9; on operands of one
  // magnitude: the first takes 129 with constant ones and 141 with normal ones.)
  auto rounds = [&](int64_t n, int64_t at_once) { return static_cast<double>((n + at_once - 1) / at_once); };
  // Rows that are not whole vectors: 0.66 and 0.36 on the 64-row tiles, as long
  // as the others on the 128-row one.  (300 x 8191 x 14336: 166 us on 128 rows, 195
  // on 64; 400 x 4097 x 8000: 50 and 84; 500 x 8191 x 4096: 88 and 85; 1000 x 1001 x
  // 1101: 17.8 and 15.7.)
  const double cost64 = tiles(64) <= n_cu ? (kAligned ? 0.22 : 0.36) : (kAligned ? 0.4 : 0.66) * rounds(tiles(64), 2 * n_cu);
  const double cost128 = 0.72 * rounds(tiles(128), n_cu);
  if constexpr (kAligned) {
    if (1.5 * rounds(tiles(256), n_cu) <= std::min(cost64, cost128))
      return launch_tiles<T, 256, 256, 2, 4, 2, kAligned>(a, stream);
  }
  if (cost128 <= cost64) return launch_tiles<T, 128, 128, 4, 2, 4, kAligned>(a, stream);
  return launch_tiles<T, 64, 64, 2, 2, 4, kAligned>(a, stream);
}

}  // namespace

hipError_t launch_proj(int dtype_bf16, ProjArgs& a, int n_cu, hipStream_t stream) {
  auto whole = [](const void* p, int64_t ld, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld % (bytes / 2) == 0;
  };
  a.rows_vec = whole(a.y, a.ldy, 8) && whole(a.residual, a.ldr, 8);
  // Rows further apart than kFarRows take the register paths, which have no 32-bit offsets.
  const bool vectors = a.d_in % 8 == 0 && whole(a.x, a.ldx, 16) && whole(a.w, a.ldw, 16) && a.ldx <= kFarRows && a.ldw <= kFarRows;
  const bool words = whole(a.x, a.ldx, 4) && whole(a.w, a.ldw, 4);
  auto run = [&](auto t) {
    using T = decltype(t);
    return vectors ? launch<T, kVectors>(a, n_cu, stream) : words ? launch<T, kWords>(a, n_cu, stream) : launch<T, kElements>(a, n_cu, stream);
  };
  return dtype_bf16 ? run(__bf16{}) : run(_Float16{});
}

}  // namespace wp
