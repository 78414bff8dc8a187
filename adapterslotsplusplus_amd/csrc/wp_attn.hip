// wp_attn.hip -- attention over packed sequences of different lengths
// (gfx950): causal, grouped heads, optional window, fp32 softmax statistics.
//
// For every query row i of a key head (the rows of one key head are its
// sequence's tokens times the query heads that share it):
//   out_i = sum_j 2^(c s_ij - m_i) v_j / l_i,   l_i = sum_j 2^(c s_ij - m_i),
// with s = q . k, c = scale * log2(e) and m_i a running bound of c s_ij, in one
// pass over the keys.
//
// The scores are computed transposed, S^T = K . Q^T (32x32x16): a lane then
// holds 16 keys of one query per tile, so maximum and sum are sums over its
// own registers (and one other lane's), and the exponentials, packed in
// register order, already are the right operand of O^T = V^T . P^T, whose
// contraction index may run over the keys in any order.  V^T's fragments come
// out of LDS by the transposing read, four keys of a column at a time, in that
// same order.
//
// Two roles.  Sequences with many rows per key head run on row tiles: a
// workgroup's waves take 32 rows each and stage 64 keys and values at a time
// in LDS for all of them.  Short ones (single tokens, drafted tokens) run on
// key chunks: the waves share out the keys, 32 at a time, and (past 32 rows)
// the rows, and each streams keys of its own.  A launch has one role where the
// host can tell, else both.  Either role splits a long key range over
// workgroups where there are too few of them, and the last one of a row tile
// to finish joins the partial results.
//
// What bounds it.  Long prompts: the matrix and the vector unit take turns at
// nearly equal work (16384 tokens, 32 heads of 128: 2000 us, 1.10 PF/s; a 64-key
// step of 32 rows takes 1024 cycles of products and about 900 of exponentials, sums
// and roundings).  Decoding over long caches: HBM (64 sequences of up to 8192
// keys, 8 key heads: 79.7 us, 4.4 TB/s).  Few and short sequences: the chain of
// latencies from the bounds over K to the join (one token over 777 keys: 11.5 us,
// of them 2.2 to find the item, 3.4 to the last product, 4 to join).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "wp_apply.h"
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
constexpr int kChunkWaves = 4;
constexpr int kChunkRows = kWaveRows * kChunkWaves;  // most query rows of a sequence that runs on key chunks
constexpr int kChunkKeys = 32;                 // keys a wave stages at a time for a key chunk
// A running bound is raised (and O and l scaled) only once a score exceeds it
// by 2^8: exponentials then stay within 2^8, far inside fp16, and most tiles
// scale nothing.
constexpr float kSlack = 8.f;
constexpr int kTiles = 1, kChunks = 2;  // the roles of a launch
constexpr int kNoSplit = 31;  // keys per split as a power of two: past every length

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

// One work item.
struct Item {
  int seq;       // -1: none
  int head;      // key head
  int tile;      // row tile of the sequence
  int chunk;     // key chunk
  int slot;      // the item's place among the partials
  int counter;   // its row tile's counter
  int stride;    // between the slots of a row tile's chunks
  int end;       // no item's id reaches this
  int64_t q0, k0;
  int n_q, n_k;
};

struct Span {
  int q0, k0, n_q, n_k;
};
// n / d, exactly for n < 2^31: the product is under 2^63.
__device__ __forceinline__ int over(int n, const Divisor& d) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * d.magic) >> d.shift);
}
__device__ __forceinline__ Span span_of(const AttnArgs& p, int b) {
  Span s;
  const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
  const int tokens = static_cast<int>(p.tokens), keys = static_cast<int>(p.keys);
  s.q0 = std::clamp(q0, 0, tokens);
  s.n_q = std::clamp(q1, s.q0, tokens) - s.q0;
  s.k0 = std::clamp(k0, 0, keys);
  s.n_k = std::clamp(k1, s.k0, keys) - s.k0;
  return s;
}

// The first key that a query at key position `pos` sees: with the windows the
// host takes, up to 2^31 - 1, pos - window + 1 need not fit 32 bits.
__device__ __forceinline__ int window_start(int pos, int window) {
  return window > 0 ? std::max(0, std::max(0, pos + 1) - window) : 0;
}

// Keys that rows [row, row + rows) of a sequence see: [first, end).
struct Range {
  int first, end;
};
__device__ __forceinline__ Range keys_of(const AttnArgs& p, int n_q, int n_k, int row, int rows) {
  Range r{0, n_k};
  if (!p.causal) return r;
  const int t0 = over(row, p.by_group), t1 = std::min(n_q - 1, over(row + rows - 1, p.by_group));
  r.end = std::clamp(t1 + n_k - n_q + 1, 0, n_k);
  r.first = std::min(window_start(t0 + n_k - n_q, p.window), r.end);
  return r;
}

// Key chunks over a whole sequence's keys for a given role.
__device__ __forceinline__ int chunks_of(int keys, int shift) {
  return std::max(1, static_cast<int>((static_cast<int64_t>(keys) + (1ll << shift) - 1) >> shift));
}
__device__ __forceinline__ int shift_of(const AttnArgs& p, int rows, bool rows_role) {
  return rows_role ? p.tile_shift : rows > p.split_rows ? kNoSplit : p.chunk_shift;
}
__device__ __forceinline__ int items_of(const AttnArgs& p, const Span& s, bool rows_role, int tile_rows, int* tiles) {
  const int rows = s.n_q * p.group;
  *tiles = 0;
  if (rows == 0 || (rows > p.chunk_rows) != rows_role) return 0;
  const Range r = keys_of(p, s.n_q, s.n_k, 0, rows);
  const int unit = rows_role ? kTileKeys : kChunkKeys;
  const int chunks = chunks_of(r.end - r.first / unit * unit, shift_of(p, rows, rows_role));
  *tiles = (rows + tile_rows - 1) / tile_rows;
  return *tiles * chunks;
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

__device__ __forceinline__ Item item_of(const AttnArgs& p, const Span& s, int lane, int head, int id, int seq, int tile, int chunk, int n_tiles,
                                        int first_tile) {
  Item it;
  it.head = head;
  it.slot = id;
  it.seq = __builtin_amdgcn_readfirstlane(seq);
  it.tile = __builtin_amdgcn_readfirstlane(tile);
  it.chunk = __builtin_amdgcn_readfirstlane(chunk);
  it.counter = __builtin_amdgcn_readfirstlane((first_tile + tile) * p.kv_heads + head);
  it.stride = __builtin_amdgcn_readfirstlane(n_tiles * p.kv_heads);
  it.q0 = __builtin_amdgcn_readlane(s.q0, lane);
  it.k0 = __builtin_amdgcn_readlane(s.k0, lane);
  it.n_q = __builtin_amdgcn_readlane(s.n_q, lane);
  it.n_k = __builtin_amdgcn_readlane(s.n_k, lane);
  return it;
}

// Row tiles that run whole, of up to 64 sequences (a lane each): the tiles
// with the most keys first, so that none of the long ones starts last.  The
// tiles of a sequence that see at least w keys are its last ones; a search over
// w finds the item's, and its place among the tiles that see exactly as many.
// (One prompt of 16384 tokens, 32 heads over 8: 2000 us, 2060 in order of the
// tiles' rows; 16 prompts of 111 to 2501 tokens: 162 either way.)
__device__ __forceinline__ Item find_by_weight(const AttnArgs& p, int tile_rows, int id) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int tiles = 0;
  Span s{0, 0, 0, 0};
  if (lane < p.n_seq) {
    s = span_of(p, lane);
    (void)items_of(p, s, true, tile_rows, &tiles);
  }
  const int lag = s.n_k - s.n_q;
  // Tiles whose last row sees at least 64 u keys.
  auto at_least = [&](int u) {
    const int w = u * kTileKeys;
    if (w > s.n_k) return 0;
    if (!p.causal) return tiles;
    const int64_t row = static_cast<int64_t>(w - lag - 1) * p.group;  // the first that sees w keys
    const int64_t below = row <= 0 ? 0 : row / tile_rows;           // tiles before that row's
    return below >= tiles ? 0 : static_cast<int>(tiles - below);
  };
  Item it;
  it.seq = -1;
  const int want = over(id, p.by_heads);
  if (want >= total_of(tiles)) return it;
  int lo = -1, hi = static_cast<int>(p.keys / kTileKeys) + 1;  // more than `want` tiles see 64 lo keys, not 64 hi
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (total_of(at_least(mid)) > want) lo = mid; else hi = mid;
  }
  const int above = at_least(lo + 1), here = (lo < 0 ? tiles : at_least(lo)) - above;
  const int rest = want - total_of(above);
  const int upto = sum_up(here);
  const int at = __builtin_ctzll(__ballot(upto > rest));
  const int from = __builtin_amdgcn_readlane(above, at) + rest -
                   (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(here, at));  // from the sequence's last tile
  const int n_tiles = __builtin_amdgcn_readlane(tiles, at);
  return item_of(p, s, at, id - want * p.kv_heads, id, at, n_tiles - 1 - from, 0, n_tiles, 0);
}

// The item of this workgroup: every wave counts through the sequences, 64 at
// a time, a lane each.
__device__ __forceinline__ Item find_item(const AttnArgs& p, bool rows_role, int tile_rows, int id) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  if (rows_role && p.tile_shift == kNoSplit && p.n_seq <= 64) return find_by_weight(p, tile_rows, id);
  Item none;
  none.seq = -1;
  const int want = over(id, p.by_heads);
  int base = 0, tile_base = 0;
  for (int b0 = 0; b0 < p.n_seq; b0 += 64) {
    const int b = b0 + lane;
    int tiles = 0, items = 0;
    Span s{0, 0, 0, 0};
    if (b < p.n_seq) {
      s = span_of(p, b);
      items = items_of(p, s, rows_role, tile_rows, &tiles);
    }
    const int sum = sum_up(items), tile_sum = sum_up(tiles);
    const unsigned long long past = __ballot(base + sum > want);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int local = want - base - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(items, at));
      const int n_tiles = __builtin_amdgcn_readlane(tiles, at);
      // Later row tiles see more keys: they go first.
      Item it = item_of(p, s, at, id - want * p.kv_heads, id, b0 + at, n_tiles - 1 - local % n_tiles, local / n_tiles, n_tiles,
                        tile_base + __builtin_amdgcn_readlane(tile_sum, at) - n_tiles);
      it.end = b0 + 64 < p.n_seq ? p.chunk_items : (base + __builtin_amdgcn_readlane(sum, 63)) * p.kv_heads;
      return it;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
    tile_base += __builtin_amdgcn_readlane(tile_sum, 63);
  }
  return none;
}

// A wave's 32 query rows and their running state.
template <typename T, int DP>
struct Rows {
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
    const int first = at + ((static_cast<int>(threadIdx.x) & 63) >> 5) * 4;
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

// K fragment of step `step`: keys row0 .. row0 + 31 of a staged tile.
template <typename T, int DP>
__device__ __forceinline__ typename VecOf<T>::v8 key_fragment(const char* keys, int row0, int step) {
  using H = Head<DP>;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int r = lane & 31, c = step * 2 + (lane >> 5);
  return *reinterpret_cast<const typename VecOf<T>::v8*>(keys + (row0 + r) * H::kRow + ((c ^ H::key_swizzle(r)) << 4));
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
  const int at = (key0 + r) * H::kRow + ((c ^ H::value_swizzle(r)) << 4) + (i & 1) * 8;
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

// Adds the infinite and NaN values of keys [at, at + n) that a query sees,
// which value_fragment<careful> left out.
template <typename T, int DP>
__device__ __forceinline__ void add_nonfinite(Rows<T, DP>& w, const char* values, int at, int n) {
  using H = Head<DP>;
  const int lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5;
  for (int r = 0; r < n; ++r) {
    const char* row = values + r * H::kRow;
    bool odd = false;
    if (lane < H::kRow / 4) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(row + lane * 4);
      odd = !finite16<T>(u & 0xFFFFu) || !finite16<T>(u >> 16);
    }
    if (!__any(odd)) continue;
    const bool sees = at + r <= w.pos && at + r >= w.low;
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

// Staging: load i of a wave fills rows (first + i) * kRowsPerLoad on of a tile
// straight in LDS, 16 bytes a lane.  A lane's offsets from the tile's first row
// are the same for every tile; the rows past the tile's last one and the
// columns past the head lie outside its bytes and are zero.
template <int DP, bool kValues, int kLoads>
struct Loads {
  using H = Head<DP>;
  int off[kLoads];
  int stride, row_bytes, first;

  __device__ __forceinline__ Loads(int64_t tok_stride, int dim, int first_load)
      : stride(static_cast<int>(tok_stride) * 2), row_bytes(dim * 2), first(first_load) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (first + i) * H::kRowsPerLoad + lane / H::kChunks;
      const int c = (lane % H::kChunks) ^ (kValues ? H::value_swizzle(r) : H::key_swizzle(r));
      off[i] = c * 8 < dim ? r * stride + c * 16 : kOutside;
    }
  }
  // The first `rows` rows (at most the tile's) at src to dst.
  __device__ __forceinline__ void stage(const void* src, int rows, char* dst) const {
    const int size = rows <= 0 ? 0 : (std::min(rows, kTileKeys) - 1) * stride + row_bytes;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_to_lds(src, dst + (first + i) * 1024, off[i], 0, size);
  }
};

template <typename T>
__device__ __forceinline__ const T* head_row(const void* base, int64_t tok, int64_t tok_stride, int64_t head_offset) {
  return static_cast<const T*>(base) + tok * tok_stride + head_offset;
}

// Exponentials of a 32-key tile, added to the lane's sum in fp32 and packed: the
// two right operands of its two 16-key steps.  The matrix cores take 16-bit
// operands: each weight is rounded to the tensors' type, once, so that O is off
// by at most half a unit of that type of sum p |v| -- what rounding the values
// themselves did.
template <typename T, int DP>
__device__ __forceinline__ void weigh(Rows<T, DP>& w, const f32x16& s, float c, typename VecOf<T>::v8 (&out)[2]) {
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
template <typename T, int DP>
__device__ __forceinline__ f32x16 scores(const Rows<T, DP>& w, const char* keys, int row0) {
  constexpr int kSteps = Head<DP>::kSteps;
  typename VecOf<T>::v8 kf[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) kf[x] = key_fragment<T, DP>(keys, row0, x);
  __builtin_amdgcn_sched_barrier(0);
  f32x16 s{};
#pragma unroll
  for (int x = 0; x < kSteps; ++x) {
    s = mfma32(kf[x % 4], w.q[x], s);
    if (x + 4 < kSteps) kf[x % 4] = key_fragment<T, DP>(keys, row0, x + 4);
    __builtin_amdgcn_sched_barrier(0);
  }
  return s;
}

// Adds 32 staged keys' weighted values to O.
template <typename T, int DP, bool kCareful>
__device__ __forceinline__ void accumulate(Rows<T, DP>& w, const char* values, int row0,
                                           const typename VecOf<T>::v8 (&e)[2]) {
  constexpr int kCols = Head<DP>::kCols, kAhead = kCols < 4 ? kCols : 4;
  auto value = [&](int i) { return value_fragment<T, DP, kCareful>(values, row0 + i / kCols * 16, i % kCols); };
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

// LDS of a workgroup.  Each buffer is an array of its own: the compiler then
// sees that a load into one leaves reads of the others alone, and does not wait
// for it.
template <int DP>
struct Staged {
  static constexpr int kBytes = kTileKeys * Head<DP>::kRow;
};
#define WP_STAGED char (&sk0)[Staged<DP>::kBytes], char (&sk1)[Staged<DP>::kBytes], char (&sv0)[Staged<DP>::kBytes], \
                  char (&sv1)[Staged<DP>::kBytes]

// Row tile: the keys [first, end) for the workgroup's rows, 64 at a time.
// While tile j is weighed and added, the scores of tile j + 1 are computed
// (they need nothing of it, so the matrix cores work beside the exponentials), and tiles j + 2
// of K and j + 1 of V are on their way.
template <typename T, int DP, int kWaves>
__device__ __forceinline__ void run_tile(const AttnArgs& p, const Item& it, Rows<T, DP>& w, float c, int first, int end,
                                         int wave_low, int wave_pos, int wave_last, int wave, WP_STAGED) {
  using H = Head<DP>;
  using V8 = typename VecOf<T>::v8;
  constexpr int kLoads = kTileKeys * H::kRow / 1024 / kWaves;
  const T* k = head_row<T>(p.k, it.k0, p.k_tok, it.head * p.k_head);
  const T* v = head_row<T>(p.v, it.k0, p.v_tok, it.head * p.v_head);
  const int64_t k_tok = p.k_tok, v_tok = p.v_tok;
  const int n_k = it.n_k;
  const Loads<DP, false, kLoads> loads_k(k_tok, p.dim, wave * kLoads);
  const Loads<DP, true, kLoads> loads_v(v_tok, p.dim, wave * kLoads);
  auto load_k = [&](int at, char* to) {
    if (at < end) loads_k.stage(k + at * k_tok, n_k - at, to);
  };
  auto load_v = [&](int at, char* to) {
    if (at < end) loads_v.stage(v + at * v_tok, n_k - at, to);
  };
  const int live_end = std::min(end, wave_last + 1);
  w.reset();
  if (first >= end) return;
  load_k(first, sk0);
  wait_vm();
  __syncthreads();
  load_k(first + kTileKeys, sk1);
  load_v(first, sv0);
  f32x16 s0 = scores(w, sk0, 0), s1 = scores(w, sk0, 32);
  constexpr std::integral_constant<bool, true> yes{};
  constexpr std::integral_constant<bool, false> no{};
  // The order of a tile's work is pinned so that products and vector work run
  // side by side throughout (two waves a SIMD in the same phase would else wait
  // for the one unit together and leave the other idle):
  //   the first half's exponentials between three quarters of the next tile's scores,
  //   the second half's between the rest of them and the first half's products with V,
  //   the next scores' maximum between the second half's products with V.
  // LDS reads go two products ahead.
  float tops = fmaxf(top_of(s0), top_of(s1));
  constexpr int kScores = 2 * H::kSteps, kFirst = kScores * 3 / 4, kValues = 2 * H::kCols;
  auto body = [&](int at, auto more, const char* knext, const char* vnow) {
    // wave_low, wave_pos: the keys that every row of the wave sees.
    if (at < wave_low || at + kTileKeys - 1 > wave_pos) {
      w.mask(s0, at);
      w.mask(s1, at + 32);
      tops = fmaxf(top_of(s0), top_of(s1));
    }
    w.raise(tops, c);
    const float base = w.m == -INFINITY ? 0.f : w.m;
    auto weigh = [&](f32x16& s, int from, int to) {
#pragma unroll
      for (int i = from; i < to; ++i) {
        s[i] = exp2_fast(fmaf(s[i], c, -base));
        w.l += s[i];
      }
    };
    auto key = [&](int i) { return key_fragment<T, DP>(knext, i / H::kSteps * 32, i % H::kSteps); };
    auto value = [&](int i) { return value_fragment<T, DP, false>(vnow, i / H::kCols * 16, i % H::kCols); };
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
  };
  auto step = [&](int at, char* kfree, const char* knext, const char* vnow, char* vnext) {
    wait_vm();
    __syncthreads();
    load_k(at + 2 * kTileKeys, kfree);
    load_v(at + kTileKeys, vnext);
    // Keys past the last one that any of the wave's rows sees are not its
    // work; the compute unit's other workgroup has the matrix cores then.
    if (at + kTileKeys < live_end)
      body(at, yes, knext, vnow);
    else if (at < live_end)
      body(at, no, knext, vnow);
  };
  for (int at = first; at < end; at += 2 * kTileKeys) {
    step(at, sk0, sk1, sv0, sv1);
    if (at + kTileKeys < end) step(at + kTileKeys, sk1, sk0, sv1, sv0);
  }
}

// run_tile, one tile after the other, with infinite and NaN values left out of
// the product and added to the rows that see them: the same sums otherwise.
template <typename T, int DP, int kWaves>
__device__ __forceinline__ void run_tile_careful(const AttnArgs& p, const Item& it, Rows<T, DP>& w, float c, int first,
                                                 int end, int wave_low, int wave_pos, int wave, char* sk, char* sv) {
  using H = Head<DP>;
  constexpr int kLoads = kTileKeys * H::kRow / 1024 / kWaves;
  const T* k = head_row<T>(p.k, it.k0, p.k_tok, it.head * p.k_head);
  const T* v = head_row<T>(p.v, it.k0, p.v_tok, it.head * p.v_head);
  const Loads<DP, false, kLoads> loads_k(p.k_tok, p.dim, wave * kLoads);
  const Loads<DP, true, kLoads> loads_v(p.v_tok, p.dim, wave * kLoads);
  w.reset();
  for (int at = first; at < end; at += kTileKeys) {
    __syncthreads();
    loads_k.stage(k + at * p.k_tok, it.n_k - at, sk);
    loads_v.stage(v + at * p.v_tok, it.n_k - at, sv);
    wait_vm();
    __syncthreads();
    f32x16 s0 = scores(w, sk, 0), s1 = scores(w, sk, 32);
    if (at < wave_low || at + kTileKeys - 1 > wave_pos) {
      w.mask(s0, at);
      w.mask(s1, at + 32);
    }
    w.raise(fmaxf(top_of(s0), top_of(s1)), c);
    typename VecOf<T>::v8 e0[2], e1[2];
    weigh(w, s0, c, e0);
    weigh(w, s1, c, e1);
    accumulate<T, DP, true>(w, sv, 0, e0);
    accumulate<T, DP, true>(w, sv, 32, e1);
    add_nonfinite(w, sv, at, kTileKeys);
  }
}

// Key chunk: a wave's keys from `at` on, 32 at a time and `step` apart.
template <typename T, int DP>
struct ChunkLoads {
  static constexpr int kLoads = kChunkKeys * Head<DP>::kRow / 1024;
  const T* k;
  const T* v;
  int64_t k_tok, v_tok;
  Loads<DP, false, kLoads> loads_k;
  Loads<DP, true, kLoads> loads_v;
  char* sk;
  char* sv;
  int end;
  __device__ __forceinline__ ChunkLoads(const AttnArgs& p, const Item& it, int end_, char* sk_, char* sv_)
      : k(head_row<T>(p.k, it.k0, p.k_tok, it.head * p.k_head)), v(head_row<T>(p.v, it.k0, p.v_tok, it.head * p.v_head)),
        k_tok(p.k_tok), v_tok(p.v_tok), loads_k(p.k_tok, p.dim, 0), loads_v(p.v_tok, p.dim, 0), sk(sk_), sv(sv_), end(end_) {}
  __device__ __forceinline__ void load_k(int at) const { loads_k.stage(k + at * k_tok, end - at, sk); }
  __device__ __forceinline__ void load_v(int at) const { loads_v.stage(v + at * v_tok, end - at, sv); }
};

// The first keys and values are on their way.  K and V take turns in flight:
// while one is read the other's next keys are coming, so each wait leaves the
// younger one's loads (a load past the end touches no memory and leaves zeros).
template <typename T, int DP, bool kCareful>
__device__ __forceinline__ void run_chunk(const ChunkLoads<T, DP>& in, Rows<T, DP>& w, float c, int at, int step,
                                          int wave_low, int wave_pos) {
  constexpr int kLoads = ChunkLoads<T, DP>::kLoads;
  w.reset();
  for (; at < in.end; at += step) {
    const int next = at + step;
    wait_vm_but<kLoads>();
    f32x16 s = scores(w, in.sk, 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    in.load_k(next);
    if (!(at >= wave_low && at + kChunkKeys - 1 <= wave_pos)) w.mask(s, at);
    w.raise(top_of(s), c);
    typename VecOf<T>::v8 e[2];
    weigh(w, s, c, e);
    wait_vm_but<kLoads>();
    accumulate<T, DP, kCareful>(w, in.sv, 0, e);
    if (kCareful) add_nonfinite(w, in.sv, at, kChunkKeys);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    in.load_v(next);
  }
  wait_vm();
}

template <typename T, int DP>
__device__ __forceinline__ bool has_nonfinite(const Rows<T, DP>& w) {
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < Head<DP>::kCols; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) z = fmaf(w.o[i][e], 0.f, z);
  return z != 0.f;  // NaN: an infinity or NaN times zero
}

// Writes four columns of a finished row (and with the first of them its lse).
template <typename T>
__device__ __forceinline__ void finish_row(const AttnArgs& p, const Item& it, int row, int d, f32x4 v, float m,
                                           float l) {
  const int tok = over(row, p.by_group), h = it.head * p.group + row - tok * p.group;
  const int pos = p.causal ? std::min(tok + it.n_k - it.n_q, it.n_k - 1) : it.n_k - 1;
  const bool sees = pos >= 0;
  if (d < p.dim)
    store4(static_cast<T*>(p.out) + (it.q0 + tok) * p.o_tok + h * p.o_head + d, sees ? v * (1.f / l) : f32x4{0.f, 0.f, 0.f, 0.f});
  if (p.lse && d == 0) p.lse[(it.q0 + tok) * p.heads + h] = sees ? fmaf(m, kLn2, logf(l)) : -INFINITY;
}

// Where a workgroup's waves meet.
template <int kWaves>
struct Shared {
  float m[kWaves][kWaveRows];
  float l[kWaves][kWaveRows];
  uint32_t last;
};

// One work item.  sk0 to sv1: LDS, Staged<DP>::kBytes each; my_k, my_v: this
// wave's halves of them on key chunks.
template <typename T, int DP, int kWaves, int kRole>
__device__ __forceinline__ void run_item(const AttnArgs& p, const Item& it, Shared<kWaves>& sh, WP_STAGED, char* my_k,
                                         char* my_v) {
  using H = Head<DP>;
  auto area = [&](int i) -> char* { return i == 0 ? sk0 : i == 1 ? sk1 : i == 2 ? sv0 : sv1; };
  constexpr bool kTile = kRole == kTiles;
  constexpr int kThreads = 64 * kWaves, kRows = kWaveRows * kWaves;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;
  const int group = p.group;
  const int n_rows = it.n_q * group;
  const int row0 = it.tile * kRows;                  // the workgroup's first row
  const int my_rows = std::min(kRows, n_rows - row0);
  const Range range = keys_of(p, it.n_q, it.n_k, row0, my_rows);
  const int shift = shift_of(p, n_rows, kTile);
  constexpr int unit = kTile ? kTileKeys : kChunkKeys;
  const int base = range.first / unit * unit;        // tiles start at whole ones
  const int chunks = chunks_of(range.end - base, shift);
  if (it.chunk >= chunks) return;
  // Bounds that fall can name more items than a launch has: a row tile then runs
  // only if all of its chunks are among them, so that its counter comes back to
  // zero and the calls after this one join what they should.
  if (it.slot + static_cast<int64_t>(chunks - 1 - it.chunk) * it.stride >= (kTile ? p.tile_items : p.chunk_items)) return;
  const int first = static_cast<int>(base + (static_cast<int64_t>(it.chunk) << shift));
  const int end = static_cast<int>(std::min<int64_t>(range.end, first + (1ll << shift)));

  // On key chunks, `share` waves take each 32 rows, every share-th 32 keys.
  const int row_log = kTile || my_rows > 2 * kWaveRows ? (kWaves == 8 ? 3 : 2) : my_rows > kWaveRows ? 1 : 0;
  const int row_waves = 1 << row_log, share = kWaves >> row_log;
  const int wave_row0 = row0 + (wave & (row_waves - 1)) * kWaveRows;
  const int row = wave_row0 + (lane & 31);
  const bool real = row < n_rows;
  const int tok = real ? over(row, p.by_group) : 0, sub = real ? row - tok * group : 0;
  const float c = p.scale == 0.f ? 1.f : fabsf(p.scale) * kLog2e;
  Rows<T, DP> w;
  {
    const T* q = head_row<T>(p.q, it.q0 + tok, p.q_tok, (it.head * group + sub) * p.q_head);
#pragma unroll
    for (int x = 0; x < H::kSteps; ++x) {
      const int d = x * 16 + half * 8;
      w.q[x] = real && d < p.dim && p.scale != 0.f ? load8(q + d) : zero8<T>();
    }
  }
  // A key chunk's first loads go out before the rest is worked out.
  const int at0 = first + (wave >> row_log) * kChunkKeys, step_keys = kChunkKeys * share;
  const ChunkLoads<T, DP> in(p, it, end, my_k, my_v);
  auto start = [&] {
    in.load_k(at0);
    in.load_v(at0);
  };
  if (!kTile) start();
  if (p.scale < 0.f) {
#pragma unroll
    for (int x = 0; x < H::kSteps; ++x) w.q[x] = negate8<T>(w.q[x]);
  }
  const int lag = it.n_k - it.n_q;
  w.pos = real ? (p.causal ? std::min(tok + lag, it.n_k - 1) : it.n_k - 1) : -1;
  w.low = p.causal ? window_start(tok + lag, p.window) : 0;
  // wave_low, wave_pos: the keys that all of the wave's rows see; wave_last: the
  // last one that any of them sees.
  int wave_pos = it.n_k - 1, wave_low = 0, wave_last = wave_row0 < n_rows ? it.n_k - 1 : -1;
  if (p.causal) {
    const int t0 = over(wave_row0, p.by_group), t1 = std::min(it.n_q - 1, over(wave_row0 + kWaveRows - 1, p.by_group));
    wave_pos = wave_row0 < n_rows ? t0 + lag : -1;
    wave_last = wave_row0 < n_rows ? t1 + lag : -1;
    wave_low = window_start(t1 + lag, p.window);
  }

  if constexpr (kTile) {
    run_tile<T, DP, kWaves>(p, it, w, c, first, end, wave_low, wave_pos, wave_last, wave, sk0, sk1, sv0, sv1);
    // Infinite or NaN values reach every row of a tile through the product, as
    // zero times them: where there are any, the pass is made again with care.
    if (__syncthreads_or(has_nonfinite(w)))
      run_tile_careful<T, DP, kWaves>(p, it, w, c, first, end, wave_low, wave_pos, wave, sk0, sv0);
  } else {
    run_chunk<T, DP, false>(in, w, c, at0, step_keys, wave_low, wave_pos);
    if (__any(has_nonfinite(w))) {
      start();
      run_chunk<T, DP, true>(in, w, c, at0, step_keys, wave_low, wave_pos);
    }
  }
  w.l += __shfl_xor(w.l, 32);

  const bool split = chunks > 1;
  const bool sees = real && w.pos >= w.low;
  // The item's partials: [rows][DP] of O, then [rows][bound, sum].
  const uint32_t slot_rows = kTile ? kRows : p.slot_rows;
  float* part = p.part + (kTile ? 0 : p.chunk_part) + static_cast<uint64_t>(it.slot) * slot_rows * (DP + 2);
  const __amdgpu_buffer_rsrc_t mine = coherent_buffer(part, slot_rows * (DP + 2) * 4u);

  if (kTile || share == 1) {
    const float inv = 1.f / w.l;
    if (!split) {
      if (!real) return;
      T* out = static_cast<T*>(p.out) + (it.q0 + tok) * p.o_tok + (it.head * group + sub) * p.o_head;
#pragma unroll
      for (int i = 0; i < H::kCols; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = i * 32 + e * 8 + half * 4;
          if (d >= p.dim) continue;
          const f32x4 v{w.o[i][e * 4], w.o[i][e * 4 + 1], w.o[i][e * 4 + 2], w.o[i][e * 4 + 3]};
          store4(out + d, sees ? v * inv : f32x4{0.f, 0.f, 0.f, 0.f});
        }
      if (p.lse && half == 0)
        p.lse[(it.q0 + tok) * p.heads + it.head * group + sub] = sees ? fmaf(w.m, kLn2, logf(w.l)) : -INFINITY;
      return;
    }
    const int r = wave * kWaveRows + (lane & 31);
    if (real) {
      if (half == 0) {
        coherent_store8(part + slot_rows * DP + 2 * r, __builtin_bit_cast(unsigned long long, f32x2{w.m, w.l}));
      }
#pragma unroll
      for (int i = 0; i < H::kCols; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          coherent_store16(mine, (r * DP + i * 32 + e * 8 + half * 4) * 4u,
                           f32x4{w.o[i][e * 4], w.o[i][e * 4 + 1], w.o[i][e * 4 + 2], w.o[i][e * 4 + 3]});
    }
  } else {
    // The waves' shares joined: each scales its O to the common bound and
    // leaves it in LDS, [row][DP] in an array of its own.
    if (half == 0) {
      sh.m[wave][lane] = w.m;
      sh.l[wave][lane] = w.l;
    }
    __syncthreads();
    float m = w.m;
    for (int i = 1; i < share; ++i) m = fmaxf(m, sh.m[(wave + i * row_waves) & (kWaves - 1)][lane & 31]);
    const float fade = m == -INFINITY ? 1.f : exp2_fast(w.m - m);
    // (Columns swizzled by the row: whole rows apart, lanes would share banks.)
    auto place = [](int r, int d) { return (r * (DP / 4) + ((d / 4) ^ (r & (DP == 96 ? 7 : 15)))) * 16; };
    char* o32 = area(wave);
    if (real)
#pragma unroll
      for (int i = 0; i < H::kCols; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<f32x4*>(o32 + place(lane & 31, i * 32 + e * 8 + half * 4)) =
              f32x4{w.o[i][e * 4], w.o[i][e * 4 + 1], w.o[i][e * 4 + 2], w.o[i][e * 4 + 3]} * fade;
    __syncthreads();
    for (int u = tid; u < my_rows * (DP / 4); u += kThreads) {
      const int r = u / (DP / 4), d = u % (DP / 4) * 4;
      const int w0 = r / kWaveRows, q = r % kWaveRows;
      float ms[kWaves], ls[kWaves];
      f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        const int x = w0 + (i < share ? i : 0) * row_waves;
        const f32x4 o = *reinterpret_cast<const f32x4*>(area(x) + place(q, d));
        ms[i] = sh.m[x][q];
        ls[i] = i < share ? sh.l[x][q] : 0.f;
        if (i < share) v += o;
      }
      float top = ms[0], l = 0.f;
#pragma unroll
      for (int i = 1; i < kWaves; ++i) top = fmaxf(top, ms[i]);
#pragma unroll
      for (int i = 0; i < kWaves; ++i) l += ls[i] * (top == -INFINITY ? 1.f : exp2_fast(ms[i] - top));
      if (split) {
        coherent_store16(mine, (r * DP + d) * 4u, v);
        if (d == 0) coherent_store8(part + slot_rows * DP + 2 * r, __builtin_bit_cast(unsigned long long, f32x2{top, l}));
      } else {
        finish_row<T>(p, it, row0 + r, d, v, top, l);
      }
    }
    if (!split) return;
  }

  // The last of the row tile's chunks to arrive joins them, in chunk order.
  wait_vm();
  __syncthreads();
  if (tid == 0) {
    uint32_t* cnt = p.counters + (kTile ? 0 : p.chunk_counters) + it.counter;
    const bool last = atomic_add_u(cnt, 1u) == static_cast<unsigned>(chunks - 1);
    if (last) atomic_store_u(cnt, 0u);
    sh.last = last ? 1u : 0u;
  }
  __syncthreads();
  if (sh.last == 0u) return;
  const int64_t step = static_cast<int64_t>(it.stride) * slot_rows * (DP + 2);  // floats between chunks' partials
  const float* part0 = part - it.chunk * step;
  for (int u = tid; u < my_rows * (DP / 4); u += kThreads) {
    const int r = u / (DP / 4), d = u % (DP / 4) * 4;
    float top = -INFINITY, l = 0.f;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    constexpr int kBatch = 8;
    for (int i0 = 0; i0 < chunks; i0 += kBatch) {
      f32x2 ml[kBatch];
      f32x4 o[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float* at = part0 + std::min(i0 + i, chunks - 1) * step;
        ml[i] = __builtin_bit_cast(f32x2, coherent_load8(at + slot_rows * DP + 2 * r));
        o[i] = coherent_load_f4(at + r * DP + d);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (i0 + i >= chunks) break;
        const float m = fmaxf(top, ml[i][0]);
        const float old = m == -INFINITY ? 1.f : exp2_fast(top - m), now = m == -INFINITY ? 1.f : exp2_fast(ml[i][0] - m);
        v = v * old + o[i] * now;
        l = l * old + ml[i][1] * now;
        top = m;
      }
    }
    finish_row<T>(p, it, row0 + r, d, v, top, l);
  }
}

// Clears the rows of no sequence: before the first bound and from the last one on.
template <typename T, int kWaves>
__device__ __forceinline__ void clear_rest(const AttnArgs& p, int bound0, int bound1) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int64_t head_rows = p.n_seq > 0 ? std::clamp<int64_t>(bound0, 0, p.tokens) : p.tokens;
  const int64_t tail = p.n_seq > 0 ? std::clamp<int64_t>(bound1, head_rows, p.tokens) : p.tokens;
  const int64_t n = (head_rows + p.tokens - tail) * p.heads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kWaves + wave; i < n; i += static_cast<int64_t>(gridDim.x) * kWaves) {
    int64_t t = i / p.heads;
    const int h = static_cast<int>(i % p.heads);
    if (t >= head_rows) t += tail - head_rows;
    T* out = static_cast<T*>(p.out) + t * p.o_tok + h * p.o_head;
    for (int d = lane; d < p.dim; d += 64) out[d] = static_cast<T>(0.f);
    if (p.lse && lane == 0) p.lse[t * p.heads + h] = -INFINITY;
  }
}

// Key chunks by themselves: as many workgroups a compute unit as LDS holds
// or the registers hold (three at heads of up to 64, else two).
template <int DP, int kRoles>
constexpr int kOccupancy = kRoles != kChunks || DP > 64 ? 2 : 3;

template <typename T, int DP, int kWaves, int kRoles>
__global__ __launch_bounds__(64 * kWaves, (kOccupancy<DP, kRoles>)) void attention_kernel(AttnArgs p) {
  constexpr int kRows = kWaveRows * kWaves, kHalf = Staged<DP>::kBytes / 2;
  __shared__ Shared<kWaves> sh;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);

  touch_kernel_args<static_cast<int>(sizeof(AttnArgs))>();
  // The outer bounds (lanes 0 and 1): a vector load, on its way together with
  // the first item's bounds and used once that is found.
  int outer = 0;
  if (p.n_seq > 0) outer = p.cu_q[threadIdx.x & 1 ? p.n_seq : 0];
  if constexpr (kRoles == kChunks) {
    __shared__ __align__(1024) char sk[2][Staged<DP>::kBytes];
    __shared__ __align__(1024) char sv[2][Staged<DP>::kBytes];
    // The grid covers the items that there usually are, the loop the most that there can be.
    int id = static_cast<int>(blockIdx.x);
    Item it = find_item(p, false, kRows, id);
    clear_rest<T, kWaves>(p, __builtin_amdgcn_readlane(outer, 0), __builtin_amdgcn_readlane(outer, 1));
    // Bounds that do not rise could name more row tiles than there are counters.
    while (id < p.chunk_items && it.seq >= 0 && it.counter < p.seq_counters) {
      run_item<T, DP, kWaves, kChunks>(p, it, sh, sk[0], sk[1], sv[0], sv[1], &sk[0][0] + wave * kHalf, &sv[0][0] + wave * kHalf);
      id += static_cast<int>(gridDim.x);
      if (id >= p.chunk_items || id >= it.end) return;
      __syncthreads();
      it = find_item(p, false, kRows, id);
    }
  } else {
    __shared__ __align__(1024) char sk0[Staged<DP>::kBytes];
    __shared__ __align__(1024) char sk1[Staged<DP>::kBytes];
    __shared__ __align__(1024) char sv0[Staged<DP>::kBytes];
    __shared__ __align__(1024) char sv1[Staged<DP>::kBytes];
    const int block = static_cast<int>(blockIdx.x);
    const bool rows_role = (kRoles & kChunks) == 0 || block < p.tile_items;
    const Item it = find_item(p, rows_role, kRows, rows_role ? block : block - p.tile_items);
    clear_rest<T, kWaves>(p, __builtin_amdgcn_readlane(outer, 0), __builtin_amdgcn_readlane(outer, 1));
    if (it.seq < 0 || it.counter >= (rows_role ? p.tile_counters : p.seq_counters)) return;
    if (rows_role) {
      run_item<T, DP, kWaves, kTiles>(p, it, sh, sk0, sk1, sv0, sv1, nullptr, nullptr);
    } else if constexpr ((kRoles & kChunks) != 0) {
      run_item<T, DP, kWaves, kChunks>(p, it, sh, sk0, sk1, sv0, sv1, (wave < 2 ? sk0 : sk1) + (wave & 1) * kHalf,
                                       (wave < 2 ? sv0 : sv1) + (wave & 1) * kHalf);
    }
  }
}

template <typename T, int DP, int kWaves, int kRoles>
hipError_t launch(const AttnArgs& a, int grid, hipStream_t stream) {
  hipLaunchKernelGGL((attention_kernel<T, DP, kWaves, kRoles>), dim3(static_cast<uint32_t>(std::max(1, grid))),
                     dim3(64 * kWaves), 0, stream, a);
  return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch_roles(const AttnArgs& a, int tile_waves, int chunk_grid, hipStream_t stream) {
  if (a.tile_items == 0) return launch<T, DP, kChunkWaves, kChunks>(a, chunk_grid, stream);
  if (tile_waves == kChunkWaves)
    return a.chunk_items == 0 ? launch<T, DP, kChunkWaves, kTiles>(a, a.tile_items, stream)
                              : launch<T, DP, kChunkWaves, kTiles | kChunks>(a, a.tile_items + a.chunk_items, stream);
  const hipError_t rc = launch<T, DP, 8, kTiles>(a, a.tile_items, stream);
  return rc != hipSuccess || a.chunk_items == 0 ? rc : launch<T, DP, kChunkWaves, kChunks>(a, chunk_grid, stream);
}

template <typename T>
hipError_t launch_head(const AttnArgs& a, int dp, int tile_waves, int chunk_grid, hipStream_t stream) {
  return dp == 64   ? launch_roles<T, 64>(a, tile_waves, chunk_grid, stream)
         : dp == 96 ? launch_roles<T, 96>(a, tile_waves, chunk_grid, stream)
                    : launch_roles<T, 128>(a, tile_waves, chunk_grid, stream);
}

}  // namespace

// Exact for every dividend under 2^31: the quotient's error is under
// dividend / 2^shift * d < 1 / d of a step.
static Divisor divisor_of(int d) {
  Divisor r{0, 31};
  while ((1ll << (r.shift - 31)) < d) ++r.shift;
  r.magic = static_cast<uint32_t>(((1ull << r.shift) + static_cast<uint64_t>(d) - 1) / static_cast<uint64_t>(d));
  return r;
}

hipError_t launch_attention(int dtype_bf16, AttnArgs& a, int n_cu, hipStream_t stream) {
  const int dp = a.dim <= 64 ? 64 : a.dim <= 96 ? 96 : 128;
  a.group = a.heads / a.kv_heads;
  a.by_group = divisor_of(a.group);
  a.by_heads = divisor_of(a.kv_heads);
  const int64_t group = a.group, rows = a.tokens * group;
  // Bounds on the work items, from the sizes the host knows: a sequence of
  // more than 128 rows has at most rows / 128 + 1 row tiles, and one of fewer
  // at most keys / chunk + 1 key chunks.
  const int64_t seqs = std::max(1, a.n_seq);
  // One sequence has one role.  Many of a few rows each (their mean at most 64,
  // and none of more than 128 if all have a token: single tokens, mostly) run on
  // key chunks alone, in a kernel without the row tiles' search and empty workgroups
  // (64 single tokens over up to 8192 keys: 79.6 us, 81.4 with both roles; 256: 193
  // and 196).  Where one could be longer the roles share a launch: drafted tokens
  // take the same either way (32 of up to 5, 8 heads a key head: 20.4 and 20.3;
  // 200 of up to 8, heads of their own keys: 50.2 and 51.9), but a prompt of 130
  // tokens among 19 single ones 35.2 us on key chunks and 26.0 on row tiles.
  // There, sequences run on key chunks up to 128 rows, or up to 32 next
  // to longer ones (32 heads of their own keys: a prompt of 128 rows takes 12.7 us
  // on key chunks, one of 129 takes 11.0 on a row tile).
  const int64_t longest = (std::max<int64_t>(0, a.tokens - seqs) + 1) * group;
  const bool few = a.n_seq <= 1 ? rows <= kChunkRows : rows <= 64 * seqs && longest <= kChunkRows;
  a.chunk_rows = few ? 0x7FFFFFFF : a.n_seq <= 1 ? 0 : rows >= kChunkRows * seqs ? kWaveRows : kChunkRows;
  const int64_t tile_seqs = few ? 0 : std::min<int64_t>(a.n_seq, rows / (a.chunk_rows + 1));
  // Row tiles of 256 rows read K and V half as often as those of 128 (a prompt of
  // 16384 tokens: 1998 us, 2060 on those), where they leave none idle.
  const int tile_waves = rows / 256 * a.kv_heads >= 2 * n_cu && rows >= 1024 * std::max(1, a.n_seq) ? 8 : 4;
  const int64_t tile_rows = kWaveRows * tile_waves;
  const int64_t tiles = tile_seqs > 0 ? rows / tile_rows + tile_seqs : 0;
  const int64_t chunk_seqs = a.chunk_rows == 0 ? 0 : std::min<int64_t>(a.n_seq, a.tokens);
  // Row tiles: enough of them for the device (two workgroups a compute unit)
  // run whole; fewer are split into ranges of at least 512 keys.
  int64_t tile_shift = kNoSplit;
  if (tiles > 0 && std::max<int64_t>(1, rows / tile_rows) * a.kv_heads < n_cu)
    for (tile_shift = 9; tile_shift < kNoSplit; ++tile_shift)
      if (tiles * ((a.keys >> tile_shift) + 2) * a.kv_heads <= 4 * n_cu) break;
  int64_t tile_items = tiles * (tile_shift == kNoSplit ? 1 : (a.keys >> tile_shift) + 2) * a.kv_heads;
  uint64_t tile_floats = tile_shift == kNoSplit ? 0 : static_cast<uint64_t>(tile_items) * tile_rows * (dp + 2);
  int64_t tile_counters = tile_shift == kNoSplit ? 0 : tiles * a.kv_heads;
  if (tile_floats * 4 > a.part_bytes / 2 || tile_counters > a.n_counters / 2) {
    tile_shift = kNoSplit;
    tile_items = tiles * a.kv_heads;
    tile_floats = 0;
    tile_counters = 0;
  }
  // Key chunks: about six workgroups a compute unit, of at least 128 keys (32
  // for each wave).
  int64_t chunk_shift = 7;
  while (chunk_shift < kNoSplit && (a.keys >> chunk_shift) * a.kv_heads > 6 * n_cu) ++chunk_shift;
  // Blocks of 128 rows: where sequences of more than 128 run on key chunks, the
  // longest could have them all.
  const int64_t blocks = few ? std::max<int64_t>(1, (rows + kChunkRows - 1) / kChunkRows) : 1;
  const int64_t usual = ((a.keys >> chunk_shift) + chunk_seqs) * a.kv_heads;
  int64_t chunk_items = 0, chunk_grid = 0;
  if (chunk_seqs > 0) {
    const int64_t counters = tile_counters + (chunk_seqs + blocks) * a.kv_heads;
    auto fits = [&](int64_t items, int64_t slot) {
      return (tile_floats + static_cast<uint64_t>(items) * slot * (dp + 2)) * 4 <= a.part_bytes && counters <= a.n_counters;
    };
    // A chunk has room for the partial results of 128 rows or, where the scratch
    // does not hold that many, of half as many or fewer, down to a token's;
    // sequences of more rows then have their keys run in one go.  (512 single tokens,
    // 32 heads over 8 of 128, one cache of 32768 keys among others of 100: 131 us
    // with room for 64 rows, 443 if no keys are split; all of 2000 keys: 692 either way.)
    int64_t slot = kChunkRows;
    const bool wide = fits(usual * blocks, slot);
    chunk_items = wide ? usual * blocks : usual + blocks * a.kv_heads;
    chunk_grid = usual;
    while (!wide && slot >= a.group && !fits(chunk_items, slot)) slot /= 2;
    if (slot < a.group && !wide) {
      chunk_shift = kNoSplit;
      chunk_items = chunk_grid = (chunk_seqs + blocks) * a.kv_heads;
    }
    a.slot_rows = static_cast<int32_t>(slot);
    a.split_rows = wide ? 0x7FFFFFFF : static_cast<int32_t>(slot);
  }
  if (tile_items + chunk_items > 0x7FFFFFFF) return hipErrorInvalidValue;
  a.tile_items = static_cast<int32_t>(tile_items);
  a.chunk_items = static_cast<int32_t>(chunk_items);
  a.tile_shift = static_cast<int32_t>(tile_shift);
  a.chunk_shift = static_cast<int32_t>(chunk_shift);
  a.chunk_part = tile_floats;
  a.tile_counters = tile_shift == kNoSplit ? 0x7FFFFFFF : static_cast<int32_t>(tile_counters);
  a.seq_counters = chunk_shift == kNoSplit ? 0x7FFFFFFF : a.n_counters - static_cast<int32_t>(tile_counters);
  a.chunk_counters = static_cast<int32_t>(tile_counters);
  return dtype_bf16 ? launch_head<__bf16>(a, dp, tile_waves, static_cast<int>(chunk_grid), stream)
                    : launch_head<_Float16>(a, dp, tile_waves, static_cast<int>(chunk_grid), stream);
}

}  // namespace wp
