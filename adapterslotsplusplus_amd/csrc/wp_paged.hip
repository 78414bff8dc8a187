// wp_paged.hip -- attention of new tokens over a paged cache (gfx950): grouped
// heads, causal, optional window with the first keys kept in sight, keys and
// values in 16 bits or e4m3 with a power of two per row, fp32 statistics.
//
//   out_i = sum_j 2^(c s_ij - m_i) v_j / l_i,   l_i = sum_j 2^(c s_ij - m_i)
// over the keys j that row i sees, s = q . k, c = scale * log2(e), m_i a running
// bound of c s_ij: one pass over the keys, by the tiles of wp_attn_core.h.
//
// Lengths are known on the device alone, and a table has room for far more keys
// than there are.  So a launch has as many workgroups as the device holds, and each
// wave works out the workgroup's share by itself, a lane for each sequence.  The cost of a row
// tile (32 or 128 rows of a key head) in keys is a linear function of the tile, cut off
// below and at the window, whose sum over a sequence has a closed form:
//   - a line of all tiles' costs, cut into equal shares wherever that is;
//   - up to 64 sequences, where there are no more tiles than workgroups and it takes no
//     longer, a line of equal pieces, one for each workgroup, that has no end of one tile and
//     start of another in a share (one token over 8192 keys 20.3 us, 34.1 without);
//   - up to 64 sequences' chunks over long caches: first stretches of whole shares (see there);
//   - many row tiles: each whole, the ones with the most keys first (see the launcher).
// 64 is where a lane holds a sequence; more share the one line (single tokens over 1 to 8192 keys,
// 4 query heads a key head of 128, 64 and 65 of them: 25.4 and 32.5 us on one key head, 31.8 and
// 35.8 on 2, 87.8 and 89.0 on 8; four chunks of 512 among 60 and 61 idle ones 403 and 426).
// A tile that several workgroups share is joined by the last of them to finish (by a
// counter of steps done), in a fixed order, so each key is read once for a tile, all
// end at about the same time, and results repeat bit for bit.
//
// Two roles.  Tiles of 128 rows: four waves of 32 rows, 64 keys and values at a
// time staged in LDS for all of them.  Up to 32 rows (single tokens, drafted
// tokens): the waves share out the keys, 32 at a time.  Launches whose sequences have no
// more rows than that on the whole have workgroups of two waves, twice as many of them: 64 single
// tokens over 1 to 8192 keys, 32 heads over 8 of 128, 85.5 us, and 98.6 in workgroups of
// four (and see the launcher).
//
// Keys and values go from their pages straight to LDS; in 8 bits they pass through
// registers, one tile ahead, and become the queries' type on their way to LDS (a power
// of two and 4 significant bits are exact in it, in fp16 where its range holds them).
// 16 keys are the unit of loads: a page holds whole ones, so that a wave's load has one
// base address.  Places of granules are listed in LDS as the first words of their
// buffers' descriptions, by lanes side by side, well before they are loaded: the tables'
// latency and the address arithmetic are off the path.
//
// What bounds it (32 heads over 8 of 128, bf16; over several cards).  Single tokens: HBM,
// 64 over 8192 keys each 381 to 388 us (5.6 TB/s), over 1 to 8192 keys 81 to 87 (4.1 to 4.3);
// 64 over 8192 keys in 8 bits 207 to 209 (5.2), near the conversions' rate.  Few: the
// chain from launch to join, 13.6 to 14.5 us over 777 keys.  Chunks: matrix and vector units as in
// wp_attn.hip, 2048 tokens over 16384 keys 489 to 504 us (1.02 to 1.05 PF/s), in 8 bits 528
// to 540: converting there takes the wave's own slots.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "wp_apply.h"
#include "wp_attn_core.h"
#include "wp_device.h"
#include "wp_paged.h"

namespace wp {
namespace {

constexpr int kTileWaves = 4;             // waves of a workgroup with row tiles among its items
constexpr int kChunkWaves = 2;            // and of one with key chunks alone
constexpr int kMostWaves = 4;
constexpr int kTiles = 1, kChunks = 2;  // the roles of a launch
// (Rows that pass through registers leave none for a tile's addresses.)
template <bool kSmall>
constexpr LaneKind kLane = kSmall ? kRenewed : kHeld;
constexpr int kGranule = 16;            // keys of one load address
constexpr int kMostWorkgroups = 1024;
constexpr int kChunkKeys = 32;          // keys of a wave's step on key chunks
constexpr int kMostPieces = 32;  // of a tile: more take longer to join than they save
constexpr float kLongestLine = 0x1p30f;
static_assert(kGranule == kMinPage, "a granule lies in one page");

// Of a workgroup of kWaves:
template <bool kTile, int kWaves>
constexpr int kStep = kTile ? kTileKeys : kChunkKeys * kWaves;  // keys of a step
template <bool kSmall, int kWaves>
constexpr int kListed = 64 * kWaves / (kSmall ? 2 : 1);  // granules whose places are listed at a time: 2 KiB a wave
template <bool kTile, bool kSmall, int kWaves>
constexpr int kSteps = kListed<kSmall, kWaves> * kGranule / kStep<kTile, kWaves>;  // steps listed at a time
template <bool kTile>
constexpr int kTileRows = kTile ? kWaveRows * kTileWaves : kWaveRows;

// ------------------------------------------------------------ the schedule --

struct Shape {
  int q0, n_q, n_k;
};
__device__ __forceinline__ Shape shape_of(const PagedArgs& p, int b) {
  const int tokens = static_cast<int>(p.tokens);
  Shape s;
  const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1];
  s.n_k = std::clamp(p.kv_lens[b], 0, p.capacity);
  s.q0 = std::clamp(q0, 0, tokens);
  s.n_q = std::clamp(q1, s.q0, tokens) - s.q0;
  return s;
}

// The line of costs.  Row tile t of a sequence sees about lag + (t + 1) * rows /
// group keys, and no more than the window, its own tokens and the first keys; it counts
// for at least 64, and as much again as 128 for its start and end.  Counted in
// keys times the group, whose sum over tiles has a closed form, and on the line
// in 2^cost_shift of them (and one for each tile), which keeps it in 31 bits.
struct Cost {
  long long lag, least, most;
  int extra, tiles, log_rows, shift;
  int pieces;  // of each tile, or 0: the line is one of costs
  int stretches;  // of keys at the start of each tile that are not on the line
  // Where tile t starts, from the sequence's start.
  __device__ __forceinline__ int before(int t) const {
    if (pieces > 0) return t * pieces;
    if (t == 0) return 0;
    if (t == 1) {
      const long long keys = lag + (1 << log_rows);
      return static_cast<int>(((keys < least ? least : keys > most ? most : keys) + extra) >> shift) + 1;
    }
    // Tiles whose line is at most `least`, and those below `most`.
    const long long low = (least - lag) >> log_rows, high = (most - lag - 1) >> log_rows;
    const long long a = low < 0 ? 0 : low > t ? t : low, b = high < a ? a : high > t ? t : high;
    const long long line = (b - a) * lag + (((b * (b + 1) - a * (a + 1)) >> 1) << log_rows);
    return static_cast<int>((a * least + line + (t - b) * most + static_cast<long long>(t) * extra) >> shift) + t;
  }
};
// `stretch`: how many steps of keys such a stretch has (0: there are none).  All
// tiles of a sequence have as many of them, before the first one's own tokens.
__device__ __forceinline__ Cost cost_of(const PagedArgs& p, const Shape& s, int stretch = 0) {
  const int rows = s.n_q * p.group;
  Cost c;
  c.log_rows = rows > p.chunk_rows ? 7 : 5;
  c.tiles = static_cast<int>((static_cast<unsigned>(rows) + (1u << c.log_rows) - 1) >> c.log_rows);
  c.lag = static_cast<long long>(p.group) * (s.n_k - s.n_q);
  c.least = 64ll * p.group;
  c.extra = 128 * p.group;
  c.most = p.window > 0 ? (static_cast<long long>(p.window) + p.sinks + 128) * p.group + (1 << c.log_rows) : (1ll << 60);
  c.shift = p.cost_shift;
  c.pieces = 0;
  c.stretches = 0;
  if (stretch > 0 && c.log_rows == 7 && s.n_k > s.n_q) {
    c.stretches = (s.n_k - s.n_q) / kTileKeys / stretch;
    // What is left of a tile with stretches is a share of it, and often the one that joins
    // them: some 20 us, 8 steps' time, 4 of them beyond a whole tile's start and end.  (16 x 128
    // tokens over caches that leave 1 to 3 steps: 518 us without, as one workgroup had
    // sixteen of those, 324.)
    if (c.stretches > 0) c.extra += 256 * p.group;
    c.lag -= static_cast<long long>(c.stretches) * stretch * kTileKeys * p.group;
  }
  return c;
}

// Sum over the wave's lanes, in the last one.
__device__ __forceinline__ float wave_sum(float v) {
  auto add = [&](auto ctrl, auto rows) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value, 0xF, true));
  };
  constexpr std::integral_constant<int, 0xF> all{};
  add(std::integral_constant<int, 0x111>{}, all);  // sum_up's moves
  add(std::integral_constant<int, 0x112>{}, all);
  add(std::integral_constant<int, 0x114>{}, all);
  add(std::integral_constant<int, 0x118>{}, all);
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
  return v;
}

// The largest of the wave's numbers.
__device__ __forceinline__ int longest_of(int v) {
#pragma unroll
  for (int i = 1; i < 64; i *= 2) v = std::max(v, __shfl_xor(v, i));
  return __builtin_amdgcn_readfirstlane(v);
}

// Row tiles that run whole, of up to 64 sequences (a lane each): the `want`-th of
// those of a key head, the tiles with the most keys first, so that none of the long
// ones starts last.  The tiles of a sequence that see at least w keys are its last
// ones; a search over w finds the tile's, and its place among those that see exactly
// as many.  seq: -1 past the last one.
__device__ __forceinline__ void tile_by_weight(const PagedArgs& p, const Shape& mine, int want, int& seq, int& tile) {
  const Cost c = cost_of(p, mine);
  const int tiles = c.tiles, lag = mine.n_k - mine.n_q;
  // Tiles whose last row sees at least 64 u keys.
  auto at_least = [&](int u) {
    const int w = u * 64;
    if (w > mine.n_k) return 0;
    const int64_t row = static_cast<int64_t>(w - lag - 1) * p.group;  // the first that sees w keys
    const int64_t below = row <= 0 ? 0 : row >> c.log_rows;         // tiles before that row's
    return below >= tiles ? 0 : static_cast<int>(tiles - below);
  };
  seq = -1;
  if (want >= total_of(tiles)) return;
  int lo = -1, hi = longest_of(mine.n_k) / 64 + 1;  // more than `want` tiles see 64 lo keys, not 64 hi
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (total_of(at_least(mid)) > want) lo = mid; else hi = mid;
  }
  const int above = at_least(lo + 1), here = (lo < 0 ? tiles : at_least(lo)) - above;
  const int rest = want - total_of(above);
  const int upto = sum_up(here);
  seq = __builtin_ctzll(__ballot(upto > rest));
  const int from = __builtin_amdgcn_readlane(above, seq) + rest -
                   (__builtin_amdgcn_readlane(upto, seq) - __builtin_amdgcn_readlane(here, seq));  // from the sequence's last tile
  tile = __builtin_amdgcn_readlane(tiles, seq) - 1 - from;
}

// The tile at place y from the sequence's start: 64 places a round.
__device__ __forceinline__ int tile_at(const Cost& c, int y) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int lo = 0, n = c.tiles;  // the tile is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 63) / 64;
    const bool upto = lane * static_cast<long long>(step) < n && c.before(lo + lane * step) <= y;
    const int k = __builtin_popcountll(__ballot(upto)) - 1;
    lo += k * step;
    n = std::min(step, n - k * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// One row tile of a key head, and what of it this workgroup does.
struct Item {
  int seq, head, tile;
  Shape s;
  int row0, rows;         // of the sequence's rows of this key head
  int low, end;           // rows see keys from `low` on, before `end`, and the first keys
  int base, sink_steps;   // step i: keys from i * kStep for the first sink_steps, then from base on
  int steps, from, to;    // all of its steps, and the workgroup's

  template <int kKeys>
  __device__ __forceinline__ int key_of(int i) const {
    return i < sink_steps ? i * kKeys : base + (i - sink_steps) * kKeys;
  }
};

// Where an item is on the line of all costs, and how the line is shared out.
struct Place {
  int start, cost;
  int total, share, near;
  int pieces;  // of each tile (Cost)
  int id;      // this workgroup's
  int stretch, whole;  // steps of a stretch, and workgroups that do one: the ones before those on the line
  int stretches;       // of the tile,
  int tiles, one;      // one workgroup for each, `tiles` apart from `one` on
  __device__ __forceinline__ int skipped() const { return stretches * stretch; }
  // Where workgroup i leaves its share of the item, if it is not the whole: two places for each
  // workgroup.  Its first item may have begun before it, its last one may go on after it,
  // and what is left of a tile with stretches goes beside the first of those.
  __device__ __forceinline__ int slot(int i, bool begins) const { return !begins ? 2 * i : stretches > 0 ? 2 * one + 1 : 2 * i + 1; }
  // Of the steps on the line, the one at which the line's point x cuts the item.  Cuts near its ends
  // are moved there: a cut costs the shares' way through memory.
  __device__ __forceinline__ int cut(int x, int steps) const {
    const int off = x - start, rest = cost - off;
    if (off <= 0) return 0;
    if (rest <= 0) return steps;
    if (std::min(off, rest) < near) return off <= rest ? 0 : steps;
    return std::min(steps, static_cast<int>(static_cast<float>(off) * __builtin_amdgcn_rcpf(static_cast<float>(cost)) * static_cast<float>(steps) + 0.01f));
  }
  __device__ __forceinline__ int from(int i) const { return static_cast<int>(std::min<long long>(total, static_cast<long long>(i - whole) * share)); }
};

// What the workgroup shares.  The item and its place are kept here, not in registers,
// while its keys are worked through.
struct Shared {
  float m[kMostWaves][kWaveRows];
  float l[kMostWaves][kWaveRows];
  Place at;
  Item item;
  int count;
  uint32_t last;
};

// The thread's number, anew to the compiler: what goes by it is worked out where
// it is needed, and not kept in registers from item to item or past the keys.
__device__ __forceinline__ int thread_number() {
  int t = static_cast<int>(threadIdx.x);
  asm volatile("" : "+v"(t));
  return t;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Item item_of(const Shared& sh) {
  const Item& i = sh.item;
  return Item{uniform(i.seq), uniform(i.head), uniform(i.tile), Shape{uniform(i.s.q0), uniform(i.s.n_q), uniform(i.s.n_k)},
              uniform(i.row0), uniform(i.rows), uniform(i.low), uniform(i.end), uniform(i.base), uniform(i.sink_steps), uniform(i.steps),
              uniform(i.from), uniform(i.to)};
}

template <bool kTile, int kWaves>
__device__ __forceinline__ void range_of(const PagedArgs& p, Item& it) {
  constexpr int kKeys = kStep<kTile, kWaves>;
  const int all = it.s.n_q * p.group;
  it.row0 = it.tile * kTileRows<kTile>;
  it.rows = std::min(kTileRows<kTile>, all - it.row0);
  const int lag = it.s.n_k - it.s.n_q;
  const int t0 = over(it.row0, p.by_group), t1 = over(it.row0 + it.rows - 1, p.by_group);
  it.end = std::clamp(t1 + lag + 1, 0, it.s.n_k);
  it.low = std::min(window_start(t0 + lag, p.window), it.end);
  it.base = it.low / kKeys * kKeys;
  const int sinks = std::min(p.sinks, it.end);
  it.sink_steps = std::min((sinks + kKeys - 1) / kKeys, it.base / kKeys);
  it.steps = std::max(1, it.sink_steps + (it.end - it.base + kKeys - 1) / kKeys);
}

// ---------------------------------------------------------- keys and values --

// A granule's place as the list holds it: the first three words of a buffer's
// description, its address and how many bytes of it there are (none: what is loaded is zero).
__device__ __forceinline__ u32x4 place_of(const void* at, int bytes) {
  const unsigned long long a = reinterpret_cast<unsigned long long>(at);
  return u32x4{static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(bytes), 0u};
}
// The buffer at a place that is the same in every lane.  (Its flags are a new number
// to the compiler each time: it would else keep the whole description from load to load, in
// lanes of vector registers.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const u32x4& place) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(place[0]), hi = __builtin_amdgcn_readfirstlane(place[1]);
  int flags = 0x00020000;
  asm volatile("" : "+s"(flags));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((static_cast<unsigned long long>(hi) << 32) | lo), 0,
                                           __builtin_amdgcn_readfirstlane(place[2]), flags);
}
// Bytes of `rows` rows, a granule's at most, the last one of `row_bytes`.
__device__ __forceinline__ int bytes_of(int rows, int stride, int row_bytes) {
  return rows <= 0 ? 0 : (std::min(rows, kGranule) - 1) * stride + row_bytes;
}

// Loads of one granule of keys or values.  16 bits: load i fills rows i *
// kRowsPerLoad on straight in LDS.  8 bits: rows to registers, 16 elements a
// lane, and from there, in the queries' type, to LDS.  Offsets from the
// granule's first row are the same for every granule; rows past the last key and columns past
// the head lie outside its bytes and are zero.
template <typename T, int DP, bool kValues, bool kSmall>
struct Granule {
  using H = Head<DP>;
  static constexpr int kLanes = kSmall ? (DP <= 64 ? 4 : 8) : H::kChunks;  // of a row
  static constexpr int kRowsPerLoad = 64 / kLanes;
  static constexpr int kLoads = kGranule / kRowsPerLoad;
  struct Held {
    u32x4 q[kLoads];
    uint32_t code[kLoads];
  };
  int off[kLoads];
  int scale_stride, lane;

  static __device__ __forceinline__ int swizzle(int r) { return kValues ? H::value_swizzle(r) : H::key_swizzle(r); }

  __device__ __forceinline__ Granule(int stride, int scale_stride_, int dim, int lane_) : scale_stride(scale_stride_), lane(lane_) {
    const int row_bytes = kSmall ? dim : 2 * dim;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kRowsPerLoad + lane / kLanes;
      const int c = kSmall ? lane % kLanes : (lane % kLanes) ^ swizzle(r);
      off[i] = c * 16 < row_bytes ? r * stride + c * 16 : kOutside;
    }
  }
  __device__ __forceinline__ void stage(const u32x4& place, char* dst) const {
    const __amdgpu_buffer_rsrc_t b = buffer_at(place);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void*)(dst + i * 1024), 16, off[i], 0, 0, 0);
  }

  __device__ __forceinline__ void fetch(const u32x4& place, const u32x4& scales, Held& h) const {
    const __amdgpu_buffer_rsrc_t r = buffer_at(place), s = buffer_at(scales);
    const int row = lane / kLanes;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      h.q[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off[i], 0, 0));
      h.code[i] = __builtin_amdgcn_raw_buffer_load_b8(s, (i * kRowsPerLoad + row) * scale_stride, 0, 0);
    }
  }

  static __device__ __forceinline__ uint32_t two(uint32_t q, float scale, std::integral_constant<bool, false>) {
    if constexpr (__is_same(T, __bf16))
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, scale, false));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q, scale, false));
  }
  static __device__ __forceinline__ uint32_t two(uint32_t q, float scale, std::integral_constant<bool, true>) {
    if constexpr (__is_same(T, __bf16))
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, scale, true));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q, scale, true));
  }
  __device__ __forceinline__ void put(const Held& h, char* dst) const {
    constexpr std::integral_constant<bool, false> low{};
    constexpr std::integral_constant<bool, true> high{};
    const int c = lane % kLanes * 2;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kRowsPerLoad + lane / kLanes;
      const float s = __builtin_bit_cast(float, h.code[i] << 23);
      char* row = dst + r * H::kRow;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t a = h.q[i][2 * e], b = h.q[i][2 * e + 1];
        *reinterpret_cast<u32x4*>(row + (((c + e) ^ swizzle(r)) << 4)) = u32x4{two(a, s, low), two(a, s, high), two(b, s, low), two(b, s, high)};
      }
    }
  }
};

// The places of a granule's keys, values and their scales.
struct Listed {
  u32x4 k, v;
};

// A workgroup's keys and values, by the list.
template <typename T, int DP, bool kSmall>
struct Source {
  using K = Granule<T, DP, false, kSmall>;
  using V = Granule<T, DP, true, kSmall>;
  const Listed* list;
  const Listed* scales;
  K keys;
  V values;

  __device__ __forceinline__ Source(const PagedArgs& p, const Listed* list_, const Listed* scales_, int lane)
      : list(list_), scales(scales_), keys(p.k_tok, p.ks_tok, p.dim, lane), values(p.v_tok, p.vs_tok, p.dim, lane) {}

  // Of granule `at` of the list; past its end (there: it is not) nothing is loaded.
  __device__ __forceinline__ void stage_k(int at, bool there, char* to) const { keys.stage(there ? list[at].k : u32x4{0u, 0u, 0u, 0u}, to); }
  __device__ __forceinline__ void stage_v(int at, bool there, char* to) const { values.stage(there ? list[at].v : u32x4{0u, 0u, 0u, 0u}, to); }
  __device__ __forceinline__ void fetch_k(int at, bool there, typename K::Held& h) const {
    keys.fetch(there ? list[at].k : u32x4{0u, 0u, 0u, 0u}, there ? scales[at].k : u32x4{0u, 0u, 0u, 0u}, h);
  }
  __device__ __forceinline__ void fetch_v(int at, bool there, typename V::Held& h) const {
    values.fetch(there ? list[at].v : u32x4{0u, 0u, 0u, 0u}, there ? scales[at].v : u32x4{0u, 0u, 0u, 0u}, h);
  }
};

// Rows of the granule at `key` up to the item's last key, 0 or less past it and
// where no row of the item sees any: steps begin before a window and end past the first
// keys, and pages out of sight need not be there any more.
__device__ __forceinline__ int rows_at(const PagedArgs& p, const Item& it, int key) {
  return key + kGranule > it.low || key < p.sinks ? it.end - key : 0;
}
// The page of the granule at `key` (0 where it has no rows).
__device__ __forceinline__ int page_of(const PagedArgs& p, const Item& it, int key) {
  return rows_at(p, it, key) > 0 ? p.table[static_cast<int64_t>(it.seq) * p.table_row + (key >> p.page_shift)] : 0;
}
// Lists the granule at `key`, in `page`: its rows, and nothing of a page outside
// the cache (which is flagged).
template <bool kSmall>
__device__ __forceinline__ void list_granule(const PagedArgs& p, const Item& it, int key, int page, Listed& list, Listed& scales) {
  const int row_bytes = kSmall ? p.dim : 2 * p.dim;
  int rows = rows_at(p, it, key);
  if (page < 0 || page >= p.n_pages) {
    if (rows > 0) flag_error(p.header, kErrIdRange);
    rows = 0;
    page = 0;
  }
  const int64_t i = page, j = key & ((1 << p.page_shift) - 1);
  list = Listed{place_of(p.k + it.head * p.k_head + i * p.k_page + j * p.k_tok, bytes_of(rows, p.k_tok, row_bytes)),
                place_of(p.v + it.head * p.v_head + i * p.v_page + j * p.v_tok, bytes_of(rows, p.v_tok, row_bytes))};
  if (kSmall)
    scales = Listed{place_of(p.k_scales + it.head * p.ks_head + i * p.ks_page + j * p.ks_tok, bytes_of(rows, p.ks_tok, 1)),
                    place_of(p.v_scales + it.head * p.vs_head + i * p.vs_page + j * p.vs_tok, bytes_of(rows, p.vs_tok, 1))};
}
// Lists the item's steps [from, to).
template <bool kTile, bool kSmall, int kWaves>
__device__ __forceinline__ void list_pages(const PagedArgs& p, const Item& it, int from, int to, int tid, Listed* list, Listed* scales) {
  constexpr int kKeys = kStep<kTile, kWaves>, kEach = kKeys / kGranule;
  const int n = (to - from) * kEach;
  for (int g = tid; g < n; g += 64 * kWaves) {
    const int key = it.key_of<kKeys>(from + g / kEach) + g % kEach * kGranule;
    list_granule<kSmall>(p, it, key, page_of(p, it, key), list[g], scales[kSmall ? g : 0]);
  }
}

// Scores of keys [at, at + 32) that the lane's query does not see become -inf.
template <typename T, int DP, LaneKind kKind>
__device__ __forceinline__ void mask_seen(const Rows<T, DP, kKind>& w, f32x16& s, int at, int sinks) {
  const int first = at + (w.lane() >> 5) * 4;
  const int up = w.pos - first, down = w.low - first, kept = sinks - first;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int key = (e >> 2) * 8 + (e & 3);
    s[e] = key <= up && (key >= down || key < kept) ? s[e] : -INFINITY;
  }
}

// What all rows of a wave see: every key of [low, pos], and of the first `sinks` up to pos.
struct Sight {
  int low, pos, sinks;
  __device__ __forceinline__ bool whole(int at, int n) const { return at + n - 1 <= pos && (at >= low || at + n <= sinks); }
};

// --------------------------------------------------------------------- roles --

// Key chunks: this wave's 32 keys of each of the item's steps [from, to), whose
// pages are listed.
template <typename T, int DP, bool kSmall, int kWaves, bool kCareful>
__device__ __forceinline__ void run_chunk(const Source<T, DP, kSmall>& in, const Item& it, Rows<T, DP, kLane<kSmall>>& w, float c,
                                          const Sight& see, int from, int to, int wave, char* sk, char* sv) {
  using Src = Source<T, DP, kSmall>;
  constexpr int kRow = Head<DP>::kRow, kKeys = kStep<false, kWaves>, kEach = kKeys / kGranule;
  auto key_of = [&](int i) { return it.key_of<kKeys>(i) + wave * kChunkKeys; };
  auto place = [&](int i) { return (i - from) * kEach + wave * 2; };
  auto weigh_in = [&](f32x16& s, int at, typename VecOf<T>::v8 (&e)[2]) {
    if (!see.whole(at, kChunkKeys)) mask_seen(w, s, at, see.sinks);
    w.raise(top_of(s), c);
    weigh(w, s, c, e);
  };
  auto add = [&](int at, const typename VecOf<T>::v8 (&e)[2]) {
    accumulate<T, DP, kCareful>(w, sv, 0, e);
    if (kCareful)
      add_nonfinite(w, sv, kChunkKeys, [&](int r) { return at + r <= w.pos && (at + r >= w.low || at + r < see.sinks); });
  };
  if constexpr (kSmall) {
    typename Src::K::Held hk[2];
    typename Src::V::Held hv[2];
    auto fetch_k = [&](int i) {
#pragma unroll
      for (int g = 0; g < 2; ++g) in.fetch_k(place(i) + g, i < to, hk[g]);
    };
    auto fetch_v = [&](int i) {
#pragma unroll
      for (int g = 0; g < 2; ++g) in.fetch_v(place(i) + g, i < to, hv[g]);
    };
    fetch_k(from);
    fetch_v(from);
    for (int i = from; i < to; ++i) {
      const int at = key_of(i);
#pragma unroll
      for (int g = 0; g < 2; ++g) in.keys.put(hk[g], sk + g * kGranule * kRow);
      fetch_k(i + 1);
      f32x16 s = scores(w, sk, 0);
      typename VecOf<T>::v8 e[2];
      weigh_in(s, at, e);
#pragma unroll
      for (int g = 0; g < 2; ++g) in.values.put(hv[g], sv + g * kGranule * kRow);
      fetch_v(i + 1);
      add(at, e);
    }
  } else {
    // K and V take turns in flight: while one is read the other's next keys are
    // coming, so each wait leaves the younger one's loads (a load of no rows
    // touches no memory and leaves zeros).
    constexpr int kLoads = 2 * Src::K::kLoads;
    auto load_k = [&](int i) {
#pragma unroll
      for (int g = 0; g < 2; ++g) in.stage_k(place(i) + g, i < to, sk + g * kGranule * kRow);
    };
    auto load_v = [&](int i) {
#pragma unroll
      for (int g = 0; g < 2; ++g) in.stage_v(place(i) + g, i < to, sv + g * kGranule * kRow);
    };
    load_k(from);
    load_v(from);
    for (int i = from; i < to; ++i) {
      const int at = key_of(i);
      wait_vm_but<kLoads>();
      f32x16 s = scores(w, sk, 0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      load_k(i + 1);
      typename VecOf<T>::v8 e[2];
      weigh_in(s, at, e);
      wait_vm_but<kLoads>();
      add(at, e);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      load_v(i + 1);
    }
    wait_vm();
  }
}

// Row tile: the item's steps [from, to), whose pages are listed, for the
// workgroup's rows.  While step i is weighed and added, the scores of step i + 1
// are computed, and steps i + 2 of K and i + 1 of V are on their way; each wave
// brings in a granule of either.
template <typename T, int DP, bool kSmall>
__device__ __forceinline__ void run_tile(const PagedArgs& p, const Source<T, DP, kSmall>& in, const Item& it, Rows<T, DP, kLane<kSmall>>& w,
                                         float c, const Sight& see, int wave, Listed* list, Listed* scales, WP_STAGED) {
  using Src = Source<T, DP, kSmall>;
  constexpr int kKeys = kStep<true, kTileWaves>, kEach = kKeys / kGranule;
  constexpr int kRing = kListed<kSmall, kTileWaves>, kHalf = kSteps<true, kSmall, kTileWaves> / 2;
  static_assert((kRing & (kRing - 1)) == 0 && kHalf >= 8 && kHalf * kEach <= 64 * kTileWaves, "half of the list is written in one go, well ahead");
  const int from = it.from, to = it.to;
  const int mine = wave * kGranule * Head<DP>::kRow;
  auto key_of = [&](int i) { return it.key_of<kKeys>(i); };
  auto place = [&](int i) { return ((i - from) * kEach & (kRing - 1)) + wave; };
  // The list is a ring: where a half of it has been worked through, the steps after the other
  // half are listed in its place, their pages read in one step and listed in the next.
  int page = 0;
  auto refill = [&](int i) {
    const int done = (i - from) & (kHalf - 1);
    if (i - from < kHalf || done > 1) return;
    // (No further than the last step: near 2^31 keys the ones past it have no number.)
    const int tid = thread_number(), first = i - done + kHalf;  // the first step to list
    if (tid >= std::min(kHalf, to - first) * kEach) return;
    const int key = it.key_of<kKeys>(first + tid / kEach) + tid % kEach * kGranule;
    if (done == 0) {
      page = page_of(p, it, key);
    } else {
      const int at = ((first - from) * kEach & (kRing - 1)) + tid;
      list_granule<kSmall>(p, it, key, page, list[at], scales[kSmall ? at : 0]);
    }
  };
  typename Src::K::Held hk;
  typename Src::V::Held hv;
  auto fetch_k = [&](int i) { in.fetch_k(place(i), i < to, hk); };
  auto fetch_v = [&](int i) { in.fetch_v(place(i), i < to, hv); };
  // Steps are asked for in their order.
  // (16 bits: a granule's place is read a step before it is used.)
  u32x4 at_k = in.list[place(from)].k, at_v = in.list[place(from)].v;
  auto load_k = [&](int i, char* buf) {
    if constexpr (kSmall) {
      in.keys.put(hk, buf + mine);
      fetch_k(i + 1);
    } else if (i < to) {
      in.keys.stage(at_k, buf + mine);
      at_k = in.list[place(std::min(i + 1, to - 1))].k;
    }
  };
  auto load_v = [&](int i, char* buf) {
    if constexpr (kSmall) {
      in.values.put(hv, buf + mine);
      fetch_v(i + 1);
    } else if (i < to) {
      in.values.stage(at_v, buf + mine);
      at_v = in.list[place(std::min(i + 1, to - 1))].v;
    }
  };
  auto meet = [&] {
    if (!kSmall) wait_vm();
    __syncthreads();
  };
  if constexpr (kSmall) {
    fetch_k(from);
    fetch_v(from);
  }
  load_k(from, sk0);
  meet();
  load_k(from + 1, sk1);
  load_v(from, sv0);
  auto next = [&](int i, char* kfree, char* vnext) {
    meet();
    refill(i);
    load_k(i + 2, kfree);
    load_v(i + 1, vnext);
  };
  f32x16 s0 = scores(w, sk0, 0), s1 = scores(w, sk0, 32);
  float tops = fmaxf(top_of(s0), top_of(s1));
  auto step = [&](int i, char* kfree, const char* knext, const char* vnow, char* vnext) {
    next(i, kfree, vnext);
    const int at = key_of(i);
    if (!see.whole(at, kKeys)) {
      mask_seen(w, s0, at, see.sinks);
      mask_seen(w, s1, at + 32, see.sinks);
      tops = fmaxf(top_of(s0), top_of(s1));
    }
    // (After the last step the next one's scores are of no use, as are steps past
    // the last key that the wave's rows see: they cost less than a second copy of this, without
    // them, costs in registers.)
    tile_body(w, s0, s1, tops, c, std::integral_constant<bool, true>{}, knext, vnow);
  };
  // Of two workgroups on a compute unit the older one goes first wherever both can, and the
  // younger one ends 17% later, alone at the end (4 x 512 tokens over 10636 keys each).  So each
  // has the right of way half of the time, by the clock (us, with and without: 2048 tokens over
  // 16384 keys 503 and 507, 4 x 512 over 16384, 9577, 2048 and 14536 418 and 423, over 8192 each 279 and 281).
  const uint32_t young = blockIdx.x >= (static_cast<uint32_t>(p.n_wg) >> 1);
  for (int i = from; i < to; i += 2) {
    if ((((static_cast<uint32_t>(__builtin_readcyclecounter()) >> 13) ^ young) & 1u) != 0)
      __builtin_amdgcn_s_setprio(1);
    else
      __builtin_amdgcn_s_setprio(0);
    step(i, sk0, sk1, sv0, sv1);
    if (i + 1 < to) step(i + 1, sk1, sk0, sv1, sv0);
  }
  __builtin_amdgcn_s_setprio(0);
}

// run_tile, one step after the other, with infinite and NaN values left out of
// the product and added to the rows that see them: the same sums otherwise.
template <typename T, int DP, bool kSmall>
__device__ __forceinline__ void run_tile_careful(const Source<T, DP, kSmall>& in, const Item& it, Rows<T, DP, kLane<kSmall>>& w, float c,
                                                 const Sight& see, int from, int to, int wave, char* sk, char* sv) {
  using Src = Source<T, DP, kSmall>;
  constexpr int kKeys = kStep<true, kTileWaves>, kEach = kKeys / kGranule;
  const int mine = wave * kGranule * Head<DP>::kRow;
  for (int i = from; i < to; ++i) {
    const int at = it.key_of<kKeys>(i), place = (i - from) * kEach + wave;
    __syncthreads();
    if constexpr (kSmall) {
      typename Src::K::Held hk;
      typename Src::V::Held hv;
      in.fetch_k(place, true, hk);
      in.fetch_v(place, true, hv);
      in.keys.put(hk, sk + mine);
      in.values.put(hv, sv + mine);
    } else {
      in.stage_k(place, true, sk + mine);
      in.stage_v(place, true, sv + mine);
      wait_vm();
    }
    __syncthreads();
    f32x16 s0 = scores(w, sk, 0), s1 = scores(w, sk, 32);
    if (!see.whole(at, kKeys)) {
      mask_seen(w, s0, at, see.sinks);
      mask_seen(w, s1, at + 32, see.sinks);
    }
    w.raise(fmaxf(top_of(s0), top_of(s1)), c);
    typename VecOf<T>::v8 e0[2], e1[2];
    weigh(w, s0, c, e0);
    weigh(w, s1, c, e1);
    accumulate<T, DP, true>(w, sv, 0, e0);
    accumulate<T, DP, true>(w, sv, 32, e1);
    add_nonfinite(w, sv, kKeys, [&](int r) { return at + r <= w.pos && (at + r >= w.low || at + r < see.sinks); });
  }
}

// Writes four columns of a finished row (and with the first of them its lse).
template <typename T>
__device__ __forceinline__ void finish_row(const PagedArgs& p, const Item& it, int row, int d, f32x4 v, float m, float l) {
  const int tok = over(row, p.by_group), h = it.head * p.group + row - tok * p.group;
  const bool sees = tok + it.s.n_k - it.s.n_q >= 0;
  const int64_t at = static_cast<int64_t>(it.s.q0) + tok;
  if (d < p.dim)
    store4(static_cast<T*>(p.out) + at * p.o_tok + h * p.o_head + d, sees ? v * (1.f / l) : f32x4{0.f, 0.f, 0.f, 0.f});
  if (p.lse && d == 0) p.lse[at * p.heads + h] = sees ? fmaf(m, kLn2, logf(l)) : -INFINITY;
}

// The workgroup's steps of one item.
template <typename T, int DP, bool kSmall, int kWaves, bool kTile, int kSlotRows>
__device__ __forceinline__ void run_item(const PagedArgs& p, Shared& sh, Listed* list, Listed* scales, WP_STAGED) {
  using H = Head<DP>;
  constexpr int kBatch = kSteps<kTile, kSmall, kWaves>, kThreads = 64 * kWaves;
  int tid = thread_number(), lane = tid & 63, half = lane >> 5;
  const int wave = uniform(tid >> 6);
  Item it = item_of(sh);
  const int group = p.group, lag = it.s.n_k - it.s.n_q;
  int row, tok, sub;
  bool real;
  const int wave_row0 = it.row0 + (kTile ? wave * kWaveRows : 0);
  auto find_row = [&] {
    row = it.row0 + (kTile ? wave * kWaveRows : 0) + (lane & 31);
    real = row < it.row0 + it.rows;
    tok = real ? over(row, p.by_group) : 0;
    sub = real ? row - tok * group : 0;
  };
  find_row();
  const float c = p.scale == 0.f ? 1.f : fabsf(p.scale) * kLog2e;
  Rows<T, DP, kLane<kSmall>> w;
  w.template hold<DP>(lane);
  {
    const T* q = static_cast<const T*>(p.q) + (static_cast<int64_t>(it.s.q0) + tok) * p.q_tok + (it.head * group + sub) * p.q_head;
#pragma unroll
    for (int x = 0; x < H::kSteps; ++x) {
      const int d = x * 16 + half * 8;
      w.q[x] = real && d < p.dim && p.scale != 0.f ? load8(q + d) : zero8<T>();
    }
  }
  if (p.scale < 0.f) {
#pragma unroll
    for (int x = 0; x < H::kSteps; ++x) w.q[x] = negate8<T>(w.q[x]);
  }
  w.pos = real ? tok + lag : -1;
  w.low = window_start(tok + lag, p.window);
  Sight see{0, -1, p.sinks};
  if (wave_row0 < it.row0 + it.rows) {
    const int t0 = over(wave_row0, p.by_group), t1 = std::min(it.s.n_q - 1, over(wave_row0 + kWaveRows - 1, p.by_group));
    see.pos = t0 + lag;
    see.low = window_start(t1 + lag, p.window);
  }
  const Source<T, DP, kSmall> in(p, list, scales, lane);
  // Key chunks: a wave's keys and values, and later its share of O.
  constexpr int kHalf = Staged<DP>::kBytes / 2;
  char* my_k = (kWaves == 2 || wave < 2 ? sk0 : sk1) + (wave & 1) * kHalf;
  char* my_v = (kWaves == 2 || wave < 2 ? sv0 : sv1) + (wave & 1) * kHalf;
  // (The first steps are listed.)
  auto pass = [&](auto careful) {
    w.reset();
    for (int i = it.from; i < it.to; i += kBatch) {
      const int to = std::min(it.to, i + kBatch);
      if (i > it.from || decltype(careful)::value) {
        __syncthreads();  // the last batch's places and tiles have been read
        list_pages<kTile, kSmall, kWaves>(p, item_of(sh), i, to, thread_number(), list, scales);
        __syncthreads();
      }
      if constexpr (!kTile)
        run_chunk<T, DP, kSmall, kWaves, decltype(careful)::value>(in, it, w, c, see, i, to, wave, my_k, my_v);
      else
        run_tile_careful(in, it, w, c, see, i, to, wave, sk0, sv0);
    }
  };
  if constexpr (kTile) {
    w.reset();
    run_tile(p, in, it, w, c, see, wave, list, scales, sk0, sk1, sv0, sv1);
  } else {
    pass(std::integral_constant<bool, false>{});
  }
  // Infinite or NaN values reach every row of a tile through the product, as
  // zero times them: where there are any, the pass is made again with care.
  if (__syncthreads_or(has_nonfinite(w))) pass(std::integral_constant<bool, true>{});
  w.l += __shfl_xor(w.l, 32);

  it = item_of(sh);
  tid = thread_number();
  lane = tid & 63;
  half = lane >> 5;
  find_row();
  const bool split = it.from > 0 || it.to < it.steps;
  constexpr uint32_t kSlot = kSlotRows * (DP + 2);  // floats: [rows][DP] of O, then [rows][bound, sum]
  float* part = p.part + static_cast<uint64_t>(uniform(sh.at.slot(sh.at.id, it.from == sh.at.skipped()))) * kSlot;
  const __amdgpu_buffer_rsrc_t mine = coherent_buffer(part, kSlot * 4u);
  if constexpr (kTile) {
    if (!split) {
      if (!real) return;
      const bool sees = tok + it.s.n_k - it.s.n_q >= 0;
      const float inv = 1.f / w.l;
      const int64_t at = static_cast<int64_t>(it.s.q0) + tok;
      T* out = static_cast<T*>(p.out) + at * p.o_tok + (it.head * group + sub) * p.o_head;
#pragma unroll
      for (int i = 0; i < H::kCols; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = i * 32 + e * 8 + half * 4;
          if (d >= p.dim) continue;
          const f32x4 v{w.o[i][e * 4], w.o[i][e * 4 + 1], w.o[i][e * 4 + 2], w.o[i][e * 4 + 3]};
          store4(out + d, sees ? v * inv : f32x4{0.f, 0.f, 0.f, 0.f});
        }
      if (p.lse && half == 0) p.lse[at * p.heads + it.head * group + sub] = sees ? fmaf(w.m, kLn2, logf(w.l)) : -INFINITY;
      return;
    }
    const int r = wave * kWaveRows + (lane & 31);
    if (real) {
      if (half == 0) coherent_store8(part + kSlotRows * DP + 2 * r, __builtin_bit_cast(unsigned long long, f32x2{w.m, w.l}));
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
#pragma unroll
    for (int i = 0; i < kWaves; ++i) m = fmaxf(m, sh.m[i][lane & 31]);
    const float fade = m == -INFINITY ? 1.f : exp2_fast(w.m - m);
    // (Columns swizzled by the row: whole rows apart, lanes would share banks.)
    auto place = [](int r, int d) { return (r * (DP / 4) + ((d / 4) ^ (r & (DP == 96 ? 7 : 15)))) * 16; };
    auto area = [&](int i) -> char* { return i == 0 ? sk0 : i == 1 ? (kWaves == 2 ? sv0 : sk1) : i == 2 ? sv0 : sv1; };
    char* o32 = area(wave);
    if (real)
#pragma unroll
      for (int i = 0; i < H::kCols; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<f32x4*>(o32 + place(lane & 31, i * 32 + e * 8 + half * 4)) =
              f32x4{w.o[i][e * 4], w.o[i][e * 4 + 1], w.o[i][e * 4 + 2], w.o[i][e * 4 + 3]} * fade;
    __syncthreads();
    for (int u = tid; u < it.rows * (DP / 4); u += kThreads) {
      const int r = u / (DP / 4), d = u % (DP / 4) * 4;
      f32x4 v{0.f, 0.f, 0.f, 0.f};
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        v += *reinterpret_cast<const f32x4*>(area(i) + place(r, d));
        top = fmaxf(top, sh.m[i][r]);
      }
#pragma unroll
      for (int i = 0; i < kWaves; ++i) l += sh.l[i][r] * (top == -INFINITY ? 1.f : exp2_fast(sh.m[i][r] - top));
      if (!split) {
        finish_row<T>(p, it, it.row0 + r, d, v, top, l);
      } else {
        if (d == 0) coherent_store8(part + kSlotRows * DP + 2 * r, __builtin_bit_cast(unsigned long long, f32x2{top, l}));
        coherent_store16(mine, (r * DP + d) * 4u, v);
      }
    }
    if (!split) return;
  }

  // The workgroup that does an item's last step joins its shares.  An item that
  // several share begins in one that no other shared item begins in: its counter's place.
  const Place at = sh.at;
  const int first = uniform(at.whole + at.start / at.share), final = uniform(at.whole + (at.start + at.cost - 1) / at.share);
  const int counter = uniform(at.stretches > 0 ? at.one : first);
  wait_vm();
  __syncthreads();
  if (tid == 0) {
    const unsigned mine = static_cast<unsigned>(it.to - it.from);
    const bool last = atomic_add_u(p.counters + counter, mine) + mine == static_cast<unsigned>(it.steps);
    if (last) atomic_store_u(p.counters + counter, 0u);
    sh.last = last ? 1u : 0u;
  }
  __syncthreads();
  if (sh.last == 0u) return;
  // Where the shares are (a workgroup may have none).
  int* slots = reinterpret_cast<int*>(sk0);
  static_assert(Staged<DP>::kBytes >= kMostWorkgroups * sizeof(int), "there is room for a slot of each workgroup");
  if (wave == 0) {
    int n = uniform(at.stretches);
    const int left = it.steps - uniform(at.skipped());
    for (int i = lane; i < n; i += 64) slots[i] = at.slot(at.one + i * at.tiles, false);
    for (int i = first; i <= final; i += 64) {
      const int id = i + lane;
      int from = 0, to = 0;
      if (id <= final) {
        from = at.cut(std::max(at.from(id), at.start), left);
        to = at.cut(std::min(at.from(id + 1), at.start + at.cost), left);
      }
      const unsigned long long some = __ballot(to > from);
      if (to > from) slots[n + __builtin_popcountll(some & ((1ull << lane) - 1))] = at.slot(id, from == 0);
      n += __builtin_popcountll(some);
    }
    if (lane == 0) sh.count = n;
  }
  __syncthreads();
  // Several loads at once: of one place in many shares (few rows), or of
  // several places in a few (a tile's).
  const int count = sh.count, places = it.rows * (DP / 4);
  const __amdgpu_buffer_rsrc_t shares = coherent_buffer(p.part, static_cast<uint32_t>(p.n_wg) * 2u * (kSlot * 4u));
  auto join = [&](auto n_places, auto n_shares) {
    constexpr int kPlaces = decltype(n_places)::value, kShares = decltype(n_shares)::value;
    for (int u0 = tid; u0 < places; u0 += kThreads * kPlaces) {
      float top[kPlaces], l[kPlaces];
      f32x4 v[kPlaces];
  #pragma unroll
      for (int x = 0; x < kPlaces; ++x) {
        top[x] = -INFINITY;
        l[x] = 0.f;
        v[x] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      for (int i0 = 0; i0 < count; i0 += kShares) {
        f32x2 ml[kShares][kPlaces];
        f32x4 o[kShares][kPlaces];
  #pragma unroll
        for (int i = 0; i < kShares; ++i) {
          const uint32_t share = static_cast<uint32_t>(slots[std::min(i0 + i, count - 1)]) * (kSlot * 4u);
  #pragma unroll
          for (int x = 0; x < kPlaces; ++x) {
            const int u = std::min(u0 + x * kThreads, places - 1), r = u / (DP / 4), d = u % (DP / 4) * 4;
            ml[i][x] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(shares, share + (kSlotRows * DP + 2 * r) * 4u, 0, kSc1));
            o[i][x] = coherent_load16(shares, share + (r * DP + d) * 4u);
          }
        }
  #pragma unroll
        for (int i = 0; i < kShares; ++i) {
          const bool there = i0 + i < count;
  #pragma unroll
          for (int x = 0; x < kPlaces; ++x) {
            const float m = there ? fmaxf(top[x], ml[i][x][0]) : top[x];
            const float old = m == -INFINITY ? 1.f : exp2_fast(top[x] - m), now = m == -INFINITY ? 1.f : exp2_fast(ml[i][x][0] - m);
            v[x] = there ? v[x] * old + o[i][x] * now : v[x];
            l[x] = there ? l[x] * old + ml[i][x][1] * now : l[x];
            top[x] = m;
          }
        }
      }
  #pragma unroll
      for (int x = 0; x < kPlaces; ++x) {
        const int u = u0 + x * kThreads, r = u / (DP / 4), d = u % (DP / 4) * 4;
        if (u < places) finish_row<T>(p, it, it.row0 + r, d, v[x], top[x], l[x]);
      }
    }
  };
  if constexpr (kTile)
    join(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
  else if (places > kThreads)  // 48 requests of up to 5 tokens, 8 heads a key head of 64: 24 us, 28.5 by the other form
    join(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
  else
    join(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
}

// Clears the rows of no sequence: before the first bound and from the last one on.
template <typename T, int kWaves>
__device__ __forceinline__ void clear_rest(const PagedArgs& p) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int64_t head_rows = p.n_seq > 0 ? std::clamp<int64_t>(p.cu_q[0], 0, p.tokens) : p.tokens;
  const int64_t tail = p.n_seq > 0 ? std::clamp<int64_t>(p.cu_q[p.n_seq], head_rows, p.tokens) : p.tokens;
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

template <int kRoles>
constexpr int kWavesOf = (kRoles & kTiles) != 0 ? kTileWaves : kChunkWaves;

template <typename T, int DP, bool kSmall, int kRoles>
__global__ __launch_bounds__(64 * kWavesOf<kRoles>, 2) void paged_kernel(PagedArgs p) {
  constexpr int kWaves = kWavesOf<kRoles>;
  constexpr int kSlotRows = (kRoles & kTiles) != 0 ? kTileRows<true> : kTileRows<false>;
  __shared__ Shared sh;
  __shared__ Listed list[kListed<kSmall, kWaves>];
  __shared__ Listed scales[kSmall ? kListed<kSmall, kWaves> : 1];
  __shared__ __align__(1024) char sk0[Staged<DP>::kBytes];
  __shared__ __align__(1024) char sv0[Staged<DP>::kBytes];
  touch_kernel_args<static_cast<int>(sizeof(PagedArgs))>();
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;

  // Every wave by itself: a lane for each sequence, 64 at a time, and the sum of
  // their costs.
  int most_cost = 0;  // of a tile
  auto cost_at = [&](int b, Shape& s) {
    s = Shape{0, 0, 0};
    if (b >= p.n_seq) return 0;
    s = shape_of(p, b);
    const Cost c = cost_of(p, s);
    const int all = c.before(c.tiles);
    if ((kRoles & kTiles) != 0 && c.tiles > 0) most_cost = std::max(most_cost, all - c.before(c.tiles - 1));
    return all * p.kv_heads;
  };
  Shape first, other;
  int mine = cost_at(lane, first);
  int sum = mine;
  float length = static_cast<float>(mine);
  for (int b = lane + 64; b < p.n_seq; b += 64) {
    const int v = cost_at(b, other);
    sum += v;
    length += static_cast<float>(v);
  }
  clear_rest<T, kWaves>(p);
  int total = total_of(sum);
  length = wave_sum(length);
  // Bounds that fall can give sequences more rows than there are, and a line
  // past its 31 bits: such a call does nothing.
  if (__builtin_amdgcn_readlane(__builtin_bit_cast(int, length), 63) > __builtin_bit_cast(int, kLongestLine)) return;
  int share = over(total, p.by_wg) + 1, pieces = 0;
  // Many row tiles run whole, one a workgroup, in the order that the device takes
  // workgroups (the host offers that, see there), if none costs more than a share of the whole: those
  // of a key head walk its keys together, on one die.
  const bool whole_tiles = (kRoles & kTiles) != 0 && static_cast<int>(gridDim.x) > p.n_wg && longest_of(most_cost) <= share;
  if (!whole_tiles && static_cast<int>(blockIdx.x) >= p.n_wg) return;
  if (p.n_seq <= 64 && !whole_tiles) {
    // A line of pieces, one for each workgroup, where that is as short: a tile's
    // keys in equal pieces, and no workgroup with an end of one item and a start of another.
    const Cost c = cost_of(p, first);
    const int step = c.log_rows == 7 ? kStep<true, kWaves> : kStep<false, kWaves>;
    const int keys = std::max(1, p.window > 0 ? static_cast<int>(std::min<long long>(first.n_k, static_cast<long long>(p.window) + p.sinks + 128)) : first.n_k);
    const float tiles = static_cast<float>(c.tiles) * p.kv_heads, all = tiles * keys;
    auto whole = [&](float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sum(v)), 63)); };
    if (whole(tiles) <= p.n_wg) {
      // The shortest pieces of which there are no more than workgroups (whole tiles are few enough).
      float size = std::max(64.f, whole(all) / p.n_wg);
      auto pieces_of = [&](float size) {
        return std::clamp(static_cast<int>(static_cast<float>(keys) * __builtin_amdgcn_rcpf(size) + 0.99f), 1, kMostPieces);
      };
      while (whole(tiles * pieces_of(size)) > p.n_wg) size *= 1.125f;
      pieces = pieces_of(size);
      const int longest = longest_of(c.tiles > 0 ? std::max(step, (keys + pieces - 1) / pieces) : 0);
      const long long slack = (kRoles & kTiles) != 0 ? 1536 : 256;
      if (static_cast<long long>(longest) * p.group > (static_cast<long long>(share) << p.cost_shift) + slack * p.group) pieces = 0;
      else share = 1;
    }
  }
  // Tiles: neighbours on the line, which read the same keys, on one die.  Chunks
  // read keys of their own, and the dies share out all kinds of items.
  const int block = static_cast<int>(blockIdx.x), dies = (kRoles & kTiles) != 0 && p.n_wg % 8 == 0 ? 8 : 1;
  int id = block % dies * (p.n_wg / dies) + block / dies;
  if (pieces > 0) {
    Cost c = cost_of(p, first);
    c.pieces = pieces;
    mine = c.tiles * pieces * p.kv_heads;
    total = total_of(mine);
  }
  // Chunks over caches of different lengths: stretches of keys as long as a share, from
  // the first key on, go to workgroups of their own, and the line is of what is left.
  // Those on the line have more ends and starts of items to do, so a stretch is ten steps
  // longer than a share (4 x 512 tokens over 16384, 9577, 2048 and 14536 keys: 440 us
  // with all on the line, 418; 16 x 128 tokens over four of each 492 and 436, over 256 to
  // 16384 keys at random 359 and 324, 268 and 221, 291 and 250, 213 and 216).  Below shares of 64 steps there
  // is nothing in it: 168 and 175 us at 55.
  int stretch = 0, whole = 0, mine_whole = 0;
  if ((kRoles & kTiles) != 0 && pieces == 0 && !whole_tiles && p.n_seq <= 64 && p.window == 0) {
    const float steps = ldexpf(static_cast<float>(share), p.cost_shift) * __builtin_amdgcn_rcpf(static_cast<float>(p.group * kTileKeys));
    stretch = static_cast<int>(std::min(steps + 11.f, 0x1p25f));
    Cost c;
    if (steps >= 64.f && __ballot((first.n_k - first.n_q) / kTileKeys >= stretch) != 0) {
      c = cost_of(p, first, stretch);
      mine_whole = c.tiles * c.stretches * p.kv_heads;
      whole = total_of(mine_whole);
    }
    if (whole > 0 && whole < p.n_wg) {
      mine = c.before(c.tiles) * p.kv_heads;
      total = total_of(mine);
      share = total / (p.n_wg - whole) + 1;
    } else {
      stretch = whole = mine_whole = 0;
    }
  }
  const long long x0_wide = static_cast<long long>(std::max(0, id - whole)) * share;
  if (x0_wide >= total && !whole_tiles) return;
  int x0 = static_cast<int>(x0_wide), x1 = static_cast<int>(std::min<long long>(total, x0_wide + share));
  int seq = -1, head, tile, start = 0;
  int part = -1, one = 0;  // which stretch, and the workgroup of the sequence's first
  Shape s{0, 0, 0};
  if (whole_tiles) {
    const int want = over(block, p.by_heads);
    head = block - want * p.kv_heads;
    if (p.n_seq <= 64) {
      tile_by_weight(p, first, want, seq, tile);
    } else {
      int base = 0;
      for (int b0 = 0; b0 < p.n_seq && seq < 0; b0 += 64) {
        int tiles = 0;
        if (b0 + lane < p.n_seq) tiles = cost_of(p, shape_of(p, b0 + lane)).tiles;
        const int up = sum_up(tiles);
        const unsigned long long past = __ballot(base + up > want);
        if (past != 0) {
          const int at = __builtin_ctzll(past);
          seq = b0 + at;
          tile = base + __builtin_amdgcn_readlane(up, at) - 1 - want;  // a sequence's last tiles see the most keys
        }
        base += __builtin_amdgcn_readlane(up, 63);
      }
    }
    if (seq < 0) return;
    s = shape_of(p, seq);
    s = Shape{uniform(s.q0), uniform(s.n_q), uniform(s.n_k)};
    // A line of one piece, the workgroup's.
    pieces = 1;
    total = share = x1 = 1;
    x0 = id = 0;
  } else {
    // The sequence at x0 (or of the stretch), its start on the line, and from there the tile.
    const bool stretched = id < whole;
    const int up_whole = stretch > 0 ? sum_up(mine_whole) : 0;
    for (int b0 = 0; b0 < p.n_seq; b0 += 64) {
      const int v = b0 == 0 ? mine : cost_at(b0 + lane, first);
      const int up = sum_up(v);
      const unsigned long long past = __ballot(stretched ? up_whole > id : start + up > x0);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        seq = b0 + at;
        start += __builtin_amdgcn_readlane(up, at) - __builtin_amdgcn_readlane(v, at);
        pieces = __builtin_amdgcn_readlane(pieces, at);
        one = __builtin_amdgcn_readlane(up_whole, at) - __builtin_amdgcn_readlane(mine_whole, at);
        s = Shape{__builtin_amdgcn_readlane(first.q0, at), __builtin_amdgcn_readlane(first.n_q, at), __builtin_amdgcn_readlane(first.n_k, at)};
        break;
      }
      start += __builtin_amdgcn_readlane(up, 63);
    }
    if (seq < 0) return;  // (lengths that change under the call)
    Cost c = cost_of(p, s, stretch);
    c.pieces = pieces;
    const int per_head = c.before(c.tiles);
    if (stretched) {  // tiles beside one another have stretches of the same keys
      const int rest = (id - one) / c.tiles;
      tile = uniform(id - one - rest * c.tiles);
      head = uniform(rest / c.stretches);
      part = uniform(rest - head * c.stretches);
      start += head * per_head;
    } else {
      head = uniform((x0 - start) / per_head);
      start += head * per_head;
      tile = tile_at(c, x0 - start);
    }
    start = uniform(start + c.before(tile));
  }
  for (;;) {
    {
      Item it;
      it.seq = seq;
      it.head = head;
      it.tile = tile;
      it.s = s;
      Cost c = cost_of(p, s, stretch);
      c.pieces = pieces;
      const bool tiled = (kRoles & kTiles) != 0 && c.log_rows == 7;
      if (tiled) range_of<true, kWaves>(p, it); else range_of<false, kWaves>(p, it);
      Place at;
      at.start = start;
      at.cost = c.before(tile + 1) - c.before(tile);
      at.total = total;
      at.share = share;
      at.near = pieces > 0 ? 0 : std::min(share >> 3, ((tiled ? 512 : 128) * p.group) >> p.cost_shift);
      at.id = id;
      at.pieces = pieces;
      at.stretch = stretch;
      at.whole = whole;
      at.stretches = c.stretches;
      at.tiles = c.tiles;
      at.one = one + head * c.tiles * c.stretches + tile;
      if (part >= 0) {
        it.from = part * stretch;
        it.to = it.from + stretch;
      } else {
        const int skipped = uniform(at.skipped());
        it.from = skipped + uniform(at.cut(x0, it.steps - skipped));
        it.to = skipped + uniform(at.cut(std::min(x1, start + at.cost), it.steps - skipped));
      }
      __syncthreads();  // what the item before left in LDS has been read
      if (tid == 0) {
        sh.item = it;
        sh.at = at;
      }
      if (tiled)
        list_pages<true, kSmall, kWaves>(p, it, it.from, std::min(it.to, it.from + kSteps<true, kSmall, kWaves>), thread_number(), list, scales);
      else
        list_pages<false, kSmall, kWaves>(p, it, it.from, std::min(it.to, it.from + kSteps<false, kSmall, kWaves>), thread_number(), list, scales);
      __syncthreads();
    }
    if (uniform(sh.item.to) > uniform(sh.item.from)) {
      if constexpr ((kRoles & kTiles) != 0) {
        __shared__ __align__(1024) char sk1[Staged<DP>::kBytes];
        __shared__ __align__(1024) char sv1[Staged<DP>::kBytes];
        if (uniform(sh.item.s.n_q) * p.group > p.chunk_rows)
          run_item<T, DP, kSmall, kWaves, true, kSlotRows>(p, sh, list, scales, sk0, sk1, sv0, sv1);
        else
          run_item<T, DP, kSmall, kWaves, false, kSlotRows>(p, sh, list, scales, sk0, sk1, sv0, sv1);
      } else {
        run_item<T, DP, kSmall, kWaves, false, kSlotRows>(p, sh, list, scales, sk0, sk0, sv0, sv0);
      }
    }
    // The next tile, key head or sequence with rows, if it is before the share's end.
    const Place at = sh.at;
    total = uniform(at.total);
    share = uniform(at.share);
    pieces = uniform(at.pieces);
    id = uniform(at.id);
    if ((kRoles & kTiles) != 0) {
      stretch = uniform(at.stretch);
      whole = uniform(at.whole);
    }
    part = -1;  // (those of a stretch end here: they are before the line)
    x0 = at.from(id);
    x1 = at.from(id + 1);
    start = uniform(at.start + at.cost);
    if (start >= x1) return;
    const Item it = item_of(sh);
    seq = it.seq;
    head = it.head;
    tile = it.tile + 1;
    s = it.s;
    const int tiles = uniform(at.tiles), of_head = tiles * uniform(at.stretches);
    one = uniform(at.one) - head * of_head - it.tile;
    if (tile < tiles) continue;
    tile = 0;
    if (++head < p.kv_heads) continue;
    head = 0;
    one += of_head * p.kv_heads;
    do {  // (there is one, as the line goes on)
      if (++seq >= p.n_seq) return;
      s = shape_of(p, seq);
    } while (cost_of(p, s).tiles == 0);
  }
}

template <typename T, int DP, bool kSmall>
hipError_t launch(const PagedArgs& a, bool tiles, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(std::max(a.n_wg, a.whole_tiles))), block(64 * (tiles ? kTileWaves : kChunkWaves));
  if (tiles)
    hipLaunchKernelGGL((paged_kernel<T, DP, kSmall, kTiles | kChunks>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((paged_kernel<T, DP, kSmall, kChunks>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T, bool kSmall>
hipError_t launch_head(const PagedArgs& a, bool tiles, hipStream_t stream) {
  return a.dim <= 64   ? launch<T, 64, kSmall>(a, tiles, stream)
         : a.dim <= 96 ? launch<T, 96, kSmall>(a, tiles, stream)
                       : launch<T, 128, kSmall>(a, tiles, stream);
}

}  // namespace

hipError_t launch_paged_attention(int dtype_bf16, PagedArgs& a, int n_cu, hipStream_t stream) {
  a.group = a.heads / a.kv_heads;
  a.by_group = divisor_of(a.group);
  const int64_t rows = a.tokens * a.group;
  // Sequences of few rows on the whole run on key chunks, in tiles of 32 rows.
  // Few sequences of many such rows, though, in workgroups of four waves, as row tiles are: half
  // as many shares of each to join (us, in four and in two, 32 heads over 8 of 128, caches of
  // 33 to 8192 keys at random: 4 of 8 tokens 40 and 41, 16 of 6 40 and 58, 32 of 8 72 and 81; 64
  // of 8 155 and 142, 200 of 3 317 and 289, 64 of 1 140 and 122, 16 of 4 41 and 44, 4 of 4 39 and 30).
  // Many over caches of one length would gain 1 to 20% by four (64 of 8 over 500, 2048 and 8192
  // keys 35 and 44, 115 and 125, 373 and 389; 4 of 4 over 2048 30 and 37, heads of 64 18 and 32), but
  // the lengths are on the device.
  const bool few = a.dim > 64 && rows >= 24ll * a.n_seq && static_cast<int64_t>(a.n_seq) * a.kv_heads <= n_cu;
  const bool tiles = few || rows > static_cast<int64_t>(kWaveRows) * std::max(1, a.n_seq);
  a.chunk_rows = tiles ? kWaveRows : 0x7FFFFFFF;
  // As many workgroups as the device holds at a time: eight waves a compute unit.
  a.n_wg = std::min(8 / (tiles ? kTileWaves : kChunkWaves) * n_cu, kMostWorkgroups);
  a.by_wg = divisor_of(a.n_wg);
  a.by_heads = divisor_of(a.kv_heads);
  // Row tiles that may run whole: where there are some for each workgroup, and sequences
  // are not short ones, whose tiles' starts take the most of it (us, whole and in shares; 32
  // heads over 8 of 128: a prompt of 16384 tokens 2095 and 2411, 8 of 2048 372 and 433, 16
  // of 512 97 and 123, 64 of 512 384 and 357, 32 of 400 151 and 139, 64 of 100 69 and 65,
  // 256 of 60 165 and 127).
  const int64_t all_tiles = (rows / kTileRows<true> + std::max(1, a.n_seq)) * a.kv_heads;
  a.whole_tiles = tiles && rows / kTileRows<true> * a.kv_heads >= 3ll * a.n_wg && a.tokens >= 448ll * a.n_seq && grid_fits(all_tiles, 64 * kTileWaves) ? static_cast<int32_t>(all_tiles) : 0;
  const int dp = a.dim <= 64 ? 64 : a.dim <= 96 ? 96 : 128;
  const uint64_t slots = 2ull * a.n_wg * (tiles ? kTileRows<true> : kTileRows<false>) * (dp + 2) * 4;
  if (slots > a.part_bytes || a.n_wg > a.n_counters) return hipErrorInvalidValue;
  // The line of costs stays under 2^30: every tile of all rows with a sequence's
  // most keys, in units that allow it.
  const double tiles_most = static_cast<double>(rows) / (tiles ? kTileRows<true> : kTileRows<false>) + std::max(1, a.n_seq);
  const double most = a.kv_heads * tiles_most * (a.group * (static_cast<double>(a.capacity) + 512) + 256.0);
  a.cost_shift = 0;
  while (a.cost_shift < 31 && std::ldexp(most, -a.cost_shift) + a.kv_heads * tiles_most > 0x1p30) ++a.cost_shift;
  if (a.cost_shift == 31) return hipErrorInvalidValue;
  if (dtype_bf16) return a.e4m3 ? launch_head<__bf16, true>(a, tiles, stream) : launch_head<__bf16, false>(a, tiles, stream);
  return a.e4m3 ? launch_head<_Float16, true>(a, tiles, stream) : launch_head<_Float16, false>(a, tiles, stream);
}

}  // namespace wp
