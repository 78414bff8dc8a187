// wp_paged.h -- rows of heads on their way into and out of a paged cache, and
// attention over it: argument structs and launchers shared by the host engine
// and the gfx950 kernels.
//
// A cache is two arrays of pages, one of keys and one of values, of page_size
// (a power of two) tokens each, a token's row of a head contiguous; slot s is
// token s % page_size of page s / page_size.  Rows are in the tensors' type, or
// e4m3 with a byte b for each row that stands for a factor of 2^(b - 127).
#pragma once

#include "wp_model.h"

namespace wp {

constexpr int kMaxRowDim = 256;
// Tokens of a launch: a grid has fewer than 2^32 threads, and so many tokens take at
// most three waves each (one for each kind).
constexpr int64_t kMostRowTokens = 1 << 24;
constexpr int kMinPage = 16;  // a wave's 16-byte loads of one kind then touch one page each

// The rows of one kind (queries, keys or values) of a launch: heads of each
// token.  In: x by token and head, or (read) the cache.  Out: y by token and
// head, or (cached) the cache.  Strides in elements.
struct HeadPart {
  const void* x;
  const void* norm;  // [dim] in the tensors' type, or null: not normalised
  void* y;
  uint8_t* scales;   // e4m3: of the cache's rows
  int64_t x_tok, x_head;
  int64_t y_page, y_tok, y_head;  // y_page: of the cache
  int64_t s_page, s_tok, s_head;
  int32_t heads, rotate, cached;
};

struct HeadArgs {
  HeadPart part[3];
  const void* positions;  // or null: nothing rotates
  const int64_t* turns;   // [rot / 2] 2^64ths of a turn a position
  const void* slots;      // or null: nothing is cached
  uint32_t* header;       // the plan header, whose error word is flagged
  int64_t tokens, n_slots;
  int32_t positions64, slots64;  // they are int64 (else int32)
  int32_t dim, rot, interleaved, e4m3, page_shift;
  float factor, eps;
  // Filled by the launchers.
  Divisor by_units;  // units of a token
  int32_t units_tok, units[3], steps;
  int32_t all;  // a unit is all of a token's heads
  uint32_t n_units;
};
// What rotate_heads, rotate_into_cache and write_cache run.
hipError_t launch_head_rows(int dtype_bf16, HeadArgs& a, int n_cu, hipStream_t stream);
// read_cache: part[i].x, x_tok, x_head, and y_page and the scales for the
// cache's strides between pages; y by token and head.
hipError_t launch_read_rows(int dtype_bf16, HeadArgs& a, int n_cu, hipStream_t stream);

// Attention of new tokens over the cache: sequence b's queries are rows
// [cu_q[b], cu_q[b + 1]) of q, its keys the first kv_lens[b] tokens of the pages
// table[b * table_row ..]; its last query stands at its last key.  A query sees the
// keys up to its own position and, with a window, only the last `window` of
// them and the first `sinks` of all.  out and lse as packed attention's.
struct PagedArgs {
  const void* q;
  void* out;
  float* lse;  // or null
  const char* k;
  const char* v;
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  const int32_t* table;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  int64_t q_tok, q_head, o_tok, o_head;
  int64_t k_page, k_head, v_page, v_head;      // bytes
  int64_t ks_page, ks_head, vs_page, vs_head;
  int64_t tokens, table_row;
  int32_t k_tok, v_tok, ks_tok, vs_tok;        // bytes
  int32_t n_pages, page_shift, capacity;       // capacity: most keys of a sequence
  int32_t n_seq, heads, kv_heads, dim, e4m3;
  float scale;
  int32_t window, sinks;
  float* part;         // partials of sequences that several workgroups share
  uint64_t part_bytes;
  uint32_t* counters;  // zero between calls
  int32_t n_counters;
  uint32_t* header;    // the plan header, whose error word is flagged
  // Filled by launch_paged_attention.
  int32_t group;       // query heads of a key head
  Divisor by_group;
  int32_t chunk_rows;  // most rows per key head of a sequence that runs on key chunks
  int32_t n_wg;
  Divisor by_wg, by_heads;
  int32_t whole_tiles;  // a workgroup for each row tile, if they may run whole
  int32_t cost_shift;
};
hipError_t launch_paged_attention(int dtype_bf16, PagedArgs& a, int n_cu, hipStream_t stream);

}  // namespace wp
