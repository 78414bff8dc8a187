// wp_model.h -- the operators around the grouped LoRA apply (projections with
// their epilogue, packed attention, token log probabilities): argument
// structs and launchers shared by the host engine and the gfx950 kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wp {

// The engine's scratch for these operators: fp32 partials and tile counters.
constexpr uint64_t kModelPartBytes = 256ull << 20;
constexpr int kModelCounters = 65536;

// Activations of wp_linear, in the order of enum wp_activation.
enum Activation : int32_t { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

// y[t, n] = rn(act(x[t] . w[n] + bias[n]) + residual[t, n]); gated: the
// weight has 2 * n_out rows and y[t, n] = rn(act(x[t] . w[n] + bias[n]) *
// (x[t] . w[n_out + n] + bias[n_out + n]) + residual[t, n]).  Strides in
// elements.
struct ProjArgs {
  const void* x;
  const void* w;
  const void* bias;      // or null
  const void* residual;  // or null
  void* y;
  int64_t ldx, ldw, ldr, ldy;
  int64_t tokens;
  int32_t d_in, n_out;
  int32_t act, gated;
  // Filled by launch_proj.
  int32_t tiles_t, tiles_n;  // tiles over tokens and over outputs
  int32_t splits, k_range;   // K-ranges of k_range columns (a multiple of 64)
  int32_t rows_vec;          // y and residual take 8-byte accesses
  float* part;               // [tile][split] fp32 partial tiles
  uint64_t part_bytes;
  uint32_t* tile_cnt;        // one counter per tile (zero between calls)
  int32_t n_cnt;
};
hipError_t launch_proj(int dtype_bf16, ProjArgs& a, int n_cu, hipStream_t stream);

// Attention over packed sequences: sequence b's queries are rows [cu_q[b],
// cu_q[b + 1]) of q and its keys rows [cu_k[b], cu_k[b + 1]) of k and v; its
// last query stands at its last key.  Query head h reads key head
// h / (heads / kv_heads).  Causal: a query sees the keys up to its own
// position and, with a window, only the last `window` of them.  out and lse
// (natural logarithm of the sum of exp(scale * q . k), fp32 [tokens, heads])
// are 0 and -inf for a query that sees no key and for rows of no sequence.
// Strides in elements; head rows are contiguous.
constexpr int kMaxHeadDim = 128;
constexpr int64_t kMaxKeyStride = 1 << 24;  // elements between two keys: 63 of them and a row stay under 2 GiB

// Division by a number that the host knows: (n * magic) >> shift.
struct Divisor {
  uint32_t magic;
  int32_t shift;
};

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;  // or null
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
  int64_t tokens, keys;  // rows of q and of k
  int32_t n_seq, heads, kv_heads, dim;
  float scale;
  int32_t causal, window;  // window 0: none
  float* part;             // partials of split key ranges
  uint64_t part_bytes;
  uint32_t* counters;      // zero between calls
  int32_t n_counters;
  // Filled by launch_attention: work items of either role (upper bounds; the
  // workgroups past the last one leave), the keys per split as a power of
  // two, and where the second role's partials and counters start.
  int32_t group;  // query heads of a key head
  Divisor by_group, by_heads;
  int32_t tile_items, chunk_items;
  int32_t tile_shift, chunk_shift;
  int32_t chunk_rows;  // most rows per key head of a sequence that runs on key chunks
  int32_t split_rows;  // and of one whose keys are split there
  int32_t slot_rows;   // rows that a key chunk has room for among the partials
  int32_t chunk_counters;
  int32_t tile_counters, seq_counters;  // how many either role has
  uint64_t chunk_part;
};
hipError_t launch_attention(int dtype_bf16, AttnArgs& a, int n_cu, hipStream_t stream);

// Per row of the logits: log softmax at the given id, the entropy of the
// softmax, the given id's rank (1 + how many logits are greater) and the `top`
// largest logits' ids (equal ones by the lower id) and log probabilities.  A
// negative id names no token: log probability and rank 0; an id past the
// vocabulary counts as none and is flagged (kErrIdRange).  Strides in elements.
constexpr int kMaxTop = 64;
struct LogprobArgs {
  const void* logits;
  const void* ids;
  int32_t ids64;  // ids are int64 (else int32)
  int32_t dtype;  // 0 fp16, 1 bf16, 2 fp32
  int64_t rows, ld;
  int32_t vocab, top;
  float* logprobs;    // [rows]
  float* entropy;     // [rows]
  int32_t* ranks;     // [rows]
  float* top_lp;      // [rows, top]
  int32_t* top_ids;   // [rows, top]
  uint32_t* header;   // the plan header, whose error word is flagged
  char* part;         // shares of rows that several workgroups read
  uint64_t part_bytes;
  uint32_t* counters; // zero between calls
  int32_t n_counters;
  int32_t parts;      // workgroups per row; filled by launch_logprobs
};
hipError_t launch_logprobs(LogprobArgs& a, int n_cu, hipStream_t stream);

}  // namespace wp
