// A paged cache of keys and values: what the kernel that fills it (rotary_kernels.hip) and those that read it (attention_kernels.hip) share.
//
// The cache is [n_pages, page_size, heads, head_dim], keys and values alike; a sequence's key number p lies in slot p % page_size of the page
// that its row of the page table names at p / page_size.  The tokens of a call lie one sequence after the other: sequence b has those
// from starts[b] to starts[b + 1] (starts NULL: one each), and they are the last of its lengths[b] keys.  What lengths, starts and the
// table hold is known on the device alone, so every kernel bounds it there: a length by the pages of a row of the table, starts by the
// tokens, and an entry of the table that is no page of the cache is not written to and stands for keys and values of zeros.
#pragma once
#include "mx_common.hpp"

namespace sarek_hip {

// n / size for 0 <= n < 2^31 by a product: size in (2^(shift - 1), 2^shift], factor = ceil(2^(31 + shift) / size) < 2^32.
struct Division {
  uint32_t factor, size, shift;
};
inline Division division_by(uint32_t size) {
  uint32_t shift = 0;
  while ((uint64_t{1} << shift) < size) ++shift;
  return {static_cast<uint32_t>(((uint64_t{1} << (31 + shift)) + size - 1) / size), size, shift};
}

struct Batch {
  const int *pages, *lengths, *starts;
  int64_t pages_stride;
  int max_pages, batch, tokens;
  int n_pages;
  Division page_size;
};

typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(2))) unsigned int place_t;

// What one launch makes of the rows and keys.
struct Pass {
  int prefix;            // rows of all sequences against the prefix, or each sequence's against its own keys
  int rows, unit;        // of a tile; keys in what a stretch has a whole number of
  int target;            // how many workgroups the card takes at once (0: no stretches, all of a sequence's keys in one)
  int spread;            // about how many it gets where these do not come out
  int least_units;       // where stretches would have fewer, half of `target`
  int all;               // everything goes into the planes, for the join
  int max_slots;
  float *o;              // [slot][kv head][row][value]
  f32x2_t *ml;           // [slot][kv head][row]
  place_t *places;       // of each token's first row: its first slot, and the number of its stretches times 256 with its row in the tile
};

struct AttentionArgs {
  Batch batch;
  const void *q, *keys, *values;
  void *out;
  float *lse;
  int64_t q_token, q_head, out_token, out_head;
  int64_t page, slot, head, extent;         // the cache's strides and size, bytes
  int heads, kv_heads, head_dim, causal;
  Division group;
  float scale;                              // times log2(e)
  const int *prefix;
  int prefix_length;
};

// The launches of one call (attention.hip plans them).
struct Launch {
  int waves;             // of 32 rows to a tile; 0: few rows
  int64_t items;         // for each kv head, at most
  Pass pass;
};
constexpr int kTileKeys = 32, kStreamKeys = 32;               // of a tile
constexpr int stream_waves(int d) { return d <= 64 ? 4 : d <= 128 ? 2 : 1; }      // of a workgroup, by the padded head
int launch_attention_bf16(const AttentionArgs &s, const Launch &own, const Launch *before, hipStream_t st);
int launch_attention_f16(const AttentionArgs &s, const Launch &own, const Launch *before, hipStream_t st);

namespace {

__device__ __forceinline__ uint32_t divided(uint32_t n, const Division &by) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * by.factor) >> (31 + by.shift));
}

// The tokens of sequence b, first and count, within the call's.
struct Tokens {
  int first, count;
};
__device__ __forceinline__ Tokens tokens_of(const Batch &s, int b) {
  if (!s.starts) return {b, b < s.tokens ? 1 : 0};
  const int first = min(max(s.starts[b], 0), s.tokens);
  return {first, min(max(s.starts[b + 1], first), s.tokens) - first};
}
// How many of a sequence's keys its row of the page table has room for.
__device__ __forceinline__ int keys_held(const Batch &s, int length) {
  return max(min(static_cast<int64_t>(length), static_cast<int64_t>(s.max_pages) * s.page_size.size), int64_t{0});
}
// The sequence of a token that all lanes of the wave ask for; batch for tokens behind the last sequence, the first one for those before it.
__device__ __forceinline__ int sequence_of(const Batch &s, int token) {
  if (!s.starts) return min(token, s.batch);
  int ended = 0;
  for (int b = 0; b < s.batch; b += 64) {
    const int mine = b + static_cast<int>(threadIdx.x & 63);
    ended += __popcll(__ballot(mine < s.batch && s.starts[min(mine, s.batch - 1) + 1] <= token));
  }
  return ended;
}

}  // namespace

int check_cache(const char *what, const sarek_hip_kv_cache *cache);
// Checks the sequences' arguments and fills in what the kernels take.
int make_batch(const char *what, const sarek_hip_kv_cache *cache, const int *pages, int64_t pages_stride, int max_pages, const int *lengths,
               const int *starts, int batch, int64_t tokens, Batch *out);
int check_heads(const char *what, const char *name, int64_t token_stride, int64_t head_stride, int64_t tokens, int heads, int head_dim,
                bool written);

#define SAREK_ATTENTION_TRY(expr)                \
  do {                                           \
    const int st_ = (expr);                      \
    if (st_ != SAREK_HIP_OK) return st_;         \
  } while (0)

}  // namespace sarek_hip
