// Attention over a paged cache (layout: attention_common.hpp): for each token and head, softmax(scale q . keys) . values.
//
// All queries that meet the same keys go together: the rows of sequence b and key head h are its tokens times the group of q's heads that
// share h, and a workgroup takes a tile of them against a stretch of the keys, in one pass over the keys with the running maximum m and
// sum l of the softmax:
//   s = scale q . k,   m' = max(m, s),   l' = l 2^(m - m') + sum 2^(s - m'),   o' = o 2^(m - m') + sum 2^(s - m') v
// in units of log2 (scale log2(e) goes into the scores).  Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T: a lane then has
// all of its scores from one row, the maximum is one exchange between lanes, and the scores are in the lanes where the second product wants
// its weights - only the order of the keys in a product differs, and V is read in that order.
//
// Two kernels.  Few rows to a sequence (single tokens) are bound by the bytes of the cache: attention_stream_kernel, 16 rows, every wave
// with its own keys and its own transfers.  Many rows are bound by the matrix unit: attention_tile_kernel, 128 rows that share what a
// workgroup brings to LDS.  Where rows are few for the card the keys are split into stretches of about the same length, and
// attention_join_kernel joins what they leave (o, m and l in float32); the tiles and stretches are laid out by every workgroup for itself
// from the lengths (find_item), which the host does not know.
#pragma once
#include <algorithm>
#include <cmath>
#include <utility>

#include "attention_common.hpp"
#include "gemm_common.hpp"

namespace sarek_hip {
namespace {

typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4_t;

// ---- which tile and stretch ----------------------------------------------------------------------------------------------------------

// Inclusive sums over the lanes of a wave, by the row and bank shifts of the data-parallel moves (8 to 20 cycles each; an exchange
// through LDS takes about 100).
template <class V> __device__ __forceinline__ V scan_wave(V v) {
  auto add = [&](auto ctrl, auto rows) {
    const int moved = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value, 0xF, true);
    v += __builtin_bit_cast(V, moved);
  };
  add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});   // row_shr:1, 2, 4, 8
  add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});   // row_bcast:15 into rows 1 and 3
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});   // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

struct Work {
  int first, count;      // tokens
  int length, held;      // keys by lengths, and of these those that the table has room for
  int tiles, units;
};
__device__ __forceinline__ Work work_of(const AttentionArgs &s, const Pass &p, int b) {
  Work w = {0, 0, 0, 0, 0, 0};
  if (p.prefix) {
    if (b != 0) return w;
    w.count = s.batch.starts ? min(max(s.batch.starts[s.batch.batch], 0), s.batch.tokens) : s.batch.batch;
    w.length = w.held = s.prefix_length;
  } else {
    if (b >= s.batch.batch) return w;
    const Tokens t = tokens_of(s.batch, b);
    w.first = t.first, w.count = t.count;
    w.length = s.batch.lengths[b];
    w.held = keys_held(s.batch, w.length);
  }
  w.tiles = (w.count * static_cast<int>(s.group.size) + p.rows - 1) / p.rows;
  w.units = (w.held + p.unit - 1) / p.unit;
  return w;
}
__device__ __forceinline__ int sequences(const AttentionArgs &s, const Pass &p) { return p.prefix ? 1 : s.batch.batch; }
__device__ __forceinline__ int stretches(int units, int at_once) { return max((units + at_once - 1) / max(at_once, 1), 1); }

constexpr int kMostStretches = 256;      // of a sequence: as many planes a row has to be joined from

struct Item {
  int b;
  int first, count, length, held;   // the sequence's, as above
  int row0;                         // the tile's first row
  int begin, end;                   // keys
  int slot;                         // of the planes; -1: straight to out
  int stretch, cut;                 // which of how many of the tile
};
// Tile and stretch number `item`; false past the last.  Every workgroup finds its own, from the lengths of all.  The last rows of a sequence
// come first: under a causal mask they have the most keys.
__device__ __forceinline__ bool find_item(const AttentionArgs &s, const Pass &p, int item, Item &it) {
  const int n = sequences(s, p), lane = threadIdx.x & 63;
  Work w = work_of(s, p, lane);
  int at_once = 1 << 30;             // units of keys to a stretch
  if (p.target != 0) {
    // All workgroups at once, if stretches of up to a third more than their even share make that; otherwise more and shorter ones, which even out
    // as they follow one another.
    uint64_t all = static_cast<uint64_t>(w.tiles) * static_cast<uint32_t>(w.units);
    for (int b = 64 + lane; b < n; b += 64) {
      const Work more = work_of(s, p, b);
      all += static_cast<uint64_t>(more.tiles) * static_cast<uint32_t>(more.units);
    }
    const float total = __builtin_bit_cast(float, lane_of(__builtin_bit_cast(int, scan_wave(static_cast<float>(all))), 63)) * static_cast<float>(s.kv_heads);
    const int target = total < static_cast<float>(p.target) * static_cast<float>(p.least_units) ? p.target / 2 : p.target;
    const auto whole = [](float units) __attribute__((always_inline)) { return max(static_cast<int>(min(ceilf(units), 1e9f)), 1); };
    const float even = total / static_cast<float>(target);
    constexpr int kTries = 5;
    int at[kTries], made[kTries];
    float part[kTries];       // of a stretch that a unit is, a little less, so that a whole number of stretches is not rounded up
#pragma unroll
    for (int j = 0; j < kTries; ++j) at[j] = whole(even * (1.f + j / 12.f)), part[j] = __builtin_amdgcn_rcpf(static_cast<float>(at[j])) * (1.f - 1e-6f), made[j] = 0;
    for (int b = 0; b < n; b += 64) {
      const Work of = b == 0 ? w : work_of(s, p, b + lane);
#pragma unroll
      for (int j = 0; j < kTries; ++j) made[j] += of.tiles * max(static_cast<int>(ceilf(static_cast<float>(of.units) * part[j])), 1);
    }
    at_once = whole(target == p.target ? total / static_cast<float>(p.spread) : even);
#pragma unroll
    for (int j = kTries - 1; j >= 0; --j)
      if (lane_of(scan_wave(made[j]), 63) * s.kv_heads <= target) at_once = at[j];
  }
  int items = 0, slots = 0;
  for (int b0 = 0; b0 < n; b0 += 64) {
    if (b0 != 0) w = work_of(s, p, b0 + lane);
    const int cut = min(stretches(w.units, at_once), kMostStretches), mine = w.tiles * cut, kept = p.all || cut > 1 ? mine : 0;
    const int upto = scan_wave(mine), slots_upto = scan_wave(kept);
    const uint64_t past = __ballot(items + upto > item);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int tiles = lane_of(w.tiles, at), units = lane_of(w.units, at);
      it.cut = lane_of(cut, at);
      const int local = item - items - lane_of(upto - mine, at), tile = tiles - 1 - local / it.cut;
      it.b = b0 + at, it.first = lane_of(w.first, at), it.count = lane_of(w.count, at);
      it.length = lane_of(w.length, at), it.held = lane_of(w.held, at);
      it.stretch = local % it.cut;
      if (local < 0 || tile < 0) return false;
      it.row0 = tile * p.rows;
      it.slot = lane_of(kept, at) ? slots + lane_of(slots_upto - kept, at) + tile * it.cut + it.stretch : -1;
      if (it.slot >= p.max_slots) return false;
      const int keys = (units + it.cut - 1) / it.cut * p.unit;
      const int last = static_cast<int>(divided(min(it.row0 + p.rows, it.count * static_cast<int>(s.group.size)) - 1, s.group));
      const int64_t sees = s.causal && !p.prefix ? static_cast<int64_t>(it.length) - it.count + last + 1 : it.held;
      it.begin = static_cast<int>(min(static_cast<int64_t>(it.stretch) * keys, static_cast<int64_t>(it.held)));
      it.end = static_cast<int>(max(min(min(sees, static_cast<int64_t>(it.held)), static_cast<int64_t>(it.begin) + keys), static_cast<int64_t>(it.begin)));
      return true;
    }
    items += lane_of(upto, 63), slots += lane_of(slots_upto, 63);
  }
  return false;
}
// For the join: where the planes of this row's token are, by the workgroup that has its first row in its first stretch.
__device__ __forceinline__ void tell_place(const Pass &p, const Item &it, int token, int row) {
  p.places[token] = u32x2_t{static_cast<uint32_t>(it.slot), it.slot < 0 ? 0u : static_cast<uint32_t>(it.cut) << 8 | static_cast<uint32_t>(row)};
}

// ---- what both kernels share -----------------------------------------------------------------------------------------------------------

// Keys and values of a tile in LDS: rows of 2 D bytes, the 16-byte pieces of a row at places turned by the key's last bits, so that neither
// 16 keys of a column of pieces (K, ds_read_b128) nor 4 or 8 keys of a pair of them (V, ds_read_b64_tr_b16) meet in a bank.
template <int D> __device__ __forceinline__ int turn_of_key(int key) { return D >= 128 ? key & 15 : key >> 1 & 7; }
template <int D> __device__ __forceinline__ int turn_of_value(int key) {
  return D >= 128 ? (key & 3) << 2 | (key >> 2 & 1) << 1 : (key >> 1 & 1) << 2 | (key >> 2 & 1) << 1;
}

__device__ const u32x4_t zero_block = {0u, 0u, 0u, 0u};

// Where the rows of keys are.  Near: as an offset of 32 bits from the head's first, past the end (where a transfer brings zeros) for what is no
// key; far, for caches past 2^32 bytes: 64 bits, negative for what is no key.
template <bool Far> struct Rows;
template <> struct Rows<false> { typedef uint32_t At; static constexpr uint32_t kNone = 0xFFFF0000u; };
template <> struct Rows<true> { typedef int64_t At; static constexpr int64_t kNone = -1; };
constexpr int64_t kNearBytes = 0xFFFF0000;

struct Table {
  const int *pages;
  int end;               // of the stretch; at least 1
};
// The page of a key; any entry of the table for what is past the end.
__device__ __forceinline__ int page_of(const AttentionArgs &s, const Table &t, int key) {
  return t.pages[divided(static_cast<uint32_t>(min(key, t.end - 1)), s.batch.page_size)];
}
template <bool Far> __device__ __forceinline__ typename Rows<Far>::At row_of(const AttentionArgs &s, const Table &t, int key, int page) {
  const uint32_t entry = divided(static_cast<uint32_t>(key), s.batch.page_size), in = static_cast<uint32_t>(key) - entry * s.batch.page_size.size;
  if (key >= t.end || static_cast<uint32_t>(page) >= static_cast<uint32_t>(s.batch.n_pages)) return Rows<Far>::kNone;
  if constexpr (Far) return page * s.page + in * s.slot;
  else return static_cast<uint32_t>(page) * static_cast<uint32_t>(s.page) + in * static_cast<uint32_t>(s.slot);
}
// One transfer: 16 bytes of a row for each lane, zeros past head_dim.
template <bool Far>
__device__ __forceinline__ void move16(const char *base, __amdgpu_buffer_rsrc_t rsrc, typename Rows<Far>::At row, int piece, int pieces, char *to) {
  if constexpr (Far) {
    const char *from = row >= 0 && piece < pieces ? base + row + piece * 16 : reinterpret_cast<const char *>(&zero_block);
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void *>(reinterpret_cast<uintptr_t>(from)),
                                     (LDS_PTR void *)to, 16, 0, 0);
  } else {
    dma16(rsrc, piece < pieces ? row + piece * 16 : Rows<false>::kNone, 0, to);
  }
}

// pack: two values of the type, rounded; pack_below: the largest below them (0 of 0), which are not negative.
__device__ __forceinline__ uint32_t before(float v) { return __builtin_elementwise_sub_sat(__float_as_uint(v), 1u); }
template <class T> struct Products;
template <> struct Products<Bf16> {
  static __device__ __forceinline__ f32x4_t mul(u32x4 a, u32x4 b, f32x4_t c) { return mfma16<true>(a, b, c); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return f32_pair_to_bf16(lo, hi); }
  static __device__ __forceinline__ float low(uint32_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t pack_below(float lo, float hi) { return __builtin_amdgcn_perm(before(hi), before(lo), 0x07060302u); }
  static constexpr uint32_t kExponent = 0x7F80u;
  static constexpr float kRaised = 0.f;
};
template <> struct Products<_Float16> {
  static __device__ __forceinline__ f32x4_t mul(u32x4 a, u32x4 b, f32x4_t c) { return mfma16<false>(a, b, c); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return f32_pair_to_f16(lo, hi); }
  static __device__ __forceinline__ float low(uint32_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v))); }
  static __device__ __forceinline__ float high(uint32_t v) { return low(v >> 16); }
  static __device__ __forceinline__ uint32_t pack_below(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(before(lo)), __uint_as_float(before(hi))));
  }
  static constexpr uint32_t kExponent = 0x7C00u;
  static constexpr float kRaised = 7.f;
};
// What is taken from a row's scores (log2) before the exponential: its maximum, less kRaised, so that weights, their sum and the weighted values are all held
// 2^kRaised times as large.  fp16 has steps of 2^-24 below 2^-14 and nothing below 2^-25: with weights of up to 1, thousands of small ones would be lost to the
// product, though not to their sum (131071 keys 18 natural units below another one, whose value is 0: 1e-4 for 2e-3).  With kLag they stay
// below 2^15 and are off by 2^-32 of the largest at most.  bf16's exponents are float32's.
template <class T> __device__ __forceinline__ float offset_of(float m, float scale) { return __builtin_fmaf(m, scale, -Products<T>::kRaised); }

// Four consecutive keys of a column of V in each lane: lane i of 16 gives the address of 8 bytes of key i / 4, columns 4 (i % 4) on, and
// gets the keys of column i.
__device__ __forceinline__ u32x2_t read_turned(const char *lds, int offset) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_PTR bf16x4_t *)(lds + offset)));
}

// Infinities and NaNs among values that some rows of the tile see and others do not: the product would bring them into all rows, 0 times
// infinity being NaN.  In tiles that some rows see in part they are set to 0 for the product, and `any` is told; behind the
// last tile they are then added to the sums of those rows that see them (what else is in such a sum does not matter).
// largest: the bits of the type's largest number, or 7FFF where all rows see the same keys and nothing is taken out.
__device__ __forceinline__ u32x4_t cleaned(u32x4_t v, uint16_t largest, uint32_t &any) {
  typedef __attribute__((ext_vector_type(2))) short s16x2_t;
  const s16x2_t most = {static_cast<short>(largest), static_cast<short>(largest)};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const s16x2_t over = (most - __builtin_bit_cast(s16x2_t, v[j] & 0x7FFF7FFFu)) >> 15;     // all ones or nothing, in 16 bits each
    any |= __builtin_bit_cast(uint32_t, over);
    v[j] &= ~__builtin_bit_cast(uint32_t, over);
  }
  return v;
}
// Four neighbouring values of a key's row from memory, the unbounded ones added to a row's sums.
template <class T> __device__ __forceinline__ void add_unbounded(const char *from, f32x4_t &sums) {
  const u32x2_t v = *reinterpret_cast<const u32x2_t *>(from);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = v[j / 2] >> (j % 2 * 16) & 0xFFFFu;
    if ((x & Products<T>::kExponent) == Products<T>::kExponent) sums[j] += Products<T>::low(x);
  }
}

// The row of q that a lane works for.
struct Row {
  bool live;
  int token, head;       // of the call
  int limit;             // the keys it sees, at most the stretch's end
};
__device__ __forceinline__ Row row_at(const AttentionArgs &s, const Pass &p, const Item &it, int kv_head, int row) {
  Row r;
  const int group = static_cast<int>(s.group.size);
  r.live = row < it.count * group;
  const int token = static_cast<int>(divided(static_cast<uint32_t>(r.live ? row : 0), s.group));
  r.token = it.first + token;
  r.head = kv_head * group + (r.live ? row : 0) - token * group;
  const int64_t sees = s.causal && !p.prefix ? static_cast<int64_t>(it.length) - it.count + token + 1 : it.held;
  r.limit = r.live ? static_cast<int>(max(min(sees, static_cast<int64_t>(it.end)), int64_t{0})) : it.end;
  return r;
}
template <class T> __device__ __forceinline__ u32x4 load_q(const AttentionArgs &s, const Row &r, int d) {
  if (!r.live || d >= s.head_dim) return u32x4{0u, 0u, 0u, 0u};
  return *reinterpret_cast<const u32x4_any *>(static_cast<const T *>(s.q) + r.token * s.q_token + r.head * s.q_head + d);
}
// Four values of a row's result.
template <class T> __device__ __forceinline__ void store_out(const AttentionArgs &s, int token, int head, int d, f32x4_t v) {
  typedef u32x2_t u32x2_any __attribute__((aligned(2)));
  if (d < s.head_dim)
    *reinterpret_cast<u32x2_any *>(static_cast<T *>(s.out) + token * s.out_token + head * s.out_head + d) =
        u32x2_t{Products<T>::pack(v[0], v[1]), Products<T>::pack(v[2], v[3])};
}
__device__ __forceinline__ void store_lse(const AttentionArgs &s, int token, int head, float m, float l) {
  if (s.lse) s.lse[static_cast<int64_t>(token) * s.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
}
// A maximum may lag behind its row by this much (log2): weights up to 2^8 times as large lose nothing, and the sums are rescaled a few times instead of
// at every new maximum.
constexpr float kLag = 8.f;

// The planes of a row: how many, and the row's place in the first of them.
struct Planes {
  int count;
  int64_t first, step;
};
__device__ __forceinline__ Planes planes_of(const AttentionArgs &s, const Pass &p, u32x2_t place, int kv_head, int in_group) {
  const int cut = static_cast<int>(place[1] >> 8), row = static_cast<int>(place[1] & 255) + in_group, slot = static_cast<int>(place[0]) + row / p.rows * cut;
  if (cut == 0 || slot < 0 || slot > p.max_slots - cut) return {0, 0, 0};      // (no place either for a token that starts out of order have left out)
  return {cut, (static_cast<int64_t>(slot) * s.kv_heads + kv_head) * p.rows + row % p.rows, static_cast<int64_t>(s.kv_heads) * p.rows};
}

// A row's sums so far, four columns of them, and what is added to them from planes: m and l and o of kAtOnce planes are asked for together.
struct Sums {
  float top, l;
  f32x4_t o;
};
template <int D, int kAtOnce> __device__ __forceinline__ void add_planes(const Pass &p, const Planes &of, int d, Sums &a) {
  for (int j0 = 0; j0 < of.count; j0 += kAtOnce) {
    f32x2_t ml[kAtOnce];
    f32x4_t o[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t at = of.first + min(j0 + u, of.count - 1) * of.step;
      ml[u] = p.ml[at];
      o[u] = *reinterpret_cast<const f32x4_t *>(p.o + at * D + d);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) asm volatile("" : "+v"(ml[u]), "+v"(o[u]));      // (all of them on their way: not each where it is used)
    float top = a.top;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) top = fmaxf(top, ml[u][0]);
    // (nothing without a key: m is minus infinity and all else 0; so is the m of a stretch whose scores are all NaN, and its l is NaN)
    const float keep = a.top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(a.top - top);
    a.top = top;
    a.l *= keep;
    a.o *= keep;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const bool there = j0 + u < of.count;      // (past the end: the last one again)
      const float weight = ml[u][0] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[u][0] - top);
      a.l += there ? weight * ml[u][1] : 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) a.o[k] += there ? weight * o[u][k] : 0.f;
    }
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------

// A wave takes every kWaves-th tile of 32 keys of the stretch by itself: its transfers go into its own part of LDS, one tile ahead, and there
// is no barrier until the waves' sums are joined at the end.  The bytes of the cache bound it: 46 sequences of 100 to 11007 keys, 8 heads of
// 128, 1.02 GB in 190 to 194 us, 5.3 TB/s (a large copy on this card: 5.1); 131071 keys of 16 heads of 64 in 99 us, 5.4.  The matrix unit is busy for 7 % of the time.  One
// token of 4095 keys: 8.0 us for 17 MB, of which about 3 are a launch's start and the way to the first transfer (lengths, page, keys).
template <class T, int D, int Used, bool Far>
__global__ __launch_bounds__(64 * stream_waves(D)) void attention_stream_kernel(AttentionArgs s, Pass p, Pass before) {
  constexpr int kWaves = stream_waves(D), kRowBytes = 2 * D, kPieces = D / 8, kKeysMoved = 64 / kPieces, kMoves = kStreamKeys / kKeysMoved;
  constexpr int kTileBytes = kStreamKeys * kRowBytes, kStage = kWaves * 2 * kTileBytes, kSteps = Used / 32, kColumns = Used / 16, kPitch = D + 4;
  static_assert(kWaves * 16 * kPitch * 4 <= kStage && 2 * kMoves < 64, "the waves' sums go into a stage; vmcnt");
  typedef typename Rows<Far>::At At;
  typedef Products<T> P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, quad = lane >> 4;
  const int kv_head = static_cast<int>(blockIdx.x) % s.kv_heads;
  Item it;
  if (!find_item(s, p, static_cast<int>(blockIdx.x) / s.kv_heads, it)) return;
  const Table table = {p.prefix ? s.prefix : s.batch.pages + it.b * s.batch.pages_stride, it.end};
  const char *const keys = static_cast<const char *>(s.keys) + kv_head * s.head, *const values = static_cast<const char *>(s.values) + kv_head * s.head;
  const uint32_t bytes = static_cast<uint32_t>(min(s.extent - kv_head * s.head, kNearBytes));
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(keys, Far ? 0u : bytes), rv = make_rsrc(values, Far ? 0u : bytes);
  const int pieces = s.head_dim / 8, tiles = (it.end - it.begin + kStreamKeys - 1) / kStreamKeys;
  auto key_of = [&](int tile) { return it.begin + tile * kStreamKeys + (lane & 31); };
  const int mine = wave * 2 * kTileBytes;      // of a stage
  auto issue = [&](char *to, At at) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int key = i * kKeysMoved + lane / kPieces;
      const At from = __shfl(at, key, 64);
      move16<Far>(keys, rk, from, lane % kPieces ^ turn_of_key<D>(key), pieces, to + (mine + i * 1024));
      move16<Far>(values, rv, from, lane % kPieces ^ turn_of_value<D>(key), pieces, to + (mine + kTileBytes + i * 1024));
    }
  };
  // Loads come in order: the row of q before the first page, a page before the transfers that it is not for.
  const Row row = row_at(s, p, it, kv_head, it.row0 + l16);
  u32x4 q[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) q[i] = load_q<T>(s, row, i * 32 + quad * 8);
  int t = wave, page = 0;
  if (t < tiles) page = page_of(s, table, key_of(t));
#pragma unroll
  for (int i = 0; i < kSteps; ++i) asm volatile("" : "+v"(q[i]));      // (waits for them here, not in the loop, where it would wait for transfers)
  if (t < tiles) {
    const At at = row_of<Far>(s, table, key_of(t), page);
    page = page_of(s, table, key_of(t + kWaves));
    asm volatile("" ::: "memory");
    issue(lds_ring<0, kStage>, at);
  }
  int least = row.limit;
#pragma unroll
  for (int x = 1; x < 16; x *= 2) least = min(least, __shfl_xor(least, x, 64));
  least = __builtin_amdgcn_readfirstlane(least);
  f32x4_t o[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) o[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;      // of this lane's row; l of this lane's keys

  const uint16_t largest = least < it.end ? P::kExponent - 1 : 0x7FFF;
  uint32_t unbounded = 0;
  // Where this lane reads: of step i and column tile c an XOR with the piece's number.  (Opaque: sums of pointers hide from the compiler which
  // array is read, and it would wait for all transfers under way.)
  int key_at = mine + l16 * kRowBytes + (quad ^ turn_of_key<D>(l16)) * 16;
  int value_at = mine + (quad * 4 + (l16 >> 2)) * kRowBytes + turn_of_value<D>(quad * 4 + (l16 >> 2)) * 16 + (l16 & 3) * 8;
  asm volatile("" : "+v"(key_at), "+v"(value_at));

  auto tile = [&](auto masked, const char *from, int key0) __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(masked)::value;
    f32x4_t score[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      score[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        score[b] = P::mul(*reinterpret_cast<const u32x4 *>(from + ((key_at ^ i << 6) + b * 16 * kRowBytes)), q[i], score[b]);
    }
    if constexpr (kMasked) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (key0 + j / 4 * 16 + quad * 4 + j % 4 >= row.limit) score[j / 4][j % 4] = -INFINITY;
    }
    float most = score[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) most = fmaxf(most, score[j / 4][j % 4]);
    most = fmaxf(most, __shfl_xor(most, 16, 64));
    most = fmaxf(most, __shfl_xor(most, 32, 64));
    if (__any((most - m) * s.scale > kLag)) {
      const float now = fmaxf(m, most), keep = now == m ? 1.f : __builtin_amdgcn_exp2f((m - now) * s.scale);
      m = now;
      l *= keep;
#pragma unroll
      for (int c = 0; c < kColumns; ++c) o[c] *= keep;
    }
    const float offset = m == -INFINITY ? 0.f : offset_of<T>(m, s.scale);
    // The weights go into the product in two parts of the type, the second what the first leaves: the matrix unit is idle for most of the time here.  They are
    // off by 2^-15 of themselves in bf16, 2^-21 in fp16 (and 2^-32 of the largest), which out's own rounding hides.  The first is below the weight, so that
    // both are positive: an infinity among the values times 0, or times parts of both signs, is NaN.  (Rounded to nearest it is half as far off, and no faster.)
    u32x4 big, small;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j / 2][j % 2 * 2], s.scale, -offset));
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j / 2][j % 2 * 2 + 1], s.scale, -offset));
      l += x + y;
      big[j] = P::pack_below(x, y);
      small[j] = P::pack(x - P::low(big[j]), y - P::high(big[j]));
    }
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      const int at = (value_at ^ c << 5) + kTileBytes;
      const u32x2_t lo = read_turned(from, at), hi = read_turned(from, at + 16 * kRowBytes);
      u32x4 a = {lo[0], lo[1], hi[0], hi[1]};
      if constexpr (kMasked) a = cleaned(a, largest, unbounded);
      o[c] = P::mul(a, big, o[c]);
      o[c] = P::mul(a, small, o[c]);
    }
  };
  auto turn = [&]<int I>(std::integral_constant<int, I>) __attribute__((always_inline)) {
    if (t + kWaves < tiles) {
      const At at = row_of<Far>(s, table, key_of(t + kWaves), page);
      page = page_of(s, table, key_of(t + 2 * kWaves));
      asm volatile("" ::: "memory");
      issue(lds_ring<1 - I, kStage>, at);
      __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(2 * kMoves));   // (the next tile's transfers may be under way)
    } else {
      __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));
    }
    asm volatile("" ::: "memory");
    const int key0 = it.begin + t * kStreamKeys;
    const char *const from = lds_ring<I, kStage>;
    if (key0 + kStreamKeys <= least) tile(std::false_type{}, from, key0);
    else tile(std::true_type{}, from, key0);
    t += kWaves;
  };
  while (t < tiles) {
    turn(std::integral_constant<int, 0>{});
    if (t < tiles) turn(std::integral_constant<int, 1>{});
  }
  if (__any(unbounded != 0)) {
    // Wave by wave the tiles are other ones: the keys from the first that is not seen by all rows on, of this wave's tiles.
    for (int first = wave; first < tiles; first += kWaves) {
      const int key0 = it.begin + first * kStreamKeys;
      if (key0 + kStreamKeys <= least) continue;
      for (int key = key0; key < min(key0 + kStreamKeys, it.end); ++key) {
        const int64_t at = row_of<true>(s, table, key, page_of(s, table, key));
        if (at < 0 || key >= row.limit) continue;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
          if (c * 16 + quad * 4 < s.head_dim) add_unbounded<T>(values + at + (c * 16 + quad * 4) * 2, o[c]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  // The waves' sums
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();
  float *const sums = reinterpret_cast<float *>(lds_ring<0, kStage>), *const ends = reinterpret_cast<float *>(lds_ring<1, kStage>);
#pragma unroll
  for (int c = 0; c < kColumns; ++c) *reinterpret_cast<f32x4_t *>(sums + (wave * 16 + l16) * kPitch + c * 16 + quad * 4) = o[c];
  if (quad == 0) ends[(wave * 16 + l16) * 2] = offset_of<T>(m, s.scale), ends[(wave * 16 + l16) * 2 + 1] = l;
  __syncthreads();
  // Threads by four columns of the rows that there are.  Where there is no other stretch the row is done, but for the prefix's planes.
  constexpr int kThreads = 64 * kWaves, kQuads = Used / 4;
  const int live = min(16, it.count * static_cast<int>(s.group.size) - it.row0);
  for (int column = threadIdx.x; column < live * kQuads; column += kThreads) {
    const int r = column / kQuads, d = column % kQuads * 4;
    if (d >= s.head_dim) continue;
    const Row to = row_at(s, p, it, kv_head, it.row0 + r);
    Sums a = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) a.top = fmaxf(a.top, ends[(w * 16 + r) * 2]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float weight = a.top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ends[(w * 16 + r) * 2] - a.top);
      a.l += weight * ends[(w * 16 + r) * 2 + 1];
      a.o += weight * *reinterpret_cast<const f32x4_t *>(sums + (w * 16 + r) * kPitch + d);
    }
    if (it.slot < 0) {
      if (before.all) add_planes<D, 16>(before, planes_of(s, before, before.places[to.token], kv_head, to.head - kv_head * static_cast<int>(s.group.size)), d, a);
      store_out<T>(s, to.token, to.head, d, a.o * (a.l == 0.f ? 0.f : 1.f / a.l));
      if (d == 0) store_lse(s, to.token, to.head, a.top, a.l);
    } else {
      const int64_t at = (static_cast<int64_t>(it.slot) * s.kv_heads + kv_head) * 16 + r;
      *reinterpret_cast<f32x4_t *>(p.o + at * D + d) = a.o;
      if (d == 0) p.ml[at] = f32x2_t{a.top, a.l};
    }
    if (p.places && it.stretch == 0 && to.head == 0 && d == 0) tell_place(p, it, to.token, r);
  }
}

// ---- many rows -----------------------------------------------------------------------------------------------------------------------

// Four or eight waves of 32 rows, two blocks of 16; tiles of 32 keys go to LDS for all of them, three ahead.  While the softmax of tile j is on the vector
// unit, the matrix unit forms the scores of tile j + 1; then come the weighted values of tile j.  Used: the values of a head, rounded up to 32 (D, the
// length of a row in LDS, is a power of two).
//
// A prompt of 8192 tokens, 32 heads on 8 of 128 (Waves 8): 514 us, 1070 TFLOP/s of what the mask leaves, right behind one another for 50 calls and more; the first ones, and
// single calls, take 540 to 640, as the clock starts low.  A matrix product reaches 1410 here.  The matrix unit is busy for 48 % of the time, at 2.1 to 2.2 GHz, the power's bound.  (In its earlier
// form:) without the exponentials it took 535 of then 567 us, without the scores' product 412, without the
// values' 460, without transfers 462: what is left is the softmax's vector instructions (4.3 to a matrix instruction) beside the matrix unit.  First without the
// scores ahead 641, with 32 x 32 matrix instructions 552 for 547; 64 rows to a wave, one wave to a SIMD, 855.
//
// The weights are rounded to 16 bits for the second product: off by up to half a step each, 2^-9 of a sum's size in bf16 where they add up at random, the size of out's own rounding (0.0022 of
// out's norm for 0.0016, in fp16 0.00028 for 0.0002).  In two parts, as in the other kernel, a prompt of 8192 takes 707 us for 514, 5 chunks of 500 73 for 64, 61 tokens behind a prefix 50 for
// 45.  l is the sum of the weights before that rounding, so lse is not touched.
constexpr int kTileRing = 4;

template <class T, int D, int Used, int Waves, bool Far>
__global__ __launch_bounds__(64 * Waves, D == 256 ? 1 : 2) void attention_tile_kernel(AttentionArgs s, Pass p) {
  constexpr int kRowBytes = 2 * D, kPieces = D / 8, kKeysMoved = 64 / kPieces, kTileBytes = kTileKeys * kRowBytes;
  constexpr int Blocks = 2, kMoves = kTileBytes / (1024 * Waves), kSteps = Used / 32, kColumns = Used / 16;
  static_assert(kMoves >= 1 && 6 * kMoves < 64, "whole transfers; vmcnt");
  typedef typename Rows<Far>::At At;
  typedef Products<T> P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, quad = lane >> 4;
  const int kv_head = static_cast<int>(blockIdx.x) % s.kv_heads;
  Item it;
  if (!find_item(s, p, static_cast<int>(blockIdx.x) / s.kv_heads, it)) return;
  const Table table = {p.prefix ? s.prefix : s.batch.pages + it.b * s.batch.pages_stride, it.end};
  const char *const keys = static_cast<const char *>(s.keys) + kv_head * s.head, *const values = static_cast<const char *>(s.values) + kv_head * s.head;
  const uint32_t bytes = static_cast<uint32_t>(min(s.extent - kv_head * s.head, kNearBytes));
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(keys, Far ? 0u : bytes), rv = make_rsrc(values, Far ? 0u : bytes);
  const int pieces = s.head_dim / 8, tiles = (it.end - it.begin + kTileKeys - 1) / kTileKeys;
  // Loads come in order: the rows of q before the first page, a page before the transfers that it is not for.
  Row row[Blocks];
  u32x4 q[Blocks][kSteps];
#pragma unroll
  for (int r = 0; r < Blocks; ++r) {
    row[r] = row_at(s, p, it, kv_head, it.row0 + wave * (16 * Blocks) + r * 16 + l16);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) q[r][i] = load_q<T>(s, row[r], i * 32 + quad * 8);
  }
  // A wave looks up the rows that it moves in a round of the ring together, a lane to each (lane kMine u + j: the j-th of its kMine keys in the u-th
  // tile), a round ahead; their pages are asked for a round before that (as loads come in order, waiting for one is waiting for all transfers
  // before it).  `ahead`: the rows of the next keys to be asked for, handed to the lanes that move them a tile before; `from`: those of the
  // last keys that were asked for, whose values are asked for one tile later.
  constexpr int kMine = kMoves * kKeysMoved, kRound = kTileRing * kTileKeys;
  static_assert(kMine * kTileRing <= 64, "a lane to each");
  const uint32_t size = s.batch.page_size.size, entries_on = divided(kRound, s.batch.page_size), slots_on = kRound - entries_on * size;
  const uint32_t last_entry = divided(static_cast<uint32_t>(max(it.end - 1, 0)), s.batch.page_size);
  const int j_mine = lane % kMine;
  int key = it.begin + lane / kMine * kTileKeys + (j_mine / kKeysMoved * Waves + wave) * kKeysMoved + j_mine % kKeysMoved, page = 0;
  uint32_t entry = divided(static_cast<uint32_t>(key), s.batch.page_size), in = static_cast<uint32_t>(key) - entry * size, in_of_page = 0;
  At rows = Rows<Far>::kNone, ahead[kMoves], from[kMoves];
  uint32_t key_piece[kMoves], value_piece[kMoves];      // bytes from a row's start; past everything where the head ends before
#pragma unroll
  for (int i = 0; i < kMoves; ++i) {
    const int k = (i * Waves + wave) * kKeysMoved + lane / kPieces, kp = lane % kPieces ^ turn_of_key<D>(k), vp = lane % kPieces ^ turn_of_value<D>(k);
    key_piece[i] = kp < pieces ? kp * 16 : Rows<false>::kNone;
    value_piece[i] = vp < pieces ? vp * 16 : Rows<false>::kNone;
    from[i] = Rows<Far>::kNone;
  }
  auto ask_for_pages = [&]() __attribute__((always_inline)) {
    page = table.pages[min(entry, last_entry)];
    in_of_page = in;
    entry += entries_on, in += slots_on;
    if (in >= size) ++entry, in -= size;
  };
  auto look_up = [&]() __attribute__((always_inline)) {      // the rows of the pages that were asked for last
    rows = Rows<Far>::kNone;
    if (key < it.end && static_cast<uint32_t>(page) < static_cast<uint32_t>(s.batch.n_pages)) rows = static_cast<At>(page) * static_cast<At>(s.page) + static_cast<At>(in_of_page) * static_cast<At>(s.slot);
    key += kRound;
    ask_for_pages();
    asm volatile("" ::: "memory");
  };
  auto hand_out = [&](int place) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) ahead[i] = __shfl(rows, place * kMine + i * kKeysMoved + lane / kPieces, 64);
  };
  auto move = [&](const char *base, __amdgpu_buffer_rsrc_t rsrc, At at, uint32_t piece, char *to) __attribute__((always_inline)) {
    if constexpr (Far) {
      const char *source = at >= 0 && piece != Rows<false>::kNone ? base + at + piece : reinterpret_cast<const char *>(&zero_block);
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void *>(reinterpret_cast<uintptr_t>(source)), (LDS_PTR void *)to, 16, 0, 0);
    } else {
      dma16(rsrc, __builtin_elementwise_add_sat(at, piece), 0, to);
    }
  };
  auto move_keys = [&](char *to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      from[i] = ahead[i];
      move(keys, rk, from[i], key_piece[i], to + ((i * Waves + wave) * 1024));
    }
  };
  auto move_values = [&](char *to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) move(values, rv, from[i], value_piece[i], to + ((i * Waves + wave) * 1024));
  };
  // Transfers come in the order K0 | V0 K1 | V1 K2 | V2 K3 | V3 K4 ...; what is behind the last tile brings zeros.
  if (tiles > 0) ask_for_pages();
#pragma unroll
  for (int r = 0; r < Blocks; ++r)
#pragma unroll
    for (int i = 0; i < kSteps; ++i) asm volatile("" : "+v"(q[r][i]));      // (waits for them here, not in the loop, where it would wait for transfers)
  if (tiles > 0) {
    look_up();
    hand_out(0), move_keys(lds_ring<10, kTileBytes>);
    move_values(lds_ring<20, kTileBytes>);
    hand_out(1), move_keys(lds_ring<11, kTileBytes>);
    move_values(lds_ring<21, kTileBytes>);
    hand_out(2), move_keys(lds_ring<12, kTileBytes>);
    move_values(lds_ring<22, kTileBytes>);
    hand_out(3), move_keys(lds_ring<13, kTileBytes>);
    look_up();
    hand_out(0);
  }
  int least = INT32_MAX, most_keys = it.begin;
#pragma unroll
  for (int r = 0; r < Blocks; ++r) least = min(least, row[r].limit), most_keys = max(most_keys, row[r].live ? row[r].limit : it.begin);
#pragma unroll
  for (int x = 1; x < 16; x *= 2) least = min(least, __shfl_xor(least, x, 64)), most_keys = max(most_keys, __shfl_xor(most_keys, x, 64));
  least = __builtin_amdgcn_readfirstlane(least), most_keys = __builtin_amdgcn_readfirstlane(most_keys);
  f32x4_t o[kColumns][Blocks], score[2][Blocks];      // score[keys 16 b on][rows 16 r on]
#pragma unroll
  for (int c = 0; c < kColumns; ++c)
#pragma unroll
    for (int r = 0; r < Blocks; ++r) o[c][r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m[Blocks], l[Blocks], bound[Blocks], offset[Blocks];    // bound: the score from which m is to follow; offset: of m, 0 before there is one
#pragma unroll
  for (int r = 0; r < Blocks; ++r) {
    score[0][r] = score[1][r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m[r] = bound[r] = -INFINITY, l[r] = offset[r] = 0.f;
  }
  const float lag = kLag / s.scale;
  const uint16_t largest = least < it.end ? P::kExponent - 1 : 0x7FFF;
  uint32_t unbounded = 0;
  // Where this lane reads, as in the other kernel
  int key_at = l16 * kRowBytes + (quad ^ turn_of_key<D>(l16)) * 16;
  int value_at = (quad * 4 + (l16 >> 2)) * kRowBytes + turn_of_value<D>(quad * 4 + (l16 >> 2)) * 16 + (l16 & 3) * 8;
  asm volatile("" : "+v"(key_at), "+v"(value_at));

  constexpr bool kEarly = Used <= 128;      // (registers)
  u32x4 fragments[2][kSteps];
  auto read_keys = [&](const char *k) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < kSteps; ++i) fragments[b][i] = *reinterpret_cast<const u32x4 *>(k + ((key_at ^ i << 6) + b * 16 * kRowBytes));
  };
  auto scores = [&](f32x4_t (&sum)[2][Blocks], int b) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < Blocks; ++r) sum[b][r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const u32x4 a = fragments[b][i];
#pragma unroll
      for (int r = 0; r < Blocks; ++r) sum[b][r] = P::mul(a, q[r][i], sum[b][r]);
    }
  };
  auto tile = [&](auto masked, const char *next, const char *v, int key0) __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(masked)::value;
    if constexpr (kEarly) {
      read_keys(next);                            // (on their way while the maxima are formed)
      __builtin_amdgcn_sched_barrier(0);
    }
    float most[Blocks];
#pragma unroll
    for (int r = 0; r < Blocks; ++r) {
      if constexpr (kMasked) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key0 + j / 4 * 16 + quad * 4 + j % 4 >= row[r].limit) score[j / 4][r][j % 4] = -INFINITY;
      }
      most[r] = score[0][r][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) most[r] = fmaxf(most[r], score[j / 4][r][j % 4]);
    }
    bool grows = false;
#pragma unroll
    for (int r = 0; r < Blocks; r += 2) {
      // Two rows' maxima over the four quads of lanes: halves exchanged with one another's, quads of a half, and back to all lanes.
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(most[r]), __float_as_uint(most[r + 1]), false, false);
      const float y = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
      const auto z = __builtin_amdgcn_permlane16_swap(__float_as_uint(y), __float_as_uint(y), false, false);
      const float w = fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1]));
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(w), __float_as_uint(w), false, false);
      most[r] = __uint_as_float(both[0]), most[r + 1] = __uint_as_float(both[1]);
      grows |= most[r] > bound[r] || most[r + 1] > bound[r + 1];
    }
    if (__any(grows)) {
#pragma unroll
      for (int r = 0; r < Blocks; ++r) {
        const float now = fmaxf(m[r], most[r]), keep = now == m[r] ? 1.f : __builtin_amdgcn_exp2f((m[r] - now) * s.scale);
        m[r] = now, bound[r] = now + lag, offset[r] = now == -INFINITY ? 0.f : offset_of<T>(now, s.scale);
        l[r] *= keep;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) o[c][r] *= keep;
      }
    }
    f32x4_t following[2][Blocks];
    if constexpr (!kEarly) read_keys(next);
    u32x4 weights[Blocks], values[kColumns];
    auto weigh = [&](int r) __attribute__((always_inline)) {
      const float less = kEarly ? offset[r] : m[r] == -INFINITY ? 0.f : offset_of<T>(m[r], s.scale);      // (registers again: heads of 256, held 195 us, formed 192)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j / 2][r][j % 2 * 2], s.scale, -less));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j / 2][r][j % 2 * 2 + 1], s.scale, -less));
        weights[r][j] = P::pack(x, y);
        l[r] += x + y;
      }
    };
    auto read_values = [&](int c) __attribute__((always_inline)) {
      const int at = value_at ^ c << 5;
      const u32x2_t lo = read_turned(v, at), hi = read_turned(v, at + 16 * kRowBytes);
      values[c] = u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    if constexpr (kEarly) {
      // Values are asked for as soon as half of the keys' registers are free, not each where it is used (16 prompts of 1000 223 to 217 us).
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        scores(following, b);
        weigh(b);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = b * kColumns / 2; c < (b + 1) * kColumns / 2; ++c) read_values(c);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      scores(following, 0), scores(following, 1);
      weigh(0), weigh(1);
    }
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      if constexpr (!kEarly) read_values(c);
      if constexpr (kMasked) values[c] = cleaned(values[c], largest, unbounded);
#pragma unroll
      for (int r = 0; r < Blocks; ++r) o[c][r] = P::mul(values[c], weights[r], o[c][r]);
    }
#pragma unroll
    for (int r = 0; r < Blocks; ++r) score[0][r] = following[0][r], score[1][r] = following[1][r];
  };
  auto turn = [&]<int I>(std::integral_constant<int, I>, auto masked, int t) __attribute__((always_inline)) {
    // The keys of tile t + 1 and the values of tile t are there when no more than the next two tiles' transfers are under way.
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(4 * kMoves));
    barrier_no_fence();
    move_values(lds_ring<20 + (I + 3) % 4, kTileBytes>);
    move_keys(lds_ring<10 + I, kTileBytes>);
    if constexpr (I == 3) look_up();
    hand_out((I + 1) % 4);
    const int key0 = it.begin + t * kTileKeys;
    if (!decltype(masked)::value || key0 < most_keys) tile(masked, lds_ring<10 + (I + 1) % 4, kTileBytes>, lds_ring<20 + I, kTileBytes>, key0);
  };
  if (tiles > 0) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(6 * kMoves));      // the first tile's keys
    barrier_no_fence();
    read_keys(lds_ring<10, kTileBytes>);
    scores(score, 0), scores(score, 1);
  }
  // Tiles that all of this wave's rows see, a whole number of rounds of the ring, and the others.
  const int whole = max(min((least - it.begin) / kTileKeys, tiles), 0) & ~3;
  for (int t = 0; t < whole; t += 4) {
    turn(std::integral_constant<int, 0>{}, std::false_type{}, t);
    turn(std::integral_constant<int, 1>{}, std::false_type{}, t + 1);
    turn(std::integral_constant<int, 2>{}, std::false_type{}, t + 2);
    turn(std::integral_constant<int, 3>{}, std::false_type{}, t + 3);
  }
  for (int t = whole; t < tiles; t += 4) {
    turn(std::integral_constant<int, 0>{}, std::true_type{}, t);
    if (t + 1 < tiles) turn(std::integral_constant<int, 1>{}, std::true_type{}, t + 1);
    if (t + 2 < tiles) turn(std::integral_constant<int, 2>{}, std::true_type{}, t + 2);
    if (t + 3 < tiles) turn(std::integral_constant<int, 3>{}, std::true_type{}, t + 3);
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));   // the last, empty transfers, before the LDS is released
  if (__any(unbounded != 0)) {
    for (int k = it.begin + whole * kTileKeys; k < it.end; ++k) {
      const int64_t at = row_of<true>(s, table, k, page_of(s, table, k));
      if (at < 0) continue;
#pragma unroll
      for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int r = 0; r < Blocks; ++r) {
          if (k < row[r].limit && c * 16 + quad * 4 < s.head_dim) add_unbounded<T>(values + at + (c * 16 + quad * 4) * 2, o[c][r]);
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  }

#pragma unroll
  for (int r = 0; r < Blocks; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
    if (!row[r].live) continue;
    const float inverse = l[r] == 0.f ? 0.f : 1.f / l[r];
    const int in_tile = wave * (16 * Blocks) + r * 16 + l16;
    const int64_t place = (static_cast<int64_t>(it.slot) * s.kv_heads + kv_head) * (16 * Blocks * Waves) + in_tile;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      const int d = c * 16 + quad * 4;
      if (it.slot < 0) store_out<T>(s, row[r].token, row[r].head, d, o[c][r] * inverse);
      else if (d < s.head_dim) *reinterpret_cast<f32x4_t *>(p.o + place * D + d) = o[c][r];
    }
    if (quad == 0) {
      if (it.slot < 0) store_lse(s, row[r].token, row[r].head, offset_of<T>(m[r], s.scale), l[r]);
      else p.ml[place] = f32x2_t{offset_of<T>(m[r], s.scale), l[r]};
      if (p.places && it.stretch == 0 && row[r].head == 0) tell_place(p, it, row[r].token, in_tile);
    }
  }
}

// ---- the stretches' sums ---------------------------------------------------------------------------------------------------------------

// D / 4 threads, `spread` times over, to a token and head: with M the largest of the planes' maxima, l = sum 2^(m - M) l, o = sum 2^(m - M) o / l,
// every part of the threads with every spread-th plane, and the parts in order.
// Latency bounds it, a row's table and then its planes: 4 to 5 us for 32 rows of 64 planes each (asked for together; one after the other 3 more).
// 2500 x 13 rows of one to three planes of 80 values 9 us.
template <class T, int D> __global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs s, Pass own, Pass before, int spread) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float sums[kGroups][D], ends[kGroups][2];
  const int group = static_cast<int>(s.group.size), part = static_cast<int>(threadIdx.x) / kLanes, d = threadIdx.x % kLanes * 4;
  const int row = static_cast<int>(blockIdx.x) * (kGroups / spread) + part / spread, token = row / s.heads, head = row - token * s.heads;
  const int end = min(s.batch.starts ? s.batch.starts[s.batch.batch] : s.batch.batch, s.batch.tokens), start = s.batch.starts ? s.batch.starts[0] : 0;
  const int held = min(token, s.batch.tokens - 1);      // (asked for before it is known whether the token is one)
  const u32x2_t place = own.places[held], place_before = before.all ? before.places[held] : u32x2_t{0u, 0u};
  Sums a = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
  int planes = 0;
  if (token >= start && token < end && d < s.head_dim) {
    const int kv_head = head / group, in_group = head - kv_head * group;
    auto add = [&](const Pass &p, Planes of) __attribute__((always_inline)) {
      planes += of.count;
      of.count = (of.count - part % spread + spread - 1) / spread, of.first += part % spread * of.step, of.step *= spread;
      if (spread > 1) add_planes<D, 8>(p, of, d, a);
      else add_planes<D, 4>(p, of, d, a);
    };
    if (before.all) add(before, planes_of(s, before, place_before, kv_head, in_group));
    add(own, planes_of(s, own, place, kv_head, in_group));
  }
  if (spread > 1) {
    *reinterpret_cast<f32x4_t *>(&sums[part][d]) = a.o;
    if (d == 0) ends[part][0] = a.top, ends[part][1] = a.l;
    __syncthreads();
    if (part % spread != 0) return;
    const float mine = a.top;
    for (int j = 1; j < spread; ++j) a.top = fmaxf(a.top, ends[part + j][0]);
    const float keep = mine == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mine - a.top);
    a.l *= keep, a.o *= keep;
    for (int j = 1; j < spread; ++j) {
      const float weight = ends[part + j][0] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ends[part + j][0] - a.top);
      a.l += weight * ends[part + j][1];
      a.o += weight * *reinterpret_cast<const f32x4_t *>(&sums[part + j][d]);
    }
  }
  if (planes == 0) return;           // the one workgroup that had the row has written it
  store_out<T>(s, token, head, d, a.o * (a.l == 0.f ? 0.f : 1.f / a.l));
  if (d == 0) store_lse(s, token, head, a.top, a.l);
}

// ---- launches --------------------------------------------------------------------------------------------------------------------------

template <class T, int D, int Used> int launch_all(const AttentionArgs &s, const Launch &own, const Launch *before, hipStream_t st) {
  const bool far = s.extent > kNearBytes;
  const Pass none = {};
  const auto one = [&](const Launch &r) {
    const Pass &then = before && !r.pass.prefix ? before->pass : none;      // (what the few rows' kernel joins with its own)
    const dim3 grid(static_cast<unsigned>(r.items * s.kv_heads));
    if (r.waves == 8) {
      if constexpr (D == 128) {
        if (far) hipLaunchKernelGGL((attention_tile_kernel<T, D, Used, 8, true>), grid, dim3(512), 0, st, s, r.pass);
        else hipLaunchKernelGGL((attention_tile_kernel<T, D, Used, 8, false>), grid, dim3(512), 0, st, s, r.pass);
      }
    } else if (r.waves == 4) {
      if (far) hipLaunchKernelGGL((attention_tile_kernel<T, D, Used, 4, true>), grid, dim3(256), 0, st, s, r.pass);
      else hipLaunchKernelGGL((attention_tile_kernel<T, D, Used, 4, false>), grid, dim3(256), 0, st, s, r.pass);
    } else {
      if (far) hipLaunchKernelGGL((attention_stream_kernel<T, D, Used, true>), grid, dim3(64 * stream_waves(D)), 0, st, s, r.pass, then);
      else hipLaunchKernelGGL((attention_stream_kernel<T, D, Used, false>), grid, dim3(64 * stream_waves(D)), 0, st, s, r.pass, then);
    }
    return check_launch("attention launch");
  };
  if (before) SAREK_ATTENTION_TRY(one(*before));
  SAREK_ATTENTION_TRY(one(own));
  if (own.pass.max_slots == 0) return SAREK_HIP_OK;
  // Rows that are few for the card take more threads each, which share the planes (one token of 4095 keys, both launches: 16.5 us, 22.7 without).
  constexpr int kGroups = 1024 / D;
  const int64_t rows = static_cast<int64_t>(s.batch.tokens) * s.heads;
  int spread = 1;
  while (spread < kGroups && rows * (D / 4) * spread < 512 * compute_units()) spread *= 2;
  hipLaunchKernelGGL((attention_join_kernel<T, D>), dim3(static_cast<unsigned>(ceil_div(rows, kGroups / spread))), dim3(256), 0, st, s, own.pass,
                     before ? before->pass : none, spread);
  return check_launch("attention join launch");
}

template <class T> int launch_type(const AttentionArgs &s, const Launch &own, const Launch *before, hipStream_t st) {
  const int d = s.head_dim;
  if (d <= 64) return launch_all<T, 64, 64>(s, own, before, st);
  if (d <= 96) return launch_all<T, 128, 96>(s, own, before, st);
  if (d <= 128) return launch_all<T, 128, 128>(s, own, before, st);
  return d <= 192 ? launch_all<T, 256, 192>(s, own, before, st) : launch_all<T, 256, 256>(s, own, before, st);
}

}  // namespace
}  // namespace sarek_hip
