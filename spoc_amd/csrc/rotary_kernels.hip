// Rotary positions, by themselves and on the way into a paged cache.
//
// Pair (a, b) of a head becomes amplitude (a cos t - b sin t, a sin t + b cos t), t = position * frequency.  The angle is formed in whole
// numbers: position times the frequency in units of 2^-64 turns, modulo one turn by the overflow, of which the upper 32 bits, rounded, are the angle as a
// signed fraction of a turn.  The table's entry is off by less than 2^-64 turns (frequencies of up to half a turn), so the angle is off by |position| 2^-64 + 2^-33 turns, up
// to 2^-32 at positions of up to 2^31, and by 2^-24 of itself, float32's rounding (a 32-bit product of both is 0.06 radians off at position 10^6).  There is no reduction
// of the argument left for the sine.
//
// Memory bounds both kernels (two products and a sum to a value); a thread takes 8 pairs of a head, two accesses of 16 bytes each way in
// 16-bit types, and where there are many tokens 4 heads, for which it forms the sines once (8192 x 32 x 128 bf16: 22 us, 6.1 TB/s; a
// thread to each head 26).  One token of 32 heads: 2.8 us, a launch.  Appending 8190 tokens of 32 and 8 + 8 heads of 128 to pages in fp16: 38 us, 5.3 TB/s;
// 16 tokens 4.5 us, the search for a token's sequence and its page before the first access.
#include <cmath>

#include "attention_common.hpp"

namespace sarek_hip {
namespace {

constexpr int kPairs = 8;

struct Heads {      // [tokens, heads, head_dim], elements
  int64_t token, head;
};
struct RotaryArgs {
  const uint64_t *turns;
  float amplitude;
  int pairs, inverse, head_dim;
  int units, copies;        // pieces of 8 pairs and of 16 values behind them in a head that is turned
};

template <class T> struct Bits { typedef uint16_t type; };
template <> struct Bits<float> { typedef uint32_t type; };

// 16 values as they are, and fewer
template <class T> __device__ __forceinline__ void load16(const T *from, u32x4_t (&v)[sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) v[i] = *reinterpret_cast<const u32x4_any *>(reinterpret_cast<const typename Bits<T>::type *>(from) + i * (16 / sizeof(T)));
}
template <class T> __device__ __forceinline__ void store16(T *to, const u32x4_t (&v)[sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) *reinterpret_cast<u32x4_any *>(reinterpret_cast<typename Bits<T>::type *>(to) + i * (16 / sizeof(T))) = v[i];
}
template <class T> __device__ __forceinline__ void copy_few(const T *from, T *to, int count) {
  typedef typename Bits<T>::type B;
  for (int i = 0; i < count; ++i) reinterpret_cast<B *>(to)[i] = reinterpret_cast<const B *>(from)[i];
}

struct Turned {
  float cos[kPairs], sin[kPairs];
};
__device__ __forceinline__ Turned angles(const RotaryArgs &r, int64_t position, int unit) {
  Turned t;
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const uint64_t turn = static_cast<uint64_t>(position) * r.turns[min(unit * kPairs + j, r.pairs - 1)] + 0x80000000u;
    sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * 0x1p-31f, &t.sin[j], &t.cos[j]);
    t.sin[j] *= r.inverse ? -r.amplitude : r.amplitude;
    t.cos[j] *= r.amplitude;
  }
  return t;
}

// Piece `unit` of heads head to head + kHeads - 1, those of them below `heads`: 8 pairs, or 16 of the values behind the pairs.  All are asked for
// before the first is written: out may be x, so the compiler would not put a load before an earlier store.  (8190 tokens of 32 and 8
// heads appended: 49.8 us, 58.7 with each head's loads behind the stores of the one before; launch and tensors among it.)
template <class T, bool Interleaved, int kHeads>
__device__ __forceinline__ void turn_pieces(const RotaryArgs &r, int64_t position, const T *x, int64_t x_head, T *out, int64_t out_head, int head, int heads,
                                            int unit) {
  const bool in_place = x == out;
  if (unit >= r.units) {
    const int at = 2 * r.pairs + (unit - r.units) * 16;
    if (in_place) return;
    if (r.head_dim - at >= 16) {
      u32x4_t v[kHeads][sizeof(T)];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) load16(x + min(head + h, heads - 1) * x_head + at, v[h]);
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
        if (head + h < heads) store16(out + (head + h) * out_head + at, v[h]);
    } else {
#pragma unroll 1
      for (int h = head; h < min(head + kHeads, heads); ++h) copy_few(x + h * x_head + at, out + h * out_head + at, r.head_dim - at);
    }
    return;
  }
  const int a_at = Interleaved ? unit * 16 : unit * kPairs, b_at = Interleaved ? a_at + 8 : a_at + r.pairs, left = r.pairs - unit * kPairs;
  auto turned = [&](const Turned &t, const Raw8<T> &ra, const Raw8<T> &rb, float (&u)[8], float (&v)[8]) __attribute__((always_inline)) {
    float a[8], b[8];
    widen8<T>(ra, a);
    widen8<T>(rb, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (Interleaved) {
        const float *const from = j < 4 ? a : b;
        float *const to = j < 4 ? u : v;
        const int k = 2 * (j & 3);
        to[k] = from[k] * t.cos[j] - from[k + 1] * t.sin[j];
        to[k + 1] = from[k] * t.sin[j] + from[k + 1] * t.cos[j];
      } else {
        u[j] = a[j] * t.cos[j] - b[j] * t.sin[j];
        v[j] = a[j] * t.sin[j] + b[j] * t.cos[j];
      }
    }
  };
  float u[8], v[8];
  if (left >= kPairs) {
    Raw8<T> ra[kHeads], rb[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const T *const from = x + min(head + h, heads - 1) * x_head;      // (past the last head: the last one again)
      ra[h] = load8(from + a_at, 8), rb[h] = load8(from + b_at, 8);
    }
    const Turned t = angles(r, position, unit);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (head + h >= heads) break;
      turned(t, ra[h], rb[h], u, v);
      store8(out + (head + h) * out_head + a_at, 8, u);
      store8(out + (head + h) * out_head + b_at, 8, v);
    }
    return;
  }
  // The last pairs, fewer than 8
  const int a_count = Interleaved ? 2 * left : left, b_count = Interleaved ? 2 * left - 8 : left;
  if constexpr (kHeads == 1) {
    const Raw8<T> ra = load8(x + head * x_head + a_at, a_count), rb = load8(x + head * x_head + b_at, b_count);
    turned(angles(r, position, unit), ra, rb, u, v);
    store8(out + head * out_head + a_at, a_count, u);
    store8(out + head * out_head + b_at, b_count, v);
    return;
  }
  const Turned t = angles(r, position, unit);
#pragma unroll 1
  for (int h = head; h < min(head + kHeads, heads); ++h) {
    turned(t, load8(x + h * x_head + a_at, a_count), load8(x + h * x_head + b_at, b_count), u, v);
    store8(out + h * out_head + a_at, a_count, u);
    store8(out + h * out_head + b_at, b_count, v);
  }
}

template <class T, bool Interleaved, int kHeads>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs r, const T *x, Heads xs, const void *__restrict__ positions,
                                                     int position_bytes, T *out, Heads os, int heads, int groups, int per_token,
                                                     int64_t pieces) {
  for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < pieces; i += gridDim.x * int64_t{256}) {
    const int64_t token = i / per_token;
    const int in = static_cast<int>(i - token * per_token), group = in / (r.units + r.copies), unit = in - group * (r.units + r.copies);
    const int64_t position = position_bytes == 8 ? static_cast<const int64_t *>(positions)[token] : static_cast<const int32_t *>(positions)[token];
    turn_pieces<T, Interleaved, kHeads>(r, position, x + token * xs.token, xs.head, out + token * os.token, os.head, group * kHeads, heads, unit);
  }
}

struct AppendArgs {
  Batch batch;
  int64_t first;
  const void *k, *v, *q;
  void *q_out, *keys, *values;
  Heads ks, vs, qs, q_outs;
  int64_t page, slot, head;         // the cache's strides
  int q_heads, heads;
  int q_pieces, k_pieces, v_pieces; // of a token, the first two for groups of kHeads heads
};

// A workgroup to up to 256 pieces of one token: the search for the token's sequence is the same for all of them.
template <class T, bool Interleaved, int kHeads>
__global__ __launch_bounds__(256) void kv_append_kernel(RotaryArgs r, AppendArgs s) {
  const int token = static_cast<int>(blockIdx.x), b = sequence_of(s.batch, token);
  if (b >= s.batch.batch) return;
  const Tokens mine = tokens_of(s.batch, b);
  if (token < mine.first) return;
  const int64_t place = static_cast<int64_t>(s.batch.lengths[b]) - mine.count + (token - mine.first);
  const uint32_t entry = place >= 0 && place < INT32_MAX ? divided(static_cast<uint32_t>(place), s.batch.page_size) : 0xFFFFFFFFu;
  int page = -1;
  if (entry < static_cast<uint32_t>(s.batch.max_pages)) page = s.batch.pages[b * s.batch.pages_stride + entry];
  const bool held = page >= 0 && page < s.batch.n_pages;
  const int64_t at = held ? page * s.page + (place - static_cast<int64_t>(entry) * s.batch.page_size.size) * s.slot : 0;
  const int per_head = r.units + r.copies;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < s.q_pieces + s.k_pieces + s.v_pieces; i += gridDim.y * blockDim.x) {
    if (i < s.q_pieces + s.k_pieces) {
      const bool of_q = i < s.q_pieces;
      const int in = of_q ? i : i - s.q_pieces, group = in / per_head, unit = in - group * per_head, heads = of_q ? s.q_heads : s.heads;
      if (!of_q && !held) continue;
      const T *const from = static_cast<const T *>(of_q ? s.q : s.k) + token * (of_q ? s.qs.token : s.ks.token);
      T *const to = of_q ? static_cast<T *>(s.q_out) + token * s.q_outs.token : static_cast<T *>(s.keys) + at;
      const int64_t from_head = of_q ? s.qs.head : s.ks.head, to_head = of_q ? s.q_outs.head : s.head;
      turn_pieces<T, Interleaved, kHeads>(r, place + s.first, from, from_head, to, to_head, group * kHeads, heads, unit);
    } else if (held) {
      const int in = i - s.q_pieces - s.k_pieces, per_v = (r.head_dim + 15) / 16, h = in / per_v, unit = in - h * per_v;
      const T *const from = static_cast<const T *>(s.v) + token * s.vs.token + h * s.vs.head + unit * 16;
      T *const to = static_cast<T *>(s.values) + at + h * s.head + unit * 16;
      if (r.head_dim - unit * 16 >= 16) {
        u32x4_t v[sizeof(T)];
        load16(from, v);
        store16(to, v);
      } else {
        copy_few(from, to, r.head_dim - unit * 16);
      }
    }
  }
}

int make_plan(const char *what, const sarek_hip_rotary_plan *plan, int head_dim, RotaryArgs *r) {
  *r = {nullptr, 1.f, 0, 0, head_dim, 0, static_cast<int>(ceil_div(head_dim, 16))};
  if (!plan) return SAREK_HIP_OK;
  if (!plan->turns) return fail(SAREK_HIP_E_INVALID_ARG, "%s: NULL pointer", what);
  if (plan->pairs < 1 || plan->pairs > head_dim / 2)
    return fail(SAREK_HIP_E_INVALID_ARG, "%s: %d pairs in a head of %d values", what, plan->pairs, head_dim);
  if (!std::isfinite(plan->amplitude)) return fail(SAREK_HIP_E_INVALID_ARG, "%s: the amplitude must be finite", what);
  *r = {plan->turns, plan->amplitude, plan->pairs, 0, head_dim, static_cast<int>(ceil_div(plan->pairs, kPairs)), static_cast<int>(ceil_div(head_dim - 2 * plan->pairs, 16))};
  return SAREK_HIP_OK;
}
// From here on (pieces of one head) a thread takes 4 heads; below that more threads, and so more loads at once, are worth the sines.  (Graphs of one
// launch, us, 4 heads to a thread / 1, heads of 128 in bf16: 16384 x 4 17.5 / 16.6, 4096 x 8 16.5 / 16.8, 4096 x 32 17.5 / 21.2, 16384 x 8 17.6 / 21.1, 16384 x 32 46.8 / 53.7.)
// Fewer than 4 heads leave a thread's places empty (16384 x 2: 16.4 / 17.8, x 3 17.4 / 16.7: no difference that stands out).
constexpr int64_t kManyPieces = 1 << 19;

}  // namespace

int check_heads(const char *what, const char *name, int64_t token_stride, int64_t head_stride, int64_t tokens, int heads, int head_dim, bool written) {
  // (what is only read may lie on itself, as an expanded tensor does)
  const bool negative = (tokens > 1 && token_stride < 0) || (heads > 1 && head_stride < 0);
  const bool overlaps = (heads > 1 && head_stride < head_dim) || (tokens > 1 && token_stride < head_dim) ||
                        (heads > 1 && tokens > 1 && token_stride < head_stride * (heads - 1) + head_dim && head_stride < token_stride * (tokens - 1) + head_dim);
  if (negative || (written && overlaps))
    return fail(SAREK_HIP_E_INVALID_ARG, "%s: %s: strides of %lld and %lld for %lld tokens of %d heads of %d", what, name,
                static_cast<long long>(token_stride), static_cast<long long>(head_stride), static_cast<long long>(tokens), heads, head_dim);
  return SAREK_HIP_OK;
}

int check_cache(const char *what, const sarek_hip_kv_cache *c) {
  if (!c || !c->keys || !c->values) return fail(SAREK_HIP_E_INVALID_ARG, "%s: NULL pointer", what);
  if (c->type != SAREK_HIP_TYPE_BF16 && c->type != SAREK_HIP_TYPE_F16) return fail(SAREK_HIP_E_INVALID_ARG, "%s: a cache holds bf16 or fp16, not type %d", what, c->type);
  if (c->n_pages < 1 || c->page_size < 1 || c->heads < 1 || c->head_dim < 1)
    return fail(SAREK_HIP_E_INVALID_ARG, "%s: a cache of %lld pages of %d, %d heads of %d", what, static_cast<long long>(c->n_pages), c->page_size, c->heads, c->head_dim);
  if (c->head_dim % 8 != 0 || c->head_dim > 256) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: heads of %d values: multiples of 8 up to 256 are served", what, c->head_dim);
  if (c->n_pages > INT32_MAX || c->page_size > (1 << 30) || c->heads > 65535)
    return fail(SAREK_HIP_E_UNSUPPORTED, "%s: a cache of 2^31 pages, pages past 2^30 or heads past 65535", what);
  if (((reinterpret_cast<uintptr_t>(c->keys) | reinterpret_cast<uintptr_t>(c->values)) & 15) != 0)
    return fail(SAREK_HIP_E_INVALID_ARG, "%s: keys and values start at multiples of 16 bytes", what);
  const int64_t strides[3] = {c->page_stride, c->slot_stride, c->head_stride}, counts[3] = {c->n_pages, c->page_size, c->heads};
  for (int i = 0; i < 3; ++i)
    if (counts[i] > 1 && (strides[i] < c->head_dim || strides[i] % 8 != 0))
      return fail(SAREK_HIP_E_INVALID_ARG, "%s: a stride of %lld in a cache of heads of %d: at least that, and a multiple of 8", what,
                  static_cast<long long>(strides[i]), c->head_dim);
  return SAREK_HIP_OK;
}

int make_batch(const char *what, const sarek_hip_kv_cache *cache, const int *pages, int64_t pages_stride, int max_pages, const int *lengths,
               const int *starts, int batch, int64_t tokens, Batch *out) {
  if (batch < 0 || tokens < 0 || max_pages < 0) return fail(SAREK_HIP_E_INVALID_ARG, "%s: batch, tokens and max_pages must not be negative", what);
  if (batch > 0 && (!lengths || (max_pages > 0 && !pages))) return fail(SAREK_HIP_E_INVALID_ARG, "%s: NULL pointer", what);
  if (batch > 1 && pages_stride < max_pages) return fail(SAREK_HIP_E_INVALID_ARG, "%s: rows of the page table are %lld apart, less than %d", what, static_cast<long long>(pages_stride), max_pages);
  if (!starts && tokens < batch) return fail(SAREK_HIP_E_INVALID_ARG, "%s: without starts each of %d sequences has a token, but there are %lld", what, batch, static_cast<long long>(tokens));
  if (static_cast<int64_t>(max_pages) * cache->page_size > (int64_t{1} << 30)) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: sequences past 2^30 keys", what);
  if (tokens >= 1 << 24 || batch > 1 << 16) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: 2^24 tokens or more than 2^16 sequences", what);
  *out = {pages, lengths, starts, pages_stride, max_pages, batch, static_cast<int>(tokens), static_cast<int>(cache->n_pages), division_by(cache->page_size)};
  return SAREK_HIP_OK;
}

}  // namespace sarek_hip

using namespace sarek_hip;

extern "C" {

int sarek_hip_rotary_turns(const double *radians, uint64_t *turns, int pairs) {
  if (pairs < 0 || (pairs > 0 && (!radians || !turns))) return fail(SAREK_HIP_E_INVALID_ARG, "rotary_turns: NULL pointer or a negative count");
  for (int i = 0; i < pairs; ++i) {
    if (!std::isfinite(radians[i])) return fail(SAREK_HIP_E_INVALID_ARG, "rotary_turns: frequency %d is not finite", i);
    const long double turn = radians[i] / 6.283185307179586476925286766559005768L, part = turn - std::floor(turn);
    const long double rounded = std::nearbyint(part * 0x1p64L);
    turns[i] = rounded < 0x1p64L ? static_cast<uint64_t>(rounded) : 0;
  }
  return SAREK_HIP_OK;
}

int sarek_hip_rotary(const sarek_hip_rotary_plan *plan, const void *x, int64_t x_token, int64_t x_head, int type, const void *positions,
                     int position_bytes, int inverse, void *out, int64_t out_token, int64_t out_head, int64_t tokens, int heads, int head_dim,
                     sarek_hip_stream stream) {
  if (!plan) return fail(SAREK_HIP_E_INVALID_ARG, "rotary: NULL pointer");
  if (!known_type(type)) return fail(SAREK_HIP_E_INVALID_ARG, "rotary: unknown type %d", type);
  if (tokens < 0 || heads < 1 || head_dim < 1) return fail(SAREK_HIP_E_INVALID_ARG, "rotary: %lld tokens of %d heads of %d", static_cast<long long>(tokens), heads, head_dim);
  if (position_bytes != 4 && position_bytes != 8) return fail(SAREK_HIP_E_INVALID_ARG, "rotary: positions of %d bytes", position_bytes);
  if (tokens > int64_t{1} << 31 || heads > 65535 || head_dim > 65536) return fail(SAREK_HIP_E_UNSUPPORTED, "rotary: more than 2^31 tokens, 65535 heads or 65536 values");
  RotaryArgs r;
  SAREK_ATTENTION_TRY(make_plan("rotary", plan, head_dim, &r));
  r.inverse = inverse != 0;
  SAREK_ATTENTION_TRY(check_heads("rotary", "x", x_token, x_head, tokens, heads, head_dim, false));
  SAREK_ATTENTION_TRY(check_heads("rotary", "out", out_token, out_head, tokens, heads, head_dim, true));
  if (tokens == 0) return SAREK_HIP_OK;
  if (!x || !positions || !out) return fail(SAREK_HIP_E_INVALID_ARG, "rotary: NULL pointer");
  if (x == out && ((tokens > 1 && x_token != out_token) || (heads > 1 && x_head != out_head)))
    return fail(SAREK_HIP_E_INVALID_ARG, "rotary: out is x with other strides");
  return by_type(type, [&]<class T>(T *) {
    const auto run = [&](auto kernel, int at_once) {
      const int groups = static_cast<int>(ceil_div(heads, at_once)), per_token = groups * (r.units + r.copies);
      const int64_t pieces = tokens * per_token;
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(pieces, 256), 1 << 20))), dim3(256), 0, as_stream(stream), r,
                         static_cast<const T *>(x), Heads{x_token, x_head}, positions, position_bytes, static_cast<T *>(out), Heads{out_token, out_head},
                         heads, groups, per_token, pieces);
      return check_launch("rotary launch");
    };
    if (tokens * heads * (r.units + r.copies) < kManyPieces || heads < 4) return plan->interleaved ? run(rotary_kernel<T, true, 1>, 1) : run(rotary_kernel<T, false, 1>, 1);
    return plan->interleaved ? run(rotary_kernel<T, true, 4>, 4) : run(rotary_kernel<T, false, 4>, 4);
  });
}

int sarek_hip_kv_append(const sarek_hip_kv_cache *cache, const void *k, int64_t k_token, int64_t k_head, const void *v, int64_t v_token,
                        int64_t v_head, const void *q, int64_t q_token, int64_t q_head, void *q_out, int64_t q_out_token, int64_t q_out_head,
                        int q_heads, const sarek_hip_rotary_plan *plan, const int *pages, int64_t pages_stride, int max_pages,
                        const int *lengths, const int *starts, int batch, int64_t tokens, int64_t first, sarek_hip_stream stream) {
  SAREK_ATTENTION_TRY(check_cache("kv_append", cache));
  AppendArgs s;
  SAREK_ATTENTION_TRY(make_batch("kv_append", cache, pages, pages_stride, max_pages, lengths, starts, batch, tokens, &s.batch));
  RotaryArgs r;
  const int d = cache->head_dim;
  SAREK_ATTENTION_TRY(make_plan("kv_append", plan, d, &r));
  SAREK_ATTENTION_TRY(check_heads("kv_append", "k", k_token, k_head, tokens, cache->heads, d, false));
  SAREK_ATTENTION_TRY(check_heads("kv_append", "v", v_token, v_head, tokens, cache->heads, d, false));
  if (!q) q_heads = 0;
  if (q) {
    if (q_heads < 1 || q_heads > 65535) return fail(SAREK_HIP_E_INVALID_ARG, "kv_append: %d heads of q", q_heads);
    SAREK_ATTENTION_TRY(check_heads("kv_append", "q", q_token, q_head, tokens, q_heads, d, false));
    SAREK_ATTENTION_TRY(check_heads("kv_append", "q_out", q_out_token, q_out_head, tokens, q_heads, d, true));
    if (q == q_out && ((tokens > 1 && q_token != q_out_token) || (q_heads > 1 && q_head != q_out_head)))
      return fail(SAREK_HIP_E_INVALID_ARG, "kv_append: q_out is q with other strides");
  }
  if (tokens == 0 || batch == 0) return SAREK_HIP_OK;
  if (!k || !v || (q && !q_out)) return fail(SAREK_HIP_E_INVALID_ARG, "kv_append: NULL pointer");
  s.first = first;
  s.k = k, s.v = v, s.q = q, s.q_out = q_out, s.keys = cache->keys, s.values = cache->values;
  s.ks = {k_token, k_head}, s.vs = {v_token, v_head}, s.qs = {q_token, q_head}, s.q_outs = {q_out_token, q_out_head};
  s.page = cache->page_stride, s.slot = cache->slot_stride, s.head = cache->head_stride;
  s.q_heads = q_heads, s.heads = cache->heads;
  return by_type(cache->type, [&]<class T>(T *) {
    const auto run = [&](auto kernel, int at_once) {
      const int per_head = r.units + r.copies;
      s.q_pieces = static_cast<int>(ceil_div(q_heads, at_once)) * per_head;
      s.k_pieces = static_cast<int>(ceil_div(s.heads, at_once)) * per_head;
      s.v_pieces = s.heads * static_cast<int>(ceil_div(d, 16));
      const int64_t all = s.q_pieces + s.k_pieces + s.v_pieces, threads = std::min<int64_t>(ceil_div(all, 64) * 64, 256);
      const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>(ceil_div(all, threads)));
      hipLaunchKernelGGL(kernel, grid, dim3(static_cast<unsigned>(threads)), 0, as_stream(stream), r, s);
      return check_launch("kv_append launch");
    };
    const bool interleaved = plan && plan->interleaved;
    if constexpr (sizeof(T) == 4) {
      return fail(SAREK_HIP_E_INVALID_ARG, "kv_append: float32");    // (check_cache has refused it)
    } else {
      if (tokens * (q_heads + s.heads) * (r.units + r.copies) < kManyPieces || std::max(q_heads, s.heads) < 4) return interleaved ? run(kv_append_kernel<T, true, 1>, 1) : run(kv_append_kernel<T, false, 1>, 1);
      return interleaved ? run(kv_append_kernel<T, true, 4>, 4) : run(kv_append_kernel<T, false, 4>, 4);
    }
  });
}

}  // extern "C"
