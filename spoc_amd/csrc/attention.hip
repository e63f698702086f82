// Attention over a paged cache: the arguments' checks, and what a call launches (the kernels: attention_kernels.hpp).
#include <algorithm>
#include <cmath>

#include "attention_common.hpp"
#include "gemm_common.hpp"
#include "tunables.hpp"

namespace sarek_hip {
namespace {

constexpr float kLog2E = 1.44269504088896f;
int padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
// What the planes of a launch take: o, m and l, and where each token's are.
int64_t plane_bytes(const sarek_hip_kv_cache *cache, const Launch &r, int64_t tokens) {
  if (r.pass.max_slots == 0) return 0;
  const int64_t planes = static_cast<int64_t>(r.pass.max_slots) * cache->heads;
  return planes * r.pass.rows * (padded(cache->head_dim) + 2) * 4 + (tokens + 1) / 2 * 16;
}
// What is launched, by what the host knows: how many tokens, sequences and keys there are at most.
//
// Kernel.  Up to 16 rows to a sequence on average: the kernel of few rows; more: tiles of 128.  (us, calls without pauses, 32 heads on 8 of 128, few rows / tiles: one
// sequence of 4095 keys, 4 rows 16.6 / 19.5; 131071 keys of 16 heads of 64, 113 / 121; 64 of 2000, 20 rows 135 / 105, 16 rows 107 / 104, 8 rows 104 / 103.  Tiles are as fast from 8 rows on
// where there are many sequences, but round the weights to 16 bits, which the kernel of few rows does not.)  One kernel for the call: a chunk among single tokens, or one in a batch of
// empty places, is not served by its own (127 tokens and a chunk of 380 265, each alone 246 and 42; a prompt of 1000 39, in a batch of 256 places 85).
// Tiles of 256: heads of 65 to 128 values, long sequences that fill the card twice.  (One prompt, tiles of 256 / 128: 8192 tokens 516 / 522, 16384 1943 /
// 1971; but 5000 229 / 217, and 16 prompts of 1000 242 / 217, for the rows past the ends and what the mask hides in a larger tile.)
//
// Stretches.  Where tiles are few for the card, the keys are cut: for as many workgroups as it takes at once if that comes out (find_item).  That is two to
// a compute unit for tiles of 128 and few rows of more than 64 values, whose transfers it takes to keep the memory busy (one token each: 8 sequences of 4000 512
// workgroups 34.6, 256 37.1, 768 41.1; 131071 keys of 16 heads 195, 210, 218), one otherwise, or where there is no room for two (the same of 64 values 118, 113, 117;
// 12 of 4000, which do not fill 512: 480 42.7, 576 56.3).  Few rows that do not come out get half as many again (61 sequences of 100 to 11007: 768 276, 512
// 293).  Tiles are cut below one to a compute unit: planes of 128 rows cost as much as 6 units of keys (2000 tokens behind 6000: uncut 238, cut 248); and for half as many
// workgroups where a stretch would have less than 12 units (64 behind 8128: 31.4, 34.9 without that; 500 behind 7692, which has more: 88.8, 95.1 with it).
// No more than 256 stretches: 30000 keys of one head, 235 of them 20.1, 469 23.0 (131071: 256 30.0, 512 33.5, 128 36.6).
// Own keys behind a prefix, few rows: a workgroup to each tile where these fill the card, which then finishes with the prefix's planes; no launch for
// the join (61 sequences of up to 500 behind 8191: 56 with the join, 47).
// Whether keys are cut goes by how many tiles there are, not by how unlike the lengths are, which the host does not know: one sequence of 131071 keys among others of 500 takes 177 in a batch
// of 90 single tokens, 2813 in one of 100, which is not cut any more.
enum { kAlone, kBehindPrefix, kPrefix };
Launch plan(const sarek_hip_kv_cache *cache, int q_heads, int64_t sequences, int64_t tokens, int64_t keys, int what) {
  const int d = cache->head_dim;
  const int64_t rows = tokens * (q_heads / cache->heads), heads = cache->heads, units_at_once = compute_units();
  const int64_t large = tunable("attention.large_rows", 25600);
  const auto large_tiles = [&] { return large == 0 || (rows / 256 * heads >= 2 * units_at_once && rows >= large * sequences); };
  Launch r;
  r.waves = rows <= 16 * sequences ? 0 : d > 64 && d <= 128 && large_tiles() ? 8 : 4;
  r.pass = {};
  r.pass.prefix = what == kPrefix;
  r.pass.rows = r.waves ? 32 * r.waves : 16;
  r.pass.unit = r.waves ? 2 * kTileKeys : kStreamKeys * stream_waves(d);
  const int64_t most_tiles = rows / r.pass.rows + sequences, tiles = std::max(rows / r.pass.rows, std::min(tokens, sequences)), units = ceil_div(keys, r.pass.unit);
  const bool two_to_a_unit = r.waves ? r.waves == 4 && d <= 128 : d > 64;
  const int64_t wanted = r.waves ? tunable("attention.tile_workgroups", 2 * compute_units()) : tunable("attention.stream_workgroups", 2 * compute_units());
  const int64_t at_once = std::clamp<int64_t>(two_to_a_unit ? wanted : wanted / 2, 0, 1 << 20);
  const int64_t spread = r.waves ? at_once : at_once * 3 / 2;
  if (units > 1 && at_once > 0 && tiles * heads < (r.waves || what == kBehindPrefix ? units_at_once : spread)) {
    r.pass.target = static_cast<int>(at_once), r.pass.spread = static_cast<int>(spread);
    r.pass.least_units = r.waves && two_to_a_unit ? 12 : 0;
  }
  r.pass.all = what == kPrefix || (what == kBehindPrefix && (r.waves || r.pass.target != 0));
  // (the number of units to a stretch comes from a float32 sum: a few items more)
  r.items = r.pass.target == 0 ? most_tiles : std::min(most_tiles + spread / heads + 8, most_tiles * units);
  r.pass.max_slots = static_cast<int>(r.pass.all ? r.items : r.pass.target == 0 ? 0 : std::min(r.items, 2 * spread / heads + 8));
  return r;
}
char *place_planes(const sarek_hip_kv_cache *cache, Launch *r, int64_t tokens, char *at) {
  if (r->pass.max_slots == 0) return at;
  const int64_t rows = static_cast<int64_t>(r->pass.max_slots) * cache->heads * r->pass.rows;
  r->pass.o = reinterpret_cast<float *>(at);
  r->pass.ml = reinterpret_cast<f32x2_t *>(at + rows * padded(cache->head_dim) * 4);
  r->pass.places = reinterpret_cast<place_t *>(at + rows * (padded(cache->head_dim) + 2) * 4);
  return at + plane_bytes(cache, *r, tokens);
}

int attention(const char *what, const sarek_hip_kv_cache *cache, const void *q, int64_t q_token, int64_t q_head, int q_heads, void *out,
              int64_t out_token, int64_t out_head, float *lse, const int *prefix_pages, int64_t prefix_length, const int *pages,
              int64_t pages_stride, int max_pages, const int *lengths, const int *starts, int batch, int64_t tokens, int causal, float scale,
              void *workspace, int64_t workspace_bytes, sarek_hip_stream stream) {
  SAREK_ATTENTION_TRY(check_cache(what, cache));
  AttentionArgs s;
  SAREK_ATTENTION_TRY(make_batch(what, cache, pages, pages_stride, max_pages, lengths, starts, batch, tokens, &s.batch));
  if (q_heads < 1 || q_heads % cache->heads != 0) return fail(SAREK_HIP_E_INVALID_ARG, "%s: %d heads of q over %d of the cache", what, q_heads, cache->heads);
  // (a launch has below 2^32 threads)
  if (q_heads > 65535 || tokens * q_heads >= int64_t{1} << 26) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: more than 65535 heads, or 2^26 tokens times heads", what);
  if (!(scale > 0.f) || !std::isfinite(scale * kLog2E)) return fail(SAREK_HIP_E_INVALID_ARG, "%s: the scale must be positive and finite", what);
  SAREK_ATTENTION_TRY(check_heads(what, "q", q_token, q_head, tokens, q_heads, cache->head_dim, false));
  SAREK_ATTENTION_TRY(check_heads(what, "out", out_token, out_head, tokens, q_heads, cache->head_dim, true));
  if (q && q == out && ((tokens > 1 && q_token != out_token) || (q_heads > 1 && q_head != out_head)))
    return fail(SAREK_HIP_E_INVALID_ARG, "%s: out is q with other strides", what);
  if (prefix_length < 0 || (prefix_length > 0 && !prefix_pages)) return fail(SAREK_HIP_E_INVALID_ARG, "%s: a prefix of %lld keys", what, static_cast<long long>(prefix_length));
  if (prefix_length > int64_t{1} << 30) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: a prefix past 2^30 keys", what);
  const int64_t need = sarek_hip_attention_workspace_bytes(cache, q_heads, batch, tokens, max_pages, prefix_length);
  if (workspace_bytes < need)
    return fail(SAREK_HIP_E_WORKSPACE, "%s: a workspace of %lld bytes, %lld are needed", what, static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  if (tokens == 0 || batch == 0) return SAREK_HIP_OK;
  if (!q || !out || (need > 0 && !workspace)) return fail(SAREK_HIP_E_INVALID_ARG, "%s: NULL pointer", what);
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return fail(SAREK_HIP_E_INVALID_ARG, "%s: a workspace starts at a multiple of 16 bytes", what);
  const int d = cache->head_dim;
  s.q = q, s.keys = cache->keys, s.values = cache->values, s.out = out, s.lse = lse;
  s.q_token = q_token, s.q_head = q_head, s.out_token = out_token, s.out_head = out_head;
  s.page = cache->page_stride * 2, s.slot = cache->slot_stride * 2, s.head = cache->head_stride * 2;
  s.extent = ((cache->n_pages - 1) * cache->page_stride + (cache->page_size - 1) * cache->slot_stride + (cache->heads - 1) * cache->head_stride + d) * 2;
  s.heads = q_heads, s.kv_heads = cache->heads, s.head_dim = d, s.causal = causal != 0;
  s.group = division_by(static_cast<uint32_t>(q_heads / cache->heads));
  s.scale = scale * kLog2E;
  s.prefix = prefix_pages, s.prefix_length = static_cast<int>(prefix_length);
  const bool shared = prefix_length > 0;
  Launch own = plan(cache, q_heads, batch, tokens, static_cast<int64_t>(max_pages) * cache->page_size, shared ? kBehindPrefix : kAlone);
  Launch before = plan(cache, q_heads, 1, tokens, prefix_length, kPrefix);
  if (std::max(own.items, before.items) * cache->heads >= int64_t{1} << 23) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: 2^23 tiles of rows or more", what);
  char *const rest = place_planes(cache, &own, tokens, static_cast<char *>(workspace));
  if (shared) place_planes(cache, &before, tokens, rest);
  const Launch *const first = shared ? &before : nullptr;
  return (cache->type == SAREK_HIP_TYPE_BF16 ? launch_attention_bf16 : launch_attention_f16)(s, own, first, as_stream(stream));
}

}  // namespace
}  // namespace sarek_hip

using namespace sarek_hip;

extern "C" {

int64_t sarek_hip_attention_workspace_bytes(const sarek_hip_kv_cache *cache, int q_heads, int batch, int64_t tokens, int max_pages, int64_t prefix_length) {
  if (!cache || cache->heads < 1 || q_heads < cache->heads || batch < 1 || tokens < 1 || max_pages < 0 || prefix_length < 0) return 0;
  const Launch own = plan(cache, q_heads, batch, tokens, static_cast<int64_t>(max_pages) * cache->page_size, prefix_length > 0 ? kBehindPrefix : kAlone);
  return plane_bytes(cache, own, tokens) + (prefix_length > 0 ? plane_bytes(cache, plan(cache, q_heads, 1, tokens, prefix_length, kPrefix), tokens) : 0);
}

int sarek_hip_attention_paged(const sarek_hip_kv_cache *cache, const void *q, int64_t q_token, int64_t q_head, int q_heads, void *out,
                              int64_t out_token, int64_t out_head, float *lse, const int *pages, int64_t pages_stride, int max_pages,
                              const int *lengths, const int *starts, int batch, int64_t tokens, int causal, float scale, void *workspace,
                              int64_t workspace_bytes, sarek_hip_stream stream) {
  return attention("attention_paged", cache, q, q_token, q_head, q_heads, out, out_token, out_head, lse, nullptr, 0, pages, pages_stride, max_pages, lengths,
                   starts, batch, tokens, causal, scale, workspace, workspace_bytes, stream);
}

int sarek_hip_attention_shared(const sarek_hip_kv_cache *cache, const void *q, int64_t q_token, int64_t q_head, int q_heads, void *out,
                               int64_t out_token, int64_t out_head, float *lse, const int *prefix_pages, int64_t prefix_length,
                               const int *pages, int64_t pages_stride, int max_pages, const int *lengths, const int *starts, int batch,
                               int64_t tokens, int causal, float scale, void *workspace, int64_t workspace_bytes, sarek_hip_stream stream) {
  return attention("attention_shared", cache, q, q_token, q_head, q_heads, out, out_token, out_head, lse, prefix_pages, prefix_length, pages, pages_stride,
                   max_pages, lengths, starts, batch, tokens, causal, scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
