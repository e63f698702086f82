// Attention over a paged cache (layout: attention_common.hpp): for each token and head, softmax(scale q . keys) . values.
#include <algorithm>
#include <cmath>

#include "attention_common.hpp"

namespace sarek_hip {
namespace {

struct AttentionArgs {
  Batch batch;
  const void *q, *keys, *values;
  void *out;
  float *lse;
  int64_t q_token, q_head, out_token, out_head;
  int64_t page, slot, head;         // the cache's strides
  int heads, group, head_dim, causal;
  float scale;
  const int *prefix;
  int prefix_length;
};

template <class T> __device__ __forceinline__ float widen(T v) { return load_one(&v); }

// One wave to a token and head, 64 keys at a time: a lane to a key for the scores, a lane to every 64th value for the weighted sum.  The
// running maximum and sum of the softmax, one pass over the keys.
template <class T>
__global__ __launch_bounds__(64) void attention_simple_kernel(AttentionArgs s) {
  __shared__ float q[256];
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, d = s.head_dim;
  const int b = sequence_of(s.batch, token);
  if (b >= s.batch.batch) return;
  const Tokens mine = tokens_of(s.batch, b);
  const int length = s.batch.lengths[b];
  int64_t sees = s.causal ? static_cast<int64_t>(length) - mine.count + (token - mine.first) + 1 : length;
  const int own = static_cast<int>(max(min(sees, static_cast<int64_t>(keys_held(s.batch, length))), int64_t{0}));
  for (int i = lane; i < d; i += 64) q[i] = load_one(static_cast<const T *>(s.q) + token * s.q_token + head * s.q_head + i);
  __syncthreads();
  float most = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < 2; ++part) {
    const int keys = part ? own : s.prefix_length;
    const int *const table = part ? s.batch.pages + b * s.batch.pages_stride : s.prefix;
    for (int k0 = 0; k0 < keys; k0 += 64) {
      const int key = k0 + lane;
      float score = -INFINITY;
      int64_t at = -1;
      if (key < keys) {
        const uint32_t entry = divided(key, s.batch.page_size);
        const int page = table[entry];
        score = 0.f;
        if (page >= 0 && page < s.batch.n_pages) {
          at = page * s.page + (key - static_cast<int64_t>(entry) * s.batch.page_size.size) * s.slot + head / s.group * s.head;
          const T *const k = static_cast<const T *>(s.keys) + at;
          for (int i = 0; i < d; ++i) score += q[i] * load_one(k + i);
        }
        score *= s.scale;
      }
      float top = score;
      for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
      const float now = fmaxf(most, top), before = now == most ? 1.f : expf(most - now);
      const float p = key < keys ? expf(score - now) : 0.f;
      float total = p;
      for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x, 64);
      sum = sum * before + total;
      most = now;
      for (int i = 0; i < 4; ++i) o[i] *= before;
      for (int j = 0; j < min(64, keys - k0); ++j) {
        const float pj = __shfl(p, j, 64);
        const int64_t aj = __shfl(at, j, 64);
        for (int i = 0; i < 4; ++i)
          if (aj >= 0 && lane + 64 * i < d) o[i] += pj * load_one(static_cast<const T *>(s.values) + aj + lane + 64 * i);
      }
    }
  }
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < d) store_one(static_cast<T *>(s.out) + token * s.out_token + head * s.out_head + lane + 64 * i, sum == 0.f ? 0.f : o[i] / sum);
  if (s.lse && lane == 0) s.lse[static_cast<int64_t>(token) * s.heads + head] = sum == 0.f ? -INFINITY : most + logf(sum);
}

int attention(const char *what, const sarek_hip_kv_cache *cache, const void *q, int64_t q_token, int64_t q_head, int q_heads, void *out,
              int64_t out_token, int64_t out_head, float *lse, const int *prefix_pages, int64_t prefix_length, const int *pages,
              int64_t pages_stride, int max_pages, const int *lengths, const int *starts, int batch, int64_t tokens, int causal, float scale,
              void *workspace, int64_t workspace_bytes, sarek_hip_stream stream) {
  SAREK_ATTENTION_TRY(check_cache(what, cache));
  AttentionArgs s;
  SAREK_ATTENTION_TRY(make_batch(what, cache, pages, pages_stride, max_pages, lengths, starts, batch, tokens, &s.batch));
  if (q_heads < 1 || q_heads % cache->heads != 0) return fail(SAREK_HIP_E_INVALID_ARG, "%s: %d heads of q over %d of the cache", what, q_heads, cache->heads);
  if (q_heads > 65535) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: more than 65535 heads", what);
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(SAREK_HIP_E_INVALID_ARG, "%s: the scale must be positive and finite", what);
  SAREK_ATTENTION_TRY(check_heads(what, "q", q_token, q_head, tokens, q_heads, cache->head_dim, false));
  SAREK_ATTENTION_TRY(check_heads(what, "out", out_token, out_head, tokens, q_heads, cache->head_dim, true));
  if (prefix_length < 0 || (prefix_length > 0 && !prefix_pages)) return fail(SAREK_HIP_E_INVALID_ARG, "%s: a prefix of %lld keys", what, static_cast<long long>(prefix_length));
  if (prefix_length > int64_t{1} << 30) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: a prefix past 2^30 keys", what);
  const int64_t need = sarek_hip_attention_workspace_bytes(cache, q_heads, batch, tokens, max_pages, prefix_length);
  if (workspace_bytes < need)
    return fail(SAREK_HIP_E_WORKSPACE, "%s: a workspace of %lld bytes, %lld are needed", what, static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  if (tokens == 0 || batch == 0) return SAREK_HIP_OK;
  if (!q || !out || (need > 0 && !workspace)) return fail(SAREK_HIP_E_INVALID_ARG, "%s: NULL pointer", what);
  s.q = q, s.keys = cache->keys, s.values = cache->values, s.out = out, s.lse = lse;
  s.q_token = q_token, s.q_head = q_head, s.out_token = out_token, s.out_head = out_head;
  s.page = cache->page_stride, s.slot = cache->slot_stride, s.head = cache->head_stride;
  s.heads = q_heads, s.group = q_heads / cache->heads, s.head_dim = cache->head_dim, s.causal = causal != 0, s.scale = scale;
  s.prefix = prefix_pages, s.prefix_length = static_cast<int>(prefix_length);
  const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>(q_heads));
  if (cache->type == SAREK_HIP_TYPE_BF16) hipLaunchKernelGGL(attention_simple_kernel<Bf16>, grid, dim3(64), 0, as_stream(stream), s);
  else hipLaunchKernelGGL(attention_simple_kernel<_Float16>, grid, dim3(64), 0, as_stream(stream), s);
  return check_launch("attention launch");
}

}  // namespace
}  // namespace sarek_hip

using namespace sarek_hip;

extern "C" {

int64_t sarek_hip_attention_workspace_bytes(const sarek_hip_kv_cache *cache, int q_heads, int batch, int64_t tokens, int max_pages, int64_t prefix_length) {
  (void)cache, (void)q_heads, (void)batch, (void)tokens, (void)max_pages, (void)prefix_length;
  return 0;
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
