// C ABI of attention (declared in include/glm53_moe.h): packed sequences with
// their gradients, the paged key-value cache and one token over it.
#include "api_util.h"
#include "attention.h"
#include "kv_cache.h"

using namespace glm53;

namespace {

// More rows than this would not be numbered in 32 bits, tiles included.
constexpr int64_t kMaxRows = int64_t{1} << 30;
constexpr int64_t kMaxSequences = int64_t{1} << 24;
constexpr int64_t kMaxGrid = int64_t{1} << 23;  // workgroups of up to 512 threads: a grid has fewer than 2^32
constexpr int64_t kMaxCopied = 4 * kMaxGrid;    // rows, four a workgroup, that one call writes to or reads from a cache
// The rows' logarithms over this are where the gradients' products start: still finite.
constexpr float kLeastScale = 0x1p-64f;
constexpr float kMostScale = 0x1p127f;  // its product with log2 e: still finite

int head_rows(const glm53_head_rows& r, int64_t heads, const char* name, bool wanted, Rows16& out) {
  CHECK_ARG(!wanted || r.data != nullptr, "null pointer argument: %s", name);
  CHECK_ARG(aligned(r.data, 16), "%s must be 16-byte aligned", name);
  for (const int64_t stride : {r.token_stride, r.head_stride})
    CHECK_ARG(stride >= 0 && stride <= kMaxRowStride && stride % 8 == 0, "%s: stride %lld is no multiple of 8 up to %lld",
              name, (long long)stride, (long long)kMaxRowStride);
  CHECK_ARG(heads * r.head_stride <= kMaxHeadSpan, "%s: %lld heads at a stride of %lld lie more than %lld elements apart", name,
            (long long)heads, (long long)r.head_stride, (long long)kMaxHeadSpan);
  out = Rows16{static_cast<const uint16_t*>(r.data), r.token_stride, r.head_stride};
  return GLM53_OK;
}

int head_shape(int64_t heads, int64_t kv_heads, int64_t dim) {
  CHECK_ARG(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "%lld query heads are not a multiple of %lld key heads",
            (long long)heads, (long long)kv_heads);
  CHECK_ARG(heads <= 65536, "more than 65536 heads");
  CHECK_ARG(dim > 0 && dim % 8 == 0 && dim <= kMaxHeadDim, "head_dim %lld is no multiple of 8 up to %lld", (long long)dim,
            (long long)kMaxHeadDim);
  return GLM53_OK;
}

int check_scale(float scale) {
  CHECK_ARG(scale >= kLeastScale && scale <= kMostScale, "scale must be from 2^-64 to 2^127");
  return GLM53_OK;
}

size_t split_bytes(const AttentionArgs& a, int splits) {
  return splits > 1 ? 2 * sizeof(float) * static_cast<size_t>(splits) * a.keys * a.kv_heads * a.dim : 0;
}

int attention_args(const glm53_attention* d, bool backward, AttentionArgs& a) {
  CHECK_ARG(d != nullptr, "attention descriptor is null");
  CHECK_ARG(d->tokens >= 0 && d->keys >= 0, "invalid shape tokens=%lld keys=%lld", (long long)d->tokens, (long long)d->keys);
  if (int rc = head_shape(d->heads, d->kv_heads, d->head_dim)) return rc;
  if (int rc = check_scale(d->scale)) return rc;
  CHECK_ARG(d->tokens < kMaxRows / d->heads && d->keys < kMaxRows / d->heads, "tokens or keys times heads reach 2^30");
  CHECK_ARG(d->offsets != nullptr || d->key_offsets == nullptr, "key_offsets without offsets");
  CHECK_ARG(d->offsets == nullptr || (d->sequences > 0 && d->sequences < kMaxSequences), "sequences must be 1 to 2^24 - 1, got %lld",
            (long long)d->sequences);
  CHECK_ARG(d->key_offsets != nullptr || d->tokens == d->keys, "keys of another number than the queries need key_offsets");
  const int64_t sequences = d->offsets != nullptr ? d->sequences : 1;
  CHECK_ARG((d->tokens * d->heads / d->kv_heads / 64 + sequences + 2) * d->kv_heads < kMaxGrid &&
                (d->keys / 64 + sequences + 2) * d->kv_heads < kMaxGrid,
            "too many tiles for a grid");
  a = AttentionArgs{};
  if (int rc = head_rows(d->q, d->heads, "q", d->tokens > 0, a.q)) return rc;
  if (int rc = head_rows(d->k, d->kv_heads, "k", d->keys > 0, a.k)) return rc;
  if (int rc = head_rows(d->v, d->kv_heads, "v", d->keys > 0, a.v)) return rc;
  a.offsets = d->offsets;
  a.key_offsets = d->key_offsets;
  a.tokens = d->tokens;
  a.keys = d->keys;
  a.sequences = static_cast<int>(sequences);
  a.kv_heads = static_cast<int>(d->kv_heads);
  a.group = static_cast<int>(d->heads / d->kv_heads);
  a.dim = static_cast<int>(d->head_dim);
  a.causal = d->causal != 0;
  a.scale = d->scale;
  a.out = static_cast<uint16_t*>(d->out);
  a.lse = d->lse;
  CHECK_ARG(d->tokens == 0 || d->out != nullptr, "null pointer argument: out");
  CHECK_ARG(aligned(d->out, 16), "out must be 16-byte aligned");
  if (!backward) return GLM53_OK;
  if (int rc = head_rows(d->d_out, d->heads, "d_out", d->tokens > 0, a.d_out)) return rc;
  CHECK_ARG(d->tokens == 0 || d->lse != nullptr, "null pointer argument: lse");
  a.d_q = static_cast<uint16_t*>(d->d_q);
  a.d_k = static_cast<uint16_t*>(d->d_k);
  a.d_v = static_cast<uint16_t*>(d->d_v);
  for (const void* p : {d->d_q, d->d_k, d->d_v}) CHECK_ARG(aligned(p, 16), "gradients must be 16-byte aligned");
  const size_t need = glm53_packed_attention_backward_workspace_bytes(d->tokens, d->heads);
  CHECK_ARG(need == 0 || (d->workspace && d->workspace_bytes >= need && aligned(d->workspace, 256)),
            "attention's gradients need a 256-byte aligned workspace of %zu bytes", need);
  a.starts = static_cast<float*>(d->workspace);
  a.splits = attention_row_splits(a);
  if (d->workspace_bytes < need + split_bytes(a, a.splits)) a.splits = 1;
  a.sums = reinterpret_cast<float*>(static_cast<uint8_t*>(d->workspace) + need);
  return GLM53_OK;
}

int cache_args(const glm53_kv_cache* c, CacheArgs& a) {
  CHECK_ARG(c != nullptr, "cache descriptor is null");
  if (int rc = head_shape(c->kv_heads, c->kv_heads, c->head_dim)) return rc;
  CHECK_ARG(c->pages > 0 && c->pages < (int64_t{1} << 31), "a cache has 1 to 2^31 - 1 pages, got %lld", (long long)c->pages);
  int log2 = 4;
  while (log2 < 16 && (int64_t{1} << log2) < c->page_size) ++log2;
  CHECK_ARG((int64_t{1} << log2) == c->page_size, "page_size %lld is no power of two from 16 to 65536", (long long)c->page_size);
  CHECK_ARG(c->sequences >= 0 && c->sequences < kMaxSequences, "sequences must be below 2^24, got %lld", (long long)c->sequences);
  CHECK_ARG(c->max_pages >= 0 && c->max_pages < (int64_t{1} << 31) && c->table_stride >= c->max_pages,
            "invalid page table: %lld pages of a sequence, %lld from one to the next", (long long)c->max_pages,
            (long long)c->table_stride);
  CHECK_ARG(c->k_pages && c->v_pages, "null pointer argument: pages");
  CHECK_ARG(c->sequences == 0 || c->max_pages == 0 || c->page_table, "null pointer argument: page_table");
  CHECK_ARG(aligned(c->k_pages, 16) && aligned(c->v_pages, 16), "pages must be 16-byte aligned");
  CHECK_ARG((c->e4m3 != 0) == (c->k_scales != nullptr) && (c->e4m3 != 0) == (c->v_scales != nullptr),
            "scales belong to an E4M3 cache");
  CHECK_ARG(aligned(c->k_scales, 16) && aligned(c->v_scales, 16), "scales must be 16-byte aligned");
  a = CacheArgs{};
  a.k = static_cast<uint8_t*>(c->k_pages);
  a.v = static_cast<uint8_t*>(c->v_pages);
  a.k_scales = c->k_scales;
  a.v_scales = c->v_scales;
  a.table = c->page_table;
  a.pages = c->pages;
  a.table_stride = c->table_stride;
  a.sequences = static_cast<int>(c->sequences);
  a.max_pages = static_cast<int>(c->max_pages);
  a.kv_heads = static_cast<int>(c->kv_heads);
  a.dim = static_cast<int>(c->head_dim);
  a.page_log2 = log2;
  a.e4m3 = c->e4m3 != 0;
  CHECK_ARG(!a.e4m3 || a.dim % 16 == 0, "an E4M3 cache needs a head_dim that is a multiple of 16, got %d", a.dim);
  return GLM53_OK;
}

}  // namespace

extern "C" {

int glm53_packed_attention(const glm53_attention* attention, void* stream) {
  AttentionArgs a;
  if (int rc = attention_args(attention, false, a)) return rc;
  if (a.tokens == 0) return GLM53_OK;
  HIP_TRY(launch_attention(a, S(stream)), "attention launch");
  return GLM53_OK;
}

size_t glm53_packed_attention_backward_workspace_bytes(int64_t tokens, int64_t heads) {
  if (tokens <= 0 || heads <= 0 || tokens >= kMaxRows / heads) return 0;
  return round_up(2 * sizeof(float) * static_cast<size_t>(tokens * heads));
}

size_t glm53_packed_attention_backward_split_bytes(int64_t tokens, int64_t keys, int64_t sequences, int64_t heads, int64_t kv_heads,
                                                   int64_t head_dim) {
  if (tokens <= 0 || keys <= 0 || heads <= 0 || tokens >= kMaxRows / heads || keys >= kMaxRows / heads || kv_heads <= 0 ||
      heads % kv_heads != 0 || head_dim <= 0 || head_dim > kMaxHeadDim || sequences >= kMaxSequences)
    return 0;
  AttentionArgs a{};
  a.tokens = tokens;
  a.keys = keys;
  a.sequences = static_cast<int>(sequences > 0 ? sequences : 1);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(heads / kv_heads);
  a.dim = static_cast<int>(head_dim);
  return split_bytes(a, attention_row_splits(a));
}

int glm53_packed_attention_backward(const glm53_attention* attention, void* stream) {
  AttentionArgs a;
  if (int rc = attention_args(attention, true, a)) return rc;
  HIP_TRY(launch_attention_backward(a, S(stream)), "attention gradient launch");
  return GLM53_OK;
}

int glm53_kv_append(const glm53_kv_cache* cache, const glm53_head_rows* k, const glm53_head_rows* v, int64_t tokens,
                    const int32_t* offsets, const int32_t* lengths, void* stream) {
  AppendArgs a{};
  if (int rc = cache_args(cache, a.cache)) return rc;
  CHECK_ARG(k != nullptr && v != nullptr, "null pointer argument: rows");
  CHECK_ARG(tokens >= 0 && tokens < kMaxCopied, "invalid number of tokens %lld", (long long)tokens);
  CHECK_ARG(offsets != nullptr || tokens == cache->sequences, "one token a sequence is %lld tokens, got %lld",
            (long long)cache->sequences, (long long)tokens);
  if (int rc = head_rows(*k, cache->kv_heads, "k", tokens > 0, a.rows_k)) return rc;
  if (int rc = head_rows(*v, cache->kv_heads, "v", tokens > 0, a.rows_v)) return rc;
  if (tokens == 0 || cache->sequences == 0) return GLM53_OK;
  CHECK_ARG(lengths != nullptr, "null pointer argument: lengths");
  a.tokens = tokens;
  a.offsets = offsets;
  a.lengths = lengths;
  HIP_TRY(launch_append(a, S(stream)), "cache append launch");
  return GLM53_OK;
}

int glm53_kv_read(const glm53_kv_cache* cache, const int32_t* offsets, int64_t rows, void* k, void* v, void* stream) {
  ReadArgs a{};
  if (int rc = cache_args(cache, a.cache)) return rc;
  CHECK_ARG(rows >= 0 && rows < kMaxCopied, "invalid number of rows %lld", (long long)rows);
  CHECK_ARG(aligned(k, 16) && aligned(v, 16), "k and v must be 16-byte aligned");
  if (rows == 0 || (k == nullptr && v == nullptr)) return GLM53_OK;
  CHECK_ARG(offsets != nullptr, "null pointer argument: offsets");
  a.offsets = offsets;
  a.rows = rows;
  a.k = static_cast<uint16_t*>(k);
  a.v = static_cast<uint16_t*>(v);
  HIP_TRY(launch_read(a, S(stream)), "cache read launch");
  return GLM53_OK;
}

size_t glm53_paged_attention_workspace_bytes(int64_t head_dim, int32_t e4m3) {
  if (head_dim <= 0 || head_dim > kMaxHeadDim) return 0;
  return round_up(decode_space(static_cast<int>(head_dim), e4m3 != 0));
}

int glm53_paged_attention(const glm53_kv_cache* cache, const glm53_head_rows* q, int64_t heads, const int32_t* lengths,
                          float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  DecodeArgs a{};
  if (int rc = cache_args(cache, a.cache)) return rc;
  if (int rc = head_shape(heads, cache->kv_heads, cache->head_dim)) return rc;
  if (int rc = check_scale(scale)) return rc;
  CHECK_ARG(q != nullptr, "null pointer argument: q");
  if (int rc = head_rows(*q, heads, "q", cache->sequences > 0, a.q)) return rc;
  if (cache->sequences == 0) return GLM53_OK;
  CHECK_ARG(lengths && out, "null pointer argument");
  CHECK_ARG(aligned(out, 16), "out must be 16-byte aligned");
  CHECK_ARG(cache->sequences * heads < kMaxGrid, "sequences times heads reach %lld", (long long)kMaxGrid);
  const size_t need = glm53_paged_attention_workspace_bytes(cache->head_dim, cache->e4m3);
  CHECK_ARG(workspace && workspace_bytes >= need && aligned(workspace, 256),
            "attention over a cache needs a 256-byte aligned workspace of %zu bytes", need);
  a.lengths = lengths;
  a.group = static_cast<int>(heads / cache->kv_heads);
  a.scale = scale;
  a.out = static_cast<uint16_t*>(out);
  a.partial = static_cast<float*>(workspace);
  HIP_TRY(launch_decode(a, S(stream)), "paged attention launch");
  return GLM53_OK;
}

}  // extern "C"
