// The C ABI of the paged cache and of attention over prompts and pages (include/qmm_decode.h): checks of arguments and the choice of kernel. No
// kernel code lives here.
#include <cmath>

#include "attention.h"

namespace qmm {
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// (`work`: the call has something to do; a table of no sequences has no address)
int view_of(const char* what, const qmm_paged_cache* c, bool work, CacheView* v) {
  if (!c || c->struct_size != sizeof(qmm_paged_cache)) return fail(QMM_ERR_NULL, "%s: a qmm_paged_cache with its struct_size is required", what);
  if (!c->k || !c->v || (work && !c->table)) return fail(QMM_ERR_NULL, "%s: the cache's k, v and table are required", what);
  if (c->elem != QMM_BF16 && c->elem != QMM_F16 && c->elem != QMM_E4M3) return fail(QMM_ERR_DTYPE, "%s: a cache holds bf16, f16 or e4m3", what);
  if (c->elem == QMM_E4M3 && (!c->k_exp || !c->v_exp)) return fail(QMM_ERR_NULL, "%s: an e4m3 cache needs its exponent bytes", what);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(QMM_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", what);
  int shift = 0;
  while (shift < 9 && (1 << shift) != c->page_size) ++shift;
  if (shift < 4 || shift > 8) return fail(QMM_ERR_UNSUPPORTED, "%s: page_size must be 16, 32, 64, 128 or 256", what);
  if (c->pages < 1 || c->kv_heads < 1 || c->table_width < 1 || c->table_stride < c->table_width) return fail(QMM_ERR_SHAPE, "%s: bad cache or table shape", what);
  if (c->pages > (1ll << 31) - 1 || c->pages * c->kv_heads > (1ll << 39) || static_cast<int64_t>(c->table_width) * c->page_size > (1ll << 30))
    return fail(QMM_ERR_TOO_LARGE, "%s: at most 2^30 positions a sequence and 2^31 - 1 pages", what);
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_exp) || !aligned16(c->v_exp)) return fail(QMM_ERR_LAYOUT, "%s: the cache must be 16-byte aligned", what);
  v->k = static_cast<uint8_t*>(c->k);
  v->v = static_cast<uint8_t*>(c->v);
  v->k_exp = static_cast<uint8_t*>(c->k_exp);
  v->v_exp = static_cast<uint8_t*>(c->v_exp);
  v->table = c->table;
  v->table_stride = c->table_stride;
  v->pages = c->pages;
  v->table_width = c->table_width;
  v->page_shift = shift;
  v->kv_heads = c->kv_heads;
  return QMM_OK;
}

// What every form of a call has: tokens, sequences, heads.
int check_attention(const char* what, const qmm_attention_args* a) {
  if (!a || a->struct_size != sizeof(qmm_attention_args)) return fail(QMM_ERR_NULL, "%s: qmm_attention_args with their struct_size are required", what);
  if (a->tokens < 0 || a->tokens > (1 << 30) || a->seqs < 0 || a->seqs > (1 << 30)) return fail(QMM_ERR_SHAPE, "%s: bad number of tokens or sequences", what);
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads) return fail(QMM_ERR_SHAPE, "%s: the key heads must divide the query heads", what);
  if (a->tokens * (a->heads / a->kv_heads) > (1ll << 31) - 256) return fail(QMM_ERR_TOO_LARGE, "%s: a key head has less than 2^31 rows of queries", what);
  if (a->heads / a->kv_heads > 64) return fail(QMM_ERR_UNSUPPORTED, "%s: at most 64 query heads per key head", what);
  if (a->head_dim != 64 && a->head_dim != 128) return fail(QMM_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", what);
  return QMM_OK;
}

// Rows of heads as copies of whole tiles want them: tokens a whole number of heads apart, no two elements in one place. (A dimension of one has no stride.)
bool lies(int64_t tokens, int64_t heads, int64_t dim, int64_t* row, int64_t* head) {
  if (tokens <= 1) *row = heads == 1 ? dim : heads * *head;
  if (heads == 1) *head = *row;
  return *row % 8 == 0 && *head % 8 == 0 && *head >= dim && *row >= heads * *head && *row % *head == 0;
}

int64_t workspace_of(const qmm_attention_args* a) {
  const int64_t rows = attend_rows_workspace(a->head_dim, attend_rows_ctas()), tc = attend_tc_workspace(a->head_dim, attend_tc_ctas());
  return rows > tc ? rows : tc;
}

int attend(const char* what, const qmm_paged_cache* cache, const CacheView* view, const qmm_attention_args* a, cudaStream_t stream) {
  if (a->elem != QMM_BF16 && a->elem != QMM_F16) return fail(QMM_ERR_DTYPE, "%s: q is bf16 or f16", what);
  if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) return fail(QMM_ERR_UNSUPPORTED, "%s: scale must be a positive number", what);
  if (a->tokens == 0 || a->seqs == 0) return QMM_OK;
  if (!a->q || !a->out) return fail(QMM_ERR_NULL, "%s: q and out are required", what);
  RowsParams p = {};
  p.q_row = a->q_row;
  p.q_head = a->q_head;
  p.k_row = a->k_row;
  p.k_head = a->k_head;
  p.v_row = a->v_row;
  p.v_head = a->v_head;
  if (!aligned16(a->q) || !aligned16(a->out) || !lies(a->tokens, a->heads, a->head_dim, &p.q_row, &p.q_head) ||
      (!view && (!lies(a->tokens, a->kv_heads, a->head_dim, &p.k_row, &p.k_head) || !lies(a->tokens, a->kv_heads, a->head_dim, &p.v_row, &p.v_head))))
    return fail(QMM_ERR_LAYOUT, "%s: 16-byte aligned tensors are wanted, strides multiples of 8, tokens a whole number of heads apart", what);
  if (!a->workspace || a->workspace_bytes < workspace_of(a)) return fail(QMM_ERR_TOO_LARGE, "%s: the workspace is too small", what);
  if (!aligned16(a->workspace)) return fail(QMM_ERR_LAYOUT, "%s: the workspace must be 16-byte aligned", what);
  p.work.cu_q = a->cu_q;
  p.work.kv_lens = a->kv_lens;
  p.work.tokens = a->tokens;
  p.work.seqs = static_cast<int32_t>(a->seqs);
  p.work.heads = a->heads;
  p.work.kv_heads = a->kv_heads;
  p.work.group = a->heads / a->kv_heads;
  p.work.causal = a->causal ? 1 : 0;
  p.work.status = device_status_word();
  if (!p.work.status) return fail(QMM_ERR_CUDA, "could not allocate the device status word");
  p.q = static_cast<const uint8_t*>(a->q);
  p.k = static_cast<const uint8_t*>(a->k);
  p.v = static_cast<const uint8_t*>(a->v);
  p.out = static_cast<uint8_t*>(a->out);
  p.notes = static_cast<JoinNote*>(a->workspace);
  p.scale_log2 = a->scale * 1.4426950408889634f;
  if (view) {
    p.cache = *view;
    p.work.longest = static_cast<int64_t>(cache->table_width) << view->page_shift;
  }
  const int64_t rows = a->cu_q ? (a->tokens * p.work.group + a->seqs - 1) / a->seqs : p.work.group;
  const int source = !view ? 0 : cache->elem == QMM_E4M3 ? 2 : 1;
  // Up to 32 rows of queries that a sequence and key head have on average the stream of mma.sync tiles is no slower, from some hundred on the kernel of 2 x 128 rows
  // several times as fast (8 sequences of 2000 to 4000 positions: 20 rows 22 against 32 us, 35 rows 24 and 24, 64 rows 36 and 36).
  const bool tc = a->cu_q && rows > 32 && !attend_cluster_ctas(p, source, rows < 65 ? static_cast<int>(rows) : 65) &&
                  (!view || (static_cast<uint64_t>(p.cache.pages) * p.work.kv_heads << p.cache.page_shift) < (1ull << 31));
  const int ctas = tc ? attend_tc_ctas() : attend_rows_ctas();
  p.partial = reinterpret_cast<float*>(p.notes + ctas);
  if (tc) return launch_attend_tc(p, a->elem, a->head_dim, source, ctas, stream);
  return launch_attend_rows(p, a->elem, a->head_dim, source, static_cast<int>(rows), stream);
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" int qmm_cache_append(const qmm_paged_cache* cache, const qmm_append_args* a, void* stream) {
  CacheView v;
  if (int rc = view_of("cache_append", cache, a && a->struct_size == sizeof(*a) && a->tokens && a->seqs, &v)) return rc;
  if (!a || a->struct_size != sizeof(qmm_append_args)) return fail(QMM_ERR_NULL, "cache_append: qmm_append_args with their struct_size are required");
  if (a->elem != QMM_BF16 && a->elem != QMM_F16) return fail(QMM_ERR_DTYPE, "cache_append: rows are bf16 or f16");
  if (cache->elem != QMM_E4M3 && cache->elem != a->elem) return fail(QMM_ERR_DTYPE, "cache_append: a 16-bit cache holds the rows' own type");
  if (a->tokens < 0 || a->tokens > (1 << 30) || a->seqs < 0 || a->seqs > (1 << 30) || a->heads < 1 || a->heads > (1 << 20))
    return fail(QMM_ERR_SHAPE, "cache_append: bad number of tokens, sequences or heads");
  if (!a->cu_q && a->tokens != a->seqs) return fail(QMM_ERR_SHAPE, "cache_append: without cu_q every sequence has one token");
  if (a->rotary_dim < 0 || a->rotary_dim > cache->head_dim || a->rotary_dim % 16) return fail(QMM_ERR_SHAPE, "cache_append: rotary_dim is a multiple of 16 up to head_dim");
  if (a->tokens == 0 || a->seqs == 0) return QMM_OK;
  if (!a->qkv || !a->q_out || !a->kv_lens || (a->rotary_dim && !a->freqs)) return fail(QMM_ERR_NULL, "cache_append: qkv, q_out, kv_lens and (with rotary_dim) freqs are required");
  if (a->row_stride % 8 || a->row_stride < (a->heads + 2 * static_cast<int64_t>(cache->kv_heads)) * cache->head_dim)
    return fail(QMM_ERR_LAYOUT, "cache_append: rows of qkv are a multiple of 8 elements apart, and no less than they are long");
  if (!aligned16(a->qkv) || !aligned16(a->q_out) || !aligned16(a->q_norm) || !aligned16(a->k_norm))
    return fail(QMM_ERR_LAYOUT, "cache_append: pointers must be 16-byte aligned");
  int* status = device_status_word();
  if (!status) return fail(QMM_ERR_CUDA, "could not allocate the device status word");
  return launch_append(v, *a, cache->head_dim, cache->elem == QMM_E4M3, status, static_cast<cudaStream_t>(stream));
}

extern "C" int qmm_cache_read(const qmm_paged_cache* cache, int64_t seqs, const int32_t* cu_kv, int64_t total, int elem, void* k_out, void* v_out,
                              void* stream) {
  CacheView v;
  if (int rc = view_of("cache_read", cache, seqs && total, &v)) return rc;
  if (elem != QMM_BF16 && elem != QMM_F16) return fail(QMM_ERR_DTYPE, "cache_read: values are bf16 or f16");
  if (cache->elem != QMM_E4M3 && cache->elem != elem) return fail(QMM_ERR_DTYPE, "cache_read: a 16-bit cache is read as its own type");
  if (seqs < 0 || seqs > (1 << 30) || total < 0 || total > (1ll << 31) - 1) return fail(QMM_ERR_SHAPE, "cache_read: bad number of sequences or rows");
  if (seqs == 0 || total == 0) return QMM_OK;
  if (!cu_kv || !k_out || !v_out) return fail(QMM_ERR_NULL, "cache_read: cu_kv, k_out and v_out are required");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(QMM_ERR_LAYOUT, "cache_read: pointers must be 16-byte aligned");
  int* status = device_status_word();
  if (!status) return fail(QMM_ERR_CUDA, "could not allocate the device status word");
  return launch_cache_read(v, seqs, cu_kv, total, cache->head_dim, elem, cache->elem == QMM_E4M3, k_out, v_out, status, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t qmm_attention_workspace_bytes(const qmm_attention_args* args) {
  if (check_attention("attention", args)) return -1;
  return workspace_of(args);
}

extern "C" int qmm_prompt_attention(const qmm_attention_args* a, void* stream) {
  if (int rc = check_attention("prompt_attention", a)) return rc;
  if (a->kv_lens) return fail(QMM_ERR_UNSUPPORTED, "prompt_attention: a prompt's keys are its own tokens' (kv_lens is NULL)");
  if (a->tokens && a->seqs) {
    if (!a->cu_q || !a->k || !a->v) return fail(QMM_ERR_NULL, "prompt_attention: cu_q, k and v are required");
    if (!aligned16(a->k) || !aligned16(a->v)) return fail(QMM_ERR_LAYOUT, "prompt_attention: k and v must be 16-byte aligned");
  }
  return attend("prompt_attention", nullptr, nullptr, a, static_cast<cudaStream_t>(stream));
}

extern "C" int qmm_paged_attention(const qmm_paged_cache* cache, const qmm_attention_args* a, void* stream) {
  CacheView v;
  if (int rc = view_of("paged_attention", cache, a && a->struct_size == sizeof(*a) && a->tokens && a->seqs, &v)) return rc;
  if (int rc = check_attention("paged_attention", a)) return rc;
  if (a->kv_heads != cache->kv_heads || a->head_dim != cache->head_dim) return fail(QMM_ERR_SHAPE, "paged_attention: the cache has other heads");
  if (cache->elem == QMM_E4M3 ? a->elem != QMM_BF16 : a->elem != cache->elem)
    return fail(QMM_ERR_DTYPE, "paged_attention: q has the type of a 16-bit cache, and is bf16 with an e4m3 one");
  if (!a->cu_q && a->tokens != a->seqs) return fail(QMM_ERR_SHAPE, "paged_attention: without cu_q every sequence has one token");
  if (a->tokens && a->seqs && !a->kv_lens) return fail(QMM_ERR_NULL, "paged_attention: kv_lens is required");
  return attend("paged_attention", cache, &v, a, static_cast<cudaStream_t>(stream));
}
