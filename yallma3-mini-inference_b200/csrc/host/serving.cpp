// C entry points of the serving operators: paged cache, attention over it,
// token log probabilities (checks, then one call into kernels/serve.h).
#include "model.h"
#include "../kernels/serve.h"

struct yl_model {
  yl::Model* m;
};
struct yl_batch {
  yl::Batch* b;
};

using namespace yl;

namespace {

uint64_t dtype_size(int dtype) { return dtype == YL_DT_F32 ? 4 : dtype == YL_DT_F16 || dtype == YL_DT_BF16 ? 2 : 0; }
bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

int check_shape(int dtype, uint32_t n_pages, uint32_t page_size, uint32_t n_kv_heads, uint32_t head_size) {
  if (!dtype_size(dtype)) return fail(YL_ERR_ARG, "unknown element type");
  if (head_size != 64 && head_size != 128) return fail(YL_ERR_UNSUPPORTED, "head_size must be 64 or 128");
  if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)))
    return fail(YL_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 256");
  if (n_kv_heads == 0 || n_kv_heads > 1024) return fail(YL_ERR_ARG, "n_kv_heads must be 1..1024");
  if (n_pages == 0 || n_pages > 0x7FFFFFFFu) return fail(YL_ERR_ARG, "n_pages must be 1..2^31-1");
  return YL_OK;
}

int make_pages(const yl_kv_pages* p, k::Pages* out) {
  if (!p || !p->k || !p->v) return fail(YL_ERR_ARG, "null cache");
  if (int rc = check_shape(p->dtype, p->n_pages, p->page_size, p->n_kv_heads, p->head_size)) return rc;
  const uint64_t per16 = 16 / dtype_size(p->dtype);
  const struct {
    uint64_t stride, n;
  } axes[3] = {{p->page_stride, p->n_pages}, {p->token_stride, p->page_size}, {p->head_stride, p->n_kv_heads}};
  for (const auto& ax : axes) {
    if (ax.stride % per16 || ax.stride >= (1ull << 36)) return fail(YL_ERR_ARG, "cache strides must be multiples of 16 bytes, below 2^36 elements");
    if (ax.n > 1 && ax.stride < p->head_size) return fail(YL_ERR_ARG, "cache strides smaller than head_size");
  }
  if (!aligned16(p->k) || !aligned16(p->v)) return fail(YL_ERR_ARG, "cache must be 16-byte aligned");
  *out = k::Pages{};
  out->k = p->k;
  out->v = p->v;
  out->n_pages = p->n_pages;
  while ((1u << out->page_shift) < p->page_size) ++out->page_shift;
  out->n_kv_heads = p->n_kv_heads;
  out->head_size = p->head_size;
  out->page_stride = p->page_stride;
  out->token_stride = p->token_stride;
  out->head_stride = p->head_stride;
  return YL_OK;
}

int make_seqs(const yl_seq_batch* b, const yl_kv_pages* p, k::Seqs* out) {
  if (!b) return fail(YL_ERR_ARG, "null batch");
  if (b->n_seqs == 0 || b->n_seqs > (1u << 20)) return fail(YL_ERR_ARG, "n_seqs must be 1..2^20");
  if (b->n_rows > (1u << 24)) return fail(YL_ERR_ARG, "more than 2^24 rows");
  if (b->table_stride == 0) return fail(YL_ERR_ARG, "empty page table");
  if (b->shared_len % p->page_size) return fail(YL_ERR_ARG, "shared_len must be a multiple of page_size");
  if (b->shared_len / p->page_size > b->table_stride) return fail(YL_ERR_RANGE, "shared_len longer than the page table");
  if (b->shared_len > k::MAX_POS) return fail(YL_ERR_RANGE, "shared_len beyond the last position");
  if (!b->row_start || !b->seq_len || !b->page_table) return fail(YL_ERR_ARG, "null batch array");
  if (((uintptr_t)b->row_start | (uintptr_t)b->seq_len | (uintptr_t)b->page_table | (uintptr_t)b->status) % 4)
    return fail(YL_ERR_ARG, "batch arrays must be 4-byte aligned");
  *out = k::Seqs{b->n_seqs, b->n_rows, b->table_stride, b->shared_len, b->row_start, b->seq_len, b->page_table,
                 b->status};
  return YL_OK;
}

int check_heads(uint32_t n_heads, uint32_t n_kv_heads) {
  if (n_heads == 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > 16)
    return fail(YL_ERR_UNSUPPORTED, "n_heads must be a multiple (at most 16x) of n_kv_heads");
  return YL_OK;
}

// Rows of a call's arrays; a call of no rows may have none.
int check_rows(const void* p, uint64_t stride, uint64_t width, uint64_t size, uint64_t n_rows, const char* what) {
  if (!p && n_rows) return fail(YL_ERR_ARG, std::string("null ") + what);
  if (stride < width || stride >= (1ull << 36)) return fail(YL_ERR_ARG, std::string(what) + ": row stride smaller than a row, or too large");
  if (!aligned16(p) || stride * size % 16) return fail(YL_ERR_ARG, std::string(what) + ": rows must be 16-byte aligned");
  return YL_OK;
}

int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return fail(YL_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return YL_OK;
}

int kv_pages_alloc(int dtype, uint32_t n_pages, uint32_t page_size, uint32_t n_kv_heads, uint32_t head_size,
                   yl_kv_pages* out) {
  if (!out) return fail(YL_ERR_ARG, "null output");
  if (int rc = check_shape(dtype, n_pages, page_size, n_kv_heads, head_size)) return rc;
  yl_kv_pages p{};
  p.dtype = dtype;
  p.n_pages = n_pages;
  p.page_size = page_size;
  p.n_kv_heads = n_kv_heads;
  p.head_size = head_size;
  p.head_stride = head_size;
  p.token_stride = (uint64_t)n_kv_heads * head_size;
  p.page_stride = page_size * p.token_stride;
  p.owned = 1;
  const uint64_t bytes = n_pages * p.page_stride * dtype_size(dtype);  // below 2^31 * 2^8 * 2^17 * 4 = 2^58
  cudaError_t e = cudaMalloc(&p.k, bytes);
  if (e == cudaSuccess) e = cudaMalloc(&p.v, bytes);
  if (e == cudaSuccess) e = cudaMemset(p.k, 0, bytes);
  if (e == cudaSuccess) e = cudaMemset(p.v, 0, bytes);
  // the zeros are there before a caller's stream, which does not wait for the
  // legacy one, writes tokens
  if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
  if (e != cudaSuccess) {
    cudaFree(p.k);
    cudaFree(p.v);
    (void)cudaGetLastError();
    return fail(e == cudaErrorMemoryAllocation ? YL_ERR_OOM : YL_ERR_CUDA,
                std::string("paged cache: ") + cudaGetErrorString(e));
  }
  *out = p;
  return YL_OK;
}

int append(void* q_out, uint64_t q_stride, const float* qkv, uint64_t qkv_stride, const yl_kv_pages* pages,
           const yl_seq_batch* batch, uint32_t n_heads, const float* rope_cs, uint32_t rope_len, int rope_mode,
           void* stream) {
  k::AppendArgs a{};
  if (int rc = make_pages(pages, &a.pages)) return rc;
  if (int rc = make_seqs(batch, pages, &a.seqs)) return rc;
  if (int rc = check_heads(n_heads, pages->n_kv_heads)) return rc;
  if (rope_mode != YL_ROPE_GGUF && rope_mode != YL_ROPE_LLAMA3) return fail(YL_ERR_ARG, "unknown rope mode");
  if (rope_cs && (!aligned16(rope_cs) || rope_len == 0)) return fail(YL_ERR_ARG, "rope table must be 16-byte aligned and not empty");
  const uint64_t hd = pages->head_size;
  if (int rc = check_rows(qkv, qkv_stride, ((uint64_t)n_heads + 2 * pages->n_kv_heads) * hd, 4, batch->n_rows, "qkv")) return rc;
  if (q_out)
    if (int rc = check_rows(q_out, q_stride, n_heads * hd, dtype_size(pages->dtype), batch->n_rows, "q_out")) return rc;
  if (batch->n_rows == 0) return YL_OK;
  a.qkv = qkv;
  a.qkv_stride = qkv_stride;
  a.q_out = q_out;
  a.q_stride = q_stride;
  a.n_heads = n_heads;
  a.cs = reinterpret_cast<const float2*>(rope_cs);
  a.rope_len = rope_len;
  a.rope_mode = rope_mode;
  return launched(k::paged_append(a, pages->dtype, (cudaStream_t)stream), "paged append");
}

int attention_workspace(const yl_kv_pages* pages, const yl_seq_batch* batch, uint32_t n_heads, k::PagedAttnArgs* a,
                        uint64_t* bytes) {
  if (int rc = make_pages(pages, &a->pages)) return rc;
  if (int rc = make_seqs(batch, pages, &a->seqs)) return rc;
  if (int rc = check_heads(n_heads, pages->n_kv_heads)) return rc;
  a->share = tunables().paged_share;
  *bytes = k::paged_attention_workspace(a->pages, a->seqs, pages->dtype, n_heads, a->share);
  return YL_OK;
}

int attention(void* output, uint64_t out_stride, int out_dtype, float* lse, const void* q, uint64_t q_stride,
              const yl_kv_pages* pages, const yl_seq_batch* batch, uint32_t n_heads, float attn_scale, void* workspace,
              uint64_t workspace_bytes, void* stream) {
  k::PagedAttnArgs a{};
  uint64_t need = 0;
  if (int rc = attention_workspace(pages, batch, n_heads, &a, &need)) return rc;
  if (out_dtype != YL_DT_F32 && out_dtype != pages->dtype)
    return fail(YL_ERR_UNSUPPORTED, "output must be f32 or of the cache's type");
  const uint64_t width = (uint64_t)n_heads * pages->head_size;
  if (int rc = check_rows(q, q_stride, width, dtype_size(pages->dtype), batch->n_rows, "q")) return rc;
  if (int rc = check_rows(output, out_stride, width, dtype_size(out_dtype), batch->n_rows, "output")) return rc;
  if ((uintptr_t)lse % 4) return fail(YL_ERR_ARG, "lse must be 4-byte aligned");
  if (!workspace || (uintptr_t)workspace % 256) return fail(YL_ERR_ARG, "workspace must be 256-byte aligned");
  if (workspace_bytes < need) return fail(YL_ERR_ARG, "workspace smaller than yl_paged_attention_workspace says");
  if (batch->n_rows == 0) return YL_OK;
  if ((uint64_t)batch->n_rows * n_heads > 0x7FFFFFFFull) return fail(YL_ERR_ARG, "more than 2^31-1 rows x heads");
  a.out = output;
  a.out_stride = out_stride;
  a.lse = lse;
  a.q = q;
  a.q_stride = q_stride;
  a.n_heads = n_heads;
  a.scale = attn_scale;
  a.workspace = workspace;
  return launched(k::paged_attention(a, pages->dtype, out_dtype == YL_DT_F32, (cudaStream_t)stream),
                  "paged attention");
}

int logprobs(const void* logits, int dtype, uint64_t row_stride, uint32_t n_rows, uint32_t vocab,
             const int32_t* tokens, float* logprobs, float* entropy, uint32_t top_k, int32_t* top_ids,
             float* top_logprobs, void* stream) {
  const uint64_t size = dtype_size(dtype);
  if (!size) return fail(YL_ERR_ARG, "unknown element type");
  if (vocab == 0 || vocab > 0x7FFFFFFFu) return fail(YL_ERR_ARG, "vocab must be 1..2^31-1");
  if (n_rows > (1u << 24)) return fail(YL_ERR_ARG, "more than 2^24 rows");
  if (row_stride < vocab || row_stride >= (1ull << 36)) return fail(YL_ERR_ARG, "row stride smaller than a row, or too large");
  if (top_k > k::LP_MAX_TOP) return fail(YL_ERR_UNSUPPORTED, "top_k must be at most 32");
  if (top_k > vocab) return fail(YL_ERR_ARG, "top_k larger than the vocabulary");
  if ((!logits && n_rows) || (uintptr_t)logits % size) return fail(YL_ERR_ARG, "logits null or not aligned to their type");
  if (n_rows && !tokens != !logprobs) return fail(YL_ERR_ARG, "tokens and logprobs go together");
  if (n_rows && top_k && (!top_ids || !top_logprobs)) return fail(YL_ERR_ARG, "top_k needs top_ids and top_logprobs");
  if (((uintptr_t)tokens | (uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_logprobs) % 4)
    return fail(YL_ERR_ARG, "outputs and tokens must be 4-byte aligned");
  if (n_rows == 0) return YL_OK;
  k::LogprobArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.n_rows = n_rows;
  a.vocab = vocab;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_k = top_k;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  return launched(k::token_logprobs(a, dtype, (cudaStream_t)stream), "token logprobs");
}

}  // namespace

extern "C" {

int yl_kv_pages_alloc(int dtype, uint32_t n_pages, uint32_t page_size, uint32_t n_kv_heads, uint32_t head_size,
                      yl_kv_pages* out) {
  return guarded([&] { return kv_pages_alloc(dtype, n_pages, page_size, n_kv_heads, head_size, out); });
}

int yl_kv_pages_free(yl_kv_pages* p) {
  if (!p) return fail(YL_ERR_ARG, "null cache");
  if (p->owned) {
    cudaFree(p->k);
    cudaFree(p->v);
  }
  p->k = p->v = nullptr;
  return YL_OK;
}

int yl_paged_append(void* q_out, uint64_t q_stride, const float* qkv, uint64_t qkv_stride, const yl_kv_pages* pages,
                    const yl_seq_batch* batch, uint32_t n_heads, const float* rope_cs, uint32_t rope_len,
                    int rope_mode, void* stream) {
  return guarded([&] {
    return append(q_out, q_stride, qkv, qkv_stride, pages, batch, n_heads, rope_cs, rope_len, rope_mode, stream);
  });
}

int yl_paged_attention_workspace(const yl_kv_pages* pages, const yl_seq_batch* batch, uint32_t n_heads,
                                 uint64_t* bytes) {
  if (!bytes) return fail(YL_ERR_ARG, "null output");
  k::PagedAttnArgs a{};
  return guarded([&] { return attention_workspace(pages, batch, n_heads, &a, bytes); });
}

int yl_paged_attention(void* output, uint64_t out_stride, int out_dtype, float* lse, const void* q, uint64_t q_stride,
                       const yl_kv_pages* pages, const yl_seq_batch* batch, uint32_t n_heads, float attn_scale,
                       void* workspace, uint64_t workspace_bytes, void* stream) {
  return guarded([&] {
    return attention(output, out_stride, out_dtype, lse, q, q_stride, pages, batch, n_heads, attn_scale, workspace,
                     workspace_bytes, stream);
  });
}

int yl_token_logprobs(const void* logits, int dtype, uint64_t row_stride, uint32_t n_rows, uint32_t vocab,
                      const int32_t* tokens, float* lp, float* entropy, uint32_t top_k, int32_t* top_ids,
                      float* top_logprobs, void* stream) {
  return guarded([&] {
    return logprobs(logits, dtype, row_stride, n_rows, vocab, tokens, lp, entropy, top_k, top_ids, top_logprobs,
                    stream);
  });
}

int yl_model_rope(const yl_model* m, const float** rope_cs, uint32_t* len) {
  if (!m || !rope_cs || !len) return fail(YL_ERR_ARG, "null argument");
  *rope_cs = reinterpret_cast<const float*>(m->m->rope_cs);
  *len = m->m->shape.ctx_len;
  return YL_OK;
}

int yl_batch_logits(const yl_batch* b, float** logits) {
  if (!b || !logits) return fail(YL_ERR_ARG, "null argument");
  *logits = b->b->logits;
  return YL_OK;
}

}  // extern "C"
