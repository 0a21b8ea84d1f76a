// Host-visible interface of the serving kernels: appending to a paged
// key/value cache, attention over it, token log probabilities. Every wrapper
// enqueues on `stream` and returns the launch error. The index arithmetic that
// decides which cache rows a kernel may touch is inline here, for host and
// device, so that it can be checked without a GPU.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#if defined(__CUDACC__)
#define YL_SHD __host__ __device__ __forceinline__
#else
#define YL_SHD inline
#endif

namespace yl {
namespace k {

enum Dt : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };

// One layer's paged cache (yl_kv_pages); strides in elements.
struct Pages {
  void* k;
  void* v;
  uint32_t n_pages, page_shift, n_kv_heads, head_size;
  uint64_t page_stride, token_stride, head_stride;
};

// The sequences of a call (yl_seq_batch).
struct Seqs {
  uint32_t n_seqs, n_rows, table_stride, shared_len;
  const uint32_t* row_start;
  const uint32_t* seq_len;
  const uint32_t* page_table;
  int* status;
};

constexpr uint32_t SMS = 148;  // of a B200; grids are cut for it
constexpr uint32_t NO_PAGE = 0xFFFFFFFFu;
constexpr int STATUS_RANGE = -6;  // YL_ERR_RANGE

// Row range of a sequence: row_start limited to n_rows and to ascending order
// of each pair, whatever the caller's array holds.
YL_SHD uint32_t row_begin(const Seqs& s, uint32_t i) {
  const uint32_t r = s.row_start[i];
  return r < s.n_rows ? r : s.n_rows;
}
YL_SHD uint32_t row_end(const Seqs& s, uint32_t i) {
  const uint32_t b = row_begin(s, i), e = row_begin(s, i + 1);
  return e > b ? e : b;
}
// Whether some row of the sequence does not see the whole shared prefix. Such a
// sequence is attended to by itself: the keys of the prefix behind its end are
// other sequences', or nobody's yet, and a weight of 0 does not hide a value
// that is not finite.
YL_SHD bool starts_inside(const Seqs& s, uint32_t i) {
  const uint32_t n = row_end(s, i) - row_begin(s, i);
  return n && (int64_t)s.seq_len[i] - n + 1 < (int64_t)s.shared_len;
}
// Positions from here on are no positions: kernels count keys, and those of the
// tile they are in, in 31 bits.
constexpr uint32_t MAX_POS = 0x7FFFFF00u;
// Positions that the page table has slots for.
YL_SHD uint32_t table_limit(const Seqs& s, const Pages& p) {
  const uint64_t n = (uint64_t)s.table_stride << p.page_shift;
  return n < MAX_POS ? (uint32_t)n : MAX_POS;
}
// Page that holds position pos of sequence seq, or NO_PAGE where the table
// has no slot for it or its entry is no page.
YL_SHD uint32_t page_of(const Seqs& s, const Pages& p, uint32_t seq, uint32_t pos) {
  const uint32_t slot = pos >> p.page_shift;
  if (slot >= s.table_stride || pos >= MAX_POS) return NO_PAGE;
  const uint32_t id = s.page_table[(uint64_t)seq * s.table_stride + slot];
  return id < p.n_pages ? id : NO_PAGE;
}
// Element offset of (page, position, head) in k and v.
YL_SHD uint64_t slot_offset(const Pages& p, uint32_t page, uint32_t pos, uint32_t head) {
  return (uint64_t)page * p.page_stride + (uint64_t)(pos & ((1u << p.page_shift) - 1)) * p.token_stride +
         (uint64_t)head * p.head_stride;
}

struct AppendArgs {
  Pages pages;
  Seqs seqs;
  const float* qkv;
  uint64_t qkv_stride;
  void* q_out;  // nullable
  uint64_t q_stride;
  uint32_t n_heads;
  const float2* cs;  // [rope_len][head_size/2], nullable
  uint32_t rope_len;
  int rope_mode;  // yl_rope_mode
};
cudaError_t paged_append(const AppendArgs& a, int dtype, cudaStream_t stream);

struct PagedAttnArgs {
  Pages pages;
  Seqs seqs;
  void* out;
  uint64_t out_stride;
  float* lse;  // nullable
  const void* q;
  uint64_t q_stride;
  uint32_t n_heads;
  float scale;
  int share;  // a pass of its own for the shared prefix: -1 where it pays, 0 never, 1 wherever it can be
  void* workspace;
};
cudaError_t paged_attention(const PagedAttnArgs& a, int dtype, bool out_f32, cudaStream_t stream);
uint64_t paged_attention_workspace(const Pages& p, const Seqs& s, int dtype, uint32_t n_heads, int share);

struct LogprobArgs {
  const void* logits;
  uint64_t row_stride;
  uint32_t n_rows, vocab;
  const int32_t* tokens;  // nullable, with logprobs
  float* logprobs;
  float* entropy;  // nullable
  uint32_t top_k;  // 0..LP_MAX_TOP
  int32_t* top_ids;
  float* top_logprobs;
};
constexpr uint32_t LP_MAX_TOP = 32;
cudaError_t token_logprobs(const LogprobArgs& a, int dtype, cudaStream_t stream);

}  // namespace k
}  // namespace yl
