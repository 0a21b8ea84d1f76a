// Causal grouped-query attention over the paged cache. One block per (row,
// head): each of its warps takes every fourth key, keeps a running maximum,
// sum and output, and the warps' parts are joined at the end.
#include "serve.cuh"

namespace yl {
namespace k {
using namespace yl::dev;

namespace {

template <typename T, typename O, int HD>
__global__ void __launch_bounds__(128) attend_kernel(PagedAttnArgs a) {
  constexpr int PER = HD / 32;
  __shared__ float part[4][HD + 2];
  const uint32_t row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t seq = warp_find_seq(a.seqs, row, lane);
  if (seq == a.seqs.n_seqs) return;
  const uint32_t back = row_end(a.seqs, seq) - row, len = a.seqs.seq_len[seq];
  const uint32_t keys = len >= back ? len - back + 1 : 0;
  const uint32_t kvh = head / (a.n_heads / a.pages.n_kv_heads);
  const T* q = static_cast<const T*>(a.q) + (uint64_t)row * a.q_stride + (uint64_t)head * HD;
  float qv[PER], o[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) qv[i] = to_f32(q[lane + 32 * i]) * a.scale, o[i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  for (uint32_t j = warp; j < keys; j += 4) {
    const uint32_t page = page_of(a.seqs, a.pages, j < a.seqs.shared_len ? 0 : seq, j);
    float kv[PER], vv[PER], s = 0.0f;
    if (page == NO_PAGE) {
      if (a.seqs.status) *a.seqs.status = STATUS_RANGE;
#pragma unroll
      for (int i = 0; i < PER; ++i) kv[i] = vv[i] = 0.0f;
    } else {
      const uint64_t at = slot_offset(a.pages, page, j, kvh);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        kv[i] = to_f32(static_cast<const T*>(a.pages.k)[at + lane + 32 * i]);
        vv[i] = to_f32(static_cast<const T*>(a.pages.v)[at + lane + 32 * i]);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) s += qv[i] * kv[i];
    s = warp_sum(s);
    const float top = fmaxf(m, s), f = m == -INFINITY ? 0.0f : expf(m - top), p = expf(s - top);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = o[i] * f + p * vv[i];
    m = top;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) part[warp][lane + 32 * i] = o[i];
  if (lane == 0) part[warp][HD] = m, part[warp][HD + 1] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.0f, f[4];
  for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][HD]);
  for (int w = 0; w < 4; ++w) {
    f[w] = part[w][HD] == -INFINITY ? 0.0f : expf(part[w][HD] - top);
    sum += f[w] * part[w][HD + 1];
  }
  for (uint32_t d = threadIdx.x; d < HD; d += 128) {
    float v = 0.0f;
    for (int w = 0; w < 4; ++w) v += f[w] * part[w][d];
    static_cast<O*>(a.out)[(uint64_t)row * a.out_stride + (uint64_t)head * HD + d] =
        from_f32<O>(keys ? v / sum : 0.0f);
  }
  if (threadIdx.x == 0 && a.lse)
    a.lse[(uint64_t)row * a.n_heads + head] = keys ? top + logf(sum) : -INFINITY;
}

template <typename T, typename O>
cudaError_t launch(const PagedAttnArgs& a, cudaStream_t stream) {
  const dim3 grid(a.seqs.n_rows, a.n_heads);
  LaunchCfg lc;
  lc.stream = stream;
  return a.pages.head_size == 128 ? launch_kernel(attend_kernel<T, O, 128>, grid, dim3(128), 0, lc, a)
                                  : launch_kernel(attend_kernel<T, O, 64>, grid, dim3(128), 0, lc, a);
}

}  // namespace

cudaError_t paged_attention(const PagedAttnArgs& a, int dtype, bool out_f32, cudaStream_t stream) {
  if (dtype == DT_F32) return launch<float, float>(a, stream);
  if (dtype == DT_F16) return out_f32 ? launch<__half, float>(a, stream) : launch<__half, __half>(a, stream);
  return out_f32 ? launch<__nv_bfloat16, float>(a, stream) : launch<__nv_bfloat16, __nv_bfloat16>(a, stream);
}

uint64_t paged_attention_workspace(const Pages&, const Seqs&, int, uint32_t) { return 256; }

}  // namespace k
}  // namespace yl
