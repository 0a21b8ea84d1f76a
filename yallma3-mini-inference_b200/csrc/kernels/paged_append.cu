// Appending rows to the paged cache: rotates queries and keys by their
// positions, rounds to the cache's type and scatters keys and values to their
// page slots, in one pass over the projection's output.
//   a' = a*c - b*s,  b' = a*s + b*c   for the pair (a, b) and the position's (c, s)
// Bound by memory: every f32 of qkv is read once and written once in the
// cache's type; a thread moves 16 elements of a head (64 bytes in), which are
// eight whole pairs in either pairing, so no value is exchanged between
// threads. One block per row: the row's sequence, position and page are looked
// up once per warp, after the row's loads are in flight. Measured on one B200:
// 7000 rows of 32+2x8 heads of 128 into f16 48.7 us (271 MB, 85 % of a copy's
// rate); 64 rows 3.2 us, one row 2.2 us (launch and three dependent lookups).
#include "serve.cuh"

namespace yl {
namespace k {
using namespace yl::dev;

namespace {

// Every product and sum rounded by itself, as in the other kernels: an f32 cache
// gets the bits that a session's own cache has.
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float a0 = a;
  a = __fsub_rn(__fmul_rn(a0, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(a0, s), __fmul_rn(b, c));
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                                pack2<T>(v[6], v[7]));
  }
}

// Elements [lo, lo+8) and [hi, hi+8) of a head: neighbours in a row when the
// pairs are (2j, 2j+1), half a head apart when they are (j, j + hd/2).
template <typename T, int HD, bool HALF>
__global__ void append_kernel(AppendArgs a) {
  constexpr uint32_t UNITS = HD / 16;
  const uint32_t row = blockIdx.x, lane = threadIdx.x & 31;
  const uint32_t first_head = a.q_out ? 0 : a.n_heads;
  const uint32_t nu = (a.n_heads + 2 * a.pages.n_kv_heads) * UNITS;
  const float* src = a.qkv + (uint64_t)row * a.qkv_stride;
  uint32_t u = first_head * UNITS + threadIdx.x;
  float x[8], y[8];
  auto load = [&](uint32_t unit) {
    const uint32_t j = unit % UNITS;
    const float* h = src + (uint64_t)(unit / UNITS) * HD;
    const float* lo = h + (HALF ? 8 * j : 16 * j);
    const float* hi = lo + (HALF ? HD / 2 : 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 p = __ldcs(reinterpret_cast<const float4*>(lo) + i);
      const float4 q = __ldcs(reinterpret_cast<const float4*>(hi) + i);
      x[4 * i] = p.x, x[4 * i + 1] = p.y, x[4 * i + 2] = p.z, x[4 * i + 3] = p.w;
      y[4 * i] = q.x, y[4 * i + 1] = q.y, y[4 * i + 2] = q.z, y[4 * i + 3] = q.w;
    }
  };
  const bool padding = row >= row_begin(a.seqs, a.seqs.n_seqs);
  if (padding) return;
  if (u < nu) load(u);
  const uint32_t seq = warp_find_seq(a.seqs, row, lane);
  if (seq == a.seqs.n_seqs) return;  // between row_start entries that are out of order
  const uint32_t back = row_end(a.seqs, seq) - row, len = a.seqs.seq_len[seq];
  // before position 0, or beyond the rotation table: the row has no place
  const bool placed = len >= back && (!a.cs || len - back < a.rope_len);
  const uint32_t pos = len - back;
  const uint32_t page = placed ? page_of(a.seqs, a.pages, seq, pos) : NO_PAGE;
  if (page == NO_PAGE && threadIdx.x == 0 && a.seqs.status) *a.seqs.status = STATUS_RANGE;
  if (!placed) return;
  for (; u < nu; u += blockDim.x) {
    if (u >= first_head * UNITS + blockDim.x) load(u);
    const uint32_t head = u / UNITS, j = u % UNITS;
    if (a.cs && head < a.n_heads + a.pages.n_kv_heads) {
      const float4* cs = reinterpret_cast<const float4*>(a.cs + (uint64_t)pos * (HD / 2) + 8 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 t = cs[i];  // two (cos, sin)
        if (HALF) {
          rotate(x[2 * i], y[2 * i], t.x, t.y);
          rotate(x[2 * i + 1], y[2 * i + 1], t.z, t.w);
        } else {
          float* v = i < 2 ? x + 4 * i : y + 4 * (i - 2);
          rotate(v[0], v[1], t.x, t.y);
          rotate(v[2], v[3], t.z, t.w);
        }
      }
    }
    T* dst;
    if (head < a.n_heads) {
      dst = static_cast<T*>(a.q_out) + (uint64_t)row * a.q_stride + (uint64_t)head * HD;
    } else {
      if (page == NO_PAGE) continue;
      const uint32_t kvh = head - a.n_heads;
      dst = kvh < a.pages.n_kv_heads
                ? static_cast<T*>(a.pages.k) + slot_offset(a.pages, page, pos, kvh)
                : static_cast<T*>(a.pages.v) + slot_offset(a.pages, page, pos, kvh - a.pages.n_kv_heads);
    }
    store8<T>(dst + (HALF ? 8 * j : 16 * j), x);
    store8<T>(dst + (HALF ? 8 * j + HD / 2 : 16 * j + 8), y);
  }
}

template <typename T, int HD>
cudaError_t launch(const AppendArgs& a, cudaStream_t stream) {
  const uint32_t heads = (a.q_out ? a.n_heads : 0) + 2 * a.pages.n_kv_heads;
  const uint32_t units = heads * (HD / 16);
  const uint32_t threads = units >= 512 ? 512 : (units + 31) / 32 * 32;
  LaunchCfg lc;
  lc.stream = stream;
  return a.rope_mode ? launch_kernel(append_kernel<T, HD, true>, dim3(a.seqs.n_rows), dim3(threads), 0, lc, a)
                     : launch_kernel(append_kernel<T, HD, false>, dim3(a.seqs.n_rows), dim3(threads), 0, lc, a);
}

}  // namespace

cudaError_t paged_append(const AppendArgs& a, int dtype, cudaStream_t stream) {
  const bool wide = a.pages.head_size == 128;
  switch (dtype) {
    case DT_F32: return wide ? launch<float, 128>(a, stream) : launch<float, 64>(a, stream);
    case DT_F16: return wide ? launch<__half, 128>(a, stream) : launch<__half, 64>(a, stream);
    default: return wide ? launch<__nv_bfloat16, 128>(a, stream) : launch<__nv_bfloat16, 64>(a, stream);
  }
}

}  // namespace k
}  // namespace yl
