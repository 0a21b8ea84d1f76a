// What the paged-attention kernels share: how a call's work is laid out on a
// line and cut into pieces (paged_attention.cu tells why), and the page loads.
#pragma once
#include <atomic>
#include <cfloat>
#include <type_traits>

#include "serve.cuh"
#include "tc.cuh"

namespace yl {
namespace k {

constexpr float LN2 = 0.6931471805599453f;
constexpr int STATUS_TIMEOUT = -7;  // YL_ERR_TIMEOUT

// One launch: over the sequences' own keys (from `from` on), or over the
// shared prefix with all rows as one sequence. A sequence whose rows do not all
// see the whole prefix (starts_inside) has all of its keys in the first.
struct Pass {
  PagedAttnArgs a;
  int dtype;
  // scores in powers of two are |scale| log2(e) (a product with q, negated where
  // the scale is negative), as the sum of two f32
  float sc, sc_lo;
  uint32_t flip;
  uint32_t from, prefix;  // first key; 1: the prefix pass (keys 0 .. shared_len)
  uint32_t group, min_chunk;
  uint32_t grid;   // blocks
  uint32_t item_cost;  // an item's own cost in key tiles (queries, first tile, output), when the line is cut
  int joined;      // every item leaves its part in the workspace
  uint4* cut;      // [grid]: the item that begins in a block and goes on in the next {first row, tokens, head, blocks}
  uint2* desc;     // joined: [n_rows][n_kv_heads] {first block, blocks << 16 | token in the tile}
  float* slots;    // [2 * grid][BM][HD + 8]: a part is O, m (in powers of two), l
  float* rowpart;  // [n_rows][n_heads][HD + 8]: items of one block, where every item leaves its part
};

template <int HD>
constexpr uint32_t PART = HD + 8;  // floats of a part, a multiple of 32 bytes
constexpr uint32_t TC_TILE = 256;  // rows of an item of attend_tc

// The pass on the 5th-generation tensor cores: items of up to TC_TILE rows,
// 16-bit types, one block per SM (paged_attention_tc.cu).
cudaError_t attend_tc(const Pass& p, bool out_f32, const LaunchCfg& lc);

// Sets a kernel's dynamic shared memory once per device.
template <typename F>
cudaError_t allow_smem(std::atomic<uint64_t>& ready, F* kernel, uint32_t bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (ready.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

namespace {
using namespace yl::dev;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A part (m, l, O) of a row that sees none of its keys has m = -inf and l = 0. One
// whose scores are all below f32's range has l = 0 too; its m is this, below any
// score, so that it weighs nothing next to other parts, and alone gives NaN.
constexpr float BELOW = -FLT_MAX;
__device__ __forceinline__ float settled(float m, float l) { return l == 0.0f && m != -INFINITY ? NAN : l; }
// 4-D tiled load of a page's part: (element, head, token in the page, page).
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t head, uint32_t tok,
                                         uint32_t page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(tok), "r"(page), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// ---- work ------------------------------------------------------------------
// A sequence as a pass sees it.
struct Rows {
  uint32_t row0, n;  // its rows
  int64_t pos0;      // position of the first
  uint32_t limit;    // keys that may be read: the prefix, or what the page table has slots for
};
__device__ __forceinline__ Rows rows_of(const Pass& p, uint32_t i) {
  const Seqs& s = p.a.seqs;
  Rows r;
  if (p.prefix) {
    r.row0 = row_begin(s, 0);
    const uint32_t e = row_begin(s, s.n_seqs);
    r.n = e > r.row0 ? e - r.row0 : 0;
    r.pos0 = 0;
    r.limit = s.shared_len;
  } else {
    r.row0 = row_begin(s, i);
    r.n = row_end(s, i) - r.row0;
    r.pos0 = (int64_t)s.seq_len[i] - r.n;
    r.limit = table_limit(s, p.a.pages);
  }
  return r;
}
// First key of the pass for these rows.
__device__ __forceinline__ uint32_t keys_begin(const Pass& p, const Rows& r) {
  return p.from && r.pos0 + 1 < (int64_t)p.from ? 0 : p.from;
}
// First key behind those that tokens [.., t) of the sequence see.
__device__ __forceinline__ uint32_t keys_end(const Pass& p, const Rows& r, uint32_t t) {
  if (p.prefix) return r.limit;
  const int64_t e = r.pos0 + (t < r.n ? t : r.n);
  return e <= 0 ? 0 : e < (int64_t)r.limit ? (uint32_t)e : r.limit;
}
// Key tiles of the row tile that ends at token t (one where it sees no key). On
// the line it takes item_cost units more, before its first tile.
template <typename S>
__device__ __forceinline__ uint32_t tiles_of(const Pass& p, const Rows& r, uint32_t t) {
  const uint32_t b = keys_begin(p, r), e = keys_end(p, r, t);
  return e > b + S::KT ? (e - b + S::KT - 1) / S::KT : 1;
}
__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ Rows rows_from_lane(const Rows& r, int src) {
  return Rows{__shfl_sync(FULL, r.row0, src), __shfl_sync(FULL, r.n, src), __shfl_sync(FULL, r.pos0, src),
              __shfl_sync(FULL, r.limit, src)};
}
// Units of a sequence on the line, per head; every lane its own sequence. Those
// of many row tiles (long prompts) are counted by the whole warp, in turn.
template <typename S>
__device__ __forceinline__ uint64_t units_per_head(const Pass& p, const Rows& r, uint32_t tpt, uint32_t lane) {
  const uint32_t tiles = (r.n + tpt - 1) / tpt;
  if (p.prefix) return (uint64_t)tiles * (tiles_of<S>(p, r, r.n) + p.item_cost);
  uint64_t n = 0;
  if (tiles <= 4)
#pragma unroll 1
    for (uint32_t t = 0; t < r.n; t += tpt) n += tiles_of<S>(p, r, t + tpt) + p.item_cost;
  for (uint32_t many = __ballot_sync(FULL, tiles > 4); many; many &= many - 1) {
    const int src = __ffs(many) - 1;
    const Rows w = rows_from_lane(r, src);
    uint64_t part = 0;
#pragma unroll 1
    for (uint32_t t = lane * tpt; t < w.n; t += 32 * tpt) part += tiles_of<S>(p, w, t + tpt) + p.item_cost;
    part = warp_sum_u64(part);
    if ((int)lane == src) n = part;
  }
  return n;
}

// Where a block's piece of the line begins.
struct Start {
  uint64_t begin, end, chunk;  // on the line
  uint32_t seq, head, t;       // sequence, head, first token of the row tile
  uint64_t g0;                 // where the item begins on the line
  int masked;                  // prefix pass: some sequence is left to the other pass
};

// a / b; 64-bit division is a long piece of code that hardly ever runs.
__device__ __noinline__ uint64_t div_long(uint64_t a, uint64_t b) { return a / b; }
__device__ __forceinline__ uint64_t div(uint64_t a, uint64_t b) {
  return (a | b) >> 32 ? div_long(a, b) : (uint32_t)a / (uint32_t)b;
}

// All threads. The sequences' units are summed a block's width at a time, once
// for the total and once more to find the piece's place, which is found at once
// where one width holds all sequences, as it mostly does. (Rolled loops: this
// runs once, and a launch between other kernels waits for every instruction.)
template <typename S>
__device__ void find_start(const Pass& p, uint32_t tpt, Start* out, uint64_t* scratch) {
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t n = p.prefix ? 1 : p.a.seqs.n_seqs;
  constexpr uint32_t NWARPS = S::THREADS / 32;
  bool masked = false;
  if (p.prefix)
#pragma unroll 1
    for (uint32_t i = tid; i < p.a.seqs.n_seqs; i += S::THREADS) masked |= starts_inside(p.a.seqs, i);
  if (tid == 0) out->seq = 0xFFFFFFFFu;
  Rows r{};
  uint64_t per_head = 0, mine = 0, first = 0;  // this thread's sequence of the width: units, and where they begin
  uint64_t total = 0, begin = 0, end = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    uint64_t base = 0;
#pragma unroll 1
    for (uint32_t c = 0; c < n; c += S::THREADS) {
      if (pass == 0 || n > S::THREADS) {
        r = c + tid < n ? rows_of(p, c + tid) : Rows{};
        per_head = units_per_head<S>(p, r, tpt, lane);
        mine = per_head * p.a.pages.n_kv_heads;
        uint64_t inc = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t v = __shfl_up_sync(FULL, inc, o);
          if ((int)lane >= o) inc += v;
        }
        __syncthreads();
        if (lane == 31) scratch[warp] = inc;
        __syncthreads();
        first = base + inc - mine;
#pragma unroll 1
        for (uint32_t w = 0; w < NWARPS; ++w) {
          if (w < warp) first += scratch[w];
          base += scratch[w];
        }
      }
      if (pass == 0) continue;
      const uint32_t here = __ballot_sync(FULL, begin >= first && begin < first + mine);
      if (!here) continue;
      // in one of this warp's sequences: all lanes look for the row tile
      const int src = __ffs(here) - 1;
      const Rows w = rows_from_lane(r, src);
      const uint64_t each = __shfl_sync(FULL, per_head, src);
      uint64_t g0 = __shfl_sync(FULL, first, src), off = begin - g0;
      const uint32_t h = (uint32_t)div(off, each);
      off -= h * each;
      g0 += h * each;
      uint32_t t = 0;
      if (p.prefix) {
        const uint32_t units = tiles_of<S>(p, w, w.n) + p.item_cost, k = (uint32_t)div(off, units);
        t = k * tpt;
        g0 += (uint64_t)k * units;
      } else if (w.n > tpt) {
#pragma unroll 1
        while (t < w.n) {  // 32 row tiles at a time
          const uint32_t mt = t + lane * tpt;
          const uint32_t units = mt < w.n ? tiles_of<S>(p, w, mt + tpt) + p.item_cost : 0;
          uint64_t upto = units;
#pragma unroll 1
          for (int o = 1; o < 32; o <<= 1) {
            const uint64_t v = __shfl_up_sync(FULL, upto, o);
            if ((int)lane >= o) upto += v;
          }
          const uint32_t in = __ballot_sync(FULL, upto > off);
          if (in) {
            const int k = __ffs(in) - 1;
            t += k * tpt;
            g0 += __shfl_sync(FULL, upto - units, k);
            break;
          }
          const uint64_t all = __shfl_sync(FULL, upto, 31);
          off -= all;
          g0 += all;
          t += 32 * tpt;
        }
      }
      if (lane == 0) {
        if (end > g0 + p.item_cost) out->seq = c + warp * 32 + src;  // else the piece ends before the item's first tile
        out->head = h;
        out->t = t;
        out->g0 = g0;
      }
    }
    if (pass == 0) {
      total = base;
      uint64_t chunk = div(total + gridDim.x - 1, gridDim.x);
      if (chunk < p.min_chunk) chunk = p.min_chunk;
      begin = chunk * blockIdx.x;
      end = begin + chunk < total ? begin + chunk : total;
      if (tid == 0) out->chunk = chunk, out->begin = begin, out->end = end;
      if (begin >= total) break;  // nothing for this block
    }
  }
  // (also the barrier that makes *out visible)
  out->masked = __syncthreads_or(masked);
}

// Walks a block's piece: one step per item that has key tiles in it, the same
// in every warp.
template <typename S>
struct Walk {
  const Pass& p;
  const uint32_t tpt;
  uint64_t begin, end, chunk, g0;
  uint32_t seq, head, t, kt0, kt1, nt;
  Rows r;

  __device__ Walk(const Pass& pass, uint32_t tokens, const Start& s)
      : p(pass), tpt(tokens), begin(s.begin), end(s.end), chunk(s.chunk), g0(s.g0), seq(s.seq), head(s.head), t(s.t) {
    r = rows_of(p, seq);
    nt = tiles_of<S>(p, r, t + tpt);
    cut();
  }
  // The item's key tiles within the piece: units [g0 + item_cost, + nt).
  __device__ bool cut() {
    const uint64_t first = g0 + p.item_cost;
    kt0 = begin > first ? (uint32_t)(begin - first) : 0;
    kt1 = end > first ? (uint32_t)(end - first < nt ? end - first : nt) : 0;
    return kt0 < kt1;
  }
  __device__ bool next() {
    g0 += nt + p.item_cost;
    if (g0 >= end) return false;
    t += tpt;
    if (t >= r.n) {
      t = 0;
      if (++head == p.a.pages.n_kv_heads) {
        head = 0;
        do {
          if (++seq >= p.a.seqs.n_seqs || p.prefix) return false;
          r = rows_of(p, seq);
        } while (r.n == 0);
      }
    }
    nt = tiles_of<S>(p, r, t + tpt);
    return cut();
  }
  __device__ uint32_t tokens() const { return r.n - t < tpt ? r.n - t : tpt; }
  __device__ uint32_t kbegin() const { return keys_begin(p, r) + kt0 * S::KT; }  // of the piece
  __device__ uint32_t kend() const { return keys_end(p, r, t + tpt); }
  // All of the item lies in this block; else how many blocks it lies in, this
  // one, where it begins, the first.
  __device__ bool whole() const { return kt1 - kt0 == nt; }
  __device__ uint32_t blocks() const {
    return kt1 == nt ? 1 : 1 + (uint32_t)div(g0 + p.item_cost + nt - end + chunk - 1, chunk);
  }
};

// Whether the prefix pass leaves this row to the other one (the row's sequence by bisection).
__device__ __forceinline__ bool left_out(const Seqs& s, uint32_t row) {
  uint32_t lo = 0, hi = s.n_seqs;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (row_begin(s, mid) <= row) lo = mid;
    else hi = mid;
  }
  return starts_inside(s, lo);
}

// (element, head, token, page), boxes of 128 bytes x 1 x `tokens` x 1, swizzled.
inline bool encode_pages(CUtensorMap* m, const Pages& p, void* base, int dtype, uint32_t tokens) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const uint64_t size = dtype == DT_F32 ? 4 : 2, ps = 1ull << p.page_shift;
  const cuuint64_t dims[4] = {p.head_size, p.n_kv_heads, ps, p.n_pages};
  // an axis of one entry has no stride to speak of
  auto bytes = [&](uint64_t stride, uint64_t n) { return (n > 1 ? stride : p.head_size) * size; };
  const cuuint64_t strides[3] = {bytes(p.head_stride, p.n_kv_heads), bytes(p.token_stride, ps),
                                 bytes(p.page_stride, p.n_pages)};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / size), 1, tokens, 1}, estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t = dtype == DT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : dtype == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return fn(m, t, 4, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}


}  // namespace
}  // namespace k
}  // namespace yl
