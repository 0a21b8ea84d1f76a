// Log probabilities of given tokens, entropy and the most likely tokens of
// rows of logits, in one pass over each row.
//
// With m = max x: S = sum of exp(x_i - m) and W = sum of exp(x_i - m) (x_i - m) give
//   logprob(t) = (x_t - m) - log S,  entropy = log S - W / S.
// Parts (m_i, S_i, W_i) of the threads, then of the blocks, join under the
// largest m: with d = m_i - m, S = sum of e^d S_i, W = sum of e^d (W_i + d S_i).
// S is 1 + S', S' the sum without the largest term, and log S = log1p(S'). So that
// log probabilities near 0 keep their digits, the sum of the one thread that has
// the 1 joins the others' without it, and, where S' is below 1/2, is taken again
// from that thread's values. What is left beside a likely token are often a few
// terms far below it. Each of them is the largest its thread has, as a
// rule, so the factors e^d of the parts are taken with differences and products
// in two f32 (the rounding of d log2(e) = -40 alone is 2^-19.5), a thread's own
// terms with one.
//
// Most likely tokens: every thread knows the largest of the values it reads.
// The k-th largest of the threads' maxima bounds the k-th largest value from
// below, and only the k threads at or above it can hold one of the k largest,
// so only their values (a few per cent of the row) are read a second time.
// Values are compared as 64-bit keys, (value in integer order, ~index), which
// are distinct, so that equals go to the lower index and nothing depends on
// the order of atomics.
//
// Bound by reading the row (4 bytes and one exponential per value): 1999 rows of
// 128256 f32 in 186 us on one B200 (5.5 TB/s); 64 rows with 20 alternatives 16 us
// (from L2; the join and the choice of the largest take about 8), one row 6.4 us.
// A row is read by a thread-block cluster of 1..8 blocks, more for few rows, so
// that one row of a large vocabulary does not wait for one SM; its parts are
// joined over distributed shared memory.
#include <cooperative_groups.h>

#include "serve.cuh"

namespace cg = cooperative_groups;

namespace yl {
namespace k {
using namespace yl::dev;

namespace {

constexpr uint32_t LP_THREADS = 256;
constexpr uint32_t LP_WARPS = LP_THREADS / 32;
constexpr uint32_t LP_CAND = 1024;  // candidates ranked at once

__device__ __forceinline__ uint64_t key_of(float x, uint32_t idx) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (uint64_t)o << 32 | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

// Exponents (in powers of two) are taken no lower in a product with their
// power: that is 0 in f32 there, and so is the product, where -inf, or the
// lowest f32, would give NaN.
constexpr float FLOOR = -256.0f;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^t, t = (x - m) log2(e), for x <= m; off by 2^-21.5 however large t is. 0, and t
// = 0, where that is below f32's normal numbers or x is -inf.
__device__ __forceinline__ float exp_below(float x, float m, float& t) {
  constexpr float LOG2E_LO = 1.92596299e-8f;  // log2(e) - LOG2E
  const float d = x - m, z = d - x, d_lo = (x - (d - z)) - (m + z);  // x - m = d + d_lo
  t = __fmul_rn(d, LOG2E);  // (rounded, whatever it is fused with below)
  if (!(t >= -126.0f)) {
    t = 0.0f;
    return 0.0f;
  }
  const float t_lo = fmaf(d_lo, LOG2E, fmaf(d, LOG2E_LO, fmaf(d, LOG2E, -t)));
  const float n = rintf(t);
  return ex2((t - n) + t_lo) * __int_as_float(((int)n + 127) << 23);
}
// Sorts a warp's 32 keys, largest in lane 0 (bitonic network).
__device__ __forceinline__ uint64_t warp_sort_desc(uint64_t v, uint32_t lane) {
#pragma unroll
  for (uint32_t size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (uint32_t j = size >> 1; j > 0; j >>= 1) {
      const uint64_t o = __shfl_xor_sync(FULL, v, j);
      const bool desc = (lane & size) == 0 || size == 32, low = (lane & j) == 0;
      v = (desc == low) == (v > o) ? v : o;
    }
  }
  return v;
}
// The 32 largest of two sorted lists (a, and b in shared memory), sorted.
__device__ __forceinline__ uint64_t warp_merge_desc(uint64_t a, const uint64_t* b, uint32_t lane) {
  const uint64_t o = b[31 - lane];
  uint64_t v = a > o ? a : o;
#pragma unroll
  for (uint32_t j = 16; j > 0; j >>= 1) {
    const uint64_t x = __shfl_xor_sync(FULL, v, j);
    v = ((lane & j) == 0) == (v > x) ? v : x;
  }
  return v;
}
// Joins `lists` sorted lists of 32 in shared memory into list 0; all threads.
__device__ __forceinline__ void join_lists(uint64_t (*list)[32], uint32_t lists, uint32_t warp, uint32_t lane) {
  for (uint32_t step = 1; step < lists; step <<= 1) {
    __syncthreads();
    const uint32_t at = warp * 2 * step;
    if (at + step < lists) list[at][lane] = warp_merge_desc(list[at][lane], list[at + step], lane);
  }
  __syncthreads();
}

template <typename T>
struct Row {
  static constexpr uint32_t PER = 16 / sizeof(T);  // values per 16-byte load
  const T* x;
  uint32_t begin, head, vecs, end;  // [begin, begin+head) one by one, then vecs loads, then to end one by one

  __device__ Row(const T* row, uint32_t b, uint32_t e) : x(row), begin(b), end(e) {
    const uint32_t mis = (uint32_t)(reinterpret_cast<uintptr_t>(row + b) & 15) / sizeof(T);
    head = mis ? PER - mis : 0;
    if (head > e - b) head = e - b;
    vecs = (e - b - head) / PER;
  }
  __device__ uint32_t vec_index(uint32_t v) const { return begin + head + v * PER; }
  __device__ void load(uint32_t v, float (&o)[PER]) const {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(x + vec_index(v)));
    const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) o[i] = to_f32(t[i]);
  }
  // Calls f(value, index) for every value that thread t reads, lane by lane
  // of a warp that takes them together.
  template <typename F>
  __device__ void each(uint32_t t, uint32_t lane, F&& f) const {
    if (lane == 0 && t < head) f(to_f32(x[begin + t]), begin + t);
    for (uint32_t v = t + lane * LP_THREADS; v < vecs; v += 32 * LP_THREADS) {
      float o[PER];
      load(v, o);
#pragma unroll
      for (uint32_t i = 0; i < PER; ++i) f(o[i], vec_index(v) + i);
    }
    const uint32_t tail = vec_index(vecs) + t;
    if (lane == 0 && tail < end) f(to_f32(x[tail]), tail);
  }
};

// A block's largest value m; S' and W: sums of 2^t and of 2^t t, t = (x - m) log2(e),
// S' without the largest term. The difference is taken first: x log2(e) may be
// beyond f32 where x is a mask of the lowest value.
struct Part {
  float m, s, w;
};

struct LpShared {
  uint64_t list[LP_WARPS][32];
  uint64_t cand[LP_CAND];
  float top_of[LP_WARPS];  // the warps' largest values
  float s[LP_WARPS], w[LP_WARPS];  // theirs, the largest term of all left out
  uint32_t group[LP_MAX_TOP];
  uint64_t red[LP_WARPS];
  uint32_t n_group, n_cand;
  Part whole, own;  // own: of the thread that has m, the largest term in it
  uint32_t owner;
  uint64_t top[32];  // this block's largest keys, in order
};

// A thread's running (m, S, W), and which of its batches of values had m.
struct Run {
  float m = -INFINITY, s = 0.0f, w = 0.0f;
  uint32_t batch = 0;

  template <uint32_t N, bool W>
  __device__ __forceinline__ void add(const float (&v)[N], uint32_t number) {
    float top[2] = {v[0], -INFINITY};
#pragma unroll
    for (uint32_t i = 1; i < N; i += 2) top[(i / 2) & 1] = i + 1 < N ? max3(top[(i / 2) & 1], v[i], v[i + 1]) : fmaxf(top[(i / 2) & 1], v[i]);
    const float mn = max3(m, top[0], top[1]), r = mn == -INFINITY ? 0.0f : mn;
    if (mn > m) {
      batch = number;
      const float d0 = fmaxf((m - r) * LOG2E, FLOOR), f = ex2(d0);
      if (W) w = f * (w + d0 * s);
      s *= f;
      m = mn;
    }
    if constexpr (N == 1) {
      const float d = (v[0] - r) * LOG2E, e = ex2(d);
      s += e;
      if (W) w = fmaf(e, fmaxf(d, FLOOR), w);
    } else {
      const float2 l2 = make_float2(LOG2E, LOG2E), r2 = make_float2(-r, -r);
      float2 es = make_float2(0.0f, 0.0f), ws = es;
#pragma unroll
      for (uint32_t i = 0; i < N; i += 2) {
        const float2 d = mul2(add2(make_float2(v[i], v[i + 1]), r2), l2), e = make_float2(ex2(d.x), ex2(d.y));
        es = add2(es, e);
        if (W) ws = fma2(e, make_float2(fmaxf(d.x, FLOOR), fmaxf(d.y, FLOOR)), ws);
      }
      s += es.x + es.y;
      if (W) w += ws.x + ws.y;
    }
  }
};

// W: the entropy is asked for.
template <typename T, bool W>
__global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(LogprobArgs a) {
  __shared__ LpShared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank();
  const uint32_t row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* x = static_cast<const T*>(a.logits) + (uint64_t)row * a.row_stride;
  // the given token's logit: asked for before the pass, so that it is there after it
  int32_t token = -1;
  float xt = 0.0f;
  if (rank == 0 && tid == 0 && a.tokens) {
    token = a.tokens[row];
    if (token >= 0 && (uint32_t)token < a.vocab) xt = to_f32(x[token]);
    else token = -1;
  }
  const uint32_t each = (a.vocab + C - 1) / C;
  const uint32_t b = min(rank * each, a.vocab), e = min(b + each, a.vocab);
  const Row<T> part(x, b, e);
  constexpr uint32_t PER = Row<T>::PER, U = 2;  // 32 bytes in flight per thread, a batch

  Run r;
  const uint32_t batches = part.vecs > tid ? (part.vecs - tid + LP_THREADS - 1) / LP_THREADS : 0;  // of one load each
  const uint32_t tail = part.vec_index(part.vecs) + tid;
  if (tid < part.head) {
    const float v[1] = {to_f32(x[part.begin + tid])};
    r.template add<1, W>(v, 0xFFFFFFFEu);
  }
  uint32_t n = 0;
  for (; n + U <= batches; n += U) {
    float o[U * PER];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) part.load(tid + (n + u) * LP_THREADS, *reinterpret_cast<float(*)[PER]>(o + u * PER));
    r.template add<U * PER, W>(o, n);
  }
  for (; n < batches; ++n) {
    float o[PER];
    part.load(tid + n * LP_THREADS, o);
    r.template add<PER, W>(o, n);
  }
  if (tail < e) {
    const float o[1] = {to_f32(x[tail])};
    r.template add<1, W>(o, 0xFFFFFFFFu);
  }
  // a NaN left its mark in the sum alone
  const bool nan = isnan(r.s);
  if (nan) r.m = INFINITY;
  const float wm = warp_max(r.m);
  if (lane == 0) sh.top_of[warp] = wm;
  __syncthreads();
  float bm = sh.top_of[0];  // the block's, and the first warp that has it
  uint32_t first = 0;
#pragma unroll
  for (uint32_t i = 1; i < LP_WARPS; ++i)
    if (sh.top_of[i] > bm) bm = sh.top_of[i], first = i;
  {
    float t, s = exp_below(r.m, bm, t), w = s * (r.w + t * r.s);
    s *= r.s;
    if (warp == first) {  // the first thread that has it keeps its sum apart
      const uint32_t owner = __ffs(__ballot_sync(FULL, r.m == bm)) - 1;
      if (lane == owner) sh.owner = tid, sh.own = {bm, s, w}, s = w = 0.0f;
    }
    s = warp_sum(s);
    if (W) w = warp_sum(w);
    if (lane == 0) sh.s[warp] = s, sh.w[warp] = w;
  }

  if (a.top_k) {
    // where the thread's largest value lies: the first of its batch that equals it
    // (a part of nothing but -inf: its first value)
    uint32_t idx = 0xFFFFFFFFu;
    if (tid < part.head && (r.batch == 0xFFFFFFFEu || r.m == -INFINITY)) idx = part.begin + tid;
    else if (batches && (r.batch < 0xFFFFFFFEu || r.m == -INFINITY)) {
      const uint32_t n0 = r.m == -INFINITY ? 0 : r.batch, n1 = min(n0 + (n0 + U <= batches && n0 % U == 0 ? U : 1u), batches);
      for (uint32_t k = n0; k < n1 && idx == 0xFFFFFFFFu; ++k) {
        float o[PER];
        part.load(tid + k * LP_THREADS, o);
#pragma unroll
        for (uint32_t i = PER; i-- > 0;)
          if (o[i] == r.m) idx = part.vec_index(tid + k * LP_THREADS) + i;
      }
    } else if (tail < e) idx = tail;
    const uint64_t mine = idx == 0xFFFFFFFFu || nan ? 0ull : key_of(r.m, idx);
    sh.list[warp][lane] = warp_sort_desc(mine, lane);
    if (tid == 0) sh.n_group = sh.n_cand = 0;
    join_lists(sh.list, LP_WARPS, warp, lane);
    // the k-th largest maximum (0 when fewer threads hold values: then all count)
    const uint64_t thr = sh.list[0][a.top_k - 1];
    if (mine && mine >= thr) sh.group[atomicAdd(&sh.n_group, 1u)] = tid;
    __syncthreads();
    const uint32_t ng = sh.n_group;  // at most top_k: the keys are distinct
    for (uint32_t g = warp; g < ng; g += LP_WARPS)
      part.each(sh.group[g], lane, [&](float val, uint32_t idx) {
        const uint64_t key = key_of(val, idx);
        if (key >= thr) {
          const uint32_t at = atomicAdd(&sh.n_cand, 1u);
          if (at < LP_CAND) sh.cand[at] = key;
        }
      });
    __syncthreads();
    const uint32_t nc = sh.n_cand;
    if (tid < 32) sh.top[tid] = 0;
    __syncthreads();
    if (nc <= LP_CAND) {
      for (uint32_t i = tid; i < nc; i += LP_THREADS) {
        const uint64_t key = sh.cand[i];
        uint32_t above = 0;
        for (uint32_t j = 0; j < nc; ++j) above += sh.cand[j] > key;
        if (above < a.top_k) sh.top[above] = key;
      }
    } else {
      // many values of few threads: take them largest first, one at a time
      uint64_t last = ~0ull;
      for (uint32_t i = 0; i < a.top_k; ++i) {
        uint64_t best = 0;
        for (uint32_t g = warp; g < ng; g += LP_WARPS)
          part.each(sh.group[g], lane, [&](float val, uint32_t idx) {
            const uint64_t key = key_of(val, idx);
            if (key < last && key > best) best = key;
          });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(FULL, best, o);
          best = best > other ? best : other;
        }
        if (lane == 0) sh.red[warp] = best;
        __syncthreads();
        for (uint32_t w = 0; w < LP_WARPS; ++w) best = sh.red[w] > best ? sh.red[w] : best;
        if (tid == 0) sh.top[i] = best;
        last = best;
        __syncthreads();
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    float s = lane < LP_WARPS ? sh.s[lane] : 0.0f, w = W && lane < LP_WARPS ? sh.w[lane] : 0.0f;
    const float rest = sh.own.s - 1.0f;
    if (bm > -INFINITY && warp_sum(s) + rest < 0.5f) {
      part.each(sh.owner, lane, [&](float v, uint32_t) {  // (equals of m are not here: S' were 1 or more)
        float t;
        const float e = exp_below(v, bm, t);
        if (v != bm) s += e, w = fmaf(e, t, w);
      });
    } else if (lane == 0) {
      s += rest, w += sh.own.w;
    }
    s = warp_sum(s);
    if (W) w = warp_sum(w);
    if (lane == 0) sh.whole = {bm, s, w};
  }
  // ---- join the cluster's blocks: every block's first warp has the row's (m, S', W) ----
  if (C > 1) cluster.sync();
  else __syncthreads();
  if (rank == 0) {
    if (a.top_k) {
      if (warp < C) sh.list[warp][lane] = C > 1 ? cluster.map_shared_rank(&sh, warp)->top[lane] : sh.top[lane];
      join_lists(sh.list, C, warp, lane);
    }
    if (warp == 0) {
      Part q = {-INFINITY, 0.0f, 0.0f};
      if (lane < C) q = C > 1 ? cluster.map_shared_rank(&sh, lane)->whole : sh.whole;
      const float m = warp_max(q.m);
      // the blocks' largest terms but one count; the first of equals stays apart
      const bool owner = (int)lane == __ffs(__ballot_sync(FULL, q.m == m)) - 1;
      float t, f = exp_below(q.m, m, t);
      if (owner) f = 1.0f, t = 0.0f;
      const float one = owner ? 0.0f : 1.0f;
      const float rest = warp_sum(f * (one + q.s)), w = W ? warp_sum(f * (q.w + t * (one + q.s))) : 0.0f;
      // NaN, +inf, or nothing above -inf: no distribution
      const bool none = isnan(rest) || fabsf(m) == INFINITY;
      const float nanf_ = __int_as_float(0x7FC00000);
      const float log_sum = log1pf(rest);
      if (lane == 0) {
        if (a.tokens) a.logprobs[row] = none || token < 0 ? nanf_ : (xt - m) - log_sum;
        if (W) a.entropy[row] = none ? nanf_ : log_sum - w * LN2 / (1.0f + rest);
      }
      if (lane < a.top_k) {
        const uint64_t key = sh.list[0][lane];
        a.top_ids[(uint64_t)row * a.top_k + lane] = none ? -1 : (int32_t)key_index(key);
        a.top_logprobs[(uint64_t)row * a.top_k + lane] = none ? nanf_ : (key_value(key) - m) - log_sum;
      }
    }
  }
  if (C > 1) cluster.sync();  // the blocks' shared memory stays until all have read it
}

template <typename T, bool W>
cudaError_t launch_w(const LogprobArgs& a, cudaStream_t stream) {
  // blocks per row: enough to have one on every SM, while each still reads
  // 4096 values or more
  uint32_t c = 1;
  while (c < 8 && (uint64_t)a.n_rows * c < SMS && a.vocab / (2 * c) >= 4096) c *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.n_rows * c);
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, W>, a);
}

template <typename T>
cudaError_t launch(const LogprobArgs& a, cudaStream_t stream) {
  return a.entropy ? launch_w<T, true>(a, stream) : launch_w<T, false>(a, stream);
}

}  // namespace

cudaError_t token_logprobs(const LogprobArgs& a, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case DT_F32: return launch<float>(a, stream);
    case DT_F16: return launch<__half>(a, stream);
    default: return launch<__nv_bfloat16>(a, stream);
  }
}

}  // namespace k
}  // namespace yl
