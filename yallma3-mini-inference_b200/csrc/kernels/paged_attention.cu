// Causal grouped-query attention over the paged cache.
//
// For a row r at position p and the keys j <= p of its sequence
//   s_j = scale q.k_j,  m = max s_j,  l = sum e^(s_j - m),  o = sum e^(s_j - m) v_j / l
// in one pass over keys and values with a running (m, l, O); parts over
// different keys join as m = max m_i, l = sum l_i e^(m_i - m), O likewise.
// Scores are kept times log2(e), so that every exponential is one ex2.
//
// Work: the rows of a sequence that share a key/value head (new tokens x query
// heads of the group) are cut into row tiles, the keys into key tiles of 16 KB;
// one (head, row tile) is an item, its key tiles are counted up to its last
// row's position. All key tiles of all items form one line that is cut into
// equal pieces, one per block: long and short sequences, few and many, load
// every SM alike. An item cut by a piece's end leaves its parts (m, l, O) in
// the workspace, and a second kernel joins them. The geometry is read from
// device memory by every block, so a captured launch follows its arrays.
//
// Shared prefix: a first launch lets the rows of all sequences attend to the
// prefix together, as rows of one sequence (its keys are read once per row
// tile, not once per sequence), a second one to the rest, or, for sequences
// that begin or end inside the prefix, to all they see; the parts are joined
// likewise. Blocks of the second start as those of the first end (programmatic
// dependent launch; it waits for the first only before it ends).
//
// Within a block one warp fetches key and value tiles page by page with TMA
// (128-byte swizzle; a page id that is none goes to a coordinate outside the
// tensor, which reads as zeros) into a ring of 16 KB buffers; the others
// multiply with mma.sync, WM warps of 16 rows each times WK warps that split
// the tile's keys and join at the item's end. Decoding has 1..16 rows per
// item and is bound by reading the cache, so WK = 4; f32 from 33 rows on WK = 1.
// f32 operands are split into two tf32 numbers and multiplied as hi*hi + hi*lo
// + lo*hi (2^-21 relative); 16-bit ones are exact, and the softmax weights are
// rounded to their type for the second product (the sum l takes them
// unrounded), f16 weights at 2^10 times their value so that small ones do not
// fall below f16's range.
//
// Measured on one B200, 32 query and 8 key heads of 128, bf16: 16 sequences of 17
// to 8000 tokens 52 us (268 MB, 5.2 TB/s; bound by HBM and the items' ends), one
// of 100000 tokens 72 us (5.7 TB/s); one token of 9 / 3 heads of 64, f32, 301 keys
// 9 us (two launches, four dependent trips to memory each); a prompt of 2000
// tokens of 32 / 8 heads of 64, f32, 433 us, of which its 3 x 8 million tf32 MMAs
// (8.2 cycles each per scheduler) would take 190: two warps per scheduler at 168
// registers wait for one another's chains. More warps with fewer registers spill:
// 3 % longer with three blocks per SM, 20 % with eight warps per block.
#include <cmath>

#include "paged_attention.cuh"

namespace yl {
namespace k {
using namespace yl::dev;

namespace {

constexpr uint32_t BUF = 16384;  // bytes of a key or value tile
template <typename T, int HD, int WM_, int WK_>
struct Shape {
  static constexpr int WM = WM_, WK = WK_, NW = WM * WK, THREADS = 32 * (NW + 1);
  static constexpr int BM = 16 * WM;
  static constexpr int ROW = HD * (int)sizeof(T);  // bytes of a row
  static constexpr int NH = ROW / 128;             // 128-byte columns
  static constexpr int KT = BUF / ROW;             // keys per tile
  static constexpr int WKEYS = KT / WK;
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int NBUF = F32 && HD == 128 && WM == 2 ? 3 : 4;  // what two blocks per SM leave room for
  static constexpr int QP = HD + 4;  // f32 queries and the warps' joining: row stride in shared memory, no bank conflicts
  static constexpr uint32_t Q_BYTES = F32 ? BM * QP * 4 : 0;
  static constexpr uint32_t M_BYTES = WK > 1 ? NW * 16 * QP * 4 : 0;
  static constexpr uint32_t SMEM = 1024 + NBUF * BUF + Q_BYTES + M_BYTES;
  static_assert(SMEM <= 113 * 1024 - 1024, "two blocks per SM");
  static_assert(WKEYS % (F32 ? 8 : 16) == 0, "whole MMA steps");
};

// ---- MMA -------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo in tf32, off by at most 2^-21 of x: hi is x rounded to 11 bits
// (in integers; cvt.rna.tf32 takes as long as an MMA), lo the exact rest, of
// which the MMA reads the upper 11 bits. A NaN whose hi would overflow to 0
// stays a NaN in lo.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void split2(uint32_t x, uint32_t y, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
  hi[0] = (x + 0x1000u) & 0xFFFFE000u, hi[1] = (y + 0x1000u) & 0xFFFFE000u;
  const float2 l = fma2(make_float2(__uint_as_float(hi[0]), __uint_as_float(hi[1])), make_float2(-1.0f, -1.0f),
                        make_float2(__uint_as_float(x), __uint_as_float(y)));
  lo[0] = __float_as_uint(l.x), lo[1] = __float_as_uint(l.y);
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ float lds(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
// Byte of 16-byte column c of row `key` in a tile.
template <typename S>
__device__ __forceinline__ uint32_t at(uint32_t key, uint32_t c) {
  return (c >> 3) * (S::KT * 128) + key * 128 + (((c & 7) ^ (key & 7)) << 4);
}

template <typename T, typename O, int HD, int WM, int WK>
__global__ void __launch_bounds__(Shape<T, HD, WM, WK>::THREADS, 2)
    attend_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ Pass p) {
  using S = Shape<T, HD, WM, WK>;
  constexpr float SHIFT = std::is_same<T, __half>::value ? 10.0f : 0.0f;
  extern __shared__ uint8_t raw[];
  __shared__ Start start;
  __shared__ uint64_t scratch[16];
  __shared__ __align__(8) uint64_t full[S::NBUF], empty[S::NBUF];
  __shared__ float ml[S::NW][16][2];
  __shared__ volatile int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  float* qs = reinterpret_cast<float*>(smem + S::NBUF * BUF);
  float* join = reinterpret_cast<float*>(smem + S::NBUF * BUF + S::Q_BYTES);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tpt = S::BM / p.group;
  uint4 goes_on = make_uint4(0, 0, 0, 0);  // (warp 0) the item that goes on in the next block

  if (threadIdx.x == 32 * S::NW) {
    prefetch_map(&map_k);
    prefetch_map(&map_v);
  }
  if (threadIdx.x == 0) {
    for (int b = 0; b < S::NBUF; ++b) {
      mbar_init(&full[b], 1);
      mbar_init(&empty[b], S::NW);
    }
    mbar_fence_init();
    abort_flag = 0;
  }
  grid_dep_launch();  // what follows may be scheduled; it waits for this grid's end
  find_start<S>(p, tpt, &start, scratch);
  const bool idle = start.seq == 0xFFFFFFFFu;
  const PagedAttnArgs& a = p.a;

  if (!idle && warp == S::NW) {
    // ---- producer: key and value tiles, page by page ----
    Walk<S> w(p, tpt, start);
    const uint32_t ps = 1u << a.pages.page_shift;
    const uint32_t tb = ps < (uint32_t)S::KT ? ps : (uint32_t)S::KT;  // tokens per load
    const uint32_t pieces = S::KT / tb;
    uint32_t n = 0, issued = 0;
    bool ok = true;
    do {
      const uint32_t kend = w.kend(), tseq = p.prefix ? 0 : w.seq;
      if (lane == 0 && !p.prefix && a.seqs.status && w.r.pos0 + (int64_t)w.r.n > (int64_t)w.r.limit)
        *a.seqs.status = STATUS_RANGE;
      uint32_t k0 = w.kbegin();
      for (uint32_t left = w.kt1 - w.kt0; left && ok; --left, k0 += S::KT) {
        const uint32_t live = kend > k0 ? min(pieces, (kend - k0 + tb - 1) / tb) : 0;  // loads with a visible key
        for (uint32_t kv = 0; kv < 2 && ok; ++kv, ++n) {
          const uint32_t b = n % S::NBUF, round = n / S::NBUF;
          // one load per lane: lane l fetches column l % NH of piece l / NH
          const uint32_t dst = smem_u32(smem) + b * BUF;
          if (n >= (uint32_t)S::NBUF) {
            if (lane == 0) ok = mbar_wait(&empty[b], (round - 1) & 1, nullptr);
            ok = __shfl_sync(FULL, ok ? 1 : 0, 0) != 0 && !abort_flag;
            ok = __all_sync(FULL, ok);
            if (!ok) break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[b], live * tb * 128 * S::NH);
          __syncwarp();
          for (uint32_t u = lane; u < live * S::NH; u += 32) {
            const uint32_t piece = u / S::NH, col = u % S::NH, pos = k0 + piece * tb;
            uint32_t page = page_of(a.seqs, a.pages, tseq, pos);
            if (page == NO_PAGE) {
              page = a.pages.n_pages;
              if (a.seqs.status) *a.seqs.status = STATUS_RANGE;
            }
            tma_page(dst + col * (S::KT * 128) + piece * tb * 128, kv ? &map_v : &map_k, col * (128 / sizeof(T)),
                     w.head, pos & (ps - 1), page, &full[b]);
          }
          issued = n + 1;
        }
      }
    } while (ok && w.next());
    if (!ok) {
      abort_flag = 1;
      if (lane == 0) {
        if (a.seqs.status) *a.seqs.status = STATUS_TIMEOUT;
        // the copies this warp issued land before the block ends
        for (uint32_t i = issued > (uint32_t)S::NBUF ? issued - S::NBUF : 0; i < issued; ++i)
          mbar_wait(&full[i % S::NBUF], (i / S::NBUF) & 1, nullptr, 200000000ull);
      }
      __syncwarp();
    }
  } else if (!idle) {
    // ---- consumers ----
    Walk<S> w(p, tpt, start);
    const uint32_t wm = warp / WK, wk = warp % WK, g = lane >> 2, t4 = lane & 3;
    const uint32_t flip = p.flip ? 0x80008000u : 0;  // sign bits of 16-bit q
    constexpr int NB = S::WKEYS / 8, OB = HD / 8;
    uint32_t n = 0;
    bool ok = true;
    do {
      const uint32_t ntok = w.tokens(), nrow = ntok * p.group, kend = w.kend();
      // this thread's rows of the tile: token and query head
      uint32_t row[2], head[2];
      int32_t lim[2];  // keys the row sees
      bool live[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t m = wm * 16 + g + 8 * i, tok = m / p.group;
        live[i] = m < nrow;
        row[i] = w.r.row0 + w.t + (live[i] ? tok : 0);
        head[i] = w.head * p.group + (live[i] ? m % p.group : 0);
        int64_t e = w.r.pos0 + w.t + tok + 1;
        if (p.prefix) {
          e = kend;
          if (start.masked && live[i] && left_out(a.seqs, row[i])) e = 0;
        }
        lim[i] = live[i] ? (int32_t)(e < 0 ? 0 : e < (int64_t)kend ? e : kend) : 0x7FFFFFFF;
      }
      // smallest of the row tile: tiles that end before it need no mask
      const uint32_t all_see = p.prefix ? (start.masked ? 0 : kend) : [&] {
        const int64_t e = w.r.pos0 + w.t + 1;
        return e < 0 ? 0u : e < (int64_t)kend ? (uint32_t)e : kend;
      }();

      uint32_t qf[S::F32 ? 1 : HD / 16][4];
      if constexpr (S::F32) {
        // (every warp is done with the item before: they met at its end)
        for (uint32_t u = threadIdx.x; u < S::BM * (HD / 4); u += 32 * S::NW) {
          const uint32_t m = u / (HD / 4), c = u % (HD / 4);
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (m < nrow)
            v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) +
                                                 (uint64_t)(w.r.row0 + w.t + m / p.group) * a.q_stride +
                                                 (uint64_t)(w.head * p.group + m % p.group) * HD + 4 * c);
          // f32 queries take the factor, in two f32, with one rounding: scores come in powers of two
          const float sc = p.flip ? -p.sc : p.sc, lo = p.flip ? -p.sc_lo : p.sc_lo;
          v = make_float4(fmaf(v.x, sc, v.x * lo), fmaf(v.y, sc, v.y * lo), fmaf(v.z, sc, v.z * lo),
                          fmaf(v.w, sc, v.w * lo));
          *reinterpret_cast<float4*>(qs + m * S::QP + 4 * c) = v;
        }
        named_bar_sync(1, 32 * S::NW);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) +
                                                                (uint64_t)row[i] * a.q_stride + (uint64_t)head[i] * HD);
#pragma unroll
          for (int s = 0; s < HD / 16; ++s) {
            qf[s][i] = live[i] ? q[8 * s + t4] ^ flip : 0;
            qf[s][2 + i] = live[i] ? q[8 * s + 4 + t4] ^ flip : 0;
          }
        }
      }
      float o[OB][4];
#pragma unroll
      for (int j = 0; j < OB; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
      const bool busy = wm * 16 < nrow;  // a warp without a row only hands the buffers on

      uint32_t k0 = w.kbegin();
      for (uint32_t left = w.kt1 - w.kt0; left && ok; --left, k0 += S::KT) {
        uint32_t b = n % S::NBUF;
        uint32_t base = smem_u32(smem) + b * BUF;
        ok = mbar_wait(&full[b], (n / S::NBUF) & 1, nullptr);
        ok = __all_sync(FULL, ok);
        if (!ok) break;
        float s[NB][4];
        if (busy) {
#pragma unroll
          for (int j = 0; j < NB; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
          if constexpr (S::F32) {
            // The tensor cores drop what falls below an accumulator's last bit, so
            // long chains lose digits: two accumulators for the large products
            // and one for the small ones, added at the end; 32 keys at a time,
            // for the registers.
            constexpr int JG = NB < 4 ? NB : 4;
#pragma unroll
            for (int j0 = 0; j0 < NB; j0 += JG) {
              float s1[JG][4], sl[JG][4];
#pragma unroll
              for (int j = 0; j < JG; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) s1[j][c] = sl[j][c] = 0.0f;
#pragma unroll 2
              for (int ks = 0; ks < HD / 16; ++ks) {  // 16 elements: two k-steps of 8
                uint32_t ah[2][4], al[2][4];
                // (split again for every tile: kept split, in shared memory, the loads
                // cost more than the arithmetic, 6 % of the time below)
                const float* q0 = qs + (wm * 16 + g) * S::QP + 16 * ks + t4;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                  for (int i = 0; i < 4; ++i) split(q0[8 * h + 8 * (i & 1) * S::QP + 4 * (i >> 1)], ah[h][i], al[h][i]);
                // (all splits, then the products across the keys: the chains are as long as they look)
                uint32_t bh[JG][2][2], bl[JG][2][2];
#pragma unroll
                for (int j = 0; j < JG; ++j) {
                  uint32_t r[4];
                  ldsm4(r, base + at<S>(wk * S::WKEYS + 8 * (j0 + j) + (lane & 7), 4 * ks + (lane >> 3)));
                  split2(r[0], r[1], bh[j][0], bl[j][0]);
                  split2(r[2], r[3], bh[j][1], bl[j][1]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                  for (int j = 0; j < JG; ++j) mma_tf32(sl[j], al[h], bh[j][h][0], bh[j][h][1]);
#pragma unroll
                  for (int j = 0; j < JG; ++j) mma_tf32(h ? s1[j] : s[j0 + j], ah[h], bh[j][h][0], bh[j][h][1]);
#pragma unroll
                  for (int j = 0; j < JG; ++j) mma_tf32(sl[j], ah[h], bl[j][h][0], bl[j][h][1]);
                }
              }
#pragma unroll
              for (int j = 0; j < JG; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[j0 + j][c] = (s[j0 + j][c] + s1[j][c]) + sl[j][c];
            }
          } else {
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
              for (int j = 0; j < NB; j += 2) {
                uint32_t r[4];
                ldsm4(r, base + at<S>(wk * S::WKEYS + 8 * j + (lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)));
                mma16<T>(s[j], qf[ks], r[0], r[1]);
                mma16<T>(s[j + 1], qf[ks], r[2], r[3]);
              }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[b]);
        ++n;
        float corr[2];
        if (busy) {
          if (k0 + S::KT > all_see) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if ((int32_t)(k0 + wk * S::WKEYS + 8 * j + 2 * t4 + (c & 1)) >= lim[c >> 1]) s[j][c] = -INFINITY;
          }
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) top[c >> 1] = fmaxf(top[c >> 1], s[j][c]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(FULL, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(FULL, top[i], 2));
            const float mn = fmaxf(m[i], S::F32 ? top[i] : top[i] * p.sc);
            const float ref = mn == -INFINITY ? 0.0f : mn - SHIFT;
            corr[i] = ex2(m[i] - (mn == -INFINITY ? 0.0f : mn));  // 0 from -inf
            m[i] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int c = 2 * i; c < 2 * i + 2; ++c) {
                // (the product with the factor is exact before the maximum is taken off)
                s[j][c] = ex2(S::F32 ? s[j][c] - ref : fmaf(s[j][c], p.sc, -ref));
                sum += s[j][c];
              }
            l[i] = l[i] * corr[i] + sum;
          }
          if (__any_sync(FULL, corr[0] != 1.0f || corr[1] != 1.0f)) {
#pragma unroll
            for (int j = 0; j < OB; ++j) {
              o[j][0] *= corr[0], o[j][1] *= corr[0];
              o[j][2] *= corr[1], o[j][3] *= corr[1];
            }
          }
        }
        b = n % S::NBUF;
        base = smem_u32(smem) + b * BUF;
        ok = mbar_wait(&full[b], (n / S::NBUF) & 1, nullptr);
        ok = __all_sync(FULL, ok);
        if (!ok) break;
        if (busy) {
          if (k0 + S::KT > kend) {
            // values behind the last visible key may be anything: their weight is 0, and 0 times NaN is not
#pragma unroll 1
            for (uint32_t u = lane; u < (uint32_t)S::WKEYS * S::NH * 8; u += 32) {
              const uint32_t key = wk * S::WKEYS + u / (S::NH * 8), c = u % (S::NH * 8);
              if (k0 + key >= kend)
                *reinterpret_cast<uint4*>(smem + b * BUF + at<S>(key, c)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();  // before the next TMA write of the buffer
            __syncwarp();
          }
          if constexpr (S::F32) {
            constexpr int JP = NB < 2 ? 1 : 2;  // 16 keys in a chain (2000 tokens of 32 / 8 heads of 64: 433 us; of 8 keys 10 % longer, of 32 no less)
#pragma unroll
            for (int j = 0; j < NB; j += JP) {
              // keys 2i of the eight are the MMA's k = i, keys 2i+1 its k = 4+i: the weights are where QK left them
              uint32_t ph[JP][4], pl[JP][4];
#pragma unroll
              for (int x = 0; x < JP; ++x) {
                split(s[j + x][0], ph[x][0], pl[x][0]);
                split(s[j + x][2], ph[x][1], pl[x][1]);
                split(s[j + x][1], ph[x][2], pl[x][2]);
                split(s[j + x][3], ph[x][3], pl[x][3]);
              }
              const uint32_t key = wk * S::WKEYS + 8 * j + 2 * t4;
#pragma unroll
              for (int d = 0; d < OB; d += 2) {  // two columns at a time: the chains are long
                uint32_t vh[JP][2][2], vl[JP][2][2];
                float t[2][4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t c = 2 * (d + e) + (g >> 2), w = (g & 3) * 4;
#pragma unroll
                  for (int x = 0; x < JP; ++x) {
                    split(lds(base + at<S>(key + 8 * x, c) + w), vh[x][e][0], vl[x][e][0]);
                    split(lds(base + at<S>(key + 8 * x + 1, c) + w), vh[x][e][1], vl[x][e][1]);
                  }
                  t[e][0] = t[e][1] = t[e][2] = t[e][3] = 0.0f;  // (added with rounding, see above)
                }
#pragma unroll
                for (int x = 0; x < JP; ++x) {
#pragma unroll
                  for (int e = 0; e < 2; ++e) mma_tf32(t[e], pl[x], vh[x][e][0], vh[x][e][1]);
#pragma unroll
                  for (int e = 0; e < 2; ++e) mma_tf32(t[e], ph[x], vl[x][e][0], vl[x][e][1]);
                }
#pragma unroll
                for (int x = 0; x < JP; ++x)
#pragma unroll
                  for (int e = 0; e < 2; ++e) mma_tf32(t[e], ph[x], vh[x][e][0], vh[x][e][1]);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                  for (int c = 0; c < 4; ++c) o[d + e][c] += t[e][c];
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < NB; j += 2) {
              const uint32_t pf[4] = {pack2<T>(s[j][0], s[j][1]), pack2<T>(s[j][2], s[j][3]),
                                      pack2<T>(s[j + 1][0], s[j + 1][1]), pack2<T>(s[j + 1][2], s[j + 1][3])};
#pragma unroll
              for (int d = 0; d < OB; d += 2) {
                uint32_t r[4];
                ldsm4t(r, base + at<S>(wk * S::WKEYS + 8 * j + (lane & 15), d + (lane >> 4)));
                mma16<T>(o[d], pf, r[0], r[1]);
                mma16<T>(o[d + 1], pf, r[2], r[3]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[b]);
        ++n;
      }
      // ---- the item's end ----
      // All consumers meet, those too whose wait ran out, and leave together or go
      // on together: nobody is left at this barrier or at the item's next ones.
      // (A warp that gave up hands no buffer on, so the others' waits for later
      // ones run out as well.) Behind it nobody reads this item's queries or the
      // join's buffers of the item before.
      ok = named_bar_all(1, 32 * S::NW, ok);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(FULL, l[i], 1);
        l[i] += __shfl_xor_sync(FULL, l[i], 2);
        if (m[i] == INFINITY) l[i] = NAN;  // finite scores whose maximum overflowed have lost their weights
        if (l[i] == 0.0f && lim[i] > (int32_t)(w.kbegin() + wk * S::WKEYS)) m[i] = BELOW;
      }
      const bool whole = w.whole();
      if (w.kt0 == 0 && warp == 0) {
        const uint32_t blocks = whole ? 0 : w.blocks();
        if (p.joined)
#pragma unroll 1
          for (uint32_t t = lane; t < ntok; t += 32)
            p.desc[(uint64_t)(w.r.row0 + w.t + t) * a.pages.n_kv_heads + w.head] = make_uint2(blockIdx.x, blocks << 16 | t);
        else if (!whole)
          goes_on = make_uint4(w.r.row0 + w.t, ntok, w.head, blocks);
      }
      float* const slot = p.slots + (uint64_t)(2 * blockIdx.x + (w.kt0 == 0 ? 1 : 0)) * S::BM * PART<HD>;
      auto part = [&](uint32_t mrow, uint32_t r, uint32_t h) {
        return whole ? p.rowpart + ((uint64_t)r * a.n_heads + h) * PART<HD> : slot + mrow * PART<HD>;
      };
      const bool direct = whole && !p.joined;
      if constexpr (WK > 1) {
        // the warps of a row group join over shared memory
        float* mine = join + warp * 16 * S::QP;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (t4 == 0) ml[warp][g + 8 * i][0] = m[i], ml[warp][g + 8 * i][1] = l[i];
        if (busy) {
#pragma unroll
          for (int d = 0; d < OB; ++d) {
            *reinterpret_cast<float2*>(mine + g * S::QP + 8 * d + 2 * t4) = make_float2(o[d][0], o[d][1]);
            *reinterpret_cast<float2*>(mine + (g + 8) * S::QP + 8 * d + 2 * t4) = make_float2(o[d][2], o[d][3]);
          }
        }
        named_bar_sync(1, 32 * S::NW);
#pragma unroll 1
        for (uint32_t u = threadIdx.x; u < nrow * (HD / 4); u += 32 * S::NW) {
          const uint32_t mr = u / (HD / 4), c = u % (HD / 4), w0 = mr / 16 * WK, rr = mr % 16;
          float top = -INFINITY, sum = 0.0f;
#pragma unroll
          for (int x = 0; x < WK; ++x) top = fmaxf(top, ml[w0 + x][rr][0]);
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < WK; ++x) {
            const float f = ex2(ml[w0 + x][rr][0] - (top == -INFINITY ? 0.0f : top));
            const float4 v = *reinterpret_cast<const float4*>(join + ((w0 + x) * 16 + rr) * S::QP + 4 * c);
            sum += f * ml[w0 + x][rr][1];
            acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
          }
          const uint32_t r = w.r.row0 + w.t + mr / p.group, h = w.head * p.group + mr % p.group;
          if (direct) {
            sum = settled(top, sum);
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            O* out = static_cast<O*>(a.out) + (uint64_t)r * a.out_stride + (uint64_t)h * HD + 4 * c;
            if constexpr (sizeof(O) == 4)
              *reinterpret_cast<float4*>(out) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            else
              *reinterpret_cast<uint2*>(out) = make_uint2(pack2<O>(acc.x * inv, acc.y * inv), pack2<O>(acc.z * inv, acc.w * inv));
            if (c == 0 && a.lse)
              a.lse[(uint64_t)r * a.n_heads + h] = sum == 0.0f ? -INFINITY : (top - SHIFT + log2f(sum)) * LN2;
          } else {
            if (top == -INFINITY) acc = make_float4(0.f, 0.f, 0.f, 0.f);  // no key seen: 0 times what was there, which may be NaN
            float* d = part(mr, r, h);
            reinterpret_cast<float2*>(d + 4 * c)[0] = make_float2(acc.x, acc.y);
            reinterpret_cast<float2*>(d + 4 * c)[1] = make_float2(acc.z, acc.w);
            if (c == 0) d[HD] = top - SHIFT, d[HD + 1] = sum;
          }
        }
      } else if (busy) {
        static_assert(WK > 1 || std::is_same<O, float>::value, "f32 alone has rows that one warp finishes");
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!live[i]) continue;
          if (direct) {
            l[i] = settled(m[i], l[i]);
            const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
            O* out = static_cast<O*>(a.out) + (uint64_t)row[i] * a.out_stride + (uint64_t)head[i] * HD + 2 * t4;
#pragma unroll
            for (int d = 0; d < OB; ++d)
              *reinterpret_cast<float2*>(out + 8 * d) = make_float2(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
            if (t4 == 0 && a.lse)
              a.lse[(uint64_t)row[i] * a.n_heads + head[i]] =
                  l[i] == 0.0f ? -INFINITY : (m[i] - SHIFT + log2f(l[i])) * LN2;
          } else {
            float* d0 = part(wm * 16 + g + 8 * i, row[i], head[i]);
#pragma unroll
            for (int d = 0; d < OB; ++d)
              *reinterpret_cast<float2*>(d0 + 8 * d + 2 * t4) =
                  m[i] == -INFINITY ? make_float2(0.f, 0.f) : make_float2(o[d][2 * i], o[d][2 * i + 1]);  // (as above)
            if (t4 == 0) d0[HD] = m[i] - SHIFT, d0[HD + 1] = l[i];
          }
        }
      }
    } while (w.next());
    if (!ok) {
      abort_flag = 1;
      if (lane == 0 && a.seqs.status) *a.seqs.status = STATUS_TIMEOUT;
    }
  }
  if (threadIdx.x == 0) p.cut[blockIdx.x] = goes_on;
  __syncthreads();
  grid_dep_wait();  // the launch before has ended when this one has
}

// ---- joining the parts -------------------------------------------------------
struct JoinArgs {
  PagedAttnArgs a;
  uint32_t group;
  struct {
    const uint4* cut;
    const uint2* desc;
    const float* slots;
    const float* rowpart;
    uint32_t grid, bm;
  } pass[2];
};

// Joins n parts of one (row, query head) and writes it out; part(i) is where
// the i-th lies. `each` warps take every each-th part and meet in shared
// memory (all of the block's threads then call this together); lanes hold
// HD/32 neighbours.
template <typename O, int HD, typename F>
__device__ __forceinline__ void join_row(const PagedAttnArgs& a, uint32_t row, uint32_t head, uint32_t n, F&& part,
                                         uint32_t first, uint32_t each, float (*meet)[PART<HD>]) {
  constexpr int PER = HD / 32;
  const uint32_t lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.0f, o[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.0f;
  constexpr uint32_t U = 4;  // parts in flight
  for (uint32_t i0 = first; i0 < n; i0 += U * each) {
    float pm[U], pl[U];
    __align__(16) float po[U][PER];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      pm[u] = -INFINITY, pl[u] = 0.0f;
#pragma unroll
      for (int e = 0; e < PER; ++e) po[u][e] = 0.0f;
      if (i0 + u * each < n) {
        const float* q = part(i0 + u * each);
        const float2 ml = *reinterpret_cast<const float2*>(q + HD);
        pm[u] = ml.x, pl[u] = ml.y;
        if constexpr (PER == 4) *reinterpret_cast<float4*>(po[u]) = *reinterpret_cast<const float4*>(q + PER * lane);
        else *reinterpret_cast<float2*>(po[u]) = *reinterpret_cast<const float2*>(q + PER * lane);
      }
    }
    const float top = fmaxf(m, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]))), ref = top == -INFINITY ? 0.0f : top;
    const float f0 = ex2(m - ref);
    m = top;
    l *= f0;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] *= f0;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const float f = ex2(pm[u] - ref);
      l += f * pl[u];
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += f * po[u][e];
    }
  }
  if (each > 1) {
    __syncthreads();  // the row before has been read
#pragma unroll
    for (int e = 0; e < PER; ++e) meet[first][PER * lane + e] = o[e];
    if (lane == 0) meet[first][HD] = m, meet[first][HD + 1] = l;
    __syncthreads();
    if (first) return;
    float top = m;
    for (uint32_t w = 1; w < each; ++w) top = fmaxf(top, meet[w][HD]);
    const float ref = top == -INFINITY ? 0.0f : top, f0 = ex2(m - ref);
    m = top;
    l *= f0;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] *= f0;
    for (uint32_t w = 1; w < each; ++w) {
      const float f = ex2(meet[w][HD] - ref);
      l += f * meet[w][HD + 1];
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += f * meet[w][PER * lane + e];
    }
  }
  l = settled(m, l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  O* out = static_cast<O*>(a.out) + (uint64_t)row * a.out_stride + (uint64_t)head * HD + PER * lane;
#pragma unroll
  for (int e = 0; e < PER; e += 2) {
    if constexpr (sizeof(O) == 4) *reinterpret_cast<float2*>(out + e) = make_float2(o[e] * inv, o[e + 1] * inv);
    else *reinterpret_cast<uint32_t*>(out + e) = pack2<O>(o[e] * inv, o[e + 1] * inv);
  }
  if (lane == 0 && a.lse) a.lse[(uint64_t)row * a.n_heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

// One pass: block x takes the item that begins in the pass's block x and goes
// on in the next; its rows go round the grid's second dimension, eight at a
// time with a warp each, or, where many blocks share them, one at a time.
template <typename O, int HD>
__global__ void __launch_bounds__(256) join_cut_kernel(JoinArgs j) {
  __shared__ float meet[8][PART<HD>];
  grid_dep_wait();
  const PagedAttnArgs& a = j.a;
  const auto& ps = j.pass[0];
  const uint4 c = ps.cut[blockIdx.x];  // {first row, tokens, head, blocks}
  const uint32_t rows = c.y * j.group, n = c.w, warp = threadIdx.x >> 5;
  const uint32_t slot = ps.bm * PART<HD>;
  auto each_part = [&](uint32_t mr) {
    const float* at = ps.slots + (2ull * blockIdx.x * ps.bm + mr) * PART<HD>;
    return [at, slot](uint32_t i) { return at + (i ? 2 * i : 1) * slot; };
  };
  if (n > 8) {
    for (uint32_t mr = blockIdx.y; mr < rows; mr += gridDim.y)
      join_row<O, HD>(a, c.x + mr / j.group, c.z * j.group + mr % j.group, n, each_part(mr), warp, 8, meet);
  } else {
    for (uint32_t mr = blockIdx.y * 8 + warp; mr < rows; mr += gridDim.y * 8)
      join_row<O, HD>(a, c.x + mr / j.group, c.z * j.group + mr % j.group, n, each_part(mr), 0, 1, meet);
  }
}

// Prefix and own parts: four warps per (row, query head).
template <typename O, int HD>
__global__ void __launch_bounds__(128) join_rows_kernel(JoinArgs j) {
  __shared__ float meet[4][PART<HD>];
  const PagedAttnArgs& a = j.a;
  const uint32_t row = blockIdx.x / a.n_heads, head = blockIdx.x % a.n_heads;
  grid_dep_wait();
  if (row < row_begin(a.seqs, 0) || row >= row_begin(a.seqs, a.seqs.n_seqs)) return;
  uint2 d[2];
  uint32_t n[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    d[p] = j.pass[p].desc[(uint64_t)row * a.pages.n_kv_heads + head / j.group];
    n[p] = d[p].y >> 16 ? d[p].y >> 16 : 1;
    // (row ranges that overlap or leave gaps: nothing outside the workspace is read)
    if (d[p].y >> 16 && ((uint64_t)d[p].x + n[p] > j.pass[p].grid || (d[p].y & 0xFFFFu) >= j.pass[p].bm / j.group)) return;
  }
  const float* at[2];
  uint32_t slot[2];  // 0: the whole item, in rowpart
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    slot[p] = d[p].y >> 16 ? j.pass[p].bm * PART<HD> : 0;
    at[p] = slot[p] ? j.pass[p].slots + (2ull * d[p].x * j.pass[p].bm + (d[p].y & 0xFFFFu) * j.group + head % j.group) * PART<HD>
                    : j.pass[p].rowpart + ((uint64_t)row * a.n_heads + head) * PART<HD>;
  }
  auto part = [&](uint32_t i) {
    const int p = i < n[0] ? 0 : 1;
    const uint32_t k = p ? i - n[0] : i;
    return (p ? at[1] : at[0]) + (k ? 2 * k : 1) * (p ? slot[1] : slot[0]);
  };
  join_row<O, HD>(a, row, head, n[0] + n[1], part, threadIdx.x >> 5, 4, meet);
}

// ---- host --------------------------------------------------------------------
// Row tile for items of `rows` rows. Decoding pads to 16 rows. 12, 16 and 32
// sequences of 4 query heads per key head over 8192 shared tokens (48, 64 and 128
// rows) took 32.9, 36.9 and 39.7 us on tcgen05 and 37.0, 39.6 and 39.7 us in
// 64-row tiles on mma.sync, which are no longer built for 16 bits; 8 of them (32
// rows) 26.7 us on mma.sync and 31.0 on tcgen05, 64 sequences of 6 rows each (24)
// 54 and 64. f32 has no tcgen05 form.
uint32_t tile_rows(uint64_t rows, int dtype) {
  if (dtype != DT_F32 && rows > 32) return TC_TILE;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}
// Two blocks per SM; two passes that both leave room for the other get one each
// and run side by side (12 sequences over 4096 f32 tokens 15 % faster than one
// after the other).
uint32_t blocks_of(uint32_t bm, bool beside) { return bm == TC_TILE || beside ? SMS : 2 * SMS; }

// What a call launches, by its counts alone.
struct Plan {
  bool shared;        // a prefix pass of its own
  bool beside;        // the two passes run side by side
  uint32_t bm[2];     // row tiles of the sequences' pass, and of the prefix pass
  uint64_t cut[2], desc[2], slots[2], rowpart[2], bytes;  // workspace offsets
};
Plan plan_of(const Pages& p, const Seqs& s, int dtype, uint32_t n_heads, int share) {
  const uint64_t group = n_heads / p.n_kv_heads, hd = p.head_size;
  const uint64_t each = ((uint64_t)s.n_rows + s.n_seqs - 1) / s.n_seqs * group;
  Plan pl{};
  pl.bm[0] = tile_rows(each, dtype);
  pl.bm[1] = tile_rows((uint64_t)s.n_rows * group, dtype);
  pl.beside = pl.bm[0] != TC_TILE && pl.bm[1] != TC_TILE;
  // A pass over the prefix for all sequences saves reading it n_seqs - 1 times
  // (from L2, as a rule) and costs its launch and the joining of every row.
  // Measured, us with and without it (8 key heads of 128, bf16, own keys 100..300):
  //   side by side:  4 x 1024 tokens 12.9 / 11.7,  8 x 1024 16.6 / 14.3,  8 x 2048 16.9 / 18.5,  4 x 16384 28 / 42
  //   on tcgen05:    16 x 1024 24.0 / 19.3,  16 x 2048 25.9 / 27.0,  64 x 512 41 / 36,  64 x 1024 42 / 51
  //   f32, head 64:  4 x 1024 12.1 / 14.3,  12 x 1024 20 / 22,  12 x 4096 35 / 56
  // Rows of a prompt share what they read by themselves: 16 sequences of 16 tokens
  // (64 rows each) behind 4096 63 / 77, of 32 tokens 93 / 81.
  const double saved = (s.n_seqs - 1.0) * s.shared_len * p.n_kv_heads * hd * (dtype == DT_F32 ? 8 : 4);
  const double worth = dtype == DT_F32 ? 8 << 20 : pl.beside ? 40 << 20 : 128 << 20;
  pl.shared = s.shared_len && s.n_seqs > 1 && each <= 64 && (share < 0 ? saved >= worth : share > 0);
  pl.beside = pl.beside && pl.shared;
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    const uint64_t o = at;
    at = (at + n + 255) / 256 * 256;
    return o;
  };
  for (int i = 0; i < (pl.shared ? 2 : 1); ++i) {
    pl.cut[i] = take(16ull * blocks_of(pl.bm[i], pl.beside));
    pl.desc[i] = pl.shared ? take((uint64_t)s.n_rows * p.n_kv_heads * 8) : 0;
    pl.slots[i] = take(2ull * blocks_of(pl.bm[i], pl.beside) * pl.bm[i] * (hd + 8) * 4);
    pl.rowpart[i] = pl.shared ? take((uint64_t)s.n_rows * n_heads * (hd + 8) * 4) : 0;
  }
  pl.bytes = at;
  return pl;
}

template <typename T, typename O, int HD, int WM, int WK>
cudaError_t launch_pass(const CUtensorMap& mk, const CUtensorMap& mv, const Pass& p, const LaunchCfg& lc) {
  using S = Shape<T, HD, WM, WK>;
  static std::atomic<uint64_t> ready{0};
  const cudaError_t e = allow_smem(ready, attend_kernel<T, O, HD, WM, WK>, S::SMEM);
  if (e != cudaSuccess) return e;
  return launch_kernel(attend_kernel<T, O, HD, WM, WK>, dim3(p.grid), dim3(S::THREADS), S::SMEM, lc, mk, mv, p);
}

template <typename T, typename O, int HD>
cudaError_t launch(const PagedAttnArgs& a, int dtype, cudaStream_t stream) {
  constexpr uint32_t KT = BUF / (HD * sizeof(T));
  const Plan pl = plan_of(a.pages, a.seqs, dtype, a.n_heads, a.share);
  const uint32_t ps = 1u << a.pages.page_shift, tokens = ps < KT ? ps : KT;
  CUtensorMap mk, mv;
  if (!encode_pages(&mk, a.pages, a.pages.k, dtype, tokens) || !encode_pages(&mv, a.pages, a.pages.v, dtype, tokens))
    return cudaErrorInvalidValue;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  JoinArgs j{};
  j.a = a;
  j.group = a.n_heads / a.pages.n_kv_heads;
  LaunchCfg lc;
  lc.stream = stream;
  for (int i = pl.shared ? 1 : 0; i >= 0; --i) {  // the prefix first
    Pass p{};
    p.a = a;
    p.dtype = dtype;
    const double sc = std::fabs((double)a.scale) * 1.4426950408889634;
    p.sc = sc < 1.2e-38 ? 1.2e-38f : (float)sc;  // not 0: times -inf it stays -inf
    p.sc_lo = std::isfinite(p.sc) ? (float)(sc - (double)p.sc) : 0.0f;
    p.flip = a.scale < 0.0f;
    p.grid = blocks_of(pl.bm[i], pl.beside);
    p.prefix = i;
    p.from = pl.shared && !i ? a.seqs.shared_len : 0;
    p.group = j.group;
    // A piece is at least so long: an f32 tile takes as long as joining its part
    // (one token against 301: pieces of 1 9.0 us, of 2 10.1); a 16-bit one of 2 is as
    // fast as of 1 and makes fewer parts (one token against 301 9.1 / 8.9, 8 sequences
    // behind 2048 16.9 / 17.0; of 3 9.9, 18.0).
    p.min_chunk = dtype == DT_F32 ? 1 : 2;
    // 16-bit items cost as much as two tiles more (with 0 / 1 / 2 / 3: 64 sequences of
    // up to 1000 tokens 51 / 42.5 / 34.2 / 33.8 us, of 6 rows each 85 / 69 / 54 / 51, an
    // 8191-token prompt on tcgen05 616 / 566 / 529 / 526); an f32 tile takes as long as
    // an item's ends (a 900-token prompt of 9 / 3 heads 58 / 42 / 48 / 48).
    p.item_cost = dtype == DT_F32 ? 1 : 2;
    p.joined = pl.shared;
    p.cut = reinterpret_cast<uint4*>(ws + pl.cut[i]);
    p.desc = reinterpret_cast<uint2*>(ws + pl.desc[i]);
    p.slots = reinterpret_cast<float*>(ws + pl.slots[i]);
    p.rowpart = reinterpret_cast<float*>(ws + pl.rowpart[i]);
    j.pass[i].cut = p.cut;
    j.pass[i].desc = p.desc;
    j.pass[i].slots = p.slots;
    j.pass[i].rowpart = p.rowpart;
    j.pass[i].grid = p.grid;
    j.pass[i].bm = pl.bm[i];
    cudaError_t e;
    if (pl.bm[i] == 16) e = launch_pass<T, O, HD, 1, 4>(mk, mv, p, lc);
    else if (pl.bm[i] == 32) e = launch_pass<T, O, HD, 2, 2>(mk, mv, p, lc);
    else if constexpr (sizeof(T) == 4) e = launch_pass<T, O, HD, 4, 1>(mk, mv, p, lc);
    else e = attend_tc(p, sizeof(O) == 4, lc);
    if (e != cudaSuccess) return e;
    lc.pdl = true;
  }
  if (pl.shared)
    return launch_kernel(join_rows_kernel<O, HD>, dim3(a.seqs.n_rows * a.n_heads), dim3(128), 0, lc, j);
  return launch_kernel(join_cut_kernel<O, HD>, dim3(blocks_of(pl.bm[0], pl.beside), pl.bm[0] == TC_TILE ? 32 : 4), dim3(256), 0, lc,
                       j);
}

template <typename T, typename O>
cudaError_t launch_hd(const PagedAttnArgs& a, int dtype, cudaStream_t stream) {
  return a.pages.head_size == 128 ? launch<T, O, 128>(a, dtype, stream) : launch<T, O, 64>(a, dtype, stream);
}

}  // namespace

cudaError_t paged_attention(const PagedAttnArgs& a, int dtype, bool out_f32, cudaStream_t stream) {
  if (dtype == DT_F32) return launch_hd<float, float>(a, dtype, stream);
  if (dtype == DT_F16)
    return out_f32 ? launch_hd<__half, float>(a, dtype, stream) : launch_hd<__half, __half>(a, dtype, stream);
  return out_f32 ? launch_hd<__nv_bfloat16, float>(a, dtype, stream)
                 : launch_hd<__nv_bfloat16, __nv_bfloat16>(a, dtype, stream);
}

uint64_t paged_attention_workspace(const Pages& p, const Seqs& s, int dtype, uint32_t n_heads, int share) {
  const Plan pl = plan_of(p, s, dtype, n_heads, share);
  return pl.bytes > 256 ? pl.bytes : 256;
}

}  // namespace k
}  // namespace yl
