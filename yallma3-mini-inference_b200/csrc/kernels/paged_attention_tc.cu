// Paged attention of items with many rows (prompts, and the rows of a whole
// batch over a shared prefix) on the 5th-generation tensor cores. The
// mathematics and the cutting of the work are paged_attention.cu's; here an
// item is two tiles of 128 rows that read the same keys, one block per SM.
//
// Per key tile of 128 keys: S = Q K^T into tensor memory (128 x 128 f32 per row
// tile, operands in 128-byte-swizzled shared memory); one thread per row reads
// its row of S, takes the exponentials and writes the weights P, rounded to 16
// bits, over the first half of S; O += P V with P as the operand from tensor
// memory, V from shared memory ([key][element], so its descriptor is that of an
// operand whose rows run along the columns of the product). The two row tiles
// take turns: while one's softmax runs, the tensor cores multiply for the
// other. A row tile's MMAs are all issued by one thread and run in its order, so
// its next S may be issued right behind the product that reads P from the same
// columns.
//
// O stays in tensor memory. It is rescaled only when a row's maximum has grown
// by more than 2^8 since the last time: until then P is taken relative to the
// old maximum (at most 2^8, 2^15 with f16's shift), which changes nothing in the
// quotient O / l. The commit that announces S of a tile covers the product of
// the tile before, so O is at rest while its rows are rescaled.
//
// Warps: 0-3 softmax of the first row tile, 4-7 of the second (warp w reads
// tensor-memory lanes 32 (w % 4) ..), 8 and 10 issue the MMAs of the first and
// the second (one's waiting is hidden behind the other's MMAs; the tensor cores
// hold only a few in advance), 9 loads Q (a box of group heads x tokens), and keys
// and values page by page, 11 only hands its registers to the softmax warps, for
// which a row of S is 128 registers. (Two threads per row, 16 softmax warps of 96
// registers, took 12 % longer for a prompt of 8191 tokens, now 529 us: they spill,
// and pairs have to agree on every tile's maximum.)
#include "paged_attention.cuh"

namespace yl {
namespace k {

namespace {

template <typename T, int HD>
struct TcShape {
  static constexpr int THREADS = 384;
  static constexpr int KT = 128;                      // keys per tile
  static constexpr int NH = HD / 64;                  // 128-byte columns of a row
  static constexpr uint32_t COL = 128 * 128;          // bytes of a column of 128 rows
  static constexpr uint32_t TILE = NH * COL;          // bytes of 128 rows
  static constexpr int NBUF = HD == 128 ? 5 : 8;      // key / value tiles in the ring
  static constexpr uint32_t SMEM = 1024 + (2 + NBUF) * TILE;
  static constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0 : 1;
  // f32 accumulators, 16-bit operands, M = 128; S: N = 128 keys; O: N = HD, its second operand along N
  static constexpr uint32_t IDESC_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t IDESC_O =
      (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((128u >> 4) << 24);
  static_assert(SMEM <= 226 * 1024, "shared memory");
  static_assert(SMEM > 114 * 1024, "one block per SM: it holds all of tensor memory");
};
constexpr uint32_t TMEM_S = 0, TMEM_O = 256, TMEM_COLS = 512;  // per row tile: 128 columns of each

// Shared-memory descriptors of 128-byte-swizzled tiles, as (upper, lower) words:
// the lower holds the address (in 16 bytes) and can be advanced by adding to it.
// Q, K: rows of 128 bytes along the summed axis, 8-row groups 1024 bytes apart.
// V [key][element]: rows of 128 bytes along N, 8-key groups 1024 bytes apart,
// 64-element columns COL apart.
constexpr uint32_t DESC_HI = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_n(uint32_t saddr, uint32_t col_bytes) {
  return (saddr >> 4) | ((col_bytes >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " YL_V32 ";" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
               "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
               "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
// Waits for the loads before; the registers pass through, so that nothing reads them earlier.
#define YL_RW32(p) "+r"(p[0]), "+r"(p[1]), "+r"(p[2]), "+r"(p[3]), "+r"(p[4]), "+r"(p[5]), "+r"(p[6]), "+r"(p[7]), \
                   "+r"(p[8]), "+r"(p[9]), "+r"(p[10]), "+r"(p[11]), "+r"(p[12]), "+r"(p[13]), "+r"(p[14]),       \
                   "+r"(p[15]), "+r"(p[16]), "+r"(p[17]), "+r"(p[18]), "+r"(p[19]), "+r"(p[20]), "+r"(p[21]),     \
                   "+r"(p[22]), "+r"(p[23]), "+r"(p[24]), "+r"(p[25]), "+r"(p[26]), "+r"(p[27]), "+r"(p[28]),     \
                   "+r"(p[29]), "+r"(p[30]), "+r"(p[31])
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&a)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : YL_RW32(a)::"memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&a)[32], uint32_t (&b)[32]) {
  tmem_wait_ld(a);
  asm volatile("" : YL_RW32(b)::"memory");
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x for x up to 127 without the special-function unit, which gives 16 results
// per clock and SM and would bound the softmax: x = n + f, |f| <= 1/2, 2^f by a
// polynomial fitted to it by least squares of the relative error on Chebyshev
// nodes (off by 2^-22.2 at most, roundings included, as ex2.approx), times 2^n.
// Below -126.5 n is -127, whose exponent field is 0: the result is 0, as it
// is for hidden keys (-inf), whose values may be anything finite. NaN stays NaN.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  constexpr float C0 = 1.00000012f, C1 = 0.693146944f, C2 = 0.240221217f, C3 = 0.0555074252f, C4 = 0.00967545994f,
                  C5 = 0.0013266971f;
  constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are n
  x = make_float2(max_nan(x.x, -127.0f), max_nan(x.y, -127.0f));
  const float2 t = add2(x, make_float2(MAGIC, MAGIC));
  const float2 n = add2(t, make_float2(-MAGIC, -MAGIC));
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 y = make_float2(C5, C5);
  y = fma2(y, f, make_float2(C4, C4));
  y = fma2(y, f, make_float2(C3, C3));
  y = fma2(y, f, make_float2(C2, C2));
  y = fma2(y, f, make_float2(C1, C1));
  y = fma2(y, f, make_float2(C0, C0));
  // n in the exponent's place: (bits of t) << 23 drops what MAGIC put above n
  const float px = __uint_as_float((__float_as_uint(t.x) << 23) + 0x3F800000u);
  const float py = __uint_as_float((__float_as_uint(t.y) << 23) + 0x3F800000u);
  return make_float2(y.x * px, y.y * py);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 bytes in one store (a thread writes its row: fewer of them, fewer trips), or two where 16 bytes is the alignment.
__device__ __forceinline__ void store32(void* to, const uint32_t* v, bool wide) {
  if (wide)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  else {
    static_cast<uint4*>(to)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    static_cast<uint4*>(to)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}
// 3-D tiled load: (element, head, row).
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t head, uint32_t row,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(smem_u32(bar))
      : "memory");
}

template <typename T, typename O, int HD>
__global__ void __launch_bounds__(384, 1)
    attend_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ CUtensorMap map_q, const __grid_constant__ Pass p) {
  using S = TcShape<T, HD>;
  constexpr float SHIFT = std::is_same<T, __half>::value ? 7.0f : 0.0f;  // weights up to 2^(SHIFT + 8)
  constexpr float GROWN = 8.0f;
  extern __shared__ uint8_t raw[];
  __shared__ Start start;
  __shared__ uint64_t scratch[16];
  __shared__ __align__(8) uint64_t full[S::NBUF], empty[S::NBUF], q_full, q_empty, s_full[2], p_full[2], o_full[2], turn[2], drain[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t q_smem = smem_u32(smem), ring = q_smem + 2 * S::TILE;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tok_tile = 128 / p.group, tpt = 2 * tok_tile;
  const PagedAttnArgs& a = p.a;
  uint4 goes_on = make_uint4(0, 0, 0, 0);  // (warp 0) the item that goes on in the next block

  if (threadIdx.x == 32 * 9) {
    prefetch_map(&map_q);
    prefetch_map(&map_k);
    prefetch_map(&map_v);
  }
  if (threadIdx.x == 0) {
    for (int b = 0; b < S::NBUF; ++b) {
      mbar_init(&full[b], 1);
      mbar_init(&empty[b], 2);
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 2);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&drain[x], 1);
      mbar_init(&turn[x], 1);
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4);
      mbar_init(&o_full[x], 1);
    }
    mbar_fence_init();
    abort_flag = 0;
  }
  grid_dep_launch();
  find_start<S>(p, tpt, &start, scratch);
  const bool idle = start.seq == 0xFFFFFFFFu;
  if (!idle && warp == 8) {
    tmem_alloc(&tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = idle ? 0 : tmem_slot;

  // 384 threads at 168 registers are launched; 256 x 200 + 128 x 104 are as many
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
  if (!idle && warp == 9) {
    // ---- loads ----
    Walk<S> w(p, tpt, start);
    const uint32_t ps = 1u << a.pages.page_shift;
    const uint32_t tb = ps < (uint32_t)S::KT ? ps : (uint32_t)S::KT, pieces = S::KT / tb;
    uint32_t n = 0, items = 0;
    bool ok = true;
    do {
      const uint32_t kend = w.kend(), tseq = p.prefix ? 0 : w.seq;
      if (lane == 0 && !p.prefix && a.seqs.status && w.r.pos0 + (int64_t)w.r.n > (int64_t)w.r.limit)
        *a.seqs.status = STATUS_RANGE;
      const uint32_t tiles = w.tokens() > tok_tile ? 2 : 1;
      if (items > 0) {
        ok = mbar_wait(&q_empty, (items - 1) & 1, nullptr);
        ok = __all_sync(FULL, ok);
        if (!ok) break;
      }
      if (lane == 0) mbar_arrive_expect_tx(&q_full, tiles * S::NH * 128 * p.group * tok_tile);
      __syncwarp();
      if (lane < tiles * S::NH) {
        const uint32_t x = lane / S::NH, c = lane % S::NH;
        tma_rows(q_smem + x * S::TILE + c * S::COL, &map_q, c * 64, w.head * p.group, w.r.row0 + w.t + x * tok_tile,
                 &q_full);
      }
      ++items;
      uint32_t k0 = w.kbegin();
      for (uint32_t left = w.kt1 - w.kt0; left && ok; --left, k0 += S::KT) {
        const uint32_t live = kend > k0 ? min(pieces, (kend - k0 + tb - 1) / tb) : 0;  // loads with a visible key
        // the tile's pages, one per lane: the same for keys and values (pieces <= 16, NH <= 2)
        const uint32_t piece = lane / S::NH, col = lane % S::NH, pos = k0 + piece * tb;
        uint32_t page = 0;
        if (piece < live) {
          page = page_of(a.seqs, a.pages, tseq, pos);
          if (page == NO_PAGE) {
            page = a.pages.n_pages;
            if (a.seqs.status) *a.seqs.status = STATUS_RANGE;
          }
        }
        for (uint32_t kv = 0; kv < 2; ++kv, ++n) {
          const uint32_t b = n % S::NBUF;
          if (n >= (uint32_t)S::NBUF) {
            ok = mbar_wait(&empty[b], (n / S::NBUF - 1) & 1, nullptr);
            ok = __all_sync(FULL, ok);
            if (!ok) break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[b], live * tb * 128 * S::NH);
          __syncwarp();
          if (piece < live)
            tma_page(ring + b * S::TILE + col * S::COL + piece * tb * 128, kv ? &map_v : &map_k, col * 64, w.head,
                     pos & (ps - 1), page, &full[b]);
        }
      }
    } while (ok && w.next());
    if (!ok) {
      abort_flag = 1;
      if (lane == 0) {
        if (a.seqs.status) *a.seqs.status = STATUS_TIMEOUT;
        // the copies this warp issued land before the block ends
        if (items) mbar_wait(&q_full, (items - 1) & 1, nullptr, 200000000ull);
        for (uint32_t i = n > (uint32_t)S::NBUF ? n - S::NBUF : 0; i < n; ++i)
          mbar_wait(&full[i % S::NBUF], (i / S::NBUF) & 1, nullptr, 200000000ull);
      }
      __syncwarp();
    }
  } else if (!idle && warp != 11) {
    // ---- MMAs of one row tile: an elected lane issues; all wait, and clear what lies behind the last key ----
    Walk<S> w(p, tpt, start);
    const uint32_t x = warp == 8 ? 0 : 1;
    uint32_t n = 0, items = 0, p_phase = 0, turns = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = __all_sync(FULL, mbar_wait(bar, parity, nullptr));
      tc_fence_after();
      return ok;
    };
    auto wait_full = [&](uint32_t i) { return wait(&full[i % S::NBUF], (i / S::NBUF) & 1); };
    // Issued by the lane that elect.sync names (not one picked by its number):
    // only then an MMA's descriptors go to its uniform registers directly, and
    // it costs the 64 cycles that the tensor cores need, not 130.
    auto qk = [&](uint32_t buf) {
      if (elect_one()) {
        const uint32_t q = desc_k(q_smem + x * S::TILE), kb = desc_k(ring + buf * S::TILE);
#pragma unroll
        for (uint32_t s = 0; s < HD / 16; ++s) {
          const uint32_t off = ((s >> 2) * S::COL + (s & 3) * 32) >> 4;
          mma_ss(tmem + TMEM_S + 128 * x, q + off, kb + off, S::IDESC_S, s > 0);
        }
        tc_commit(&s_full[x]);
      }
    };
    auto pv = [&](uint32_t buf, bool first, bool last) {
      if (elect_one()) {
        const uint32_t vb = desc_n(ring + buf * S::TILE, S::COL);
#pragma unroll
        for (uint32_t s = 0; s < S::KT / 16; ++s)
          mma_ts(tmem + TMEM_O + 128 * x, tmem + TMEM_S + 128 * x + 8 * s, vb + s * (16 * 128 >> 4), S::IDESC_O,
                 s > 0 || !first);
        if (last) tc_commit(&o_full[x]);
      }
    };
    // a buffer is free when both row tiles' MMAs are through with it; a tile without rows has none
    auto release = [&](uint64_t* bar, bool mine) {
      if (elect_one()) {
        if (mine) tc_commit(bar);
        else mbar_arrive(bar);
      }
    };
    do {
      const uint32_t kend = w.kend(), nt = w.kt1 - w.kt0;
      const bool mine = x == 0 || w.tokens() > tok_tile;
      if (mine && !wait(&q_full, items & 1)) break;
      if (!wait_full(n)) break;
      if (mine) qk(n % S::NBUF);
      release(&empty[n % S::NBUF], mine);
      if (nt == 1) release(&q_empty, mine);
      uint32_t k0 = w.kbegin();
      for (uint32_t i = 0; i < nt; ++i, k0 += S::KT) {
        const uint32_t v = n + 1, kn = n + 2;
        const bool more = i + 1 < nt;
        if (!wait_full(v)) break;
        if (mine && k0 + S::KT > kend) {
          // values behind the last visible key may be anything: their weight is 0, and 0 times NaN is not
          // (both warps write the same zeros, each before its own products)
          uint8_t* vb = smem + (2 + v % S::NBUF) * S::TILE;
          const uint32_t from = kend > k0 ? kend - k0 : 0;
#pragma unroll 1
          for (uint32_t u = lane; u < (S::KT - from) * 8 * S::NH; u += 32) {
            const uint32_t c = u / ((S::KT - from) * 8), o = u % ((S::KT - from) * 8);
            *reinterpret_cast<uint4*>(vb + c * S::COL + from * 128 + o * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        }
        if (more && !wait_full(kn)) break;
        if (mine && !wait(&p_full[x], p_phase)) break;
        // The row tiles' MMAs alternate, each tile's at one go: mixed, both
        // tiles' S would be there at the same time, both softmaxes would run
        // together, and the tensor cores would wait for both (10 % longer at 8191 rows).
        if ((x == 1 || turns > 0) && !wait(&turn[x], (turns - 1 + x) & 1)) break;
        ++turns;
        if (mine) {
          p_phase ^= 1;
          pv(v % S::NBUF, i == 0, !more);
          if (more) qk(kn % S::NBUF);
        }
        if (elect_one()) mbar_arrive(&turn[x ^ 1]);
        release(&empty[v % S::NBUF], mine);
        if (more) release(&empty[kn % S::NBUF], mine);
        if (i + 2 == nt) release(&q_empty, mine);
        n += 2;
      }
      if (!ok) break;
      ++items;
    } while (w.next());
    if (!ok) {
      abort_flag = 1;
      if (lane == 0 && a.seqs.status) *a.seqs.status = STATUS_TIMEOUT;
    }
    if (elect_one()) tc_commit(&drain[x]);  // every MMA of this warp has completed when this flips
    mbar_wait(&drain[x], 0, nullptr);
    __syncwarp();
  }
  } else {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
  if (!idle) {
    // ---- softmax: one thread per row ----
    Walk<S> w(p, tpt, start);
    const uint32_t x = warp >> 2, quarter = (warp & 3) << 21;  // lane 32 * (warp % 4) in the address's upper half
    const uint32_t ts = tmem + TMEM_S + 128 * x + quarter, to = tmem + TMEM_O + 128 * x + quarter;
    const uint32_t m = 32 * (warp & 3) + lane;
    const float sc = p.sc;
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    do {
      const uint32_t all = w.tokens(), t0 = x * tok_tile, kend = w.kend();
      const uint32_t tok = m / p.group + t0, gh = m % p.group;
      if (warp == 0 && w.kt0 == 0) {
        const uint32_t blocks = w.whole() ? 0 : w.blocks();
        if (p.joined)
#pragma unroll 1
          for (uint32_t t = lane; t < all; t += 32)
            p.desc[(uint64_t)(w.r.row0 + w.t + t) * a.pages.n_kv_heads + w.head] = make_uint2(blockIdx.x, blocks << 16 | t);
        else if (blocks)
          goes_on = make_uint4(w.r.row0 + w.t, all, w.head, blocks);
      }
      if (all <= t0) continue;  // this row tile has no rows (no barrier of it moves)
      const bool live = m < tok_tile * p.group && tok < all;
      const bool busy = __any_sync(FULL, live);
      const uint32_t row = w.r.row0 + w.t + (live ? tok : 0), head = w.head * p.group + gh;
      // keys this row sees, and those that every row of the tile sees
      int64_t e = w.r.pos0 + w.t + tok + 1, e0 = w.r.pos0 + w.t + t0 + 1;
      if (p.prefix) {
        e = e0 = kend;
        if (start.masked) {
          e0 = 0;
          if (live && left_out(a.seqs, row)) e = 0;
        }
      }
      const uint32_t lim = e < 0 ? 0 : e < (int64_t)kend ? (uint32_t)e : kend;
      const uint32_t all_see = e0 < 0 ? 0 : e0 < (int64_t)kend ? (uint32_t)e0 : kend;
      float mx = -INFINITY, l = 0.0f;  // the maximum that O and l are taken relative to, in powers of two

      uint32_t k0 = w.kbegin();
      for (uint32_t kt = w.kt0; kt < w.kt1; ++kt, k0 += S::KT) {
        ok = mbar_wait(&s_full[x], s_phase, nullptr);
        ok = __all_sync(FULL, ok);
        if (!ok) break;
        s_phase ^= 1;
        tc_fence_after();
        if (busy) {
          uint32_t r[4][32];
          auto load = [&] {
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, r[c]);
            tmem_wait_ld(r[0], r[1]);
            tmem_wait_ld(r[2], r[3]);
            if (__builtin_expect(p.flip != 0, 0)) {
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i) r[c][i] ^= 0x80000000u;
            }
            if (__any_sync(FULL, k0 + S::KT > all_see)) {
              const uint32_t left = lim > k0 ? lim - k0 : 0;  // visible keys of the tile
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (32u * c + i >= left) r[c][i] = 0xFF800000u;
            }
          };
          load();
          // Weights and the tile's maximum in one go, relative to the maximum so
          // far; if that turns out to have grown by more than GROWN in a row of
          // the warp, which is rare after an item's first tile, O and l are
          // rescaled and the weights taken again.
          uint32_t pk[4][16];
          float2 sum[4];
          float t[4];
          auto weights = [&](float ref) {
            const float2 sc2 = make_float2(sc, sc), ref2 = make_float2(-ref, -ref);
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = make_float2(0.0f, 0.0f), t[c] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float2 s2 = make_float2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1]));
                const float2 e = fma2(s2, sc2, ref2);
                const float2 w2 = (i + c) % 4 == 3 ? exp2_fma(e) : make_float2(ex2(e.x), ex2(e.y));
                t[c] = max3(t[c], s2.x, s2.y);
                sum[c] = add2(sum[c], w2);
                pk[c][i] = pack2<T>(w2.x, w2.y);
              }
          };
          if (kt == w.kt0) {  // no maximum yet: the tile's first
#pragma unroll
            for (int c = 0; c < 4; ++c) t[c] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; i += 2)
#pragma unroll
              for (int c = 0; c < 4; ++c) t[c] = max3(t[c], __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
            mx = max3(fmaxf(t[0], t[1]), t[2], t[3]) * sc;
          }
          weights(mx == -INFINITY ? 0.0f : mx - SHIFT);
          const float top = fmaxf(mx, max3(fmaxf(t[0], t[1]), t[2], t[3]) * sc);
          if (__any_sync(FULL, top > mx + GROWN)) {
            const float f = ex2(mx - (top == -INFINITY ? 0.0f : top));  // 0 from -inf
            l *= f;
            mx = top;
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(to + 32 * c, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st32(to + 32 * c, o);
            }
            load();  // (the row and its weights together are more than a thread's registers)
            weights(mx == -INFINITY ? 0.0f : mx - SHIFT);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_st16(ts + 16 * c, pk[c]);
          l += ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) + ((sum[2].x + sum[2].y) + (sum[3].x + sum[3].y));
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      if (!ok) break;

      // ---- the item's end ----
      ok = mbar_wait(&o_full[x], o_phase, nullptr);
      ok = __all_sync(FULL, ok);
      if (!ok) break;
      o_phase ^= 1;
      tc_fence_after();
      if (mx == INFINITY) l = NAN;  // finite scores whose maximum overflowed have lost their weights
      if (l == 0.0f && lim > w.kbegin()) mx = BELOW;
      if (busy) {
        const bool whole = w.whole(), direct = whole && !p.joined;
        if (direct) l = settled(mx, l);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float* part = whole ? p.rowpart + ((uint64_t)row * a.n_heads + head) * PART<HD>
                            : p.slots + ((uint64_t)(2 * blockIdx.x + (w.kt0 == 0 ? 1 : 0)) * TC_TILE + tok * p.group + gh) * PART<HD>;
        O* out = static_cast<O*>(a.out) + (uint64_t)row * a.out_stride + (uint64_t)head * HD;
        const bool wide = (reinterpret_cast<uintptr_t>(a.out) | (a.out_stride * sizeof(O))) % 32 == 0;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
          tmem_wait_ld(o);
          if (live) {
            if (direct) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
              if constexpr (sizeof(O) == 2) {
                uint32_t v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = pack2<O>(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
#pragma unroll
                for (int i = 0; i < 16; i += 8) store32(out + 32 * c + 2 * i, v + i, wide);
              } else {
#pragma unroll
                for (int i = 0; i < 32; i += 8) store32(out + 32 * c + i, o + i, wide);
              }
            } else {
              if (mx == -INFINITY) {  // no key seen: 0 times what was there, which may be NaN
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0;
              }
#pragma unroll
              for (int i = 0; i < 32; i += 8) store32(part + 32 * c + i, o + i, true);
            }
          }
        }
        if (live) {
          if (!direct) part[HD] = mx - SHIFT, part[HD + 1] = l;
          else if (a.lse) a.lse[(uint64_t)row * a.n_heads + head] = l == 0.0f ? -INFINITY : (mx - SHIFT + log2f(l)) * LN2;
        }
      }
      tc_fence_before();  // O has been read before the next item's first product, which waits for its weights
    } while (w.next());
    if (!ok) abort_flag = 1;
  }
  if (threadIdx.x == 0) p.cut[blockIdx.x] = goes_on;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!idle && warp == 8) tmem_dealloc(tmem, TMEM_COLS);
  grid_dep_wait();  // the launch before has ended when this one has
}

bool encode_rows(CUtensorMap* m, const Pass& p) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const uint32_t hd = p.a.pages.head_size;
  const cuuint64_t dims[3] = {hd, p.a.n_heads, p.a.seqs.n_rows};
  const cuuint64_t strides[2] = {hd * 2ull, p.a.q_stride * 2};
  const cuuint32_t box[3] = {64, p.group, 128 / p.group}, estr[3] = {1, 1, 1};
  return fn(m, p.dtype == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
            const_cast<void*>(p.a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename O, int HD>
cudaError_t launch(const Pass& p, const LaunchCfg& lc) {
  using S = TcShape<T, HD>;
  static std::atomic<uint64_t> ready{0};
  const cudaError_t e = allow_smem(ready, attend_tc_kernel<T, O, HD>, S::SMEM);
  if (e != cudaSuccess) return e;
  const uint32_t ps = 1u << p.a.pages.page_shift, tokens = ps < (uint32_t)S::KT ? ps : (uint32_t)S::KT;
  CUtensorMap mk, mv, mq;
  if (!encode_pages(&mk, p.a.pages, p.a.pages.k, p.dtype, tokens) ||
      !encode_pages(&mv, p.a.pages, p.a.pages.v, p.dtype, tokens) || !encode_rows(&mq, p))
    return cudaErrorInvalidValue;
  return launch_kernel(attend_tc_kernel<T, O, HD>, dim3(p.grid), dim3(S::THREADS), S::SMEM, lc, mk, mv, mq, p);
}
template <typename T, typename O>
cudaError_t launch_hd(const Pass& p, const LaunchCfg& lc) {
  return p.a.pages.head_size == 128 ? launch<T, O, 128>(p, lc) : launch<T, O, 64>(p, lc);
}

}  // namespace

cudaError_t attend_tc(const Pass& p, bool out_f32, const LaunchCfg& lc) {
  if (p.dtype == DT_F16) return out_f32 ? launch_hd<__half, float>(p, lc) : launch_hd<__half, __half>(p, lc);
  return out_f32 ? launch_hd<__nv_bfloat16, float>(p, lc) : launch_hd<__nv_bfloat16, __nv_bfloat16>(p, lc);
}

}  // namespace k
}  // namespace yl
