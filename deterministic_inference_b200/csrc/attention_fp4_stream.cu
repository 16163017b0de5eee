// Attention of few rows over a cache in 4-bit floating point, the form for heads of 64 and 128 and bfloat16 queries (attention_fp4.cu has
// the formula and the forms for the rest).  A sequence's rows (new token, query head of the kv group), ROWS at a time, against a
// run of its keys, by one CTA, in tiles of 128 keys.
//   S^T = K Q^T on the tensor cores' block-scaled 4-bit products (tcgen05.mma kind::mxf4nvf4): the keys' codes and block scales
//     enter as they lie in the cache, nothing of them is converted.  A query row is the sum of four rows in 4 bits, each the quantised rest
//     of those before it, in a unit of a quarter (a column of the product each): an element is off by 2^-14.8 of its block's largest
//     in the root mean square and by 2^-10 at most (each row leaves 0.1771 of it, a sixth and e4m3's rounding of the scale), by 2^-24
//     of the row's largest where the block is so far below that its scales vanish.
//     Lane k of the accumulator holds key k's products with all of them; a thread, who has a key, adds the four up, joins the
//     key's and the value's powers of two and makes the weights of its key.
//   O^T = V^T P^T on mma.sync (m16n8k16, A = 16 dimensions x 16 keys): a warp has the 32 keys whose weights its threads made, so that
//     they pass through the warp's own shared memory only.  A thread has the block of dimensions from 16 g on, of four keys: the
//     codes of two keys are interleaved (two instructions a word), so that a byte is a pair of keys, and become float16 (one
//     instruction a pair), times the two block scales.  Keys 2 and 3, 6 and 7 of each eight change places, so that no two rows
//     that are read at a time share banks.
// The outputs' weights 2^(a + E_v - D + LIFT) (the references of attention_fp4.cuh, a warp's own) are rounded to float16 (11 digits): at
// most 2^15, so that what lies 2^-29 below the largest still has all digits.  Sums are in float32, the warps' own until the end of the
// run, where they are added in the order of the warps.
//
// What bounds it: instructions, some 300 for 32 keys of a warp (130 of them conversions and scales of values; with keys converted the
// same way some 700), and the chain of a tile, some 3,000 cycles of which three or four CTAs an SM run side by side: an instruction issues
// in 54 % of the cycles.  With the merge, 32 / 8 heads of 128: 64 requests of up to 4,096 keys 53 us, 3.3 TB/s; 64 / 8 heads, four of 32,000
// keys 56 us, 2.7 TB/s; 16 / 8 heads, 16 drafts of 5 tokens on up to 1,500 keys 26 us; one of 2,048 keys 8.9 us.
//
// Roles in a CTA: warps 0-3 as above, warp 4 copies (TMA, a box a page; scales by cp.async), warp 5 issues the scores' products, warp
// 6 finds the next work items, warp 7 adds the four warps' sums of an item up under the next one.  The first group of warps gets a
// part of the second's registers.
// Work items: (sequence, kv head, tile of rows, run of keys), a CTA takes a contiguous range of them.  The length of a run
// follows from the sequence's own lengths, so a row's bits do not depend on the rest of the step.
#include <cuda.h>

#include "attention_fp4.cuh"

namespace {

__device__ int dib_attention_fp4_error_word = 0;

constexpr int ST_THREADS = 256, ST_ITEMS = 4, ST_PARTS = 4;
constexpr int ST_COPY_WARP = 4, ST_SCORE_WARP = 5, ST_WALK_WARP = 6;      // and 7: sums
// a stage: codes of keys and values (rows of 64 bytes, swizzled), block scales of keys (two tiles of 128 rows x 64 values, as the products
// take them) and values (a row a key), exponents
constexpr int ST_V = SP_TILE * 64, ST_KS = 2 * ST_V, ST_VS = ST_KS + 1024, ST_KE = ST_VS + SP_TILE * 8, ST_VE = ST_KE + SP_TILE,
              ST_STAGE = (ST_VE + SP_TILE + 511) / 512 * 512;

__device__ __forceinline__ void mbar_init(unsigned long long* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_2d(unsigned dst, const CUtensorMap* map, int c0, int c1, unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<unsigned long long>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Issued by one lane, in code that the whole warp runs: what they are given stays in uniform registers.
__device__ __forceinline__ unsigned elect_one() {
  unsigned is;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t"
      "}\n" : "=r"(is));
  return is;
}
__device__ __forceinline__ void tc_commit(unsigned elected, unsigned long long* bar) {
  asm volatile(
      "{\n\t"
      ".reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
      "}\n" ::"r"(smem_u32(bar)), "r"(elected)
      : "memory");
}
// a tile of 128 rows' scales of 64 values (512 bytes) into four columns of tensor memory
__device__ __forceinline__ void tc_copy_scales(unsigned elected, unsigned tmem, unsigned long long desc) {
  asm volatile(
      "{\n\t"
      ".reg .pred e;\n\t"
      "setp.ne.b32 e, %2, 0;\n\t"
      "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t"
      "}\n" ::"r"(tmem), "l"(desc), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tc_mma(unsigned elected, unsigned tmem_d, unsigned long long desc_a, unsigned long long desc_b,
                                       unsigned idesc, unsigned scales_a, unsigned scales_b, unsigned accum) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 e, %7, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
      "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scales_a), "r"(scales_b), "r"(accum), "r"(elected)
      : "memory");
}
// Waits for tc_ld16, whose N registers are handed on here: arithmetic on them must not be moved ahead of the wait.
template <int N> __device__ __forceinline__ void tc_wait_ld(unsigned (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}
// 16 consecutive columns of this thread's lane; valid after tc_wait_ld()
__device__ __forceinline__ void tc_ld16(unsigned taddr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// K-major rows of 64 bytes, 64-byte swizzle: 8-row groups 512 bytes apart
__device__ __forceinline__ unsigned long long operand_desc(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((unsigned long long)(512u >> 4) << 32) | (1ull << 46) |
         (4ull << 61);
}
// 32 rows of 16 bytes, one after the other: 8-row groups 128 bytes apart
__device__ __forceinline__ unsigned long long scales_desc(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(128u >> 4) << 32) | (1ull << 46);
}
// kind::mxf4nvf4: e2m1 operands, both K-major, unsigned e4m3 scales, 64 values an instruction
__host__ __device__ constexpr unsigned make_idesc(int m, int n) {
  return (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 7) << 27);
}
__device__ __forceinline__ float warp_top(float v) {      // the largest of the warp's values, NaN aside
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
template <int N> __device__ __forceinline__ void regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// A work item as it is handed from the warp that walks the CTA's items to the others.
struct __align__(16) StreamItem {
  int seq, q_begin, n, kv_len;      // the sequence: index, first token, new tokens, keys
  int i, kvh, tile, local;          // sequence of the launch, kv head, tile of rows, number of the item in its sequence
  int seen, at, end, splits;        // its keys: [seen, end), those of the run that some row sees; its tiles from `at` on, a multiple
                                    // of 128; runs of the sequence
  int fresh, tiles, lo_all, hi_all;        // other query rows than the item before; tiles of keys, 0: there are no more
                                           // items; the keys that every row sees
};

template <bool V> struct Flag {
  static constexpr bool value = V;
};
template <int ROWS> struct StreamShape {
  static constexpr int STAGES = 2;
  static constexpr int NT = (ROWS + 7) / 8, N = ROWS * ST_PARTS;      // tiles of 8 rows, columns of the scores
  static constexpr int SFK = 2 * N, SFQ = SFK + 8, TMEM = SFQ + 8 <= 64 ? 64 : SFQ + 8 <= 128 ? 128 : 256;
  static constexpr int QUERIES = (STAGES * ST_STAGE + 1023) / 1024 * 1024;              // [2][N][64], swizzled
  static constexpr int QSCALES = QUERIES + 2 * N * 64;                // [2] two tiles of 512 bytes
  static constexpr int WEIGHTS = QSCALES + 2 * 1024;                  // [4 warps][NT][32 keys][8 rows] float16
  static constexpr int SUMS = WEIGHTS + 4 * NT * 512;                 // [4 warps][ROWS][132]
  static constexpr int TOPS = SUMS + 4 * ROWS * 132 * 4;              // [4 warps][ROWS] references (at, D)
  static constexpr int PARTS = TOPS + 4 * ROWS * 8;                   // [4 warps][ROWS][16 lanes] parts of the sums of weights
  static constexpr int FOUND = PARTS + 4 * ROWS * 64;                 // [4 warps][ROWS + 4] D of the rows, whether one is not 0
  static constexpr int UNITS = FOUND + 4 * (ROWS + 4) * 4;            // [2][ROWS] of the scores
  static constexpr int SEEN = UNITS + 2 * ROWS * 4;                   // [2][2][ROWS] first and last key
  static constexpr int ITEMS = SEEN + 2 * 2 * ROWS * 4;
  static constexpr int BARS = ITEMS + ST_ITEMS * 64;
  static constexpr int SEQS = BARS + 32 * 8;                          // [sequences] int4, then the work before each
  static constexpr size_t fixed = SEQS + 16 + 1024;
  // CTAs an SM; they are launched with 64, 80 or 128 registers a thread, and the groups' shares add up to twice that
  static constexpr int CTAS = ROWS <= 4 ? 4 : ROWS <= 8 ? 3 : 2;
  static constexpr int REGS_MANY = ROWS <= 4 ? 88 : ROWS <= 8 ? 104 : 200, REGS_FEW = ROWS <= 4 ? 40 : 56;
};

template <int ROWS, int D>
__global__ void __launch_bounds__(ST_THREADS, StreamShape<ROWS>::CTAS)
attention_stream_kernel(const __grid_constant__ CUtensorMap map, const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out,
                        const __grid_constant__ SplitArgs a, const int box_rows, const int late) {
  using SH = StreamShape<ROWS>;
  constexpr int NT = SH::NT, N = SH::N, STAGES = SH::STAGES;
  extern __shared__ unsigned char smem_raw[];
  // (an offset, not a rounded address: what is known to be shared memory is read and written with 32-bit addresses)
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  StreamItem* items = reinterpret_cast<StreamItem*>(smem + SH::ITEMS);
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + SH::BARS);
  unsigned long long* full = bars;             // [3] a tile's keys, values, scales and exponents have arrived
  unsigned long long* empty = bars + 3;        // [3] all of it has been read
  unsigned long long* s_full = bars + 6;       // [2] its scores are in tensor memory
  unsigned long long* s_empty = bars + 8;      // [2] they have been read
  unsigned long long* q_full = bars + 10;      // [2] an item's query rows are in shared memory
  unsigned long long* q_empty = bars + 12;     // [2] they have been read
  unsigned long long* sum_full = bars + 14;    // the four warps' sums of an item are in shared memory
  unsigned long long* sum_empty = bars + 15;   // they have been read
  unsigned long long* item_full = bars + 16;   // [ST_ITEMS] an item's record is there
  unsigned long long* item_empty = bars + 16 + ST_ITEMS;      // [ST_ITEMS] it has been read by every role
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 16 + 2 * ST_ITEMS);
  int4* seqs = reinterpret_cast<int4*>(smem + SH::SEQS);
  long long* first = reinterpret_cast<long long*>(seqs + a.seq_count);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int G = a.Hq / a.Hkv;
  if (threadIdx.x == 0) prefetch_tensormap(&map);
  // ---- the work before each sequence (metadata alone, which no kernel of a step writes)
  for (int i = threadIdx.x; i < a.seq_count; i += ST_THREADS) {
    const int4 m = load_seq(a, i);
    const SplitSeq s = split_seq<ROWS>(a, m);
    seqs[i] = m;
    first[i + 1] = s.items(a.Hkv) * s.item_work();
  }
  if (threadIdx.x == 0) first[0] = 0;
  if (threadIdx.x == 32) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 33);
      mbar_init(&empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
      mbar_init(&q_full[i], 4);
      mbar_init(&q_empty[i], 1);
    }
    mbar_init(sum_full, 4);
    mbar_init(sum_empty, 1);
    for (int i = 0; i < ST_ITEMS; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 7);      // copy, scores, sums, four that compute
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ST_SCORE_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((unsigned)SH::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  __syncthreads();
  // (with its tensor memory taken: the blocks of the kernel that follows wait for this grid, and must not hold what one of it waits for)
  if (!late) pdl_trigger();
  if (warp == 0) {
    long long base = 0;
    for (int i0 = 0; i0 < a.seq_count; i0 += 32) {
      long long v = i0 + lane < a.seq_count ? first[i0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (i0 + lane < a.seq_count) first[i0 + lane + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_wait(q);
  bool ok = true;

  if (warp >= 4) {
  regs_give<SH::REGS_FEW>();
  if (warp == ST_COPY_WARP) {
    // ---- copies: lane l has the keys 4l .. 4l + 3 of a tile; the first lane of each page sends for its rows
    const int page_mask = (1 << a.page_shift) - 1, half = a.Hkv << a.page_shift;
    constexpr int row_scales = D >> 4;      // half: rows of a page's keys
    int n = 0, stage = 0;
    unsigned phase = 1;      // (the ring's first round finds it empty)
    for (int k = 0; ok; ++k) {
      const int slot = k % ST_ITEMS;
      ok = mbar_wait_brief(&item_full[slot], (k / ST_ITEMS) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int seq = items[slot].seq, kvh = items[slot].kvh, at = items[slot].at, end = items[slot].end, tiles = items[slot].tiles;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (tiles == 0) break;
      const int* table = a.block_table + (long long)seq * a.max_blocks;
      for (int kb = at; kb < end; kb += SP_TILE, ++n) {
        const int key = kb + lane * 4, off = key & page_mask;
        int page = -1;
        if (key < end) page = table[key >> a.page_shift];
        const bool have = page >= 0 && page < a.num_pages;
        const unsigned senders = __ballot_sync(0xffffffffu, have && (lane == 0 || off == 0));
        if (n >= STAGES) ok = mbar_wait_brief(&empty[stage], phase);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&full[stage], __popc(senders) * box_rows * 128);
        __syncwarp();
        const int row = have ? page * 2 * half + (kvh << a.page_shift) + off : 0;
        const unsigned to = smem_u32(smem) + stage * ST_STAGE;
        if (senders >> lane & 1) {
          tma_load_2d(to + lane * 256, &map, 0, row, &full[stage]);
          tma_load_2d(to + ST_V + lane * 256, &map, 0, row + half, &full[stage]);
        }
        // (keys that are not there, and those on a page that is none of the pool's: scales and exponents of zero)
        const unsigned char* ks = a.scales + (long long)row * row_scales;
        const unsigned char* vs = a.scales + (long long)(have ? row + half : 0) * row_scales;
        const int r = lane * 4;
        const unsigned tile = to + ST_KS + (r & 31) * 16 + (r >> 5) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          cp_async4(tile + e * 16, ks + e * row_scales, have ? 4 : 0);
          if (row_scales == 8) cp_async4(tile + 512 + e * 16, ks + e * row_scales + 4, have ? 4 : 0);
        }
        cp_async16(to + ST_VS + r * row_scales, vs, have ? 16 : 0);
        if (row_scales == 8) cp_async16(to + ST_VS + r * row_scales + 16, vs + 16, have ? 16 : 0);
        cp_async4(to + ST_KE + r, a.exponents + row, have ? 4 : 0);
        cp_async4(to + ST_VE + r, a.exponents + (have ? row + half : 0), have ? 4 : 0);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[stage])) : "memory");
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok)      // given up: what was sent for arrives before this memory is another's
      for (int m = max(n - STAGES, 0); m < n; ++m) mbar_wait_brief(&full[m % STAGES], (m / STAGES) & 1);
  } else if (warp == ST_SCORE_WARP) {
    // ---- scores: a tile ahead of the weights
    const unsigned elected = elect_one(), base = smem_u32(smem);
    constexpr unsigned idesc = make_idesc(128, N);
    constexpr int k_steps = D >> 6;
    int n = 0, q_used = -1, stage = 0;
    unsigned phase = 0;
    for (int k = 0; ok; ++k) {
      const int slot = k % ST_ITEMS;
      ok = __all_sync(0xffffffffu, mbar_wait_brief(&item_full[slot], (k / ST_ITEMS) & 1));
      if (!ok) break;
      const int tiles = items[slot].tiles, fresh = items[slot].fresh;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (tiles == 0) break;
      if (fresh) {
        if (q_used >= 0) tc_commit(elected, &q_empty[q_used & 1]);
        ++q_used;
        ok = __all_sync(0xffffffffu, mbar_wait_brief(&q_full[q_used & 1], (q_used >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        for (int s = 0; s < k_steps; ++s)
          tc_copy_scales(elected, tmem + SH::SFQ + 4 * s, scales_desc(base + SH::QSCALES + (q_used & 1) * 1024 + s * 512));
      }
      const unsigned long long qd = operand_desc(base + SH::QUERIES + (q_used & 1) * N * 64);
      for (int t = tiles; t > 0 && ok; --t, ++n) {
        ok = __all_sync(0xffffffffu, mbar_wait_brief(&full[stage], phase) &&
                                         (n < 2 || mbar_wait_brief(&s_empty[n & 1], ((n >> 1) - 1) & 1)));
        if (!ok) break;
        tc_fence_after();
        proxy_fence();      // the scales came by cp.async and are read by the tensor core
        const unsigned at = base + stage * ST_STAGE;
        const unsigned long long kd = operand_desc(at), sd = scales_desc(at + ST_KS);
        for (int s = 0; s < k_steps; ++s) tc_copy_scales(elected, tmem + SH::SFK + 4 * s, sd + s * (512 >> 4));
        for (int s = 0; s < k_steps; ++s)
          tc_mma(elected, tmem + (n & 1) * N, kd + s * 2, qd + s * 2, idesc, tmem + SH::SFK + 4 * s, tmem + SH::SFQ + 4 * s, s > 0);
        tc_commit(elected, &s_full[n & 1]);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == ST_WALK_WARP) {
    // ---- the walk over this CTA's items, a contiguous range of equal work
    const long long total = first[a.seq_count];
    const int place = block_place(a);
    const long long from_work = total / gridDim.x * place + total % gridDim.x * place / gridDim.x;
    const long long to_work = total / gridDim.x * (place + 1) + total % gridDim.x * (place + 1) / gridDim.x;
    int i = 0, old_i = -1, old_kvh = -1, old_tile = -1, item = 0;
    SplitSeq s = {};
    if (total > 0) {
      for (int hi = a.seq_count - 1; i < hi;) {      // the sequence in which the range begins
        const int mid = (i + hi + 1) >> 1;
        if (first[mid] <= from_work) i = mid; else hi = mid - 1;
      }
      s = split_seq<ROWS>(a, seqs[i]);
      const int each = s.item_work();
      item = (int)((from_work - first[i] + each - 1) / each);       // the first item that begins in it
    }
    for (int k = 0; ok;) {
      const int slot = k % ST_ITEMS;
      StreamItem it = {};              // (as it is: no more items)
      bool more = false;
      while (total > 0 && i < a.seq_count) {
        if (item < s.items(a.Hkv)) {
          more = first[i] + (long long)item * s.item_work() < to_work;
          break;
        }
        item = 0;
        if (++i < a.seq_count) s = split_seq<ROWS>(a, seqs[i]);
      }
      if (more) {
        const int local = item++, unit = s.splits > 1 ? local / s.splits : local, run_at = (local - unit * s.splits) * s.split;
        it.seq = s.seq; it.q_begin = s.q_begin; it.n = s.n; it.kv_len = s.kv_len;
        it.i = i; it.local = local; it.splits = s.splits;
        it.kvh = s.tiles > 1 ? unit / s.tiles : unit;
        it.tile = unit - it.kvh * s.tiles;
        const int p0 = s.kv_len - s.n;
        int tok0 = 0, tok1 = s.n - 1;
        if (s.tiles > 1) {
          tok0 = it.tile * ROWS / G;
          tok1 = (min((it.tile + 1) * ROWS, s.n * G) - 1) / G;
        }
        it.seen = max(run_at, first_visible_key(p0 + tok0, a.window));
        it.end = min(run_at + s.split, p0 + tok1 + 1);
        it.at = it.seen & ~(SP_TILE - 1);
        if (it.end <= it.seen) {
          if (s.splits == 1) {             // a sequence of one run: rows that see no key are zeros, from here
            const int rows = min(ROWS, s.n * G - it.tile * ROWS);
            for (int e = lane; e < rows * D; e += 32) {
              const int row = it.tile * ROWS + e / D, tok = row / G;
              Elem<__nv_bfloat16>::store(out + ((long long)(s.q_begin + tok) * a.Hq + it.kvh * G + row - tok * G) * D + e % D, 0.f);
            }
          }
          continue;
        }
        it.tiles = (it.end - it.at + SP_TILE - 1) / SP_TILE;
        it.lo_all = max(run_at, first_visible_key(p0 + tok1, a.window));
        it.hi_all = min(it.end - 1, p0 + tok0);
        it.fresh = i != old_i || it.kvh != old_kvh || it.tile != old_tile;
        old_i = i; old_kvh = it.kvh; old_tile = it.tile;
      }
      if (k >= ST_ITEMS) ok = mbar_wait_brief(&item_empty[slot], ((k / ST_ITEMS) - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        items[slot] = it;
        mbar_arrive(&item_full[slot]);
      }
      ++k;
      if (it.tiles == 0) break;
    }
  } else {
    // ---- an item's sums: a lane four places of a row; finished where the sequence has one run, else partial results for the merge
    const float* sums = reinterpret_cast<const float*>(smem + SH::SUMS);
    const float2* tops = reinterpret_cast<const float2*>(smem + SH::TOPS);
    const float* parts = reinterpret_cast<const float*>(smem + SH::PARTS);
    const int d0 = dim_of(lane * 4), d1 = dim_of(lane * 4 + 2);
    for (int k = 0; ok; ++k) {
      const int slot = k % ST_ITEMS;
      ok = mbar_wait_brief(&item_full[slot], (k / ST_ITEMS) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const StreamItem it = items[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (it.tiles == 0) break;
      const int row0 = it.tile * ROWS, rows = min(ROWS, it.n * G - row0);
      ok = mbar_wait_brief(sum_full, k & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // A lane finds what the warps' sums of a row are taken times, f those of the weights, fo those of the outputs; it is handed to the
      // others, a row after another.
      const long long to = ((long long)it.i * a.max_items + it.local) * ROWS;
      auto finish = [&](const float (&f)[4], const float (&fo)[4], const float top_d, auto odd) {
#pragma unroll 1
        for (int r = 0; r < rows; ++r) {
          float sum = 0.f;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float w = __shfl_sync(0xffffffffu, f[x], r);
            const float4 v = *reinterpret_cast<const float4*>(sums + (x * ROWS + r) * 132 + lane * 4);
            if (lane < 16) sum = fmaf(w, parts[(x * ROWS + r) * 16 + lane], sum);
            if (odd.value) w = __shfl_sync(0xffffffffu, fo[x], r);
            y.x = fmaf(w, v.x, y.x); y.y = fmaf(w, v.y, y.y);
            y.z = fmaf(w, v.z, y.z); y.w = fmaf(w, v.w, y.w);
          }
          sum = warp_sum(sum);
          if (it.splits == 1) {
            const int tok = (row0 + r) / G;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            __nv_bfloat16* dst = out + ((long long)(it.q_begin + tok) * a.Hq + it.kvh * G + row0 + r - tok * G) * D;
            y.x *= inv; y.y *= inv; y.z *= inv; y.w *= inv;
            if (odd.value) {
              const float d = __shfl_sync(0xffffffffu, top_d, r);
              y.x = times_power(y.x, d); y.y = times_power(y.y, d);
              y.z = times_power(y.z, d); y.w = times_power(y.w, d);
            }
            if (d0 < D) store_two<__nv_bfloat16>(dst + d0, y.x, y.y);
            if (d1 < D) store_two<__nv_bfloat16>(dst + d1, y.z, y.w);
          } else if (it.local < a.max_items) {
            *reinterpret_cast<float4*>(a.part_o + (to + r) * 128 + lane * 4) = y;
            if (lane == 0) a.part_ml[to + r].z = sum;
          }
        }
      };
      float2 refs[4];
      float f[4], top = UNSET, top_d = 0.f;
      bool odd = false;      // some D is not 0
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        refs[x] = tops[x * ROWS + lane % ROWS];
        top = fmaxf(top, refs[x].x);
        odd |= refs[x].y != 0.f;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) f[x] = fast_exp2(refs[x].x - top);
      if (!__any_sync(0xffffffffu, odd)) {
        finish(f, f, 0.f, Flag<false>());
      } else {
        float fo[4];
        top_d = UNSET;
#pragma unroll
        for (int x = 0; x < 4; ++x) top_d = fmaxf(top_d, rintf(refs[x].x - top + refs[x].y));
#pragma unroll
        for (int x = 0; x < 4; ++x) fo[x] = fast_exp2(refs[x].x - top + refs[x].y - top_d);
        finish(f, fo, top_d, Flag<true>());
      }
      if (it.splits > 1 && it.local < a.max_items && lane < rows) *reinterpret_cast<float2*>(a.part_ml + to + lane) = make_float2(top, top_d);
      __syncwarp();
      if (lane == 0) mbar_arrive(sum_empty);
    }
  }
  } else {
    regs_take<SH::REGS_MANY>();
    // ---- weights and outputs: thread = key of the warp's 32, then a block of dimensions and pairs of rows
    constexpr int row_scales = D >> 4;
    const int g = lane >> 2, t = lane & 3;
    const unsigned tm = tmem + ((unsigned)(warp * 32) << 16);
    unsigned char* weights = smem + SH::WEIGHTS + warp * NT * 512;
    float* sums = reinterpret_cast<float*>(smem + SH::SUMS) + warp * ROWS * 132;
    float2* tops = reinterpret_cast<float2*>(smem + SH::TOPS) + warp * ROWS;
    float* parts = reinterpret_cast<float*>(smem + SH::PARTS) + warp * ROWS * 16;
    float* found = reinterpret_cast<float*>(smem + SH::FOUND) + warp * (ROWS + 4);
    int n = 0, q_used = -1, done = 0, stage = 0;
    unsigned phase = 0;
    for (int k = 0; ok; ++k) {
      const int slot = k % ST_ITEMS;
      ok = mbar_wait_brief(&item_full[slot], (k / ST_ITEMS) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const StreamItem it = items[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (it.tiles == 0) break;
      const int row0 = it.tile * ROWS, rows = min(ROWS, it.n * G - row0);
      if (it.fresh) {
        // ---- the query rows: half a warp has a row, a lane 8 of its dimensions.  (How a rest is rounded is of no account: the next
        // part has what is left.)
        ++q_used;
        const int hl = lane & 15, qbuf = q_used & 1;
        uint4 raw[(ROWS + 7) / 8];
#pragma unroll
        for (int x = 0; x < (ROWS + 7) / 8; ++x) {
          const int r = x * 8 + warp * 2 + (lane >> 4), tok = (row0 + r) / G;
          raw[x] = make_uint4(0, 0, 0, 0);
          if (r < rows && hl * 8 < D)
            raw[x] = *reinterpret_cast<const uint4*>(q + ((long long)(it.q_begin + tok) * a.Hq + it.kvh * G + row0 + r - tok * G) * D + hl * 8);
        }
        if (q_used >= 2) ok = mbar_wait_brief(&q_empty[qbuf], ((q_used >> 1) - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        unsigned char* codes = smem + SH::QUERIES + qbuf * N * 64;
        unsigned char* scales = smem + SH::QSCALES + qbuf * 1024;
        float* units = reinterpret_cast<float*>(smem + SH::UNITS) + qbuf * ROWS;
        int* seen = reinterpret_cast<int*>(smem + SH::SEEN) + qbuf * 2 * ROWS;
#pragma unroll
        for (int x8 = 0; x8 < (ROWS + 7) / 8; ++x8) {
          const int r = x8 * 8 + warp * 2 + (lane >> 4);
          const unsigned w[4] = {raw[x8].x, raw[x8].y, raw[x8].z, raw[x8].w};
          float x[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          }
          unsigned top = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, fp4_magnitude(x[e]));
#pragma unroll
          for (int s = 1; s < 16; s <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
          // in units of the row's 2^E, at most 2,688 (a row that holds an infinity or a NaN: its scores are NaN)
          const unsigned exponent = fp4_row_exponent(top);
          const float down = fp4_down(exponent);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = exponent == FP4_NO_NUMBER ? 0.f : x[e] * down;
#pragma unroll
          for (int p = 0; p < ST_PARTS; ++p) {
            float most = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            const unsigned scale = fp4_scale_code(most * (1.f / 6.f));
            const float b = fp4_scale_value(scale), inv = __fdividef(1.f, fmaxf(b, 0x1p-20f));
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[e] * inv;
            const unsigned code = fp4_pack8(y);
            const int col = p * ROWS + r;
            if (r < ROWS) {
              *reinterpret_cast<unsigned*>(codes + col * 64 + (((hl >> 2) ^ (col >> 1 & 3)) << 4) + (hl & 3) * 4) = code;
              if ((hl & 1) == 0) scales[(hl >> 3) * 512 + (col & 31) * 16 + (col >> 5) * 4 + (hl >> 1 & 3)] = (unsigned char)scale;
            }
            // the rest in units of a quarter: it is a sixth of the largest at most.  (The codes by way of a shuffle: taken straight
            // from the conversion to them, the conversion back gave the upper four as zeros, nvcc 12.9.)
            fp4_values8(__shfl_sync(0xffffffffu, code, lane), b, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (x[e] - y[e]) * 4.f;
          }
          if (hl == 0 && r < ROWS) {
            const int pos = it.kv_len - it.n + (row0 + r) / G;
            units[r] = exponent == FP4_NO_NUMBER ? __uint_as_float(0x7fc00000u) : fp4_unit(exponent) * (a.scale * LOG2E);
            seen[r] = first_visible_key(pos, a.window);
            seen[ROWS + r] = r < rows ? pos : -1;
          }
        }
        proxy_fence();      // the rows are read by the tensor core
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[qbuf]);
        // (what belongs to the rows is every warp's)
        ok = mbar_wait_brief(&q_full[qbuf], (q_used >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      const float* units = reinterpret_cast<const float*>(smem + SH::UNITS) + (q_used & 1) * ROWS;
      const int* row_seen = reinterpret_cast<const int*>(smem + SH::SEEN) + (q_used & 1) * 2 * ROWS;
      float ref[ROWS], l[ROWS], o[8][NT][4];
      if (lane <= ROWS) found[lane] = 0.f;
      __syncwarp();
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        ref[r] = UNSET;
        l[r] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[d][nt][0] = o[d][nt][1] = o[d][nt][2] = o[d][nt][3] = 0.f;
#pragma unroll 1
      for (int kb = it.at; kb < it.end; kb += SP_TILE, ++n) {
        const int buf = n & 1;
        ok = mbar_wait_brief(&full[stage], phase) && mbar_wait_brief(&s_full[buf], (n >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const unsigned char* st = smem + stage * ST_STAGE;
        const int in_tile = warp * 32 + lane, key = kb + in_tile;
        const bool plain = kb >= it.lo_all && kb + SP_TILE - 1 <= it.hi_all;        // every row sees every key
        // ---- scores and the value's power of two.  An exponent of no number, the key's or the value's, makes those of the rows that see
        // it NaN.
        float z[ROWS];
        {
          unsigned v[N];
#pragma unroll
          for (int c = 0; c < N; c += 16) tc_ld16(tm + buf * N + c, v + c);
          tc_wait_ld(v);
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            z[r] = fmaf(fmaf(fmaf(__uint_as_float(v[3 * ROWS + r]), 0.25f, __uint_as_float(v[2 * ROWS + r])), 0.25f,
                             __uint_as_float(v[ROWS + r])), 0.25f, __uint_as_float(v[r]));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[buf]);
        const unsigned ke = st[ST_KE + in_tile], ve = st[ST_VE + in_tile];
        const float ks = fp4_unit(ve == FP4_NO_NUMBER ? ve : ke), lv = (float)(int)ve - 127.f;
        float back = off_value(ve), less = -1.f;      // (0 where the references are off the scores already)
        const bool odd = found[ROWS] != 0.f;
        bool over = odd || !is_tame(ve);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          z[r] = fmaf(z[r], ks * units[r], lv);
          if (!plain && (key < it.seen || key >= it.end || key < row_seen[r] || key > row_seen[ROWS + r])) z[r] = -INFINITY;
          over |= z[r] > ref[r] + (LIFT + RAISE);
        }
        if (__any_sync(0xffffffffu, over)) {
          const bool wild = !is_tame(ve) && (plain || (key >= it.seen && key < it.end)), first = kb == it.at;
          bool apart = odd || __any_sync(0xffffffffu, wild);
          float f[NT * 8];
#pragma unroll
          for (int r = 0; r < NT * 8; ++r) f[r] = 1.f;
          if (!apart) {
            float most = 0.f;
            if (first) {      // (a row that sees none of the tile's keys while another does: below)
#pragma unroll
              for (int r = 0; r < ROWS; ++r) {
                ref[r] = warp_top(z[r]) - LIFT;
                most = fmaxf(most, fabsf(ref[r]));
              }
            } else {
#pragma unroll
              for (int r = 0; r < ROWS; ++r) {
                const float top = warp_top(z[r]);
                if (top > ref[r] + (LIFT + RAISE)) {
                  const float to = top - LIFT;
                  most = fmaxf(most, fabsf(to));
                  if (fabsf(to) < FAR) {
                    f[r] = fast_exp2(ref[r] - to);
                    l[r] *= f[r];
                    ref[r] = to;
                  }
                }
              }
            }
            apart = most >= FAR;
            if (apart && first) {
#pragma unroll
              for (int r = 0; r < ROWS; ++r) ref[r] = UNSET;
            }
          }
          if (apart) {
            // Values or scores far from one another: the tile's part of the sums of weights from here, a row at a time, by way of the
            // sums' memory (unrolled, it costs those that never come here: 6 of 78 us for 16 drafts on 4,096 keys, 32 heads).
            if (done > 0) ok = mbar_wait_brief(sum_empty, (done - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
              sums[r * 132 + lane] = z[r];
              sums[r * 132 + 32 + lane] = l[r];
              if (lane == 0) *reinterpret_cast<float2*>(sums + r * 132 + 64) = make_float2(ref[r], f[r]);
            }
            __syncwarp();
            bool any_d = false;
#pragma unroll 1
            for (int r = 0; r < ROWS; ++r) {
              float* row = sums + r * 132;
              const float2 was = *reinterpret_cast<const float2*>(row + 64);
              const float at = row[lane], score = at - lv, old = odd ? found[r] : 0.f;
              const bool fresh = was.x == UNSET, wide = __any_sync(0xffffffffu, wild && at > -INFINITY);
              float top = warp_top(at), to = top > was.x + (LIFT + RAISE) ? top - LIFT : was.x, d = old, y = at - to;
              float f_l = fast_exp2(was.x - to), f_o = f_l;
              if (old != 0.f || (fabsf(to) >= FAR && to != UNSET) || wide) {
                const float base = fresh ? 0.f : was.x;
                top = warp_top(score - base);
                const float by = top > (fresh ? -INFINITY : HIGH) ? rintf(top) - LIFT : 0.f;
                to = base + by;
                d -= by;
                top = warp_top(score - to + lv);
                if (fresh || top - d > LIFT + RAISE) d = top > -INFINITY ? rintf(top) - LIFT : 0.f;
                y = score - to + (lv - d);
                f_l = fresh ? 0.f : fast_exp2(-by);
                f_o = fresh ? 0.f : fast_exp2(old - by - d);
              }
              const float sum = row[32 + lane] * f_l;
              row[lane] = y;
              row[32 + lane] = d != 0.f || wild ? sum + fast_exp2(score - to) : fmaf(fast_exp2(y), back, sum);
              any_d |= d != 0.f;
              __syncwarp();
              if (lane == 0) {
                *reinterpret_cast<float2*>(row + 64) = make_float2(to, was.y * f_o);
                found[r] = d;
              }
            }
            __syncwarp();
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
              const float2 is = *reinterpret_cast<const float2*>(sums + r * 132 + 64);
              z[r] = sums[r * 132 + lane];
              l[r] = sums[r * 132 + 32 + lane];
              ref[r] = is.x;
              f[r] = is.y;
            }
            __syncwarp();
            back = less = 0.f;
            if (lane == 0) found[ROWS] = any_d ? 1.f : 0.f;
            __syncwarp();
          }
          if (!first) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float f0 = t < 2 ? (t == 0 ? f[nt * 8] : f[nt * 8 + 2]) : (t == 2 ? f[nt * 8 + 4] : f[nt * 8 + 6]);
              const float f1 = t < 2 ? (t == 0 ? f[nt * 8 + 1] : f[nt * 8 + 3]) : (t == 2 ? f[nt * 8 + 5] : f[nt * 8 + 7]);
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                o[d][nt][0] *= f0; o[d][nt][2] *= f0;
                o[d][nt][1] *= f1; o[d][nt][3] *= f1;
              }
            }
          }
        }
        // ---- weights, through the warp's own shared memory, as B operands
        unsigned two[NT * 4];
#pragma unroll
        for (int r = 0; r < NT * 8; r += 2) {
          float w[2] = {0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (r + c < ROWS) {
              w[c] = fast_exp2(fmaf(ref[(r + c) % ROWS], less, z[(r + c) % ROWS]));
              l[(r + c) % ROWS] = fmaf(w[c], back, l[(r + c) % ROWS]);
            }
          two[r / 2] = pack_half(w[0], w[1]);
        }
        unsigned pw[2][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<uint4*>(weights + nt * 512 + (lane ^ (lane >> 1 & 1)) * 16) =
              make_uint4(two[4 * nt], two[4 * nt + 1], two[4 * nt + 2], two[4 * nt + 3]);
        __syncwarp();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                       : "=r"(pw[0][nt][0]), "=r"(pw[0][nt][1]), "=r"(pw[1][nt][0]), "=r"(pw[1][nt][1])
                       : "r"(smem_u32(weights) + nt * 512 + lane * 16)
                       : "memory");
        // ---- outputs
        const int place = ((g >> 1 ^ t) << 4) + (g & 1) * 8;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int ra = warp * 32 + m * 16 + (2 * t ^ (t & 1)), rb = ra ^ 1;      // and 8 keys on
          const uint2 va = *reinterpret_cast<const uint2*>(st + ST_V + ra * 64 + place);
          const uint2 vb = *reinterpret_cast<const uint2*>(st + ST_V + rb * 64 + place);
          const uint2 vc = *reinterpret_cast<const uint2*>(st + ST_V + (ra + 8) * 64 + place);
          const uint2 vd = *reinterpret_cast<const uint2*>(st + ST_V + (rb + 8) * 64 + place);
          unsigned sab = 0, scd = 0;
          if (g < row_scales) {
            const unsigned char* vs = st + ST_VS + g;
            sab = vs[ra * row_scales] | (unsigned)vs[rb * row_scales] << 8;
            scd = vs[(ra + 8) * row_scales] | (unsigned)vs[(rb + 8) * row_scales] << 8;
          }
          if (!plain) {      // keys that no row sees: whatever is held there, nothing comes of it
            const int ka = kb + ra, kc = kb + rb;
            if (ka < it.seen || ka >= it.end) sab &= 0xff00u;
            if (kc < it.seen || kc >= it.end) sab &= 0x00ffu;
            if (ka + 8 < it.seen || ka + 8 >= it.end) scd &= 0xff00u;
            if (kc + 8 < it.seen || kc + 8 >= it.end) scd &= 0x00ffu;
          }
          sab = scales_to_half(sab);
          scd = scales_to_half(scd);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const unsigned xa = y ? va.y : va.x, xb = y ? vb.y : vb.x, xc = y ? vc.y : vc.x, xd = y ? vd.y : vd.x;
            // bytes of (this key's code, the next key's code) of the even and the odd dimensions
            unsigned e0[4], e1[4], f0[4], f1[4];
            codes_to_half((xa & 0x0f0f0f0fu) | (xb << 4 & 0xf0f0f0f0u), e0);
            codes_to_half((xa >> 4 & 0x0f0f0f0fu) | (xb & 0xf0f0f0f0u), e1);
            codes_to_half((xc & 0x0f0f0f0fu) | (xd << 4 & 0xf0f0f0f0u), f0);
            codes_to_half((xc >> 4 & 0x0f0f0f0fu) | (xd & 0xf0f0f0f0u), f1);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const unsigned a0 = mul_half(e0[x], sab), a1 = mul_half(e1[x], sab), a2 = mul_half(f0[x], scd), a3 = mul_half(f1[x], scd);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma(o[4 * y + x][nt], a0, a1, a2, a3, pw[m][nt][0], pw[m][nt][1]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      const float d_of_lane = found[lane % ROWS];
      // ---- this warp's sums of the run
      if (done > 0) ok = mbar_wait_brief(sum_empty, (done - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float v = l[r] + __shfl_xor_sync(0xffffffffu, l[r], 16);
        if (lane < 16) parts[r * 16 + lane] = v;
        if (lane == r) tops[r] = make_float2(ref[r], d_of_lane);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = nt * 8 + 2 * t + c;
          if (r < ROWS)
#pragma unroll
            for (int d = 0; d < 8; ++d)
              *reinterpret_cast<float2*>(sums + r * 132 + d * 16 + g * 2) = make_float2(o[d][nt][c], o[d][nt][2 + c]);
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(sum_full);
      ++done;
    }
  }
  if (!ok) atomicExch(&dib_attention_fp4_error_word, 1);
  // (A grid that fills the GPU lets the kernel that follows come from here on: earlier, its blocks would take places among this
  // grid's own.)
  if (late) pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (warp == ST_SCORE_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)SH::TMEM));
}

// ---- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess &&
        r == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}
// The cache's codes as rows of D / 2 bytes; boxes of box_rows x 64 bytes (what lies beyond the row reads as zero), swizzled.
bool make_cache_map(CUtensorMap* map, const void* data, long long rows, int D, int box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)D / 2, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)D / 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int ROWS, int D>
int launch_stream(const CUtensorMap& map, const void* q, void* out, SplitArgs a, int box_rows, int max_rows, int runs, int sm_count,
                  cudaStream_t st) {
  using SH = StreamShape<ROWS>;
  auto kern = attention_stream_kernel<ROWS, D>;
  const size_t smem = SH::fixed + (size_t)a.seq_count * 24 + 8;
  constexpr int MOST = 200 * 1024;
  if (smem > MOST) return DIB_BAD_SIZE;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    // (all of an SM's memory as shared memory for both kernels: an SM that is set up otherwise would take fewer CTAs until it is empty)
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
        cudaFuncSetAttribute(attention_split_merge_kernel<__nv_bfloat16, ROWS>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared) != cudaSuccess)
      return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  // the grid is what runs at a time: by shared memory (228 KB an SM, 1 KB of each block's own), registers, tensor memory
  const int by_smem = (int)(228 * 1024 / (smem + 1024));
  int per_sm = by_smem < SH::CTAS ? by_smem : SH::CTAS;
  per_sm = per_sm < 512 / SH::TMEM ? per_sm : 512 / SH::TMEM;
  const long long most = (long long)a.max_items * a.seq_count, grid = (long long)sm_count * (per_sm < 1 ? 1 : per_sm);
  a.sms = most >= grid ? sm_count : 0;
  dib_launch(kern, dim3((unsigned)(grid < most ? grid : most)), dim3(ST_THREADS), smem, st, map, reinterpret_cast<const __nv_bfloat16*>(q),
             reinterpret_cast<__nv_bfloat16*>(out), a, box_rows, most >= grid ? 1 : 0);
  DIB_CHECK_LAUNCH();
  if (runs) {
    const long long blocks = merge_blocks((long long)max_rows * a.Hkv, runs);
    if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
    dib_launch(attention_split_merge_kernel<__nv_bfloat16, ROWS>, dim3((unsigned)blocks, a.seq_count), dim3(SM_WARPS * 32), 0, st,
               reinterpret_cast<__nv_bfloat16*>(out), a);
    DIB_CHECK_LAUNCH();
  }
  return DIB_OK;
}

}  // namespace

extern "C" {

int dib_attention_fp4_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dib_attention_fp4_error_word, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int dib_attention_fp4_status_clear() {
  const int v = 0;
  return cudaMemcpyToSymbol(dib_attention_fp4_error_word, &v, sizeof(int)) == cudaSuccess ? 0 : -1;
}

// As dib_fp4_attention_split (attention_fp4.cu), for bfloat16 queries (dtype 1), heads of 64 or 128 and 4, 8 or 16 rows a tile.
int dib_fp4_attention_stream(const void* q, void* out, const void* data, const void* scales, const void* exponents, long long num_pages,
                             const void* block_table, int max_blocks, const void* cu_q_lens, const void* seq_lens,
                             const void* seq_list, int seq_first, int seq_count, int max_rows, int tile_rows, void* part_o,
                             void* part_ml, int max_items, int runs, int Hq, int Hkv, int D, int page_size, float scale,
                             int window, int dtype, int sm_count, cudaStream_t st) {
  if (dtype != 1) return DIB_BAD_DTYPE;
  if (seq_count < 0 || seq_count > 4096 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || (D != 64 && D != 128) || page_size < 4 ||
      (page_size & (page_size - 1)) != 0 || num_pages * 2 * Hkv * page_size >= (1ll << 31) || max_items < 1 || sm_count < 1 ||
      (tile_rows != 4 && tile_rows != 8 && tile_rows != 16))
    return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(q) |
        reinterpret_cast<uintptr_t>(out)) & 15) != 0 || (reinterpret_cast<uintptr_t>(exponents) & 3) != 0)
    return DIB_BAD_ALIGN;
  if (seq_count == 0 || max_rows == 0) return DIB_OK;
  SplitArgs a = cache_args(data, scales, exponents, num_pages, block_table, max_blocks, cu_q_lens, seq_lens, Hq, Hkv, D, scale, window);
  a.seq_list = reinterpret_cast<const int*>(seq_list);
  a.seq_first = seq_first;
  a.seq_count = seq_count;
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  a.part_o = reinterpret_cast<float*>(part_o);
  a.part_ml = reinterpret_cast<float4*>(part_ml);
  a.max_items = max_items;
  const int box_rows = page_size < SP_TILE ? page_size : SP_TILE;
  CUtensorMap map;
  if (!make_cache_map(&map, data, num_pages * 2 * Hkv * page_size, D, box_rows)) return DIB_LAUNCH_FAILED;
  auto launch = D == 128 ? (tile_rows == 4 ? launch_stream<4, 128> : tile_rows == 8 ? launch_stream<8, 128> : launch_stream<16, 128>)
                         : (tile_rows == 4 ? launch_stream<4, 64> : tile_rows == 8 ? launch_stream<8, 64> : launch_stream<16, 64>);
  return launch(map, q, out, a, box_rows, max_rows, runs, sm_count, st);
}

}  // extern "C"
