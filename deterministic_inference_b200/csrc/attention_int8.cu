// Attention of a step's new tokens over a paged cache in 8-bit integers (cache_int8.cu): query row i of head h, at
// position p, over the keys j of its sequence that it sees (j <= p, and j > p - window with a window):
//   s_j = scale * ks_j * (q . kc_j),   o = sum_j exp(s_j - m) vs_j vc_j / sum_j exp(s_j - m),
// kc, vc the codes of a key and a value, ks, vs their scales.  The scales never touch the codes: a key's joins its score,
// a value's the probability.  A row that sees no key is zeros.  A sequence's new tokens are its last ones.
//
// Forms: split (one new token, a few drafted ones, and every float32 portion: the cache is streamed once), one for every shape
// (heads above 128, pages that are not a power of two), and attention_int8_prompt.cu for bfloat16 portions of prompts.
#include <cuda.h>

#include "common.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
__device__ int dib_attention_int8_error_word = 0;

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_2d(unsigned dst, const CUtensorMap* map, int c0, int c1, unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<unsigned long long>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- split form
// A sequence's rows (new token, query head of the kv group), ROWS at a time, against a run of its keys, by one CTA, in
// tiles of 128 keys.  Both products run on the tensor cores' 8-bit integers (tcgen05.mma kind::i8) and read keys and
// values from shared memory as the copies left them: nothing is converted, whatever the number of rows.
//   S^T = K Q^T:  A = the keys' tile (128 keys x 128 bytes, K-major), B = the query rows as integers against their largest
//     element, each the sum of PARTS bytes of 7 bits (2 for bfloat16 queries, 4 for float32), a column of B a byte.
//     Lane k of the accumulator holds key k's exact integer dot products with all rows.
//   O^T = V^T P^T: A = the values' tile read MN-major (128 dimensions), B = the weights w = p vs, p = 2^(s - L), as
//     integers against the tile's largest one of the row, again PARTS bytes each (MN-major, a thread writes its key's).
//     Lane d holds dimension d's integers for all rows.
// The largest weight of 128 keys becomes an integer between 2^13 and 2^14 (2^27 and 2^28): each is off by 2^-14 (2^-28) of it at
// most, 0.8 % of a tile's sum if all erred alike; errors of either sign in a sum of many that matter are 2^-10 of it.  A query's elements are off by
// 2^-15 of the row's largest, which is more than bfloat16's own step for those below 2^-7 of it.  The
// integers are then scaled and added up in float32.  L, the reference of a row's probabilities, follows the tiles'
// largest weights and is raised only when they have left it by 2^20: float32 holds what lies between.
//
// What bounds it: the bytes of keys and values for up to 4 rows, the threads above.  A thread has a key (then a dimension)
// and ROWS rows: some 20 instructions a key and row, a quarter of what mma.sync on converted codes takes.  Three CTAs an SM
// (two above 8 rows), each with a tile on its way and one in use, cover the trips between copy, tensor core and threads.  An
// item's beginning and end cost as much as a tile or two, through instructions that are not in the cache any more: they are
// kept few.  Heads of 128, 8 kv heads: 64 requests of up to 4,096 keys, 4 rows each, 67.3 us (312 MB at 4.6 TB/s); four of
// 32,000, 8 rows, 58.7 us (270 MB at 4.6 TB/s), of which the last CTA is 7 us behind the median and the merge takes 6; sixteen of up to 1,500
// with 10 rows 26.0 us (31 MB), with 20 rows at 4,096 keys 73 us (tiles of 24 rows; 104 us in tiles of 32); one of 2,048, 8.8 us.
//
// Roles in a CTA: warps 0-3 softmax (TMEM lane = key, dimension), warp 4 copies (TMA, a box a page; scales by cp.async),
// warp 5 issues the scores' products, warp 7 the outputs', warp 6 finds the next work items and makes their query rows.
// Registers are handed out to groups of four warps: the second group gives a part of its own to the first (setmaxnreg).
// Work items: (sequence, kv head, tile of rows,
// run of keys), a CTA takes a contiguous range of them.  The length of a run follows from the sequence's own lengths, so a
// row's bits do not depend on the rest of the step (those of a float32 portion do on its own rows: where its prompt was cut).
constexpr int SP_TILE = 128, SP_THREADS = 256, SP_STAGES = 2, SP_ITEMS = 4;
constexpr int SP_COPY_WARP = 4, SP_SCORE_WARP = 5, SP_OUTPUT_WARP = 7;      // and 6: items and query rows

// Keys of a run: two tiles (one: 72 -> 77 us for 64 decoding requests of up to 4,096 keys, as an item's beginning and end
// cost about a tile, and no gain for one request of 2,048), four for more than 4 rows, whose beginning and end cost more (32
// requests of 4,096 keys and 64 heads: 69 -> 62 us, sixteen of 1,500 with five drafted tokens 32 -> 29; but one of those
// 15.5 -> 17.7), and for long sequences, where the partial results would grow; with many rows a run gets longer still, as
// their partial results do with the rows.
__host__ __device__ __forceinline__ int split_keys(int kv_len, int rows) {
  const int base = kv_len <= 16384 && rows <= 4 ? 256 : 512;
  const int tiles = (rows + 31) / 32;
  return tiles <= 2 ? base : base * tiles;
}

// What a work item takes, in tiles of 128 keys: its own, and one for its beginning and end.  (Of a run longer than the sequence
// those of the sequence, as a run grows with the rows; but not below 512, so that short sequences' items do not share a CTA
// while others have none.)
__device__ __forceinline__ int item_work(int split, int kv_len) {
  return (min(split, max(kv_len, 512)) + SP_TILE - 1) / SP_TILE + 1;
}

__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
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
__device__ __forceinline__ void tc_mma_i8(unsigned elected, unsigned tmem_d, unsigned long long desc_a, unsigned long long desc_b,
                                          unsigned idesc, unsigned accum) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accum), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 8 consecutive columns of this thread's lane; valid after tc_wait_ld()
__device__ __forceinline__ void tc_ld8(unsigned taddr, int (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
// Matrix descriptors: rows of 128 bytes, 128-byte swizzle, 8-row groups 1,024 bytes apart (K-major: a row is a key or a
// query byte column; MN-major: a row is a key, its bytes the dimensions); and MN-major without swizzle: 16 columns x 8 keys
// in 128 bytes, the next 8 keys 128 bytes on, the next 16 columns 2,048.
__device__ __forceinline__ unsigned long long desc_sw128(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((unsigned long long)(1024u >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
__device__ __forceinline__ unsigned long long desc_columns16(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(128u >> 4) << 16) |
         ((unsigned long long)(2048u >> 4) << 32) | (1ull << 46);
}
// kind::i8: 32-bit integer accumulator, signed bytes; A and B MN-major or not
constexpr unsigned idesc_i8(int m, int n, int mn_major) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((unsigned)mn_major << 15) | ((unsigned)mn_major << 16) |
         ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
}
__device__ __forceinline__ float warp_top(float v) {      // the largest of the warp's values, NaN aside
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// An integer y, |y| <= 127 * 128^(PARTS - 1) and rounded here, as the sum of part[i] * 128^(PARTS - 1 - i), a signed byte
// each (in the low byte of a word): adding 1.5 * 2^23 rounds to an integer and leaves it in the low bits.
template <int PARTS> __device__ __forceinline__ void split7(float y, unsigned (&part)[PARTS]) {
  constexpr float MAGIC = 12582912.f;
  float unit = PARTS == 4 ? 2097152.f : 128.f;
#pragma unroll
  for (int i = 0; i < PARTS - 1; ++i) {
    const float z = fmaf(y, 1.f / unit, MAGIC);
    part[i] = __float_as_uint(z);
    y = fmaf(z - MAGIC, -unit, y);
    unit *= 0.0078125f;
  }
  part[PARTS - 1] = __float_as_uint(y + MAGIC);
}
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// the number that PARTS exact sums of part products stand for
template <int PARTS, int STRIDE> __device__ __forceinline__ float join7(const int* acc) {
  const float high = (float)(acc[0] * 128 + acc[STRIDE]);
  return PARTS == 4 ? fmaf(high, 16384.f, (float)(acc[2 * STRIDE] * 128 + acc[3 * STRIDE])) : high;
}

struct SplitArgs {
  const float* scales;          // [pages, 2, Hkv, page_size]
  const int* block_table;       // [B, max_blocks]
  const int* cu_q_lens;
  const int* seq_lens;
  const int* seq_list;          // the sequences of this launch, or null: seq_first ..
  int seq_first, seq_count, max_blocks;
  int Hq, Hkv, D, page_shift, window, box_rows;
  int num_pages;
  float scale;
  float* part_o;                // [seq_count, max_items, ROWS, D]
  float2* part_ml;              // [seq_count, max_items, ROWS]: reference (log 2), sum
  int max_items;
  int late;                     // the grid fills the GPU: the kernel that follows waits for its end
};
// A sequence of the launch and how it is cut.
struct SplitSeq {
  int seq, q_begin, n, kv_len, tiles, split, splits;
};
template <int ROWS> __device__ __forceinline__ SplitSeq split_seq(const SplitArgs& a, int i) {
  SplitSeq s;
  s.seq = a.seq_list != nullptr ? a.seq_list[i] : a.seq_first + i;
  s.q_begin = a.cu_q_lens[s.seq];
  s.n = a.cu_q_lens[s.seq + 1] - s.q_begin;
  s.kv_len = min(a.seq_lens[s.seq], (int)min((long long)a.max_blocks << a.page_shift, 0x7fffffc0ll));
  const int rows = s.n * (a.Hq / a.Hkv);
  s.tiles = (rows + ROWS - 1) / ROWS;
  s.split = split_keys(s.kv_len, rows);
  s.splits = s.n > 0 ? max(1, (s.kv_len + s.split - 1) / s.split) : 0;
  return s;
}

// A work item as it is handed from the warp that walks the CTA's items to the others.
struct __align__(16) SplitItem {
  int seq, q_begin, n, kv_len;      // the sequence: index, first token, new tokens, keys
  int i, kvh, tile, local;          // sequence of the launch, kv head, tile of rows, number of the item in its sequence
  int seen, at, end, splits;        // its keys: [seen, end), those of the run that some row sees; its tiles from `at` on, a multiple
                                    // of 128; runs of the sequence
  int fresh, tiles, lo_all, hi_all;        // other query rows than the item before; tiles of keys, 0: there are no more
                                           // items; the keys that every row sees
};

__device__ __forceinline__ float4 four_floats(const float4& v) { return v; }
__device__ __forceinline__ float4 four_floats(const uint2& v) {      // four bfloat16
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                     __uint_as_float(v.y & 0xffff0000u));
}
template <typename T> struct FourOf { using type = uint2; };
template <> struct FourOf<float> { using type = float4; };

template <typename T, int ROWS> struct SplitShape {
  using Four = typename FourOf<T>::type;
  static constexpr int PARTS = sizeof(T) == 4 ? 4 : 2;
  static constexpr int N = ROWS * PARTS < 16 ? 16 : ROWS * PARTS;      // byte columns of a product's B (16 at least)
  static constexpr int TMEM = N == 16 ? 64 : N == 32 ? 128 : 256;      // S twice, O; a power of two
  static constexpr int STAGE = 2 * SP_TILE * 128;              // keys, values
  static constexpr int SCALES = SP_STAGES * STAGE;             // [stages][2][128] float32
  static constexpr int QUERIES = SCALES + SP_STAGES * 1024;    // [2][N][128], swizzled
  static constexpr int WEIGHTS = QUERIES + 2 * N * 128;        // [N / 16][128 keys][16]
  static constexpr int ROWDATA = WEIGHTS + N * 128;            // [2][3][ROWS]: unit, first and last key seen
  static constexpr int TOPS = ROWDATA + 2 * 3 * ROWS * 4;      // [2][4 warps][ROWS + 4]
  static constexpr int SUMS = TOPS + 2 * 4 * (ROWS + 4) * 4;   // [4 warps][ROWS]
  static constexpr int ITEMS = SUMS + 4 * ROWS * 4;            // [SP_ITEMS]
  static constexpr int BARS = ITEMS + SP_ITEMS * 64;
  static constexpr int FIRST = BARS + 32 * 8;
  static constexpr size_t fixed = FIRST + 16 + 1024;
  // CTAs an SM (what shared memory allows); they are launched with 80 (128) registers a thread, and the groups' shares
  // add up to twice that
  static constexpr int CTAS = N == 16 ? 3 : 2, REGS_MANY = N == 16 ? 112 : 200, REGS_FEW = N == 16 ? 48 : 56;
};

template <int N> __device__ __forceinline__ void regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int ROWS>
__global__ void __launch_bounds__(SP_THREADS, SplitShape<T, ROWS>::CTAS)
attention_split_kernel(const __grid_constant__ CUtensorMap map, const T* __restrict__ q, T* __restrict__ out,
                       const __grid_constant__ SplitArgs a) {
  using SH = SplitShape<T, ROWS>;
  constexpr int PARTS = SH::PARTS, N = SH::N;
  constexpr float MOST = PARTS == 4 ? 127.f * 2097152.f : 127.f * 128.f;      // of the integers
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* scales = reinterpret_cast<float*>(smem + SH::SCALES);
  float* row_data = reinterpret_cast<float*>(smem + SH::ROWDATA);
  float* tops = reinterpret_cast<float*>(smem + SH::TOPS);
  float* sums = reinterpret_cast<float*>(smem + SH::SUMS);
  SplitItem* items = reinterpret_cast<SplitItem*>(smem + SH::ITEMS);
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + SH::BARS);
  unsigned long long* k_full = bars;           // [2] a tile's keys and both kinds of scales have arrived
  unsigned long long* v_full = bars + 2;       // [2] its values have
  unsigned long long* s_full = bars + 4;       // [2] its scores are in tensor memory, its keys have been read
  unsigned long long* s_empty = bars + 6;      // [2] its scores and scales have been read
  unsigned long long* p_full = bars + 8;       // its weights are in shared memory, and O has been read
  unsigned long long* o_full = bars + 9;       // its outputs are in tensor memory, its values and weights have been read
  unsigned long long* v_empty = bars + 10;     // [2] its values have been read
  unsigned long long* q_full = bars + 12;      // [2] an item's query rows are in shared memory
  unsigned long long* q_empty = bars + 14;     // [2] they have been read
  unsigned long long* item_full = bars + 16;   // [SP_ITEMS] an item's record is there
  unsigned long long* item_empty = bars + 16 + SP_ITEMS;      // [SP_ITEMS] it has been read by every role
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 16 + 2 * SP_ITEMS);
  int* softmax_left = reinterpret_cast<int*>(tmem_slot + 1);      // softmax warps that have ended
  int* first = reinterpret_cast<int*>(smem + SH::FIRST);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) prefetch_tensormap(&map);
  if (!a.late) pdl_trigger();
  // ---- the work before each sequence (metadata alone, which no kernel of a step writes); all of it stays below 2^31, which the
  // host sees to
  for (int i = threadIdx.x; i < a.seq_count; i += SP_THREADS) {
    const SplitSeq s = split_seq<ROWS>(a, i);
    first[i + 1] = s.tiles * s.splits * a.Hkv * item_work(s.split, s.kv_len);
  }
  if (threadIdx.x == 0) first[0] = 0;
  if (threadIdx.x == 32) {
    *softmax_left = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 33);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 5);
    }
    mbar_init(p_full, 4);
    mbar_init(o_full, 1);
    for (int i = 0; i < SP_ITEMS; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 7);      // copy, scores, outputs, four softmax warps
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == SP_SCORE_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((unsigned)SH::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  __syncthreads();
  if (warp == 0) {
    int base = 0;
    for (int i0 = 0; i0 < a.seq_count; i0 += 32) {
      int v = i0 + lane < a.seq_count ? first[i0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
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
  const int G = a.Hq / a.Hkv;
  pdl_wait(q);
  bool ok = true;

  if (warp >= 4) {
  regs_give<SH::REGS_FEW>();
  if (warp == SP_COPY_WARP) {
    // ---- copies: lane l has the keys 4l .. 4l + 3 of a tile; the first lane of each page sends for its rows.  Keys are
    // free again once the scores are made, long before the values: keys go a tile ahead of them.
    const int page_mask = (1 << a.page_shift) - 1, half = a.Hkv << a.page_shift;      // rows of a page's keys
    int n = 0, v_sent = 0, v_row = 0;      // tiles whose keys, whose values were sent for; the values' row of the tile before
    unsigned v_senders = 0;
    auto send_values = [&](int m) {        // of tile m
      if (m >= SP_STAGES) ok = mbar_wait_brief(&v_empty[m & 1], ((m >> 1) - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      if (lane == 0) mbar_expect_tx(&v_full[m & 1], __popc(v_senders) * a.box_rows * 128);
      __syncwarp();
      if (v_senders >> lane & 1)
        tma_load_2d(smem_u32(smem) + (m & 1) * SH::STAGE + SP_TILE * 128 + lane * 512, &map, 0, v_row, &v_full[m & 1]);
      v_sent = m + 1;
    };
    for (int k = 0; ok; ++k) {
      const int slot = k % SP_ITEMS;
      ok = mbar_wait_brief(&item_full[slot], (k / SP_ITEMS) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int seq = items[slot].seq, kvh = items[slot].kvh, at = items[slot].at, end = items[slot].end, tiles = items[slot].tiles;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (tiles == 0) break;
      const int* table = a.block_table + (long long)seq * a.max_blocks;
      for (int kb = at; kb < end; kb += SP_TILE, ++n) {
        const int key = kb + lane * 4, off = key & page_mask, stage = n & 1;
        int page = -1;
        if (key < end) page = table[key >> a.page_shift];
        const bool have = page >= 0 && page < a.num_pages;
        const unsigned senders = __ballot_sync(0xffffffffu, have && (lane == 0 || off == 0));
        if (n >= SP_STAGES)       // (the scores made, and the scales read: those of the tile two before this one)
          ok = mbar_wait_brief(&s_full[stage], ((n >> 1) - 1) & 1) && mbar_wait_brief(&s_empty[stage], ((n >> 1) - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&k_full[stage], __popc(senders) * a.box_rows * 128);
        __syncwarp();
        const int row = page * 2 * half + (kvh << a.page_shift) + off;
        if (senders >> lane & 1) tma_load_2d(smem_u32(smem) + stage * SH::STAGE + lane * 512, &map, 0, row, &k_full[stage]);
        // (keys that are not there, and those on a page that is none of the pool's: scales of zero)
        const unsigned sc = smem_u32(scales) + stage * 1024 + lane * 16, bytes = have ? 16 : 0;
        const float* from = a.scales + (have ? row : 0);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(sc), "l"(from), "r"(bytes) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(sc + 512), "l"(from + half), "r"(bytes) : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&k_full[stage])) : "memory");
        if (n > 0) send_values(n - 1);
        v_row = row + half;
        v_senders = senders;
      }
    }
    if (ok && n > 0) send_values(n - 1);
    if (!ok) {      // given up: what was sent for arrives before this memory is another's
      for (int m = max(n - SP_STAGES, 0); m < n; ++m) mbar_wait_brief(&k_full[m & 1], (m >> 1) & 1);
      for (int m = max(v_sent - SP_STAGES, 0); m < v_sent; ++m) mbar_wait_brief(&v_full[m & 1], (m >> 1) & 1);
    }
  } else if (warp == SP_SCORE_WARP) {
    // ---- scores: a tile ahead of the softmax
    {
      const unsigned elected = elect_one();
      constexpr unsigned idesc = idesc_i8(128, N, 0);
      const unsigned base = smem_u32(smem);
      int n = 0, q_used = -1;
      for (int k = 0; ok; ++k) {
        const int slot = k % SP_ITEMS;
        ok = __all_sync(0xffffffffu, mbar_wait_brief(&item_full[slot], (k / SP_ITEMS) & 1));
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
        }
        const unsigned long long qd = desc_sw128(base + SH::QUERIES + (q_used & 1) * N * 128);
        for (int t = tiles; t > 0 && ok; --t, ++n) {
          ok = __all_sync(0xffffffffu, mbar_wait_brief(&k_full[n & 1], (n >> 1) & 1) && (n < 2 || mbar_wait_brief(&s_empty[n & 1], ((n >> 1) - 1) & 1)));
          if (!ok) break;
          tc_fence_after();
          const unsigned long long kd = desc_sw128(base + (n & 1) * SH::STAGE);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) tc_mma_i8(elected, tmem + (n & 1) * N, kd + ks * 2, qd + ks * 2, idesc, ks > 0);
          tc_commit(elected, &s_full[n & 1]);
        }
      }
    }
  } else if (warp == SP_OUTPUT_WARP) {
    // ---- outputs, as soon as a tile's weights are there
    {
      const unsigned elected = elect_one();
      constexpr unsigned idesc = idesc_i8(128, N, 1);
      const unsigned base = smem_u32(smem);
      const unsigned long long weights = desc_columns16(base + SH::WEIGHTS);
      int n = 0;
      for (int k = 0; ok; ++k) {
        const int slot = k % SP_ITEMS;
        ok = __all_sync(0xffffffffu, mbar_wait_brief(&item_full[slot], (k / SP_ITEMS) & 1));
        if (!ok) break;
        const int tiles = items[slot].tiles;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[slot]);
        if (tiles == 0) break;
        for (int t = tiles; t > 0 && ok; --t, ++n) {
          ok = __all_sync(0xffffffffu, mbar_wait_brief(&v_full[n & 1], (n >> 1) & 1) && mbar_wait_brief(p_full, n & 1));
          if (!ok) break;
          tc_fence_after();
          const unsigned long long vd = desc_sw128(base + (n & 1) * SH::STAGE + SP_TILE * 128);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            tc_mma_i8(elected, tmem + 2 * N, vd + ks * (4096 >> 4), weights + ks * (512 >> 4), idesc, ks > 0);
          tc_commit(elected, o_full);
          tc_commit(elected, &v_empty[n & 1]);
        }
      }
    }
  } else {
    // ---- the walk over this CTA's items, a contiguous range of equal work, and the query rows: a lane has 4 of a row's
    // dimensions
    const long long total = first[a.seq_count];
    const int from_work = (int)(total * blockIdx.x / gridDim.x), to_work = (int)(total * (blockIdx.x + 1) / gridDim.x);
    int i = 0, item = 0, old_i = -1, old_kvh = -1, old_tile = -1, made = 0;
    for (int hi = a.seq_count - 1; i < hi;) {      // the sequence in which the range begins
      const int mid = (i + hi + 1) >> 1;
      if (first[mid] <= from_work) i = mid; else hi = mid - 1;
    }
    if (total > 0) {
      const SplitSeq s = split_seq<ROWS>(a, i);
      const int each = item_work(s.split, s.kv_len);
      item = (from_work - first[i] + each - 1) / each;       // the first item that begins in it
    }
    for (int k = 0; ok; ++item) {
      SplitItem it = {};              // (as it is: no more items)
      bool more = false;
      SplitSeq s;
      for (; i < a.seq_count; ++i, item = 0) {
        s = split_seq<ROWS>(a, i);
        if (item < s.tiles * s.splits * a.Hkv) {
          more = first[i] + item * item_work(s.split, s.kv_len) < to_work;
          break;
        }
      }
      if (more) {
        const int local = item;
        const int unit = s.splits > 1 ? local / s.splits : local;
        it.seq = s.seq; it.q_begin = s.q_begin; it.n = s.n; it.kv_len = s.kv_len;
        it.i = i; it.local = local; it.splits = s.splits;
        const int run_at = (local - unit * s.splits) * s.split;
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
            for (int e = lane; e < rows * a.D; e += 32) {
              const int row = it.tile * ROWS + e / a.D, tok = row / G;
              Elem<T>::store(out + ((long long)(s.q_begin + tok) * a.Hq + it.kvh * G + row - tok * G) * a.D + e % a.D, 0.f);
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
      // the query rows' loads, some rows at a time, go out ahead of the copies that the record sets off
      const int row0 = it.tile * ROWS, rows = min(ROWS, it.n * G - row0);
      constexpr int AHEAD = 4;      // (few, and not unrolled further: instructions that a warp runs seldom cost the others theirs)
      typename SH::Four raw[AHEAD];        // 4 elements of a row
      int tok = row0 / G, head = row0 - tok * G;      // of the next row to be loaded
      const T* src = q + ((long long)(it.q_begin + tok) * a.Hq + it.kvh * G + head) * a.D + lane * 4;
      auto load_rows = [&](int from) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          raw[u] = typename SH::Four();
          if (from + u < rows && lane * 4 < a.D) raw[u] = *reinterpret_cast<const typename SH::Four*>(src);
          src += a.D;
          if (++head == G) {
            head = 0;
            src += (long long)(a.Hq - G) * a.D;
          }
        }
      };
      if (it.fresh) load_rows(0);
      const int slot = k % SP_ITEMS;
      if (k >= SP_ITEMS) ok = mbar_wait_brief(&item_empty[slot], ((k / SP_ITEMS) - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        items[slot] = it;
        mbar_arrive(&item_full[slot]);
      }
      ++k;
      if (it.tiles == 0) break;
      if (!it.fresh) continue;
      const int buf = made & 1;
      if (made >= 2) ok = mbar_wait_brief(&q_empty[buf], ((made >> 1) - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      unsigned char* dst = smem + SH::QUERIES + buf * N * 128;
      float* data = row_data + buf * 3 * ROWS;
      unsigned my_bits = 0;      // of the row that is this lane's number
      float my_up = 1.f;
#pragma unroll 1
      for (int from = 0; from < ROWS; from += AHEAD) {
        if (from > 0) load_rows(from);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int r = from + u;
          const float4 x4 = four_floats(raw[u]);
          const float x[4] = {x4.x, x4.y, x4.z, x4.w};
          unsigned bits = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) bits = max(bits, __float_as_uint(x[e]) & 0x7fffffffu);
          bits = __reduce_max_sync(0xffffffffu, bits);
          const float top = fmaxf(__uint_as_float(bits), 0x1p-100f), up = __fdividef(MOST * (1.f - 0x1p-20f), top);
          unsigned part[4][PARTS];
#pragma unroll
          for (int e = 0; e < 4; ++e) split7<PARTS>(x[e] * up, part[e]);
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            const int col = p * ROWS + r;
            *reinterpret_cast<unsigned*>(dst + col * 128 + (((lane >> 2) ^ (col & 7)) << 4) + (lane & 3) * 4) =
                low_bytes(part[0][p], part[1][p], part[2][p], part[3][p]);
          }
          if (lane == r) {
            my_bits = bits;
            my_up = up;
          }
        }
      }
      if (lane < ROWS) {      // lane r: what belongs to row r
        // (a row that holds an infinity or a NaN: its unit is NaN, and so is all that comes of it)
        const int pos = it.kv_len - it.n + (row0 + lane) / G;
        data[lane] = my_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a.scale * LOG2E, my_up);
        data[ROWS + lane] = __int_as_float(first_visible_key(pos, a.window));
        data[2 * ROWS + lane] = __int_as_float(lane < rows ? pos : -1);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the rows are read by the tensor core
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[buf]);
      ++made;
    }
  }
  } else {
    regs_take<SH::REGS_MANY>();
    // ---- softmax: thread = key of the tile, then dimension
    constexpr float UNSET = -1e30f;      // the reference of a row that has seen no key
    constexpr int R8 = ROWS < 8 ? ROWS : 8;
    const int key_of = threadIdx.x;
    const unsigned tm = tmem + ((unsigned)(warp * 32) << 16);
    float L[ROWS], l[ROWS], o[ROWS], f[ROWS];      // f: what the pending tile's integers are multiplied by
    int n = 0, q_used = -1;
    // PARTS x R8 columns from `col` on, as numbers: rows r8 .. of an accumulator
    auto load_rows = [&](unsigned acc_col, int r8, float (&y)[R8]) {
      if (ROWS == 4 && PARTS == 2) {
        int acc[8];
        tc_ld8(tm + acc_col, acc);
        tc_wait_ld();
#pragma unroll
        for (int r = 0; r < R8; ++r) y[r] = join7<2, 4>(&acc[r]);
      } else {
        int acc[PARTS][8];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) tc_ld8(tm + acc_col + p * ROWS + r8, acc[p]);
        tc_wait_ld();
#pragma unroll
        for (int r = 0; r < R8; ++r) y[r] = join7<PARTS, 8>(&acc[0][r]);
      }
    };
    auto add_outputs = [&](int m) {      // tile m's integers
      ok = mbar_wait_brief(o_full, m & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
#pragma unroll
      for (int r8 = 0; r8 < ROWS; r8 += R8) {
        float y[R8];
        load_rows(2 * N, r8, y);
#pragma unroll
        for (int r = 0; r < R8; ++r) o[r8 + r] = fmaf(y[r], f[r8 + r], o[r8 + r]);
      }
    };
    // The rows of the item whose tiles have all been added: finished where the sequence has one run, else partial
    // results for the merge.  (Done under the next item's first tile, whose scores do not wait for it.)
    int d_rows = 0, d_splits = 0, d_local = 0, d_head = 0, d_row0 = 0, d_begin = 0;
    long long d_at = 0;
    auto finish = [&]() {
#pragma unroll
      for (int r8 = 0; r8 < ROWS; r8 += R8) {
        // sums of R8 rows over a warp: exchanges that halve the rows a lane has, then whole sums
        float v[R8];
#pragma unroll
        for (int r = 0; r < R8; ++r) v[r] = l[r8 + r];
        int of = 16;
#pragma unroll
        for (int h = R8 / 2; h > 0; h >>= 1, of >>= 1) {
          const bool up = lane & of;
#pragma unroll
          for (int r = 0; r < h; ++r) {
            const float give = up ? v[r] : v[r + h], keep = up ? v[r + h] : v[r];
            v[r] = keep + __shfl_xor_sync(0xffffffffu, give, of);
          }
        }
#pragma unroll
        for (int x = 16 / R8; x > 0; x >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], x);
        if ((lane & (32 / R8 - 1)) == 0) sums[warp * ROWS + r8 + lane / (32 / R8)] = v[0];
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float sum[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; r += 4) {
        const float4 w0 = *reinterpret_cast<const float4*>(sums + r), w1 = *reinterpret_cast<const float4*>(sums + ROWS + r);
        const float4 w2 = *reinterpret_cast<const float4*>(sums + 2 * ROWS + r), w3 = *reinterpret_cast<const float4*>(sums + 3 * ROWS + r);
        sum[r] = (w0.x + w1.x) + (w2.x + w3.x); sum[r + 1] = (w0.y + w1.y) + (w2.y + w3.y);
        sum[r + 2] = (w0.z + w1.z) + (w2.z + w3.z); sum[r + 3] = (w0.w + w1.w) + (w2.w + w3.w);
      }
      if (d_splits == 1) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          if (r >= d_rows) break;
          const int row = d_row0 + r, tok = row / G;
          if (key_of < a.D)
            Elem<T>::store(out + ((long long)(d_begin + tok) * a.Hq + d_head + row - tok * G) * a.D + key_of,
                           sum[r] == 0.f ? 0.f : o[r] / sum[r]);
        }
      } else if (d_local < a.max_items) {
        float* dst = a.part_o + d_at * a.D + key_of;
        if (key_of < a.D) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r, dst += a.D)
            if (r < d_rows) *dst = o[r];
        }
        if (key_of == 0) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            if (r < d_rows) a.part_ml[d_at + r] = make_float2(L[r], sum[r]);
        }
      }
    };
    for (int k = 0; ok; ++k) {
      const int slot = k % SP_ITEMS;
      ok = mbar_wait_brief(&item_full[slot], (k / SP_ITEMS) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const SplitItem it = items[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (it.tiles == 0) break;
      const int row0 = it.tile * ROWS, rows = min(ROWS, it.n * G - row0);
      if (it.fresh) {
        if (q_used >= 0 && lane == 0) mbar_arrive(&q_empty[q_used & 1]);
        ++q_used;
        ok = mbar_wait_brief(&q_full[q_used & 1], (q_used >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      const float* data = row_data + (q_used & 1) * 3 * ROWS;
      for (int kb = it.at; kb < it.end; kb += SP_TILE, ++n) {
        const int buf = n & 1;
        ok = mbar_wait_brief(&k_full[buf], (n >> 1) & 1) && mbar_wait_brief(&s_full[buf], (n >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        // scores, in units of log 2.  A scale that is no finite number, the key's or the value's, makes the key's scores NaN in
        // the rows that see it, and the value's is zero then: a row that does not see it multiplies it by a probability of zero.
        const float vs_raw = scales[buf * 256 + 128 + key_of], ks_raw = scales[buf * 256 + key_of];
        const float no_number = (ks_raw - ks_raw) + (vs_raw - vs_raw), ks = ks_raw + no_number;
        const int key = kb + key_of;
        const bool plain = kb >= it.lo_all && kb + SP_TILE - 1 <= it.hi_all;        // every row sees every key
        const bool there = key >= it.seen && key < it.end;
        const float vs = there && no_number == 0.f ? vs_raw : 0.f, lv = there ? fmaxf(__log2f(vs), -120.f) : -INFINITY;
        float s[ROWS];
#pragma unroll
        for (int r8 = 0; r8 < ROWS; r8 += R8) {
          float y[R8];
          load_rows(buf * N, r8, y);
#pragma unroll
          for (int r = 0; r < R8; r += 4) {
            const float4 unit = *reinterpret_cast<const float4*>(data + r8 + r);
            s[r8 + r] = y[r] * (ks * unit.x); s[r8 + r + 1] = y[r + 1] * (ks * unit.y);
            s[r8 + r + 2] = y[r + 2] * (ks * unit.z); s[r8 + r + 3] = y[r + 3] * (ks * unit.w);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[buf]);
        if (!plain) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            if (!there || key < __float_as_int(data[ROWS + r]) || key > __float_as_int(data[2 * ROWS + r])) s[r] = -INFINITY;
        }
        // the tile's largest weight of each row, and the largest value scale of the keys that all rows see: what one row sees
        // has no part in another's reference
        float top[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) top[r] = warp_top(s[r] + lv);
        float size = warp_top(key >= it.lo_all && key <= it.hi_all ? lv : -INFINITY);
        float* mine = tops + (buf * 4) * (ROWS + 4);
        if (lane == 0) {
#pragma unroll
          for (int r = 0; r < ROWS; r += 4)
            *reinterpret_cast<float4*>(mine + warp * (ROWS + 4) + r) = make_float4(top[r], top[r + 1], top[r + 2], top[r + 3]);
          mine[warp * (ROWS + 4) + ROWS] = size;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
        for (int w = 0; w < 4; ++w) size = fmaxf(size, mine[w * (ROWS + 4) + ROWS]);
        if (size == -INFINITY) size = 0.f;
#pragma unroll
        for (int r = 0; r < ROWS; r += 4) {
          float4 v = *reinterpret_cast<const float4*>(mine + r);
#pragma unroll
          for (int w = 1; w < 4; ++w) {
            const float4 u = *reinterpret_cast<const float4*>(mine + w * (ROWS + 4) + r);
            v.x = fmaxf(v.x, u.x); v.y = fmaxf(v.y, u.y); v.z = fmaxf(v.z, u.z); v.w = fmaxf(v.w, u.w);
          }
          top[r] = v.x; top[r + 1] = v.y; top[r + 2] = v.z; top[r + 3] = v.w;
        }
        // the tile before this one: its outputs are there as a rule
        if (n > 0) add_outputs(n - 1);
        if (!ok) break;
        if (kb == it.at) {
          if (n > 0) finish();
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            L[r] = UNSET;
            l[r] = o[r] = 0.f;
          }
          d_rows = rows; d_splits = it.splits; d_local = it.local; d_head = it.kvh * G; d_row0 = row0; d_begin = it.q_begin;
          d_at = ((long long)it.i * a.max_items + it.local) * ROWS;
        }
        bool rises = false;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) rises |= top[r] - size > L[r] + 20.f;
        if (rises) {      // (the same in every thread)
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float about = top[r] - size;        // near the largest score: below it by the scales' spread at most
            if (about > L[r] + 20.f) {
              const float factor = fast_exp2(L[r] - about);
              L[r] = about;
              l[r] *= factor;
              o[r] *= factor;
            }
          }
        }
        // weights
        unsigned pw[N / 4];
#pragma unroll
        for (int c = 0; c < N / 4; ++c) pw[c] = 0;
#pragma unroll
        for (int r4 = 0; r4 < ROWS; r4 += 4) {
          unsigned part[4][PARTS];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = r4 + e;
            // a power of two that brings the row's largest weight near the integers' largest, and back: 2^floor(L - top)
            const float x = floorf(fminf(L[r] - top[r], 96.f));
            const int ex = (int)(__float_as_uint(x + 12582912.f) << 23);
            const float up = __int_as_float(ex + (127 << 23));
            f[r] = __int_as_float((127 << 23) - ex) * (1.f / MOST);
            const float p = fast_exp2(s[r] - L[r]);
            l[r] += p;
            split7<PARTS>((p * (up * MOST)) * vs, part[e]);
          }
#pragma unroll
          for (int p = 0; p < PARTS; ++p) pw[(p * ROWS + r4) / 4] = low_bytes(part[0][p], part[1][p], part[2][p], part[3][p]);
        }
#pragma unroll
        for (int c = 0; c < N / 16; ++c)
          *reinterpret_cast<uint4*>(smem + SH::WEIGHTS + c * 2048 + key_of * 16) =
              make_uint4(pw[c * 4], pw[c * 4 + 1], pw[c * 4 + 2], pw[c * 4 + 3]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
    }
    if (ok && n > 0) {
      add_outputs(n - 1);
      if (ok) finish();
    }
    // A warp that has given up arrives at the four warps' barrier, which has no limit of its own, until the others have left it:
    // they come to the end of their item, or to a wait for what this warp no longer does.
    if (lane == 0) atomicAdd(softmax_left, 1);
    if (!ok) {
      for (int i = 0; i < 4096; ++i) {
        const int left = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile int*>(softmax_left), 0);
        if (left == 4) break;
        asm volatile("bar.arrive 1, 128;" ::: "memory");
        __nanosleep(1000000);
      }
    }
  }
  if (!ok) atomicExch(&dib_attention_int8_error_word, 1);
  // A grid that fills the GPU lets the kernel that follows come from here on, not earlier: a block of it that lies between
  // two of this grid's CTAs, or of the next step's, leaves an SM's shared memory in pieces that hold two CTAs instead of
  // three, and the CTAs that find no place start when others end (four contexts of 32,000 keys: 75 us instead of 64; but
  // one of 2,048, which does not fill it, 9.9 us instead of 9.0).
  if (a.late) pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (warp == SP_SCORE_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)SH::TMEM));
}

// The runs' results of a row: out = sum_r 2^(L_r - top) O_r / sum_r 2^(L_r - top) l_r.  A block a row: warp w takes the
// runs w, w + 4, ... in their order, a lane 4 dimensions; the four warps' sums are added in the order of the warps.
constexpr int SM_WARPS = 4;
template <typename T, int ROWS>
__global__ void __launch_bounds__(SM_WARPS * 32)
attention_split_merge_kernel(T* __restrict__ out, const __grid_constant__ SplitArgs a) {
  const float* part_o = a.part_o;
  const float2* part_ml = a.part_ml;
  __shared__ float4 s_o[SM_WARPS][32];
  __shared__ float s_top[SM_WARPS], s_sum[SM_WARPS];
  if (!a.late) pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.y, G = a.Hq / a.Hkv;
  const SplitSeq s = split_seq<ROWS>(a, i);
  const int n_rows = s.n * G, id = blockIdx.x;     // rows of a kv head
  // (every block waits, the one without work too: a grid none of whose blocks has waited ends ahead of the attention, and the
  // kernel that follows takes this one's end for the attention's)
  if (s.splits <= 1 || id >= n_rows * a.Hkv || s.splits * s.tiles * a.Hkv > a.max_items) {
    pdl_wait();
    return;
  }
  const int kvh = id / n_rows, row = id - kvh * n_rows, tile = row / ROWS, r = row % ROWS;
  const int p0 = s.kv_len - s.n;
  const int tok0 = tile * ROWS / G, tok1 = min((tile + 1) * ROWS - 1, n_rows - 1) / G;
  // the runs that hold keys which some row of the tile sees
  const int k_lo = first_visible_key(p0 + tok0, a.window), k_hi = p0 + tok1;
  const int s0 = k_lo / s.split, s1 = k_hi < k_lo ? s0 - 1 : min(k_hi / s.split, s.splits - 1);
  const long long base = ((long long)i * a.max_items + (long long)(kvh * s.tiles + tile) * s.splits) * ROWS + r;
  const bool in = lane * 4 < a.D;
  pdl_wait(part_o, part_ml);
  float top = -INFINITY;
  for (int run = s0 + (int)threadIdx.x; run <= s1; run += SM_WARPS * 32) top = fmaxf(top, part_ml[base + (long long)run * ROWS].x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  constexpr int AHEAD = 8;
  // the first results are on their way while the references are compared
  float4 v[AHEAD];
  float2 ml[AHEAD];
  auto load = [&](int from) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int run = from + u * SM_WARPS;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      ml[u] = make_float2(-INFINITY, 0.f);
      if (run <= s1) {
        const long long at = base + (long long)run * ROWS;
        ml[u] = part_ml[at];
        if (in) v[u] = *reinterpret_cast<const float4*>(part_o + at * a.D + lane * 4);
      }
    }
  };
  load(s0 + warp);
  top = warp_max(top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  const float ref = top == -INFINITY ? 0.f : top;
  for (int from = s0 + warp; from <= s1; from += AHEAD * SM_WARPS) {
    if (from != s0 + warp) load(from);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const float w = fast_exp2(ml[u].x - ref);
      sum = fmaf(w, ml[u].y, sum);
      o.x = fmaf(w, v[u].x, o.x); o.y = fmaf(w, v[u].y, o.y);
      o.z = fmaf(w, v[u].z, o.z); o.w = fmaf(w, v[u].w, o.w);
    }
  }
  s_o[warp][lane] = o;
  if (lane == 0) s_sum[warp] = sum;
  if (a.late) pdl_trigger();       // (as in the split kernel)
  __syncthreads();
  if (warp != 0 || !in) return;
  float4 y = s_o[0][lane];
  sum = s_sum[0];
#pragma unroll
  for (int k = 1; k < SM_WARPS; ++k) {
    const float4 z = s_o[k][lane];
    y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
    sum += s_sum[k];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int tok = row / G;
  T* dst = out + ((long long)(s.q_begin + tok) * a.Hq + kvh * G + row - tok * G) * a.D + lane * 4;
  Elem<T>::store(dst, y.x * inv);
  Elem<T>::store(dst + 1, y.y * inv);
  Elem<T>::store(dst + 2, y.z * inv);
  Elem<T>::store(dst + 3, y.w * inv);
}

// ---------------------------------------------------------------- the form for every shape
// Head sizes up to 256, any page size and group ratio: a warp takes a (token, head), a lane a key of 32 at a time for
// the scores, then a lane D / 32 dimensions for the values.  Bound by a warp's chain over the keys: 2,048 keys of heads of 256
// 1.3 ms, for one request as for sixteen.
constexpr int ANY_WARPS = 4;

template <typename T>
__global__ void __launch_bounds__(ANY_WARPS * 32)
attention_any_kernel(const T* __restrict__ q, T* __restrict__ out, const signed char* __restrict__ data,
                     const float* __restrict__ scales, const int* __restrict__ block_table, int max_blocks,
                     const int* __restrict__ token_seq, const int* __restrict__ cu_q_lens,
                     const int* __restrict__ seq_lens, int T_, int Hq, int Hkv, int D, int page_size, long long num_pages,
                     float scale, int window) {
  pdl_prologue(q, data, scales);
  __shared__ float sq[ANY_WARPS][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * ANY_WARPS + warp;
  const bool in = item < (long long)T_ * Hq;
  const int token = in ? (int)(item / Hq) : 0, h = in ? (int)(item % Hq) : 0, kvh = h / (Hq / Hkv);
  if (in)
    for (int d = lane; d < D; d += 32) sq[warp][d] = Elem<T>::load(q + item * D + d) * scale * LOG2E;
  __syncwarp();
  if (!in) return;
  const int seq = token_seq[token];
  const int pos = seq_lens[seq] - (cu_q_lens[seq + 1] - token);      // a sequence's new tokens are its last ones
  const int lo = first_visible_key(pos, window), hi = (int)min((long long)pos, (long long)max_blocks * page_size - 1);
  const int* bt = block_table + (long long)seq * max_blocks;
  float m = -INFINITY, l = 0.f, o[8] = {};
  for (int k0 = lo; k0 <= hi; k0 += 32) {
    const int key = k0 + lane;
    const bool seen = key <= hi;
    const long long page = seen ? bt[key / page_size] : -1;
    const bool have = page >= 0 && page < num_pages;      // (a page that is none of the pool's: keys and values of zeros)
    const long long krow = ((page * 2) * Hkv + kvh) * page_size + key % page_size;
    const long long vrow = have ? krow + (long long)Hkv * page_size : -1;
    float s = seen ? 0.f : -INFINITY;
    if (have) {
      float dot = 0.f;
      const uint4* p = reinterpret_cast<const uint4*>(data + krow * D);
      for (int c = 0; c < D / 16; ++c) {
        const uint4 v = p[c];
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) dot = fmaf((float)(signed char)(w[i >> 2] >> (8 * (i & 3))), sq[warp][c * 16 + i], dot);
      }
      s = dot * scales[krow];
    }
    const float top = fmaxf(m, warp_max(s));
    const float p = seen ? exp2f(s - (top == -INFINITY ? 0.f : top)) : 0.f;
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - top);
    const float vs = have ? scales[vrow] : 0.f;
    l = l * alpha + warp_sum(p);
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= alpha;
    const int n = min(32, hi - k0 + 1);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j) * __shfl_sync(0xffffffffu, vs, j);
      const long long row = __shfl_sync(0xffffffffu, vrow, j);
      if (row < 0) continue;
      const signed char* vp = data + row * D;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i * 32 + lane < D) o[i] = fmaf(pj, (float)vp[i * 32 + lane], o[i]);
    }
  }
  const bool none = hi < lo;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < D) Elem<T>::store(out + item * D + i * 32 + lane, none ? 0.f : o[i] / l);
}

// ---------------------------------------------------------------- host side
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
// The cache as rows of D bytes; boxes of box_rows x 128 bytes (what lies beyond D reads as zero), swizzled.
bool make_cache_map(CUtensorMap* map, const void* data, long long rows, int D, int box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)D};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(data), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int ROWS>
int launch_split(const CUtensorMap& map, const void* q, void* out, SplitArgs a, int max_rows, int merge, int sm_count,
                 cudaStream_t st) {
  using SH = SplitShape<T, ROWS>;
  auto kern = attention_split_kernel<T, ROWS>;
  const size_t smem = SH::fixed + ((size_t)a.seq_count + 1) * 4;
  if (smem > 200 * 1024) return DIB_BAD_SIZE;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    // (All of an SM's memory as shared memory for both kernels: an SM that is set up otherwise, by the merge of the layer
    // before, would take two CTAs until it is empty, and a CTA that starts late ends late.)
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
        cudaFuncSetAttribute(attention_split_merge_kernel<T, ROWS>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared) != cudaSuccess)
      return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  // the grid is what runs at a time: by shared memory (228 KB an SM, 1 KB of each block's own), registers, tensor memory
  const int by_smem = (int)(228 * 1024 / (smem + 1024)), by_regs = SH::CTAS, by_tmem = 512 / SH::TMEM;
  int per_sm = by_smem < by_regs ? by_smem : by_regs;
  per_sm = per_sm < by_tmem ? per_sm : by_tmem;
  const long long most = (long long)a.max_items * a.seq_count, grid = (long long)sm_count * (per_sm < 1 ? 1 : per_sm);
  a.late = most >= grid;
  dib_launch(kern, dim3((unsigned)(grid < most ? grid : most)), dim3(SP_THREADS), smem, st, map, reinterpret_cast<const T*>(q),
             reinterpret_cast<T*>(out), a);
  DIB_CHECK_LAUNCH();
  if (merge) {
    const long long blocks = (long long)max_rows * a.Hkv;
    if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
    dib_launch(attention_split_merge_kernel<T, ROWS>, dim3((unsigned)blocks, a.seq_count), dim3(SM_WARPS * 32), 0, st,
               reinterpret_cast<T*>(out), a);
    DIB_CHECK_LAUNCH();
  }
  return DIB_OK;
}

}  // namespace

extern "C" {

int dib_attention_int8_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dib_attention_int8_error_word, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int dib_attention_int8_status_clear() {
  const int v = 0;
  return cudaMemcpyToSymbol(dib_attention_int8_error_word, &v, sizeof(int)) == cudaSuccess ? 0 : -1;
}

// Keys of a run of the split form, for a sequence of kv_len keys and `rows` rows (new tokens x query heads of a kv head).
int dib_int8_attention_split_keys(int kv_len, int rows) { return split_keys(kv_len, rows); }

// The split form, for the sequences seq_list[0 .. seq_count) or (null) seq_first ...: heads up to 128, pages of a
// power of two of rows, 4 at least.  max_rows: the most rows (new tokens x query heads of a kv head) of one of them; tile_rows: 8,
// 16 or (bfloat16) 4, 24 or 32 rows a tile; max_items: the most (tiles x runs x kv heads) of one; part_o float32 [seq_count, max_items,
// tile_rows, D] and part_ml [.., 2] take partial results where merge is not 0 (some sequence may have two runs).  The work
// of all of them, (tiles of rows) x (kv heads) x (runs) x (tiles of keys of a run, and one), is below 2^31.
int dib_int8_attention_split(const void* q, void* out, const void* data, const void* scales, long long num_pages,
                             const void* block_table, int max_blocks, const void* cu_q_lens, const void* seq_lens,
                             const void* seq_list, int seq_first, int seq_count, int max_rows, int tile_rows, void* part_o,
                             void* part_ml, int max_items, int merge, int Hq, int Hkv, int D, int page_size, float scale,
                             int window, int dtype, int sm_count, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  const bool pages_fit = page_size >= 4 && (page_size & (page_size - 1)) == 0;
  if (seq_count < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || D < 16 || D > 128 || D % 16 != 0 || page_size < 1 || !pages_fit ||
      num_pages * 2 * Hkv * page_size >= (1ll << 31) || seq_count > 65535 || max_items < 1 || sm_count < 1 ||
      (tile_rows != 8 && tile_rows != 16 && ((tile_rows != 4 && tile_rows != 24 && tile_rows != 32) || dtype != 1)))
    return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(q) |
        reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (seq_count == 0 || max_rows == 0) return DIB_OK;
  SplitArgs a;
  a.scales = reinterpret_cast<const float*>(scales);
  a.block_table = reinterpret_cast<const int*>(block_table);
  a.cu_q_lens = reinterpret_cast<const int*>(cu_q_lens);
  a.seq_lens = reinterpret_cast<const int*>(seq_lens);
  a.seq_list = reinterpret_cast<const int*>(seq_list);
  a.seq_first = seq_first;
  a.seq_count = seq_count;
  a.max_blocks = max_blocks;
  a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.window = window;
  a.page_shift = 0;
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  a.box_rows = page_size < SP_TILE ? page_size : SP_TILE;
  a.scale = scale;
  a.part_o = reinterpret_cast<float*>(part_o);
  a.part_ml = reinterpret_cast<float2*>(part_ml);
  a.max_items = max_items;
  a.num_pages = (int)num_pages;
  CUtensorMap map;
  if (!make_cache_map(&map, data, num_pages * 2 * Hkv * page_size, D, a.box_rows)) return DIB_LAUNCH_FAILED;
  using B = __nv_bfloat16;
  if (dtype == 1) {
    if (tile_rows == 4) return launch_split<B, 4>(map, q, out, a, max_rows, merge, sm_count, st);
    if (tile_rows == 8) return launch_split<B, 8>(map, q, out, a, max_rows, merge, sm_count, st);
    if (tile_rows == 16) return launch_split<B, 16>(map, q, out, a, max_rows, merge, sm_count, st);
    if (tile_rows == 24) return launch_split<B, 24>(map, q, out, a, max_rows, merge, sm_count, st);
    return launch_split<B, 32>(map, q, out, a, max_rows, merge, sm_count, st);
  }
  if (tile_rows == 8) return launch_split<float, 8>(map, q, out, a, max_rows, merge, sm_count, st);
  return launch_split<float, 16>(map, q, out, a, max_rows, merge, sm_count, st);
}

int dib_int8_attention_any(const void* q, void* out, const void* data, const void* scales, const void* block_table,
                           int max_blocks, const void* token_seq, const void* cu_q_lens, const void* seq_lens, int T,
                           int Hq, int Hkv, int D, int page_size, long long num_pages, float scale, int window, int dtype,
                           cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (T < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || D < 16 || D > 256 || D % 16 != 0 || page_size < 1) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(data) & 15) != 0) return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const long long blocks = ((long long)T * Hq + ANY_WARPS - 1) / ANY_WARPS;
  if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
  const signed char* d = reinterpret_cast<const signed char*>(data);
  const float* s = reinterpret_cast<const float*>(scales);
  const int *bt = reinterpret_cast<const int*>(block_table), *ts = reinterpret_cast<const int*>(token_seq),
            *cu = reinterpret_cast<const int*>(cu_q_lens),
            *sl = reinterpret_cast<const int*>(seq_lens);
  if (dtype == 1)
    dib_launch(attention_any_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(ANY_WARPS * 32), 0, st,
               reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<__nv_bfloat16*>(out), d, s, bt, max_blocks, ts,
               cu, sl, T, Hq, Hkv, D, page_size, num_pages, scale, window);
  else
    dib_launch(attention_any_kernel<float>, dim3((unsigned)blocks), dim3(ANY_WARPS * 32), 0, st,
               reinterpret_cast<const float*>(q), reinterpret_cast<float*>(out), d, s, bt, max_blocks, ts, cu, sl, T, Hq,
               Hkv, D, page_size, num_pages, scale, window);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

}  // extern "C"
