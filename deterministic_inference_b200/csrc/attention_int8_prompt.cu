// Attention of a prompt's portion over a paged cache in 8-bit integers (cache_int8.cu; formulas in attention_int8.cu), for
// bfloat16 queries, whatever a portion's rows (and drafted tokens of many): S = Q K^T and O = P V by tcgen05.mma kind::f16, accumulators in tensor memory, a thread a
// query row for the softmax.
//
// Numbers.  Keys enter the first product as their codes, which float16 holds exactly, queries in float16 times a power of
// two of their row (exact: bfloat16 has fewer bits); a key's scale (times the softmax's) joins its column of the scores in
// float32.  Values enter the second product as code times scale in float16 (11 bits, two roundings of 2^-12), in units of a
// power of two, the probabilities in float16; their sum is taken in float32 before that.  Against 64 bits the output is off by
// its own rounding to bfloat16, 0.0017 of its norm (with bfloat16 probabilities it was 0.0024, with bfloat16 values too
// 0.0028).  The unit stays while a tile's scales lie within 2^-13 .. 2^8 of it and is the tile's own otherwise; the outputs so far
// are then multiplied by a power of two, so that no bit depends on it.  A tile whose own scales lie more than 2^17 apart is
// "wide": codes in bfloat16, exactly, and the scales joined to probabilities in bfloat16, whose range is float32's.
//
// Six warps turn a key tile's bytes (fetched by TMA, a box a page) into swizzled 16-bit tiles, once for the 256 rows of the
// two query tiles that share them.
//
// Two query tiles A and B of 128 rows (tokens x heads of a kv group) of one sequence a CTA.  Roles: warps 0-3 softmax of A,
// 4-7 of B (a row's 128 scores in registers; probabilities go back to tensor memory over the scores, half a tile at a time, and
// are the second product's operand from there), warp 9 issues the products (in code that all its lanes run, which keeps
// descriptors in uniform registers: 641 -> 566 us at 3,000 tokens on 4,096), warp 8 sends for bytes and scales, warps 10-15 convert.
// The products of the two tiles are staggered, each tile's softmax runs under the other's products.  Once a tile has had
// its last key tile (or there is no B) the other runs alone and takes its score columns as a second buffer.
// Tensor memory: S/P of A columns 0.., of B 128.., O of A 256.., of B 384...
//
// Keys are cut at multiples of 4,096 (chunks of constant size from key 0); a query tile that reaches over a cut has a CTA a
// chunk, and a second kernel adds the partial results in chunk order.  Key tiles are anchored at key 0, cuts depend on
// positions alone and units are powers of two, so a row's bits do not depend on the step (but for a tile of which it does not
// see all keys and some that it does not see make the tile wide).
//
// What bounds it: 2.5 us a key tile for both query tiles, of which the products need 1.1.  A query tile's chain is its
// scores' way out of tensor memory, scales, maximum, exponentials, packing (some 700 instructions a warp) and the next
// products; the schedulers are shared with the conversion, and with the instruction cache: what a warp runs seldom is kept
// short or out of the way.  A CTA's beginning and end cost 9 us more.  One CTA an SM (213 KB).  Two threads a row were
// slower (635 -> 852 us: registers spilled), as were exponentials shared with the FMA pipe (506 -> 518).
// 2,048 tokens, 32 / 8 heads of 128: 56.4 us, 610 TFLOP/s.  3,000 tokens on 5,000 keys beside 24 decodes: 471 us.
#include <cuda.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace {

constexpr int TILE = 128, SOFTMAX_WARPS = 8, COPY_WARP = 8, MMA_WARP = 9, CONVERTERS = 6;
constexpr int THREADS = 512;
constexpr int REGS_FEW = 64, REGS_MANY = 192;         // 256 * 64 + 256 * 192 = 512 * 128
constexpr int TILE_BYTES = 128 * 128 * 2, HALF_BYTES = 128 * 64 * 2;      // a bfloat16 tile: two halves of 64 columns
constexpr int RAW_BYTES = 128 * 128;
constexpr float NEG_BIG = -1e30f;
constexpr float LOG2E = 1.4426950408889634f;

// shared memory: queries of A and B (later their outputs); a ring of 16-bit tiles and one of bytes, keys and values in turn;
// scales; the query rows' units
constexpr int RING = 3, SLOTS = 4;
constexpr int S_KV = 2 * TILE_BYTES, S_RAW = S_KV + RING * TILE_BYTES, S_SCALES = S_RAW + RING * RAW_BYTES;
constexpr int S_INFO = S_SCALES + SLOTS * 1024, S_ROWS = S_INFO + SLOTS * 32;
constexpr int S_BARS = S_ROWS + 2 * TILE * 4, S_TOTAL = S_BARS + 32 * 8;
constexpr int S_DYNAMIC = S_TOTAL + 1024;

__device__ int dib_attention_int8_prompt_error_word = 0;

template <int N> __device__ __forceinline__ void regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
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
// 8 bytes that a whole warp reads: two wavefronts, where 16 bytes are more than four (3,000 tokens on 4,096: 510 us, 534)
__device__ __forceinline__ float2 load_shared2(unsigned addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float two_to(int n) { return __int_as_float((n + 127) << 23); }      // -126 <= n <= 127
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
__device__ __forceinline__ void tc_mma(unsigned elected, unsigned tmem_d, unsigned long long desc_a, unsigned long long desc_b,
                                       unsigned idesc, unsigned accum) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accum), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(unsigned elected, unsigned tmem_d, unsigned tmem_a, unsigned long long desc_b,
                                          unsigned idesc, unsigned accum) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accum), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_ld32(unsigned taddr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tc_st32(unsigned taddr, const unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31, %32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tc_ld8(unsigned taddr, unsigned (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tc_st8(unsigned taddr, const unsigned (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Descriptors (rows of 128 bytes, 128-byte swizzle, 8-row groups 1,024 bytes apart): K-major; MN-major, the next 64 columns
// half a tile on.
__device__ __forceinline__ unsigned long long desc_k_major(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ unsigned long long desc_mn_major(unsigned addr) {
  return desc_k_major(addr) | ((unsigned long long)(HALF_BYTES >> 4) << 16);
}
// kind::f16: float32 accumulator, A and B both float16 or both bfloat16
constexpr unsigned idesc_f16(int m, int n, bool bf16, int b_mn_major) {
  return (1u << 4) | ((unsigned)bf16 << 7) | ((unsigned)bf16 << 10) | ((unsigned)b_mn_major << 16) | ((unsigned)(n >> 3) << 17) |
         ((unsigned)(m >> 4) << 24);
}
// byte offset of (row, 16-byte piece c of the row's 128 elements) in a tile of 16-bit numbers
__device__ __forceinline__ int piece_off(int row, int c) {
  return (c >> 3) * HALF_BYTES + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}
// Two codes of a word as float16, exactly: a byte with its sign turned, under the exponent byte 0x64, is 1024 + 128 + code.
__device__ __forceinline__ unsigned codes_f16(unsigned turned, unsigned sel) {
  const unsigned a = __byte_perm(turned, 0x64646464u, sel);
  const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&a), __half2half2(__ushort_as_half(0x6480)));      // 1152
  return *reinterpret_cast<const unsigned*>(&c);
}
// Two codes of a word as bfloat16, exactly: low 7 bits and sign bit of a byte under the exponent byte 0x43 are 128 + low and
// 128 + 128 sign, and a code is the first minus the second.
__device__ __forceinline__ unsigned codes_bf16(unsigned word, unsigned sel) {
  const unsigned a = __byte_perm(word & 0x7f7f7f7fu, 0x43434343u, sel), b = __byte_perm(word & 0x80808080u, 0x43434343u, sel);
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const unsigned*>(&d);
}
__device__ __forceinline__ unsigned times_f16(unsigned codes, __half2 scale) {
  const __half2 y = __hmul2_rn(*reinterpret_cast<const __half2*>(&codes), scale);
  return *reinterpret_cast<const unsigned*>(&y);
}

// What the keys of a tile have in common.  value_exp: the values' scales are in units of 2^value_exp, the outputs too.
// wide: they are too far apart for float16.  nan: the keys that are no numbers, bit l of word j key 4 l + j.
struct TileInfo {
  unsigned nan[4], any_nan;
  int wide, value_exp, pad;
};

struct PromptArgs {
  const float* scales;          // [pages, 2, Hkv, page_size]
  const int* block_table;       // [B, max_blocks]
  const int* cu_q_lens;
  const int* seq_lens;
  const int* units;             // [5][unit_stride], of which `count`: sequence, first token of A, of B (or -1), chunk, place of
                                // A's first token in the partial results
  int count, unit_stride, max_blocks, Hq, Hkv, D, page_shift, num_pages, window, chunk_tiles, max_chunks;
  float scale;
  float* part_o;                // [places, Hq, max_chunks, 128]
  float2* part_ml;              // [places, Hq, max_chunks]: reference (log 2), sum
};

__global__ void __launch_bounds__(THREADS, 1)
attention_prompt_kernel(const __grid_constant__ CUtensorMap map, const __nv_bfloat16* __restrict__ q,
                        __nv_bfloat16* __restrict__ out, const __grid_constant__ PromptArgs a) {
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
  unsigned char* sQ = smem;
  unsigned char* sKV = smem + S_KV;
  unsigned char* raw = smem + S_RAW;
  float* scales = reinterpret_cast<float*>(smem + S_SCALES);          // [SLOTS][keys', values' of 128]
  float* row_units = reinterpret_cast<float*>(smem + S_ROWS);         // [2][TILE]; NaN: the row holds an infinity or a NaN
  TileInfo* infos = reinterpret_cast<TileInfo*>(smem + S_INFO);       // [SLOTS]
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + S_BARS);
  unsigned long long* raw_full = bars;            // [RING] a tile's bytes have arrived
  unsigned long long* raw_empty = bars + 3;       // [RING] they have been converted (a warp each)
  unsigned long long* full = bars + 6;            // [RING] a tile is there in 16 bits (a warp each)
  unsigned long long* empty = bars + 9;           // [RING] both products have read it
  unsigned long long* sc_full = bars + 12;        // [SLOTS] the scales of a key tile are there
  unsigned long long* sc_empty = bars + 16;       // [SLOTS] its outputs have been made
  unsigned long long* s_full = bars + 20;         // [A, B] the query tile's scores are in tensor memory
  unsigned long long* p_full = bars + 22;         // [2][2] half of its probabilities are, and O is rescaled (a warp each)
  unsigned long long* o_final = bars + 26;        // [2] its last product has completed
  unsigned long long* pv_done = bars + 28;        // an output product of the tile that runs alone has completed
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 30);
  if (threadIdx.x == 0) prefetch_tensormap(&map);
  pdl_trigger();
  if (smem - smem_dyn + S_TOTAL > S_DYNAMIC) {      // (the memory is aligned to 1,024 as a rule)
    if (threadIdx.x == 0) atomicExch(&dib_attention_int8_prompt_error_word, 2);
    pdl_wait();
    return;
  }
  const int unit = a.count - 1 - blockIdx.y, kvh = blockIdx.x;        // the longest first
  const int G = a.Hq / a.Hkv, npt = TILE / G;                         // tokens of a query tile
  const unsigned g_up = 65536u / G + 1;      // r / G for r < 128, exactly: 128 G < 65536
  auto token_of = [&](int r) { return (int)(r * g_up >> 16); };
  const int seq = a.units[unit];
  const int tokx[2] = {a.units[a.unit_stride + unit], a.units[2 * a.unit_stride + unit]};
  const int chunk = a.chunk_tiles > 0 ? a.units[3 * a.unit_stride + unit] : 0;
  const int q_begin = a.cu_q_lens[seq], q_len = a.cu_q_lens[seq + 1] - q_begin;
  const int kv_len = min(a.seq_lens[seq], (int)min((long long)a.max_blocks << a.page_shift, 0x7fffff00ll));
  const int prefix = kv_len - q_len;
  const int* bt = a.block_table + (long long)seq * a.max_blocks;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  // Per query tile: its tokens and the key tiles of this chunk that it needs.
  int ntok[2], jf[2], jl[2];
  bool whole[2];
  const int c_lo = chunk * a.chunk_tiles, c_hi = a.chunk_tiles > 0 ? c_lo + a.chunk_tiles - 1 : 0x7fffffff;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int t0 = tokx[x];
    ntok[x] = t0 >= 0 ? max(0, min(npt, q_len - t0)) : 0;
    const int last_pos = prefix + t0 + ntok[x] - 1;
    const int f = first_visible_key(prefix + t0, a.window) / TILE;
    const int l = ntok[x] > 0 && last_pos >= 0 ? last_pos / TILE : -1;      // an empty tile is never active
    whole[x] = a.chunk_tiles <= 0 || f / a.chunk_tiles == l / a.chunk_tiles;
    jf[x] = max(f, c_lo);
    jl[x] = min(l, c_hi);
    if (l < 0 && ntok[x] > 0 && chunk == 0) {      // its rows lie before the first key: zeros
      pdl_wait();
      for (int e = threadIdx.x; e < ntok[x] * G * a.D; e += THREADS) {
        const int row = e / a.D;
        out[((long long)(q_begin + t0 + row / G) * a.Hq + kvh * G + row % G) * a.D + e % a.D] = __float2bfloat16_rn(0.f);
      }
    }
  }
  const bool any0 = jl[0] >= jf[0], any1 = jl[1] >= jf[1];
  if (!any0 && !any1) {           // nothing of this chunk concerns the pair
    pdl_wait();                   // (a grid none of whose blocks has waited would end ahead of the kernel in front)
    return;
  }
  const int j0 = any0 && any1 ? min(jf[0], jf[1]) : (any0 ? jf[0] : jf[1]);
  const int ntiles = max(any0 ? jl[0] : -1, any1 ? jl[1] : -1) - j0 + 1;
  // (arrays indexed by a running x would live in local memory)
  auto active = [&](int x, int i) { return j0 + i >= (x ? jf[1] : jf[0]) && j0 + i <= (x ? jl[1] : jl[0]); };
  // From key tile solo_from on query tile solo_x is alone; the other one has had n_other key tiles.
  const int solo_x = (any1 && (!any0 || jl[1] >= jl[0])) ? 1 : 0;
  const int n_other = (solo_x ? any0 : any1) ? jl[1 - solo_x] - jf[1 - solo_x] + 1 : 0;
  const int solo_from = max((solo_x ? any0 : any1) ? jl[1 - solo_x] - j0 + 1 : 0, jf[solo_x] - j0);

  bool ok = true;
  // ---- bytes of key tile i: lane l has the keys 4l .. 4l + 3, the first lane of each page sends.  Item 2i is the keys,
  // 2i + 1 the values.
  const int page_mask = (1 << a.page_shift) - 1, half_rows = a.Hkv << a.page_shift, box_rows = min(1 << a.page_shift, TILE);
  auto row_of = [&](int i) {      // this lane's row of the cache for its keys of key tile i, or -1
    const int key = (j0 + i) * TILE + lane * 4;
    if (i >= ntiles || key >= kv_len) return -1;
    const int page = bt[key >> a.page_shift];
    return page >= 0 && page < a.num_pages ? page * 2 * half_rows + (kvh << a.page_shift) + (key & page_mask) : -1;
  };
  auto send = [&](int item, int row) {
    const bool sends = row >= 0 && (lane == 0 || (lane * 4 & page_mask) == 0);
    const unsigned senders = __ballot_sync(0xffffffffu, sends);
    const int at = item % RING;
    if (lane == 0) mbar_expect_tx(&raw_full[at], __popc(senders) * box_rows * 128);
    __syncwarp();
    if (sends)
      tma_load_2d(smem_u32(raw) + at * RAW_BYTES + lane * 512, &map, 0, row + (item & 1) * half_rows, &raw_full[at]);
  };
  int row_now = -1;
  if (warp == COPY_WARP) {
    if (lane == 0) {
      for (int i = 0; i < RING; ++i) {
        mbar_init(&raw_full[i], 1);
        mbar_init(&raw_empty[i], CONVERTERS);
        mbar_init(&full[i], CONVERTERS);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < SLOTS; ++i) {
        mbar_init(&sc_full[i], 1);
        mbar_init(&sc_empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[2 * i], SOFTMAX_WARPS / 2);
        mbar_init(&p_full[2 * i + 1], SOFTMAX_WARPS / 2);
        mbar_init(&o_final[i], 1);
      }
      mbar_init(pv_done, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    row_now = row_of(0);
  }
  const __nv_bfloat16* qp = q;
  pdl_wait(qp);
  if (warp == COPY_WARP) {
    send(0, row_now);
    send(1, row_now);
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  // Both query tiles -> shared memory, swizzled, 16 lanes a row: times the power of two that takes the row's largest value to
  // 2^4 .. 2^5 (exact in float16 down to 2^-21 of that); rows beyond a tile's tokens and dimensions beyond D are zero.  (A
  // thread a row took 5 us: the lines do not stay in what L1 has left.)
  {
    constexpr int PER_THREAD = 2 * TILE * 16 / THREADS;
    const int ch = threadIdx.x & 15;
    uint4 v[PER_THREAD];
#pragma unroll
    for (int it = 0; it < PER_THREAD; ++it) {
      const int row = it * (THREADS / 16) + (threadIdx.x >> 4), x = row >> 7;
      const int tl = token_of(row & 127), g = (row & 127) - tl * G;
      v[it] = make_uint4(0, 0, 0, 0);
      if (tl < (x ? ntok[1] : ntok[0]) && ch * 8 < a.D)
        v[it] = *reinterpret_cast<const uint4*>(
            qp + ((long long)(q_begin + (x ? tokx[1] : tokx[0]) + tl) * a.Hq + kvh * G + g) * a.D + ch * 8);
    }
#pragma unroll
    for (int it = 0; it < PER_THREAD; ++it) {
      const int row = it * (THREADS / 16) + (threadIdx.x >> 4), x = row >> 7;
      const unsigned w[4] = {v[it].x, v[it].y, v[it].z, v[it].w};
      unsigned top = 0;      // the largest magnitude, in the high half
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fff0000u, w[e] << 16 & 0x7fff0000u));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int expo = max((int)(top >> 23), 5);                    // (2^126 at most below)
      const bool finite = top < 0x7f800000u;
      const float to_unit = two_to(131 - expo);
      unsigned y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = finite ? pack_f16(__uint_as_float(w[e] << 16) * to_unit, __uint_as_float(w[e] & 0xffff0000u) * to_unit) : 0u;
      *reinterpret_cast<uint4*>(sQ + x * TILE_BYTES + piece_off(row & 127, ch)) = make_uint4(y[0], y[1], y[2], y[3]);
      if (ch == 0) row_units[row] = finite ? two_to(expo - 131) : __int_as_float(0x7fc00000);
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the queries are read by the tensor core
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp >= COPY_WARP) {
  regs_give<REGS_FEW>();
  if (warp == MMA_WARP) {
    {
      const unsigned elected = elect_one();
      constexpr unsigned idesc_s = idesc_f16(TILE, TILE, false, 0);
      // Descriptors are made once: a step inside a tile is an addition to the low bits, which hold the address.
      const unsigned long long q_desc = desc_k_major(smem_u32(sQ)), k_desc = desc_k_major(smem_u32(sKV)),
                               v_desc = desc_mn_major(smem_u32(sKV));
      auto issue_s = [&](int x, int buf, int i) {      // scores of query tile x, key tile i -> columns of buf
        const unsigned long long qd = q_desc + x * (TILE_BYTES >> 4), kd = k_desc + (2 * i % RING) * (TILE_BYTES >> 4);
#pragma unroll
        for (int ks = 0; ks < TILE / 16; ++ks) {
          const unsigned long long at = (unsigned long long)(((ks >> 2) * HALF_BYTES + (ks & 3) * 32) >> 4);
          tc_mma(elected, tmem + buf * 128, qd + at, kd + at, idesc_s, ks > 0);
        }
        tc_commit(elected, &s_full[buf]);
      };
      int uses[2] = {0, 0};     // completed phases of p_full
      // outputs of query tile x from the probabilities in buf, each half as soon as it is there
      auto issue_o = [&](int x, int buf, int i) {
        const unsigned long long vd = v_desc + ((2 * i + 1) % RING) * (TILE_BYTES >> 4);
        const bool first = j0 + i == (x ? jf[1] : jf[0]);
        const unsigned idesc_o = infos[i % SLOTS].wide ? idesc_f16(TILE, TILE, true, 1) : idesc_f16(TILE, TILE, false, 1);
        const int turn = (buf ? uses[1]++ : uses[0]++) & 1;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ok = __all_sync(0xffffffffu, mbar_wait_brief(&p_full[2 * buf + half], turn));
          if (!ok) return;
          tc_fence_after();
#pragma unroll
          for (int ks = half * 4; ks < half * 4 + 4; ++ks)
            tc_mma_ts(elected, tmem + 256 + x * 128, tmem + buf * 128 + ks * 8, vd + (unsigned long long)((ks * 16 * 128) >> 4),
                      idesc_o, !first || ks > 0);
        }
      };
      auto want = [&](int item) {
        ok = __all_sync(0xffffffffu, mbar_wait_brief(&full[item % RING], (item / RING) & 1));
        tc_fence_after();
        return ok;
      };
      if (want(0)) {
        if (active(0, 0)) issue_s(0, 0, 0);
        if (active(1, 0)) issue_s(1, 1, 0);
        tc_commit(elected, &empty[0]);
      }
      const int paired_end = min(ntiles, solo_from);
      for (int i = 0; i < paired_end && ok; ++i) {
        if (!want(2 * i + 1) || (i + 1 < ntiles && !want(2 * i + 2))) break;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (active(x, i)) {
            issue_o(x, x, i);
            if (!ok) break;
            if (j0 + i == jl[x]) tc_commit(elected, &o_final[x]);
          }
          if (x == 1) {
            tc_commit(elected, &empty[(2 * i + 1) % RING]);
            tc_commit(elected, &sc_empty[i % SLOTS]);
          }
          if (i + 1 < ntiles && active(x, i + 1)) issue_s(x, x, i + 1);
          if (x == 1 && i + 1 < ntiles) tc_commit(elected, &empty[(2 * i + 2) % RING]);
        }
      }
      // ---- one query tile alone: its scores of key tile i are in buffer (i - solo_from) & 1 (0: its own columns); those of
      // i + 1 go to the other one before the probabilities of i are waited for
      for (int i = solo_from; i < ntiles && ok; ++i) {
        const int x = solo_x, buf = ((i - solo_from) & 1) ? 1 - x : x;
        if (i + 1 < ntiles) {
          if (!want(2 * i + 2)) break;
          issue_s(x, 1 - buf, i + 1);
          tc_commit(elected, &empty[(2 * i + 2) % RING]);
        }
        if (!want(2 * i + 1)) break;
        issue_o(x, buf, i);
        if (!ok) break;
        tc_commit(elected, &empty[(2 * i + 1) % RING]);
        tc_commit(elected, &sc_empty[i % SLOTS]);
        tc_commit(elected, pv_done);
        if (i == ntiles - 1) tc_commit(elected, &o_final[x]);
      }
    }
  } else if (warp == COPY_WARP) {
    // ---- bytes, and the scales of this lane's keys (zero for keys that the sequence does not have), which are asked for a
    // tile ahead
    int sent = 2;
    float ks[4], vs[4];
    auto load_scales = [&](int row) {
      float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
      if (row >= 0) {
        k = *reinterpret_cast<const float4*>(a.scales + row);
        v = *reinterpret_cast<const float4*>(a.scales + row + half_rows);
      }
      ks[0] = k.x; ks[1] = k.y; ks[2] = k.z; ks[3] = k.w;
      vs[0] = v.x; vs[1] = v.y; vs[2] = v.z; vs[3] = v.w;
    };
    load_scales(row_now);
    int row_next = row_of(1);
    const float unit = a.scale * LOG2E;
    constexpr int UNSET = -1000;
    int value_exp = UNSET;      // (not known before a scale that is not zero)
    // what some row sees; the other keys of a tile are somebody else's, or not there yet
    const int seen_from = first_visible_key(prefix + (any0 ? tokx[0] : tokx[1]), a.window);
    const int seen_to = prefix + (any1 ? tokx[1] + ntok[1] : tokx[0] + ntok[0]);
    for (int i = 0; i < ntiles && ok; ++i) {
      if (i >= SLOTS) ok = mbar_wait_brief(&sc_empty[i % SLOTS], (i / SLOTS - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int key = (j0 + i) * TILE + lane * 4;
      unsigned bad[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // a key or a value that is no number shows in the sums of the rows that see it
        const float both = (ks[j] - ks[j]) + (vs[j] - vs[j]);
        const bool seen = key + j >= seen_from && key + j < seen_to, is_nan = seen && both != both;
        bad[j] = __ballot_sync(0xffffffffu, is_nan);
        ks[j] *= unit;
        if (!seen || is_nan) ks[j] = vs[j] = 0.f;
        if (fabsf(vs[j]) < 0x1p-106f) vs[j] = 0.f;      // (a row of values below 2^-99, such as zeros: it reads back as zeros)
      }
      float top = 0.f, bottom = INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        top = fmaxf(top, fabsf(vs[j]));
        if (vs[j] != 0.f) bottom = fminf(bottom, fabsf(vs[j]));
      }
      const int top_exp = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127;
      const int bottom_exp = (int)(__reduce_min_sync(0xffffffffu, __float_as_uint(bottom)) >> 23) - 127;
      // A unit takes the largest scale to 2^4 .. 2^5; scales of 2^-13 .. 2^8 leave float16 all of its bits for the values.
      bool wide = false;
      if (top_exp > -127) {
        wide = top_exp - bottom_exp > 17;
        if (value_exp == UNSET || top_exp - value_exp > (wide ? 40 : 7)) value_exp = top_exp - 4;
        if (!wide && bottom_exp - value_exp < -13) {
          // (float32 holds the outputs so far in a unit up to 2^80 smaller)
          if (value_exp - (top_exp - 4) > 80) wide = true; else value_exp = top_exp - 4;
        }
      }
      const float to_unit = value_exp == UNSET ? 0.f : two_to(-value_exp);
      float* slot = scales + (i % SLOTS) * 256 + lane * 4;
      *reinterpret_cast<float4*>(slot) = make_float4(ks[0], ks[1], ks[2], ks[3]);
      *reinterpret_cast<float4*>(slot + 128) = make_float4(vs[0] * to_unit, vs[1] * to_unit, vs[2] * to_unit, vs[3] * to_unit);
      if (lane == 0) {
        TileInfo n;
        n.any_nan = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) n.any_nan |= n.nan[j] = bad[j];
        n.wide = wide;
        n.value_exp = value_exp == UNSET ? 0 : value_exp;
        n.pad = 0;
        infos[i % SLOTS] = n;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc_full[i % SLOTS]);
      if (i + 1 < ntiles) {
        load_scales(row_next);
        row_now = row_next;
        row_next = row_of(i + 2);
        for (int item = 2 * i + 2; item < 2 * i + 4 && ok; ++item) {
          if (item >= RING) ok = mbar_wait_brief(&raw_empty[item % RING], (item / RING - 1) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) {
            send(item, row_now);
            sent = item + 1;
          }
        }
      }
    }
    // the last bytes that were sent for have arrived before this block's memory is another's
    for (int item = max(0, sent - RING); item < sent; ++item)
      if (!mbar_wait_brief(&raw_full[item % RING], (item / RING) & 1)) ok = false;
  } else {
    // ---- conversion.  A warp has the even or the odd 64 codes of some groups of 8 rows; eight lanes a pair of rows r, r ^ 5,
    // whose pieces lie in different banks in the bytes' swizzle and in the 16-bit tile's.  Warps 12 and 13 have half of the
    // groups: the others are two to a scheduler.
    const int r8 = lane & 4 ? (lane >> 3) ^ 5 : lane >> 3, p = (warp & 1) * 4 + (lane & 3);
    const int g_from = warp < 12 ? 0 : warp < 14 ? 4 : 12, g_to = warp < 12 ? 4 : warp < 14 ? 12 : 16;
    const int src_off = r8 * 128 + ((p ^ r8) << 4), dst_off0 = piece_off(r8, 2 * p), dst_off1 = piece_off(r8, 2 * p + 1);
    // codes times a scale (keys': 1, exactly) in float16; wide: codes in bfloat16
    auto convert8 = [&](const unsigned char* src, unsigned char* dst, __half2 scale, int g8, auto wide) {
      const uint4 w = *reinterpret_cast<const uint4*>(src + src_off + g8 * 1024);
      const unsigned word[4] = {w.x, w.y, w.z, w.w};
      unsigned y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const unsigned sel = half ? 0x4342 : 0x4140;
          y[2 * e + half] = wide.value ? codes_bf16(word[e], sel) : times_f16(codes_f16(word[e] ^ 0x80808080u, sel), scale);
        }
      *reinterpret_cast<uint4*>(dst + dst_off0 + g8 * 1024) = make_uint4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<uint4*>(dst + dst_off1 + g8 * 1024) = make_uint4(y[4], y[5], y[6], y[7]);
    };
    for (int item = 0, at = 0, turn = 0; item < 2 * ntiles && ok; ++item) {
      const int slot = (item >> 1) % SLOTS;
      ok = (!(item & 1) || mbar_wait_brief(&sc_full[slot], ((item >> 1) / SLOTS) & 1)) && mbar_wait_brief(&raw_full[at], turn) &&
           (item < RING || mbar_wait_brief(&empty[at], turn ^ 1));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const float* vs = scales + slot * 256 + 128;
      const unsigned char* src = raw + at * RAW_BYTES;
      unsigned char* dst = sKV + at * TILE_BYTES;
      // (loops as short as they can be: what a warp runs seldom costs the others their instructions)
      const bool values = item & 1;
      if (__builtin_expect(values && infos[slot].wide, 0)) {
#pragma unroll 1
        for (int g8 = g_from; g8 < g_to; ++g8) convert8(src, dst, __half2(), g8, std::true_type());
      } else {
#pragma unroll 1
        for (int g8 = g_from; g8 < g_to; ++g8)
          convert8(src, dst, __float2half2_rn(values ? vs[g8 * 8 + r8] : 1.f), g8, std::false_type());
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the tile is read by the tensor core, the bytes are
      __syncwarp();                                                    // written by the next copy
      if (lane == 0) {
        mbar_arrive(&full[at]);
        mbar_arrive(&raw_empty[at]);
      }
      if (++at == RING) {
        at = 0;
        turn ^= 1;
      }
    }
  }
  } else {
    regs_take<REGS_MANY>();
    // ---- softmax: thread r of group x owns row r of query tile x
    const int x = threadIdx.x >> 7, r = threadIdx.x & 127;
    const int tl = token_of(r), g = r - tl * G;
    const int tok0 = x ? tokx[1] : tokx[0], i_first = (x ? jf[1] : jf[0]) - j0, i_last = (x ? jl[1] : jl[0]) - j0;
    const bool valid = tl < (x ? ntok[1] : ntok[0]);
    // (rows behind the sequence's last token see what a token there would see: no warp goes through the tests for masked
    // keys for their sake)
    const int hi = prefix + tok0 + tl, lo = first_visible_key(hi, a.window);
    const unsigned lane_base = (unsigned)((warp & 3) * 32) << 16;
    const unsigned tmem_o = tmem + lane_base + 256 + x * 128;
    float row_unit = row_units[threadIdx.x], m_ref = NEG_BIG, l = 0.f;
    if (row_unit != row_unit) {      // its queries are zeros: the sum makes its result NaN
      l = row_unit;
      row_unit = 1.f;
    }
    int uses_own = 0, uses_other = n_other;      // completed phases of s_full of the own columns and of the other's
    const int my_solo = x == solo_x ? solo_from : 0x7fffffff;
    const float2 unit2 = make_float2(row_unit, row_unit);
    int value_exp = 0;
    for (int i = i_first; i <= i_last && ok; ++i) {
      const bool borrowed = i >= my_solo && ((i - my_solo) & 1);
      const int buf = borrowed ? 1 - x : x;
      const unsigned tmem_s = tmem + lane_base + buf * 128;
      ok = mbar_wait_brief(&sc_full[i % SLOTS], (i / SLOTS) & 1) && mbar_wait_brief(&s_full[buf], (borrowed ? uses_other : uses_own) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (borrowed) ++uses_other; else ++uses_own;
      tc_fence_after();
      const int kbase = (j0 + i) * TILE, first = lo - kbase, last = hi - kbase;      // visible: [first, last]
      const unsigned ks = smem_u32(scales + (i % SLOTS) * 256);
      const TileInfo* info = infos + i % SLOTS;
      unsigned v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tc_ld32(tmem_s + c * 32, v[c]);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float2 y = __fmul2_rn(make_float2(__uint_as_float(v[c][k]), __uint_as_float(v[c][k + 1])),
                                      load_shared2(ks + (c * 32 + k) * 4));
          v[c][k] = __float_as_uint(y.x);
          v[c][k + 1] = __float_as_uint(y.y);
        }
      if (__builtin_expect(first > 0 || last < TILE - 1, 0)) {
        // keys outside [first, last]: one subtraction and one unsigned comparison each
        const int first_vis = last >= first ? first : (1 << 20);
        const unsigned span = last >= first ? (unsigned)(last - first) : 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if ((unsigned)(c * 32 + k - first_vis) > span) v[c][k] = 0xff800000u;
      }
      float m4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) m4[c] = fmaxf(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]));
#pragma unroll
      for (int k = 2; k < 32; k += 2)
#pragma unroll
        for (int c = 0; c < 4; ++c) m4[c] = max3(m4[c], __uint_as_float(v[c][k]), __uint_as_float(v[c][k + 1]));
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * row_unit;
      if (__builtin_expect(info->any_nan, 0)) {      // a visible key that is no number: so is the row's result
        for (int k = max(first, 0); k <= min(last, TILE - 1); ++k)
          if (info->nan[k & 3] >> (k >> 2) & 1) l = __int_as_float(0x7fc00000);
      }
      const int old_exp = value_exp;
      value_exp = info->value_exp;
      const bool wide_tile = info->wide != 0, moved = i > i_first && value_exp != old_exp;
      // the reference rises only when it must (or at the first visible key)
      float factor = 1.0f;
      bool rescale = false;
      if (mx > m_ref + 8.0f) {
        rescale = m_ref > -1e29f;
        factor = rescale ? fast_exp2(m_ref - mx) : 0.f;
        m_ref = mx;
        l *= factor;
      }
      // O of this tile is rescaled when a row of the warp raised its reference, or the values' unit moved.  Its last product
      // completed before these scores did, except where the tile runs alone: the product of i - 1 is waited for there.
      if (__builtin_expect(__any_sync(0xffffffffu, rescale) || moved, 0)) {
        const float by = (rescale ? factor : 1.f) * (moved ? two_to(max(old_exp - value_exp, -126)) : 1.f);
        if (i > my_solo) {
          ok = mbar_wait_brief(pv_done, (i - 1 - my_solo) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          unsigned o[8];
          tc_ld8(tmem_o + c * 8, o);
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
          tc_st8(tmem_o + c * 8, o);
        }
      }
      const float offset = m_ref <= -1e29f ? 0.f : -m_ref;
      const float2 off2 = make_float2(offset, offset);
      float2 s8[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      auto weights = [&](int half, auto wide) {      // (wide: the values' scales join the probabilities)
#pragma unroll
        for (int k = 0; k < 64; k += 2) {
          const int c = half * 2 + (k >> 5);
          const float2 y = __ffma2_rn(make_float2(__uint_as_float(v[c][k & 31]), __uint_as_float(v[c][(k & 31) + 1])), unit2, off2);
          const float2 p = make_float2(fast_exp2(y.x), fast_exp2(y.y));      // (exactly zero for a masked score)
          s8[(k >> 1) & 3] = __fadd2_rn(s8[(k >> 1) & 3], p);
          if (wide.value) {
            const float2 w = __fmul2_rn(p, load_shared2(ks + (128 + half * 64 + k) * 4));
            v[half][k >> 1] = pack_bf16(w.x, w.y);
          } else {
            v[half][k >> 1] = pack_f16(p.x, p.y);
          }
        }
      };
      auto hand_over = [&](int half) {
        tc_st32(tmem_s + half * 32, v[half]);      // probabilities over the scores they came from
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * buf + half]);
      };
      if (__builtin_expect(wide_tile, 0)) {
        weights(0, std::true_type());
        hand_over(0);
        weights(1, std::true_type());
      } else {
        weights(0, std::false_type());
        hand_over(0);
        weights(1, std::false_type());
      }
      hand_over(1);
      l += ((s8[0].x + s8[0].y) + (s8[1].x + s8[1].y)) + ((s8[2].x + s8[2].y) + (s8[3].x + s8[3].y));
    }
    if (ok && i_last >= i_first) {
      ok = mbar_wait_brief(&o_final[x], 0);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      // Outputs by way of the query tile, which nobody reads any more: a warp's 32 rows, then whole rows to memory.
      unsigned char* stage = sQ + x * TILE_BYTES + (warp & 3) * 8192;
      const bool partial = !(x ? whole[1] : whole[0]);      // this chunk's: O as accumulated (against m_ref), m_ref, l
      const float inv = l == 0.f ? 0.f : 1.0f / l, value_unit = two_to(value_exp);
      const int my_ntok = x ? ntok[1] : ntok[0], row0 = (warp & 3) * 32;
      // row rr of this tile as a row of the output, or of the partial results, whose first token is `first`; -1: none
      auto row_of_lane = [&](int first, int rr) {
        const int t = token_of(rr);
        return t < my_ntok ? (long long)(first + t) * a.Hq + kvh * G + rr - t * G : -1ll;
      };
      if (ok && partial) {
        const int place0 = a.units[4 * a.unit_stride + unit] + tok0 - tokx[0];      // of this tile's first token
        if (valid) a.part_ml[((long long)(place0 + tl) * a.Hq + kvh * G + g) * a.max_chunks + chunk] = make_float2(m_ref, l);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {      // 64 dimensions at a time
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            unsigned o[32];
            tc_ld32(tmem_o + half * 64 + c * 32, o);
            tc_wait_ld();
            auto value = [&](int e) { return __float_as_uint(__uint_as_float(o[e]) * value_unit); };
#pragma unroll
            for (int ch = 0; ch < 8; ++ch)
              *reinterpret_cast<uint4*>(stage + lane * 256 + ((c * 8 + ch) ^ (lane & 7)) * 16) =
                  make_uint4(value(ch * 4), value(ch * 4 + 1), value(ch * 4 + 2), value(ch * 4 + 3));
          }
          __syncwarp();
#pragma unroll 4
          for (int rr = lane >> 4; rr < 32; rr += 2) {
            const long long row = row_of_lane(place0, row0 + rr);
            if (row >= 0)
              *reinterpret_cast<uint4*>(a.part_o + (row * a.max_chunks + chunk) * TILE + half * 64 + (lane & 15) * 4) =
                  *reinterpret_cast<const uint4*>(stage + rr * 256 + ((lane & 15) ^ (rr & 7)) * 16);
          }
          __syncwarp();
        }
      } else if (ok) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          unsigned o[32];
          tc_ld32(tmem_o + c * 32, o);
          tc_wait_ld();
          auto value = [&](int e) { return __uint_as_float(o[e]) * inv * value_unit; };
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
            *reinterpret_cast<uint4*>(stage + lane * 256 + ((c * 4 + ch) ^ (lane & 7)) * 16) =
                make_uint4(pack_bf16(value(ch * 8), value(ch * 8 + 1)), pack_bf16(value(ch * 8 + 2), value(ch * 8 + 3)),
                           pack_bf16(value(ch * 8 + 4), value(ch * 8 + 5)), pack_bf16(value(ch * 8 + 6), value(ch * 8 + 7)));
        }
        __syncwarp();
#pragma unroll 4
        for (int rr = lane >> 4; rr < 32; rr += 2) {
          const long long row = row_of_lane(q_begin + tok0, row0 + rr);
          if (row >= 0 && (lane & 15) * 8 < a.D)
            *reinterpret_cast<uint4*>(out + row * a.D + (lane & 15) * 8) =
                *reinterpret_cast<const uint4*>(stage + rr * 256 + ((lane & 15) ^ (rr & 7)) * 16);
        }
      }
    }
  }
  if (!ok) atomicExch(&dib_attention_int8_prompt_error_word, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// Rows whose keys span several chunks: out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c in chunk order, over the chunks of
// the row's query tile.  A warp a (token, head), a lane four dimensions; rows that the attention finished cost a look at
// their lengths.  entries [4][entry_stride]: sequence, first token, end, place of the first token's partial results.
__global__ void __launch_bounds__(256)
attention_prompt_merge_kernel(__nv_bfloat16* __restrict__ out, const __grid_constant__ PromptArgs a,
                              const int* __restrict__ entries, int entry_stride) {
  const float* part_o = a.part_o;
  const float2* part_ml = a.part_ml;
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int seq = entries[blockIdx.y], tok_begin = entries[entry_stride + blockIdx.y], tok_end = entries[2 * entry_stride + blockIdx.y];
  const int q_begin = a.cu_q_lens[seq], q_len = a.cu_q_lens[seq + 1] - q_begin;
  const int id = blockIdx.x * 8 + (threadIdx.x >> 5), h = id % a.Hq, tok = tok_begin + id / a.Hq;
  pdl_wait(part_o, part_ml);
  if (tok >= min(tok_end, q_len)) return;
  const int kv_len = min(a.seq_lens[seq], (int)min((long long)a.max_blocks << a.page_shift, 0x7fffff00ll));
  const int npt = TILE / (a.Hq / a.Hkv), tok0 = tok / npt * npt;
  const int first_pos = kv_len - q_len + tok0, last_pos = first_pos + min(npt, q_len - tok0) - 1;
  if (last_pos < 0) return;
  const int c0 = first_visible_key(first_pos, a.window) / TILE / a.chunk_tiles;
  const int c1 = min(last_pos / TILE / a.chunk_tiles, a.max_chunks - 1);
  if (c0 >= c1) return;     // finished by the attention itself
  const long long row = (long long)(entries[3 * entry_stride + blockIdx.y] + tok - tok_begin) * a.Hq + h;
  part_o += row * a.max_chunks * TILE + lane * 4;
  part_ml += row * a.max_chunks;
  float top = NEG_BIG;
  for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, part_ml[c].x);
  top = warp_max(top);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const float2 ml = part_ml[c];
    const float4 v = *reinterpret_cast<const float4*>(part_o + (long long)c * TILE);
    const float w = fast_exp2(ml.x - top);
    sum = fmaf(w, ml.y, sum);
    o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
  }
  if (lane * 4 >= a.D) return;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  *reinterpret_cast<uint2*>(out + ((long long)(q_begin + tok) * a.Hq + h) * a.D + lane * 4) =
      make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
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

}  // namespace

extern "C" {

int dib_attention_int8_prompt_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dib_attention_int8_prompt_error_word, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int dib_attention_int8_prompt_status_clear() {
  const int v = 0;
  return cudaMemcpyToSymbol(dib_attention_int8_prompt_error_word, &v, sizeof(int)) == cudaSuccess ? 0 : -1;
}

// q, out bfloat16 [T, Hq, D], heads up to 128, up to 128 query heads a kv head, pages of a power of two of rows, 4 at least.
// units int32 [5, unit_stride], `count` of each row: sequence, first tokens of A and B (128 / (Hq / Hkv) tokens each; -1: no B),
// chunk, place of A's first token in the partial results (B follows A); the longest last.
// chunk_tiles: 0, or the key tiles of a chunk: then part_o float32 [places, Hq, max_chunks, 128] and part_ml [.., 2] take partial
// results, which are added up for entry_count entries, int32 [4, entry_stride]: sequence, first token, end, place of the first
// token (max_tokens: the most of one).
int dib_int8_attention_prompt(const void* q, void* out, const void* data, const void* scales, long long num_pages,
                              const void* block_table, int max_blocks, const void* cu_q_lens, const void* seq_lens,
                              const void* units, int count, int unit_stride, const void* entries, int entry_count,
                              int entry_stride, int max_tokens, void* part_o, void* part_ml, int chunk_tiles, int max_chunks,
                              int Hq, int Hkv, int D, int page_size, float scale, int window, cudaStream_t st) {
  if (count < 0 || count > 65535 || unit_stride < count || entry_count < 0 || entry_count > 65535 || entry_stride < entry_count ||
      Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || Hq / Hkv > TILE || D < 16 || D > 128 || D % 16 != 0 || page_size < 4 || (page_size & (page_size - 1)) != 0 ||
      num_pages * 2 * Hkv * page_size >= (1ll << 31) || chunk_tiles < 0 || max_chunks < 1)
    return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(q) |
        reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (count == 0) return DIB_OK;
  PromptArgs a;
  a.scales = reinterpret_cast<const float*>(scales);
  a.block_table = reinterpret_cast<const int*>(block_table);
  a.cu_q_lens = reinterpret_cast<const int*>(cu_q_lens);
  a.seq_lens = reinterpret_cast<const int*>(seq_lens);
  a.units = reinterpret_cast<const int*>(units);
  a.count = count; a.unit_stride = unit_stride; a.max_blocks = max_blocks; a.Hq = Hq; a.Hkv = Hkv; a.D = D;
  a.page_shift = 0;
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  a.num_pages = (int)num_pages;
  a.window = window; a.chunk_tiles = chunk_tiles; a.max_chunks = max_chunks;
  a.scale = scale;
  a.part_o = reinterpret_cast<float*>(part_o);
  a.part_ml = reinterpret_cast<float2*>(part_ml);
  CUtensorMap map;
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return DIB_LAUNCH_FAILED;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)(num_pages * 2 * Hkv * page_size)};
  const cuuint64_t strides[1] = {(cuuint64_t)D};
  const cuuint32_t box[2] = {128, (cuuint32_t)(page_size < TILE ? page_size : TILE)};
  const cuuint32_t estr[2] = {1, 1};
  if (enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(data), dims, strides, box, estr,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return DIB_LAUNCH_FAILED;
  static_assert(S_DYNAMIC <= 232448, "shared memory");
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(attention_prompt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S_DYNAMIC) != cudaSuccess)
      return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  dib_launch(attention_prompt_kernel, dim3(Hkv, count), dim3(THREADS), S_DYNAMIC, st, map,
             reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<__nv_bfloat16*>(out), a);
  DIB_CHECK_LAUNCH();
  if (chunk_tiles > 0) {
    const long long blocks = ((long long)max_tokens * Hq + 7) / 8;
    if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
    dib_launch(attention_prompt_merge_kernel, dim3((unsigned)blocks, entry_count), dim3(256), 0, st,
               reinterpret_cast<__nv_bfloat16*>(out), a, reinterpret_cast<const int*>(entries), entry_stride);
    DIB_CHECK_LAUNCH();
  }
  return DIB_OK;
}

}  // extern "C"
