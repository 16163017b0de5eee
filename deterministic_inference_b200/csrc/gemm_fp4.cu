// Matrix product of rows in 4-bit floating point (fp4.cuh): y[m, n] = ux[m] * uw[n] * sum_k (cx bx)[m, k] * (cw bw)[n, k], c the
// e2m1 codes, b the e4m3 scales of blocks of 16 values, u = 2^E of the row.  Codes and block scales enter the tensor cores as
// they are (tcgen05.mma kind::mxf4nvf4, a scale for each 16 values of either operand, 64 values an instruction, sums in
// float32); the rows' powers of two are exact and join the sum in the epilogue, which rounds once.
//
// Every form adds a row's k up in one order: k is cut into parts by its own length (Parts), a part is summed in one accumulator,
// 64 values at a time from its first to its last, and the parts' sums are added in their order in float32.  So a row's
// bits depend on the row and the weight alone, not on the other rows, the tile or the form.
//
// Operands by TMA, 256 values (128 bytes, 128-byte swizzle) of each row a stage, with the block scales in tiles of 128 rows
// x 64 values (512 bytes, rows_fp4.cu), through a ring of mbarrier-guarded stages.  The products' warp copies a stage's scales
// from shared into tensor memory (tcgen05.cp), in order with the products, so that one buffer does.
//
// Few rows: a cluster has a tile of 128 channels, each of its CTAs a part of k; the channels are the products' 128 lanes, the tokens
// their columns.  Many rows: tiles of 128 tokens x BN channels, or 256 x 192 for a pair of CTAs.
//
// What bounds it: few rows, the weight's bytes (8 x 24,576 x 4,096 11.6 us, 4.9 TB/s; 8 x 4,096 x 12,288 8.0 us, 3.5 TB/s, the rest
// the cluster's start and sums); many rows, the tiles' operands from L2 (2,048 x 24,576 x 4,096 101 us among others, 97 by itself,
// 4.3 PFLOP/s: 1.06 GB at 10.9 TB/s; the copies without products take as long, the products without copies 67 us).
#include <cuda.h>

#include "fp4.cuh"

namespace {

constexpr int BM = 128, BK = 256, ROW_BYTES = BK / 2, UMMA_K = 64;      // tokens of a tile and CTA, values of a stage, of an instruction
constexpr int THREADS = 384, EPI_WARP0 = 4, EPI_WARPS = 8, MAX_STAGES = 16, MAX_PARTS = 8;
constexpr int SCALES = 2048;                            // a stage's block scales of 128 rows: four tiles along k
constexpr int EPI_STAGE_BYTES = 32 * 128;               // a warp's 32 rows of 32 values, twice in bfloat16
constexpr int SMEM_MOST = 232448 - 1024;                // (1 KB left to static shared memory)
__device__ int dib_gemm_fp4_error_word = 0;

// How k, num_kb stages, is cut into parts: eight stages each at least, eight parts at most, the first ones a stage longer than the
// others where that does not go even.  (Parts of four: 8 x 4,096 x 4,096 5.4 us instead of 6.3, but 8 x 24,576 x 4,096 22.9 instead
// of 11.7, and 2,048 x 24,576 x 4,096 127 instead of 101: with many rows each part is read from tensor memory.  One part: 8 x 4,096
// x 12,288 20.4 us instead of 8.3.)
struct Parts {
  int parts, each, longer;      // stages of a part, number of parts that have one more
  explicit Parts(int num_kb) {
    parts = num_kb / 8 < 1 ? 1 : num_kb / 8 > MAX_PARTS ? MAX_PARTS : num_kb / 8;
    each = num_kb / parts;
    longer = num_kb % parts;
  }
  __device__ __forceinline__ int begin(int part) const { return part * each + min(part, longer); }
};

// A CTA's share of a tile: rows of channels that it fetches, tiles of channels' scales (64-channel tiles that begin in the middle of a
// tile of 128 scales among them), columns of tensor memory.
template <int BN, bool PAIR> struct Shape {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int B_TILES = BN == 192 ? 2 : 1;
  static constexpr int STAGE = (B_ROWS + BM) * ROW_BYTES + (1 + B_TILES) * SCALES;
  static constexpr int STAGES = (SMEM_MOST - 1024 - EPI_WARPS * EPI_STAGE_BYTES) / STAGE < MAX_STAGES
                                    ? (SMEM_MOST - 1024 - EPI_WARPS * EPI_STAGE_BYTES) / STAGE : MAX_STAGES;
  static constexpr int SMEM = 1024 + STAGES * STAGE + EPI_WARPS * EPI_STAGE_BYTES;
  static constexpr int SFA = 2 * BN, SFB = SFA + 16, COLUMNS = SFB + 16 * B_TILES;
  static constexpr int TMEM = COLUMNS <= 256 ? 256 : 512;
};

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(unsigned cluster_address) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_address) : "memory");
}
// A copy into this CTA's shared memory whose bytes are counted by the barrier at a cluster address, which in the pair may
// be the other CTA's.
template <bool PAIR>
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int c0, int c1, unsigned bar) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
// the same of a box of three dimensions, its first coordinate 0
template <bool PAIR>
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c1, int c2, unsigned bar) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(reinterpret_cast<unsigned long long>(map)), "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
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
template <bool PAIR> __device__ __forceinline__ void tc_commit(unsigned elected, unsigned long long* bar) {
  if (PAIR)
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "setp.ne.b32 e, %2, 0;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t"
        "}\n" ::"r"(smem_u32(bar)), "h"((unsigned short)3), "r"(elected)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "setp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "}\n" ::"r"(smem_u32(bar)), "r"(elected)
        : "memory");
}
// A tile of 128 rows' scales of 64 values (512 bytes) into four columns of tensor memory, for all four quarters of its lanes; in
// the pair, each CTA's own from the same place of its shared memory.
template <bool PAIR> __device__ __forceinline__ void tc_copy_scales(unsigned elected, unsigned tmem, unsigned long long desc) {
  if (PAIR)
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "setp.ne.b32 e, %2, 0;\n\t"
        "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t"
        "}\n" ::"r"(tmem), "l"(desc), "r"(elected)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "setp.ne.b32 e, %2, 0;\n\t"
        "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t"
        "}\n" ::"r"(tmem), "l"(desc), "r"(elected)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tc_mma(unsigned elected, unsigned tmem_d, unsigned long long desc_a, unsigned long long desc_b,
                                       unsigned idesc, unsigned scales_a, unsigned scales_b, unsigned accum) {
  if (PAIR)
    asm volatile(
        "{\n\t"
        ".reg .pred p, e;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 e, %7, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scales_a), "r"(scales_b), "r"(accum), "r"(elected)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred p, e;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 e, %7, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scales_a), "r"(scales_b), "r"(accum), "r"(elected)
        : "memory");
}
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
// Waits for tc_ld8 and tc_ld32, whose registers are handed on here: arithmetic on them must not be moved ahead of the wait.
template <int N> __device__ __forceinline__ void tc_wait_ld(unsigned (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}
// 8 consecutive columns of this thread's lane; valid after tc_wait_ld()
__device__ __forceinline__ void tc_ld8(unsigned taddr, unsigned (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
// K-major rows of 128 bytes, 128-byte swizzle: 8-row groups 1,024 bytes apart
__device__ __forceinline__ unsigned long long operand_desc(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((unsigned long long)(1024u >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// 32 rows of 16 bytes, one after the other: 8-row groups 128 bytes apart
__device__ __forceinline__ unsigned long long scales_desc(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(128u >> 4) << 32) | (1ull << 46);
}
// kind::mxf4nvf4: e2m1 operands, both K-major, unsigned e4m3 scales, 64 values an instruction
__host__ __device__ constexpr unsigned make_idesc(int m, int n) {
  return (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 7) << 27);
}
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned cluster_addr(unsigned local, unsigned rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}

// ---------------------------------------------------------------- many rows
struct Args {
  Parts k;
  const float* ux;      // [M]
  const float* uw;      // [N]
  void* out;            // [M, N]
  int M, N, num_kb, m_tiles, n_tiles;
  int by_lines;         // rows of the output do not lie on 16 bytes: no TMA stores
};

// A warp's 32 token rows from row0 on and COLS columns from n0 on, 32 columns at a time: a lane turns its row's sums into the
// output's type, stages them (swizzled) and the copy engine writes whole rows, clipped at M and N.  (Written straight from the
// registers, a row's 32 bytes at a time, 2,048 x 24,576 x 4,096 took 13 us more.)
template <typename OutT, int COLS>
__device__ __forceinline__ void store_rows(const float (&acc)[COLS], const CUtensorMap* map_out, unsigned char* staging, int& turn_buffer,
                                           int lane, int row0, int n0, const Args& a) {
  constexpr int WORDS = 32 * (int)sizeof(OutT) / 4, CHUNKS = WORDS / 4, PITCH = WORDS * 4;      // of 32 columns
  constexpr int BUFFERS = EPI_STAGE_BYTES / (32 * PITCH);      // 2 or 1, in turn
  const float ux = row0 + lane < a.M ? a.ux[row0 + lane] : 0.f;
  // (the swizzle of rows of 64 bytes goes by every other row)
  const int turn = sizeof(OutT) == 2 ? lane >> 1 & 3 : lane & 7;
#pragma unroll
  for (int col = 0; col < COLS; col += 32) {
    const int n = n0 + col;
    if (n >= a.N) return;
    unsigned char* stage = staging + (BUFFERS == 2 ? turn_buffer * (32 * PITCH) : 0);
    turn_buffer ^= 1;
    unsigned y[WORDS];
    const float* uw = a.uw + n;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float4 w;
      if (n + 32 <= a.N) {
        w = *reinterpret_cast<const float4*>(uw + 4 * j);
      } else {
        const int left = a.N - n - 4 * j;
        w = make_float4(left > 0 ? uw[4 * j] : 0.f, left > 1 ? uw[4 * j + 1] : 0.f, left > 2 ? uw[4 * j + 2] : 0.f,
                        left > 3 ? uw[4 * j + 3] : 0.f);
      }
      const float y0 = fp4_times_units(acc[col + 4 * j], ux, w.x), y1 = fp4_times_units(acc[col + 4 * j + 1], ux, w.y);
      const float y2 = fp4_times_units(acc[col + 4 * j + 2], ux, w.z), y3 = fp4_times_units(acc[col + 4 * j + 3], ux, w.w);
      if (sizeof(OutT) == 2) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(y0, y1), hi = __floats2bfloat162_rn(y2, y3);
        y[(2 * j) % WORDS] = *reinterpret_cast<const unsigned*>(&lo);
        y[(2 * j + 1) % WORDS] = *reinterpret_cast<const unsigned*>(&hi);
      } else {
        y[(4 * j) % WORDS] = __float_as_uint(y0);
        y[(4 * j + 1) % WORDS] = __float_as_uint(y1);
        y[(4 * j + 2) % WORDS] = __float_as_uint(y2);
        y[(4 * j + 3) % WORDS] = __float_as_uint(y3);
      }
    }
    // the buffer's store before this one must have read it
    if (lane == 0) {
      if (BUFFERS == 2) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      *reinterpret_cast<uint4*>(stage + lane * PITCH + ((c ^ turn) << 4)) =
          make_uint4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
    if (!a.by_lines) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tma_store_2d(map_out, stage, n, row0);
    } else {
      __syncwarp();
      OutT* out = reinterpret_cast<OutT*>(a.out);
      const int byte = lane * (int)sizeof(OutT);
      for (int r = 0; r < 32 && row0 + r < a.M; ++r) {
        const int t = sizeof(OutT) == 2 ? r >> 1 & 3 : r & 7;
        if (n + lane < a.N)
          out[(long long)(row0 + r) * a.N + n + lane] =
              *reinterpret_cast<const OutT*>(stage + r * PITCH + (((byte >> 4) ^ t) << 4) + (byte & 15));
      }
      __syncwarp();
    }
  }
}

// Persistent, one CTA an SM (or a pair of CTAs on two, cta_group::2: each fetches its own 128 tokens and half of the channels).  The
// accumulator lies twice in tensor memory, so that one part is added up in registers, and a tile stored, under the products of
// the next.  Roles: warps 0, 2 and 3 copy, warp 1 issues the products, warps 4-11 are the epilogue.
// PAIR: `full` of the first CTA counts both CTAs' copies, its commits signal `empty` and `acc_full` in both, `acc_empty` of the
// first takes an arrival of every epilogue warp of both.
template <typename OutT, int BN, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws,
                const __grid_constant__ CUtensorMap map_out, const __grid_constant__ Args a) {
  using SH = Shape<BN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1, B_ROWS = SH::B_ROWS, STAGES = SH::STAGES, STAGE = SH::STAGE;
  // a stage: channels, tokens, scales of tokens, of channels
  constexpr int A_AT = B_ROWS * ROW_BYTES, AS_AT = A_AT + BM * ROW_BYTES, BS_AT = AS_AT + SCALES;
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long full[STAGES], empty[STAGES];
  __shared__ unsigned long long acc_full[2], acc_empty[2];      // a part's accumulator is complete; the epilogue has read it
  __shared__ unsigned tmem_slot;
  // (an offset, not a rounded address: what is known to be shared memory is read and written with 32-bit addresses)
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  unsigned char* epi_stage = smem + STAGES * STAGE;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_xs);
    prefetch_tensormap(&map_ws);
    prefetch_tensormap(&map_out);
  }
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_rank() : 0;
  const int group = blockIdx.x / CTAS, groups = gridDim.x / CTAS;
  const int tiles = a.m_tiles * a.n_tiles;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 3);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CTAS * EPI_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((unsigned)SH::TMEM));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((unsigned)SH::TMEM));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
  }
  tc_fence_before();
  __syncthreads();
  // (with its tensor memory taken: the blocks of the kernel that follows wait for this grid, and must not hold what one of it waits for)
  if (!PAIR) pdl_trigger();
  if (PAIR) cluster_sync_all();       // both CTAs' barriers and tensor memory exist before either is used
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  bool ok = true;

  // (168 registers a thread at the launch: the first four warps give up most of theirs to the eight that add up)
  if (warp < EPI_WARP0) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
  if (warp != 1) {
    if (lane == 0) {
      // ---- copies, of channels (warp 0), tokens (2) and scales (3): one thread issues them no faster than 150 cycles apiece.  The ring
      // runs on across the tiles: load number c is k-block c % num_kb of this CTA's tile number c / num_kb.  Tiles in the order of
      // their channels, so that the CTAs side by side share them.
      const int my_tiles = tiles > group ? (tiles - group + groups - 1) / groups : 0;
      const int total = my_tiles * a.num_kb;
      const unsigned full0 = PAIR ? cluster_addr(smem_u32(full), 0) : smem_u32(full);
      const int bytes = CTAS * (warp == 0 ? B_ROWS * ROW_BYTES : warp == 2 ? BM * ROW_BYTES : (1 + SH::B_TILES) * SCALES);
      auto load_w = [&](int s, int n0, int kb) {
        if (warp == 0) tma_load_2d<PAIR>(smem + s * STAGE, &map_w, kb * ROW_BYTES, n0 + rank * B_ROWS, full0 + s * 8);
        // (a tile of scales behind the last reads as zeros)
        if (warp == 3) tma_load_3d<PAIR>(smem + s * STAGE + BS_AT, &map_ws, kb * 4, n0 / 128, full0 + s * 8);
      };
      auto load_x = [&](int s, int m0, int kb) {
        if (warp == 2) tma_load_2d<PAIR>(smem + s * STAGE + A_AT, &map_x, kb * ROW_BYTES, m0, full0 + s * 8);
        if (warp == 3) tma_load_3d<PAIR>(smem + s * STAGE + AS_AT, &map_xs, kb * 4, m0 / 128, full0 + s * 8);
      };
      const int pre = total < STAGES ? total : STAGES;
      for (int c = 0; c < pre; ++c) {      // weights are constants: the first stages' go out before the wait
        if (rank == 0) mbar_expect_tx(&full[c], bytes);
        load_w(c, (group + (c / a.num_kb) * groups) / a.m_tiles * BN, c % a.num_kb);
      }
      pdl_wait();
      for (int c = 0; c < pre; ++c)
        load_x(c, (group + (c / a.num_kb) * groups) % a.m_tiles * (CTAS * BM) + rank * BM, c % a.num_kb);
      int c = pre, s = 0, t = group + (pre / a.num_kb) * groups, kb = pre % a.num_kb;
      int m0 = t % a.m_tiles * (CTAS * BM) + rank * BM, n0 = t / a.m_tiles * BN;
      unsigned phase = 0;
      for (; c < total; ++c) {
        ok = mbar_wait_brief(&empty[s], phase);
        if (!ok) break;
        if (rank == 0) mbar_expect_tx(&full[s], bytes);
        load_w(s, n0, kb);
        load_x(s, m0, kb);
        if (++s == STAGES) {
          s = 0;
          phase ^= 1;
        }
        if (++kb == a.num_kb) {
          kb = 0;
          t += groups;
          m0 = t % a.m_tiles * (CTAS * BM) + rank * BM;
          n0 = t / a.m_tiles * BN;
        }
      }
      // given up: what was sent for arrives before this memory is another's (the pair's second CTA stays until the first, whose
      // barriers count for both, has waited)
      if (!ok && rank == 0)
        for (int i = c - STAGES; i < c; ++i) mbar_wait_brief(&full[i % STAGES], (i / STAGES) & 1);
    }
  } else {
    if (rank == 0) {
      // ---- products
      const unsigned elected = elect_one();
      constexpr unsigned idesc = make_idesc(CTAS * BM, BN);
      int local = 0, s = 0;      // parts so far, place in the ring
      unsigned phase = 0;
      for (int t = group; t < tiles && ok; t += groups) {
        // (channels that begin in the middle of a tile of scales: its last two columns are theirs)
        const unsigned sfb = tmem + SH::SFB + (BN % 128 != 0 ? ((t / a.m_tiles) * (BN / 64) & 1) * 2 : 0);
        for (int part = 0; part < a.k.parts && ok; ++part, ++local) {
          const int buf = local & 1, end = a.k.begin(part + 1);
          unsigned accum = 0;
          if (local >= 2) {      // the epilogue must have read this buffer's earlier part
            ok = __all_sync(0xffffffffu, mbar_wait_brief(&acc_empty[buf], ((local >> 1) - 1) & 1));
            if (!ok) break;
            tc_fence_after();
          }
          for (int kb = a.k.begin(part); kb < end; ++kb) {
            ok = __all_sync(0xffffffffu, mbar_wait_brief(&full[s], phase));
            if (!ok) break;
            tc_fence_after();
            const unsigned base = smem_u32(smem + s * STAGE);
            const unsigned long long db = operand_desc(base), da = operand_desc(base + A_AT), ds = scales_desc(base + AS_AT);
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k) {
              tc_copy_scales<PAIR>(elected, tmem + SH::SFA + 4 * k, ds + k * (512 >> 4));
#pragma unroll
              for (int i = 0; i < SH::B_TILES; ++i)
                tc_copy_scales<PAIR>(elected, tmem + SH::SFB + 4 * (SH::B_TILES * k + i), ds + (((1 + i) * SCALES + k * 512) >> 4));
            }
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k) {
              tc_mma<PAIR>(elected, tmem + buf * BN, da + k * (32 >> 4), db + k * (32 >> 4), idesc, tmem + SH::SFA + 4 * k,
                           sfb + 4 * SH::B_TILES * k, accum);
              accum = 1;
            }
            tc_commit<PAIR>(elected, &empty[s]);
            if (++s == STAGES) {
              s = 0;
              phase ^= 1;
            }
          }
          if (ok) tc_commit<PAIR>(elected, &acc_full[buf]);
        }
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ---- epilogue of this CTA's 128 token rows: warps 4-7 the first half of the columns, 8-11 the second
    pdl_wait();
    constexpr int COLS = BN / 2;
    const int quarter = warp & 3, col0 = ((warp - EPI_WARP0) >> 2) * COLS;
    const unsigned src = tmem + ((unsigned)(quarter * 32) << 16) + col0;
    const unsigned acc_empty0 = PAIR ? cluster_addr(smem_u32(acc_empty), 0) : smem_u32(acc_empty);
    unsigned char* staging = epi_stage + (warp - EPI_WARP0) * EPI_STAGE_BYTES;
    int local = 0, turn_buffer = 0;
    for (int t = group; t < tiles && ok; t += groups) {
      float acc[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
#pragma unroll 1
      for (int part = 0; part < a.k.parts; ++part, ++local) {
        const int buf = local & 1;
        ok = mbar_wait_brief(&acc_full[buf], (local >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);      // tcgen05.ld below is warp-wide
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < COLS; h += 32) {
          unsigned v[32];
          tc_ld32(src + buf * BN + h, v);
          tc_wait_ld(v);
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[h + j] += __uint_as_float(v[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty0 + buf * 8);
      }
      const int row0 = (t % a.m_tiles) * CTAS * BM + rank * BM + quarter * 32;
      if (ok && row0 < a.M) store_rows<OutT, COLS>(acc, &map_out, staging, turn_buffer, lane, row0, (t / a.m_tiles) * BN + col0, a);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  if (!ok) atomicExch(&dib_gemm_fp4_error_word, 1);
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();       // the other CTA's products and arrivals may still touch this one
  if (warp == 1) {
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)SH::TMEM));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)SH::TMEM));
  }
}

// ---------------------------------------------------------------- few rows
// Up to 128 tokens.  A cluster has a tile of 128 channels, its CTA number r the part r of k, whose sums lie in lanes (channels) x
// columns (tokens); then each CTA adds up all parts of some tokens' channels from the others' shared memory and writes them.
// Bound by memory: a CTA's ring is small enough that two or three share an SM (and its tensor memory), one of which streams
// weights while another begins or ends, or the next kernel's first weights arrive under this one's end.
// Roles: warp 0 copies channels, warp 2 tokens, warp 1 issues the products, warps 3-6 take the sums; all write.
constexpr int FEW_THREADS = 224, FEW_TOKENS = 128, SUM_ROW = 132 * 4;      // (16 bytes off: no two rows share banks)
struct FewArgs {
  Parts k;
  const float* ux;
  const float* uw;
  void* out;
  int M, N, num_kb;
  int cols, stages, tmem;      // tokens rounded up to 8, stages of the ring, columns of tensor memory
  int by_values;               // rows of the output do not lie on four values
};
__host__ __device__ __forceinline__ int few_stage(int cols) { return (128 + cols) * ROW_BYTES + 2 * SCALES; }
__device__ __forceinline__ float4 load_cluster(unsigned addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store4(float* to, const float (&y)[4]) { *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]); }
__device__ __forceinline__ void store4(__nv_bfloat16* to, const float (&y)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]), b = __floats2bfloat162_rn(y[2], y[3]);
  *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

template <typename OutT>
__global__ void __launch_bounds__(FEW_THREADS)
gemm_fp4_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                    const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws,
                    const __grid_constant__ FewArgs a) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long full[MAX_STAGES], empty[MAX_STAGES], acc_full;
  __shared__ unsigned tmem_slot;
  // (an offset, not a rounded address: what is known to be shared memory is read and written with 32-bit addresses)
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  // a stage: channels, scales of channels, of tokens, tokens
  constexpr int WS_AT = 128 * ROW_BYTES, XS_AT = WS_AT + SCALES, X_AT = XS_AT + SCALES;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_xs);
    prefetch_tensormap(&map_ws);
  }
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int parts = a.k.parts, rank = (int)cluster_rank(), tile = blockIdx.x / parts, n0 = tile * 128;
  const int kb0 = a.k.begin(rank), count = a.k.begin(rank + 1) - kb0;
  const int stage = few_stage(a.cols);
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((unsigned)a.tmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  pdl_trigger();      // (as in the kernel above)
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  bool ok = true;
  if (warp == 0 || warp == 2) {
    if (lane == 0) {
      const int bytes = warp == 0 ? 128 * ROW_BYTES + SCALES : a.cols * ROW_BYTES + SCALES;
      auto load = [&](int c, int s) {
        unsigned char* to = smem + s * stage;
        mbar_expect_tx(&full[s], bytes);
        if (warp == 0) {
          tma_load_2d<false>(to, &map_w, (kb0 + c) * ROW_BYTES, n0, smem_u32(&full[s]));
          tma_load_3d<false>(to + WS_AT, &map_ws, (kb0 + c) * 4, tile, smem_u32(&full[s]));
        } else {
          tma_load_2d<false>(to + X_AT, &map_x, (kb0 + c) * ROW_BYTES, 0, smem_u32(&full[s]));
          tma_load_3d<false>(to + XS_AT, &map_xs, (kb0 + c) * 4, 0, smem_u32(&full[s]));
        }
      };
      if (warp == 2) pdl_wait();      // (weights are constants: they do not wait for the kernel in front)
      int s = 0;
      unsigned phase = 1;             // (the ring's first round finds it empty)
      int c = 0;
      for (; c < count; ++c) {
        ok = c < a.stages || mbar_wait_brief(&empty[s], phase);
        if (!ok) break;
        load(c, s);
        if (++s == a.stages) {
          s = 0;
          phase ^= 1;
        }
      }
      if (!ok)      // (as in the kernel above)
        for (int i = c - a.stages; i < c; ++i) mbar_wait_brief(&full[i % a.stages], (i / a.stages) & 1);
    }
  } else if (warp == 1) {
    const unsigned elected = elect_one(), idesc = make_idesc(128, a.cols);
    const unsigned sfa = tmem + a.cols, sfb = sfa + 16;
    int s = 0;
    unsigned phase = 0;
    for (int c = 0; c < count; ++c) {
      ok = __all_sync(0xffffffffu, mbar_wait_brief(&full[s], phase));
      if (!ok) break;
      tc_fence_after();
      const unsigned base = smem_u32(smem) + s * stage;
      const unsigned long long da = operand_desc(base), db = operand_desc(base + X_AT), ds = scales_desc(base + WS_AT);
#pragma unroll
      for (int k = 0; k < BK / UMMA_K; ++k) {
        tc_copy_scales<false>(elected, sfa + 4 * k, ds + k * (512 >> 4));
        tc_copy_scales<false>(elected, sfb + 4 * k, ds + ((SCALES + k * 512) >> 4));
      }
#pragma unroll
      for (int k = 0; k < BK / UMMA_K; ++k)
        tc_mma<false>(elected, tmem, da + k * (32 >> 4), db + k * (32 >> 4), idesc, sfa + 4 * k, sfb + 4 * k, (c > 0 || k > 0) ? 1u : 0u);
      tc_commit<false>(elected, &empty[s]);
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (ok) tc_commit<false>(elected, &acc_full);
  } else {
    // ---- sums to shared memory, over the ring: all of its copies have been read
    ok = mbar_wait_brief(&acc_full, 0);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    if (ok) {
      const int quarter = warp & 3;
      float* to = reinterpret_cast<float*>(smem) + quarter * 32 + lane;
#pragma unroll 2
      for (int col = 0; col < a.cols; col += 8) {
        unsigned v[8];
        tc_ld8(tmem + ((unsigned)(quarter * 32) << 16) + col, v);
        tc_wait_ld(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) to[(col + j) * (SUM_ROW / 4)] = __uint_as_float(v[j]);
      }
    }
  }
  if (!ok) atomicExch(&dib_gemm_fp4_error_word, 1);
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  pdl_wait();
  // ---- four channels of a token a thread
  const unsigned base = smem_u32(smem);
  const int all = a.M * 32, each = (all + parts - 1) / parts, end = min(all, (rank + 1) * each);
  for (int e = rank * each + threadIdx.x; e < end; e += FEW_THREADS) {
    const int token = e >> 5, n = n0 + (e & 31) * 4;
    if (n >= a.N) continue;
    const unsigned at = base + token * SUM_ROW + (e & 31) * 16;
    float4 v[MAX_PARTS];
#pragma unroll
    for (int r = 0; r < MAX_PARTS; ++r)
      if (r < parts) v[r] = load_cluster(cluster_addr(at, r));
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < MAX_PARTS; ++r)
      if (r < parts) {
        sum.x += v[r].x; sum.y += v[r].y; sum.z += v[r].z; sum.w += v[r].w;
      }
    const float ux = a.ux[token], s4[4] = {sum.x, sum.y, sum.z, sum.w};
    const int left = a.N - n;
    OutT* out = reinterpret_cast<OutT*>(a.out) + (long long)token * a.N + n;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = j < left ? fp4_times_units(s4[j], ux, a.uw[n + j]) : 0.f;
    if (!a.by_values && left >= 4) {
      store4(out, y);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) Elem<OutT>::store(out + j, y[j]);
    }
  }
  cluster_sync_all();       // the others may still read this one's sums
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)a.tmem));
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
// A row-major matrix [rows, cols] of `type`, boxes of box_rows x box_cols; what lies outside reads as zero and is not written.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, int size, const void* ptr, long long rows, long long cols, int box_cols,
              int box_rows, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)cols * size};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool make_codes_map(CUtensorMap* map, const void* codes, long long rows, int bytes, int box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, rows, bytes, ROW_BYTES, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Tiles of scales, 512 bytes each; a box is the four of a stage along k, of `tiles` tiles of rows.
bool make_scales_map(CUtensorMap* map, const void* ptr, long long rows, int k_tiles, int tiles) {
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[3] = {128, (cuuint64_t)k_tiles, (cuuint64_t)((rows + 127) / 128)};
  const cuuint64_t strides[2] = {512, (cuuint64_t)k_tiles * 512};
  const cuuint32_t box[3] = {128, 4, (cuuint32_t)tiles}, estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  Launch(int grid, int threads, int smem, int cluster, cudaStream_t st) {
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = dib_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }
};

struct Operands {
  const void *x, *xs, *ux, *w, *ws, *uw;
  void* out;
  int M, N, K, sm_count;
};

template <typename OutT, int BN, bool PAIR> int launch_form(const Operands& o, cudaStream_t st) {
  using SH = Shape<BN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1;
  static_assert(SH::STAGES >= 3 && SH::COLUMNS <= SH::TMEM, "shared and tensor memory");
  const int row_bytes = (o.K + 31) / 32 * 16, k_tiles = fp4_k_tiles(o.K);
  const Parts k(k_tiles / 4);
  Args a = {k};
  a.ux = reinterpret_cast<const float*>(o.ux);
  a.uw = reinterpret_cast<const float*>(o.uw);
  a.out = o.out;
  a.M = o.M; a.N = o.N;
  a.num_kb = k_tiles / 4;
  a.m_tiles = (o.M + CTAS * BM - 1) / (CTAS * BM);
  a.n_tiles = (o.N + BN - 1) / BN;
  a.by_lines = ((long long)o.N * sizeof(OutT)) % 16 != 0 || reinterpret_cast<uintptr_t>(o.out) % 16 != 0;
  const long long tiles = (long long)a.m_tiles * a.n_tiles;
  // (loads are counted in 32 bits)
  if (o.sm_count < CTAS || tiles > (1ll << 24) || (tiles / (o.sm_count / CTAS) + 1) * a.num_kb > (1ll << 30)) return DIB_BAD_SIZE;
  CUtensorMap mx, mw, mxs, mws, mo;
  const CUtensorMapDataType type = sizeof(OutT) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  if (!make_codes_map(&mx, o.x, o.M, row_bytes, BM) || !make_codes_map(&mw, o.w, o.N, row_bytes, SH::B_ROWS) ||
      !make_scales_map(&mxs, o.xs, o.M, k_tiles, 1) || !make_scales_map(&mws, o.ws, o.N, k_tiles, SH::B_TILES))
    return DIB_LAUNCH_FAILED;
  if (a.by_lines) mo = mx;      // (not used)
  else if (!make_map(&mo, type, sizeof(OutT), o.out, o.M, o.N, 32, 32, sizeof(OutT) == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B))
    return DIB_LAUNCH_FAILED;
  auto kern = gemm_fp4_kernel<OutT, BN, PAIR>;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SH::SMEM) != cudaSuccess) return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  const int groups = (int)(tiles < o.sm_count / CTAS ? tiles : o.sm_count / CTAS);
  Launch launch(CTAS * groups, THREADS, SH::SMEM, CTAS, st);
  if (cudaLaunchKernelEx(&launch.cfg, kern, mx, mw, mxs, mws, mo, a) != cudaSuccess) return DIB_LAUNCH_FAILED;
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// CTAs that share an SM, by shared memory
int few_per_sm(int cols) { return cols <= 32 ? 3 : 2; }

template <typename OutT> int launch_few(const Operands& o, cudaStream_t st) {
  const int row_bytes = (o.K + 31) / 32 * 16, k_tiles = fp4_k_tiles(o.K);
  const Parts k(k_tiles / 4);
  FewArgs a = {k};
  a.ux = reinterpret_cast<const float*>(o.ux);
  a.uw = reinterpret_cast<const float*>(o.uw);
  a.out = o.out;
  a.M = o.M; a.N = o.N;
  a.num_kb = k_tiles / 4;
  a.cols = (o.M + 7) / 8 * 8;
  a.tmem = a.cols + 32 <= 64 ? 64 : a.cols + 32 <= 128 ? 128 : 256;
  a.by_values = o.N % 4 != 0 || reinterpret_cast<uintptr_t>(o.out) % (4 * sizeof(OutT)) != 0;
  const int stage = few_stage(a.cols), parts = k.parts, longest = k.each + (k.longer > 0);
  // (228 KB an SM, 1 KB of each block's own and 1 KB for its barriers)
  const int per_sm = few_per_sm(a.cols);
  a.stages = (228 * 1024 / per_sm - 3 * 1024) / stage;
  if (a.stages > longest) a.stages = longest;
  if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
  const int ring = a.stages * stage, sums = a.cols * SUM_ROW, smem = 1024 + (ring > sums ? ring : sums);
  const long long n_tiles = ((long long)o.N + 127) / 128;
  if (n_tiles * parts > 0x7fffffffll) return DIB_BAD_SIZE;
  CUtensorMap mx, mw, mxs, mws;
  if (!make_codes_map(&mx, o.x, o.M, row_bytes, a.cols) || !make_codes_map(&mw, o.w, o.N, row_bytes, 128) ||
      !make_scales_map(&mxs, o.xs, o.M, k_tiles, 1) || !make_scales_map(&mws, o.ws, o.N, k_tiles, 1))
    return DIB_LAUNCH_FAILED;
  auto kern = gemm_fp4_few_kernel<OutT>;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 116 * 1024) != cudaSuccess) return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  Launch launch((int)n_tiles * parts, FEW_THREADS, smem, parts, st);
  if (cudaLaunchKernelEx(&launch.cfg, kern, mx, mw, mxs, mws, a) != cudaSuccess) return DIB_LAUNCH_FAILED;
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// Form forced for measurements and tests (-1: the choice of `form`): 0, 1, 2 tiles of 128 x 64, 128 x 128, 128 x 192, 3 the pair, 4 (up
// to 128 rows) clusters that share k.
int& forced_form() {
  static int v = -1;
  return v;
}
// Of the forms the one whose time, in us, is estimated lowest, from lines through measured times (148 SMs, stages of 256 values):
//   tiles      each round of tiles takes its stages; 4,096 x 4,096, 256 rows: 128 x 64 9.1, 128 x 128 9.8, 128 x 192 12.0, pair 13.8;
//              2,048 rows: 34.4, 25.6, 24.9, 26.1; 24,576 x 4,096: 182, 120, 107, 101; 128 rows of it, bound by the weight: 18.2,
//              18.2, 17.3
//   clusters   8, 32, 64, 128 rows of 4,096 x 4,096 5.4, 6.4, 7.6, 10.3; of 4,096 x 12,288 8.2, 8.7, 10.4, 13.0; of 24,576 x 4,096
//              11.6, 13.2, 20.6, 25.8; of 1,024 x 1,024 3.8, 5.1, 6.9, 10.5 (128 x 64: 4.4, 4.5, 4.6, 4.8)
// (The form never changes a bit of the result.)
int form(int M, int N, int K, int sm_count) {
  if (forced_form() >= 0 && (forced_form() < 4 || M <= FEW_TOKENS)) return forced_form();
  const int num_kb = fp4_k_tiles(K) / 4;
  const float weight = 0.5625f * (float)N * (float)K;      // bytes
  float best = 1e30f;
  int choice = 0;
  auto consider = [&](int form, float us) {
    if (us < best) {
      best = us;
      choice = form;
    }
  };
  auto tiles = [&](int form, int bm, int bn, int ctas, float base, float stage) {
    const long long n = (long long)((M + bm - 1) / bm) * ((N + bn - 1) / bn), at_once = sm_count / ctas;
    const float run = stage * (float)((n + at_once - 1) / at_once) * (float)num_kb, read = weight / 4.6e6f;
    const float busy = (float)(n < at_once ? n : at_once) / (float)at_once;
    consider(form, base + 1.2f * busy + (run > read ? run : read));
  };
  tiles(0, BM, 64, 1, 2.8f, 0.28f);
  tiles(1, BM, 128, 1, 3.4f, 0.325f);
  tiles(2, BM, 192, 1, 4.f, 0.445f);
  if (M > BM && sm_count >= 2) tiles(3, 2 * BM, 192, 2, 7.f, 0.4f);
  if (M <= FEW_TOKENS) {
    const Parts k(num_kb);
    const int cols = (M + 7) / 8 * 8;
    const float at_once = (float)(sm_count * few_per_sm(cols)), n = (float)((N + 127) / 128) * (float)k.parts;
    consider(4, (2.9f + 0.2f * (float)(k.each + (k.longer > 0)) + weight / 7.9e6f) * (n > at_once ? n / at_once : 1.f) +
                    (float)(cols - 8) * (0.02f + 0.036f / (float)k.parts));
  }
  return choice;
}

template <typename OutT> int launch(const Operands& o, cudaStream_t st) {
  switch (form(o.M, o.N, o.K, o.sm_count)) {
    case 0: return launch_form<OutT, 64, false>(o, st);
    case 1: return launch_form<OutT, 128, false>(o, st);
    case 2: return launch_form<OutT, 192, false>(o, st);
    case 4: return launch_few<OutT>(o, st);
    default: return launch_form<OutT, 192, true>(o, st);
  }
}

}  // namespace

extern "C" {

int dib_gemm_fp4_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dib_gemm_fp4_error_word, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int dib_gemm_fp4_status_clear() {
  const int v = 0;
  return cudaMemcpyToSymbol(dib_gemm_fp4_error_word, &v, sizeof(int)) == cudaSuccess ? 0 : -1;
}
void dib_gemm_fp4_force_form(int form) { forced_form() = form; }

// out[M, N] (out_dtype 0 float32, 1 bfloat16) = x w^T; x, w: codes [rows, Kp / 2], Kp = K rounded up to 32, xs, ws their block scales
// in tiles, ux, uw float32 [rows].
int dib_gemm_fp4(const void* x, const void* xs, const void* ux, const void* w, const void* ws, const void* uw, void* out, int M, int N,
                 int K, int out_dtype, int sm_count, cudaStream_t st) {
  if (out_dtype != 0 && out_dtype != 1) return DIB_BAD_DTYPE;
  if (M < 0 || N < 0 || K < 1 || K > (1 << 24) || sm_count < 1) return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(xs) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(ws) |
        reinterpret_cast<uintptr_t>(uw)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (M == 0 || N == 0) return DIB_OK;
  // (rows of the scales' map)
  if ((long long)((M > N ? M : N) / 128 + 2) * fp4_k_tiles(K) > 0x7fffffffll) return DIB_BAD_SIZE;
  const Operands o = {x, xs, ux, w, ws, uw, out, M, N, K, sm_count};
  if (out_dtype == 1) return launch<__nv_bfloat16>(o, st);
  return launch<float>(o, st);
}

// The same with x [M, K] of values (x_dtype 0 float32, 1 bfloat16; rows `stride` values apart), which `quantize`
// (dib_fp4_quantize_rows of the rows' library) first turns into tiles of scales, codes and units in `work`, one behind the other.
int dib_fp4_linear(int (*quantize)(const void*, long long, void*, void*, void*, long long, int, int, int, cudaStream_t),
                   const void* x, long long stride, int x_dtype, int K, void* work, const void* w, const void* ws, const void* uw,
                   void* out, int M, int N, int out_dtype, int sm_count, cudaStream_t st) {
  if (M < 0 || K < 1) return DIB_BAD_SIZE;
  char* codes = reinterpret_cast<char*>(work) + (long long)(M + 127) / 128 * fp4_k_tiles(K) * 512;
  char* units = codes + (long long)M * ((K + 31) / 32 * 16);
  const int rc = quantize(x, stride, codes, work, units, M, K, x_dtype, sm_count, st);
  if (rc != DIB_OK) return rc;
  return dib_gemm_fp4(codes, work, units, w, ws, uw, out, M, N, K, out_dtype, sm_count, st);
}

}  // extern "C"
