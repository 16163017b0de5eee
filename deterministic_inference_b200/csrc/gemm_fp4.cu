// Matrix product of rows in 4-bit floating point (fp4.cuh): y[m, n] = ux[m] * uw[n] * sum_k (cx bx)[m, k] * (cw bw)[n, k], c the
// e2m1 codes, b the e4m3 scales of blocks of 16 values, u = 2^E of the row.  Codes and block scales enter the tensor cores as
// they are (tcgen05.mma kind::mxf4nvf4, a scale for each 16 values of either operand, 64 values an instruction, sums in
// float32); the rows' powers of two are exact and join the sum in the epilogue, which rounds once.
//
// Every form adds a row's k up in one order, 64 values at a time from the first to the last, in one accumulator: a row's bits
// depend on the row and the weight alone, not on the other rows, the tile or the form.  So k is never shared among CTAs.
//
// Operands by TMA, 256 values (128 bytes, 128-byte swizzle) of each row a stage, with the block scales in tiles of 128 rows
// x 64 values (512 bytes, rows_fp4.cu), through a ring of mbarrier-guarded stages.  The products' warp copies a stage's scales
// from shared into tensor memory (tcgen05.cp, in order with the products, so that one buffer does); the accumulator lies twice
// in tensor memory, so that a tile's epilogue runs under the products of the next.  Roles: warp 0 copies, warp 1 issues the
// products, warps 4-11 are the epilogue.  One CTA an SM on tiles of 128 tokens x BN channels (fewer tokens are fetched where there
// are fewer), or a pair of CTAs (cta_group::2) on tiles of 256 x 192, each of which fetches its own tokens and half of the
// channels.
#include <cuda.h>

#include "fp4.cuh"

namespace {

constexpr int BM = 128, BK = 256, ROW_BYTES = BK / 2, UMMA_K = 64;      // tokens of a tile and CTA, values of a stage, of an instruction
constexpr int THREADS = 384, EPI_WARP0 = 4, EPI_WARPS = 8, MAX_STAGES = 16;
constexpr int SCALES_A = 2048;                          // a stage's block scales of 128 rows: four tiles along k
constexpr int EPI_STAGE_BYTES = 32 * 128;               // a warp's 32 rows of 128 bytes
constexpr int SMEM_MOST = 232448 - 1024;                // (1 KB left to static shared memory)
__device__ int dib_gemm_fp4_error_word = 0;

// A CTA's share of a tile: rows of channels that it fetches, tiles of channels' scales (64-channel tiles that begin in the middle of a
// tile of 128 scales among them), columns of tensor memory.
template <int BN, bool PAIR> struct Shape {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int B_TILES = BN == 192 ? 2 : 1;
  static constexpr int SCALES = SCALES_A + B_TILES * 2048;
  static constexpr int FIXED = B_ROWS * ROW_BYTES + SCALES;             // of a stage, before its tokens
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
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
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
constexpr unsigned make_idesc(int m, int n) {
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

struct Args {
  const float* ux;      // [M]
  const float* uw;      // [N]
  void* out;            // [M, N]
  int M, N, num_kb, m_tiles, n_tiles;
  int a_rows, stages;   // token rows that a CTA fetches, stages of the ring
  int by_lines;         // rows of the output do not lie on 16 bytes: no TMA stores
};

// A warp's 32 token rows from row0 on and COLS columns from n0 + col0 on, in blocks of 128 bytes a row: a lane turns its row's
// sums into the output's type, stages them (swizzled) and the copy engine writes whole rows, clipped at M and N.
template <typename OutT, int COLS>
__device__ __forceinline__ void store_rows(unsigned src, const CUtensorMap* map_out, unsigned char* stage, int lane, int row0,
                                           int n0, int col0, const Args& a) {
  constexpr int PER_BLOCK = 128 / (int)sizeof(OutT);
  const float ux = row0 + lane < a.M ? a.ux[row0 + lane] : 0.f;
#pragma unroll 1
  for (int col = col0; col < col0 + COLS; col += PER_BLOCK) {
    if (n0 + col >= a.N) return;
    // the store before this one must have read the staging block
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int h = 0; h < PER_BLOCK; h += 32) {
      unsigned v[32];
      tc_ld32(src + col + h, v);
      const float* uw = a.uw + n0 + col + h;
      float4 w[8];
      if (n0 + col + h + 32 <= a.N) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const float4*>(uw + 4 * j);
      } else {
        const int left = a.N - (n0 + col + h);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[j] = make_float4(4 * j < left ? uw[4 * j] : 0.f, 4 * j + 1 < left ? uw[4 * j + 1] : 0.f,
                             4 * j + 2 < left ? uw[4 * j + 2] : 0.f, 4 * j + 3 < left ? uw[4 * j + 3] : 0.f);
      }
      tc_wait_ld();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y0 = __uint_as_float(v[4 * j]) * ux * w[j].x, y1 = __uint_as_float(v[4 * j + 1]) * ux * w[j].y;
        const float y2 = __uint_as_float(v[4 * j + 2]) * ux * w[j].z, y3 = __uint_as_float(v[4 * j + 3]) * ux * w[j].w;
        if (sizeof(OutT) == 2) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(y0, y1), hi = __floats2bfloat162_rn(y2, y3);
          v[2 * j] = *reinterpret_cast<const unsigned*>(&lo);
          v[2 * j + 1] = *reinterpret_cast<const unsigned*>(&hi);
        } else {
          v[4 * j] = __float_as_uint(y0); v[4 * j + 1] = __float_as_uint(y1);
          v[4 * j + 2] = __float_as_uint(y2); v[4 * j + 3] = __float_as_uint(y3);
        }
      }
#pragma unroll
      for (int c = 0; c < (int)sizeof(OutT) * 2; ++c)
        *reinterpret_cast<uint4*>(stage + lane * 128 + (((h * (int)sizeof(OutT) / 16 + c) ^ (lane & 7)) << 4)) =
            make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    }
    if (!a.by_lines) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tma_store_2d(map_out, stage, n0 + col, row0);
    } else {
      __syncwarp();
      OutT* out = reinterpret_cast<OutT*>(a.out);
      for (int r = 0; r < 32 && row0 + r < a.M; ++r)
#pragma unroll
        for (int e = lane; e < PER_BLOCK; e += 32)
          if (n0 + col + e < a.N) {
            const int byte = e * (int)sizeof(OutT);
            out[(long long)(row0 + r) * a.N + n0 + col + e] =
                *reinterpret_cast<const OutT*>(stage + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15));
          }
      __syncwarp();
    }
  }
}

// PAIR: two CTAs on a tile of 256 tokens x BN channels; `full` of the first CTA counts both CTAs' copies, its commits
// signal `empty` and `acc_full` in both, `acc_empty` of the first takes an arrival of every epilogue warp of both.
template <typename OutT, int BN, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws,
                const __grid_constant__ CUtensorMap map_out, const __grid_constant__ Args a) {
  using SH = Shape<BN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1, B_ROWS = SH::B_ROWS;
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long full[MAX_STAGES], empty[MAX_STAGES];
  __shared__ unsigned long long acc_full[2], acc_empty[2];      // a tile's accumulator is complete; the epilogue has read it
  __shared__ unsigned tmem_slot;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  // A stage: channels, scales of tokens and of channels, tokens.  The products read 128 token rows whatever was fetched: those
  // behind the last stage's lie in the epilogue's memory; what they make of them is never read.
  const int stage_bytes = SH::FIXED + a.a_rows * ROW_BYTES, stages = a.stages;
  unsigned char* epi_stage = smem + stages * stage_bytes;
  if (!PAIR) pdl_trigger();
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
  const int tiles = a.m_tiles * a.n_tiles, k_tiles = a.num_kb * 4;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
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
  if (PAIR) cluster_sync_all();       // both CTAs' barriers and tensor memory exist before either is used
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      // ---- copies.  The ring runs on across the tiles: load number c is k-block c % num_kb of this CTA's tile number
      // c / num_kb.  Tiles in the order of their channels, so that the CTAs side by side share them.
      const int my_tiles = tiles > group ? (tiles - group + groups - 1) / groups : 0;
      const int total = my_tiles * a.num_kb;
      const unsigned full0 = PAIR ? cluster_addr(smem_u32(full), 0) : smem_u32(full);
      auto load_w = [&](int c, int s, int t, int kb) {
        const int n0 = (t / a.m_tiles) * BN;
        unsigned char* b = smem + s * stage_bytes;
        tma_load_2d<PAIR>(b, &map_w, kb * ROW_BYTES, n0 + rank * B_ROWS, full0 + s * 8);
        // (a tile of scales behind the last reads as zeros)
#pragma unroll
        for (int i = 0; i < SH::B_TILES; ++i)
          tma_load_2d<PAIR>(b + B_ROWS * ROW_BYTES + SCALES_A + i * 2048, &map_ws, 0, (n0 / 128 + i) * k_tiles + kb * 4, full0 + s * 8);
      };
      auto load_x = [&](int c, int s, int t, int kb) {
        const int m0 = (t % a.m_tiles) * CTAS * BM + rank * BM;
        unsigned char* b = smem + s * stage_bytes;
        tma_load_2d<PAIR>(b + B_ROWS * ROW_BYTES, &map_xs, 0, m0 / 128 * k_tiles + kb * 4, full0 + s * 8);
        tma_load_2d<PAIR>(b + SH::FIXED, &map_x, kb * ROW_BYTES, m0, full0 + s * 8);
      };
      const int pre = total < stages ? total : stages;
      for (int c = 0; c < pre; ++c) {      // weights are constants: the first stages' go out before the wait
        if (rank == 0) mbar_expect_tx(&full[c], CTAS * stage_bytes);
        load_w(c, c, group + (c / a.num_kb) * groups, c % a.num_kb);
      }
      pdl_wait();
      for (int c = 0; c < pre; ++c) load_x(c, c, group + (c / a.num_kb) * groups, c % a.num_kb);
      int c = pre, s = pre == stages ? 0 : pre, t = group + (pre / a.num_kb) * groups, kb = pre % a.num_kb;
      unsigned phase = 0;
      for (; c < total; ++c) {
        ok = mbar_wait_brief(&empty[s], phase);
        if (!ok) break;
        if (rank == 0) mbar_expect_tx(&full[s], CTAS * stage_bytes);
        load_w(c, s, t, kb);
        load_x(c, s, t, kb);
        if (++s == stages) {
          s = 0;
          phase ^= 1;
        }
        if (++kb == a.num_kb) {
          kb = 0;
          t += groups;
        }
      }
      // given up: what was sent for arrives before this memory is another's (the pair's second CTA stays until the first, whose
      // barriers count for both, has waited)
      if (!ok && rank == 0)
        for (int i = c - stages; i < c; ++i) mbar_wait_brief(&full[i % stages], (i / stages) & 1);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---- products
      const unsigned elected = elect_one();
      constexpr unsigned idesc = make_idesc(CTAS * BM, BN);
      int local = 0, s = 0;
      unsigned phase = 0;
      for (int t = group; t < tiles && ok; t += groups, ++local) {
        const int buf = local & 1;
        // (channels that begin in the middle of a tile of scales: its last two columns are theirs)
        const unsigned sfb = tmem + SH::SFB + (BN % 128 != 0 ? ((t / a.m_tiles) * (BN / 64) & 1) * 2 : 0);
        if (local >= 2) {      // the epilogue must have read this buffer's earlier tile
          ok = __all_sync(0xffffffffu, mbar_wait_brief(&acc_empty[buf], ((local >> 1) - 1) & 1));
          if (!ok) break;
          tc_fence_after();
        }
        for (int kb = 0; kb < a.num_kb; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait_brief(&full[s], phase));
          if (!ok) break;
          tc_fence_after();
          const unsigned base = smem_u32(smem + s * stage_bytes);
          const unsigned long long db = operand_desc(base), da = operand_desc(base + SH::FIXED);
          const unsigned long long ds = scales_desc(base + B_ROWS * ROW_BYTES);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            tc_copy_scales<PAIR>(elected, tmem + SH::SFA + 4 * k, ds + k * (512 >> 4));
#pragma unroll
            for (int i = 0; i < SH::B_TILES; ++i)
              tc_copy_scales<PAIR>(elected, tmem + SH::SFB + 4 * (SH::B_TILES * k + i), ds + ((SCALES_A + i * 2048 + k * 512) >> 4));
          }
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            tc_mma<PAIR>(elected, tmem + buf * BN, da + k * (32 >> 4), db + k * (32 >> 4), idesc, tmem + SH::SFA + 4 * k,
                         sfb + 4 * SH::B_TILES * k, (kb > 0 || k > 0) ? 1u : 0u);
          tc_commit<PAIR>(elected, &empty[s]);
          if (++s == stages) {
            s = 0;
            phase ^= 1;
          }
        }
        if (ok) tc_commit<PAIR>(elected, &acc_full[buf]);
      }
    }
  } else if (warp >= EPI_WARP0) {
    // ---- epilogue of this CTA's 128 token rows: warps 4-7 the first half of the columns, 8-11 the second
    pdl_wait();
    const int quarter = warp & 3, half = (warp - EPI_WARP0) >> 2;
    const unsigned lane_base = (unsigned)(quarter * 32) << 16;
    const unsigned acc_empty0 = PAIR ? cluster_addr(smem_u32(acc_empty), 0) : smem_u32(acc_empty);
    int local = 0;
    for (int t = group; t < tiles; t += groups, ++local) {
      const int buf = local & 1;
      bool got = ok && mbar_wait_brief(&acc_full[buf], (local >> 1) & 1);
      got = __all_sync(0xffffffffu, got);      // tcgen05.ld below is warp-wide
      if (!got) {
        ok = false;
        break;
      }
      tc_fence_after();
      // (in whole blocks of 128 bytes; bfloat16 tiles of 64 or 192 channels are one and three: the first half has the odd one)
      constexpr int BLOCK = 128 / (int)sizeof(OutT), BLOCKS = BN / BLOCK, FIRST = (BLOCKS + 1) / 2 * BLOCK;
      const int row0 = (t % a.m_tiles) * CTAS * BM + rank * BM + quarter * 32, n0 = (t / a.m_tiles) * BN;
      const unsigned src = tmem + buf * BN + lane_base;
      unsigned char* staging = epi_stage + (warp - EPI_WARP0) * EPI_STAGE_BYTES;
      if (row0 < a.M) {
        if (half == 0) store_rows<OutT, FIRST>(src, &map_out, staging, lane, row0, n0, 0, a);
        else if (BN > FIRST) store_rows<OutT, BN - FIRST>(src, &map_out, staging, lane, row0, n0, FIRST, a);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + buf * 8);
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
// tiles of scales, 512 bytes a row; a box is the four of a stage
bool make_scales_map(CUtensorMap* map, const void* tiles, long long rows, int k_tiles) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, tiles, (rows + 127) / 128 * k_tiles, 128, 128, 4, CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct Operands {
  const void *x, *xs, *ux, *w, *ws, *uw;
  void* out;
  int M, N, K, sm_count;
};

// token rows that a CTA of the single form fetches
int fetched_rows(int M) { return M <= 8 ? 8 : M <= 32 ? 32 : M <= 64 ? 64 : BM; }

template <typename OutT, int BN, bool PAIR> int launch_form(const Operands& o, cudaStream_t st) {
  using SH = Shape<BN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1;
  const int row_bytes = (o.K + 31) / 32 * 16, k_tiles = fp4_k_tiles(o.K);
  Args a;
  a.ux = reinterpret_cast<const float*>(o.ux);
  a.uw = reinterpret_cast<const float*>(o.uw);
  a.out = o.out;
  a.M = o.M; a.N = o.N;
  a.num_kb = k_tiles / 4;
  a.m_tiles = (o.M + CTAS * BM - 1) / (CTAS * BM);
  a.n_tiles = (o.N + BN - 1) / BN;
  a.by_lines = ((long long)o.N * sizeof(OutT)) % 16 != 0 || reinterpret_cast<uintptr_t>(o.out) % 16 != 0;
  a.a_rows = PAIR ? BM : fetched_rows(o.M);
  const int stage = SH::FIXED + a.a_rows * ROW_BYTES, epilogue = EPI_WARPS * EPI_STAGE_BYTES;
  a.stages = (SMEM_MOST - 1024 - epilogue) / stage;
  if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
  const size_t smem = 1024 + (size_t)a.stages * stage + epilogue;
  static_assert(EPI_WARPS * EPI_STAGE_BYTES >= (BM - 8) * ROW_BYTES, "token rows behind the last stage's");
  static_assert((SMEM_MOST - 1024 - EPI_WARPS * EPI_STAGE_BYTES) / (SH::FIXED + BM * ROW_BYTES) >= 3, "stages");
  static_assert(SH::COLUMNS <= SH::TMEM, "tensor memory");
  const long long tiles = (long long)a.m_tiles * a.n_tiles;
  // (loads are counted in 32 bits)
  if (o.sm_count < CTAS || tiles > (1ll << 24) || (tiles / (o.sm_count / CTAS) + 1) * a.num_kb > (1ll << 30)) return DIB_BAD_SIZE;
  CUtensorMap mx, mw, mxs, mws, mo;
  const CUtensorMapDataType type = sizeof(OutT) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  if (!make_codes_map(&mx, o.x, o.M, row_bytes, a.a_rows) || !make_codes_map(&mw, o.w, o.N, row_bytes, SH::B_ROWS) ||
      !make_scales_map(&mxs, o.xs, o.M, k_tiles) || !make_scales_map(&mws, o.ws, o.N, k_tiles))
    return DIB_LAUNCH_FAILED;
  if (a.by_lines) mo = mx;      // (not used)
  else if (!make_map(&mo, type, sizeof(OutT), o.out, o.M, o.N, 128 / (int)sizeof(OutT), 32, CU_TENSOR_MAP_SWIZZLE_128B))
    return DIB_LAUNCH_FAILED;
  auto kern = gemm_fp4_kernel<OutT, BN, PAIR>;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST) != cudaSuccess) return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  const int groups = (int)(tiles < o.sm_count / CTAS ? tiles : o.sm_count / CTAS);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CTAS * groups);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = dib_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, mx, mw, mxs, mws, mo, a) != cudaSuccess) return DIB_LAUNCH_FAILED;
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// Form forced for measurements and tests (-1: the choice of `form`): 0, 1, 2 tiles of 128 x 64, 128 x 128, 128 x 192, 3 the pair.
int& forced_form() {
  static int v = -1;
  return v;
}
// The form in which the busiest SM fetches the fewest bytes: rounds of tiles times the bytes of a stage.  (The form never changes a
// bit of the result.)
int form(int M, int N, int sm_count) {
  if (forced_form() >= 0) return forced_form();
  long long best = 1ll << 62;
  int choice = 0;
  auto consider = [&](int form, int bm, int bn, int ctas, int bytes) {
    const long long tiles = (long long)((M + bm - 1) / bm) * ((N + bn - 1) / bn), at_once = sm_count / ctas;
    const long long cost = (tiles + at_once - 1) / at_once * bytes;
    if (cost <= best) {
      best = cost;
      choice = form;
    }
  };
  const int tokens = fetched_rows(M) * ROW_BYTES;
  consider(0, BM, 64, 1, Shape<64, false>::FIXED + tokens);
  consider(1, BM, 128, 1, Shape<128, false>::FIXED + tokens);
  consider(2, BM, 192, 1, Shape<192, false>::FIXED + tokens);
  if (M > BM && sm_count >= 2) consider(3, 2 * BM, 192, 2, Shape<192, true>::FIXED + BM * ROW_BYTES);
  return choice;
}

template <typename OutT> int launch(const Operands& o, cudaStream_t st) {
  switch (form(o.M, o.N, o.sm_count)) {
    case 0: return launch_form<OutT, 64, false>(o, st);
    case 1: return launch_form<OutT, 128, false>(o, st);
    case 2: return launch_form<OutT, 192, false>(o, st);
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
int dib_fp4_linear(int (*quantize)(const void*, long long, void*, void*, void*, long long, int, int, cudaStream_t), const void* x,
                   long long stride, int x_dtype, int K, void* work, const void* w, const void* ws, const void* uw, void* out, int M,
                   int N, int out_dtype, int sm_count, cudaStream_t st) {
  if (M < 0 || K < 1) return DIB_BAD_SIZE;
  char* codes = reinterpret_cast<char*>(work) + (long long)(M + 127) / 128 * fp4_k_tiles(K) * 512;
  char* units = codes + (long long)M * ((K + 31) / 32 * 16);
  const int rc = quantize(x, stride, codes, work, units, M, K, x_dtype, st);
  if (rc != DIB_OK) return rc;
  return dib_gemm_fp4(codes, work, units, w, ws, uw, out, M, N, K, out_dtype, sm_count, st);
}

}  // extern "C"
