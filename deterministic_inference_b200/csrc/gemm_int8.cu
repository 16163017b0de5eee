// Matrix product in 8-bit integers: y[m, n] = sx[m] * sw[n] * sum_k x[m, k] * w[n, k], x and w int8 (K-major, rows of Kp
// bytes, a multiple of 16), the sum an exact 32-bit integer for K up to 133,144 (127^2 K < 2^31).  Because it is exact,
// the order in which it is added up (warps, runs of k, tile shapes) never changes a bit of the result: a row's bits
// depend on the row and the weight alone.
//
// Few rows: the weight is streamed once from memory straight into the registers of mma.sync (m16n8k32: 16 output
// channels x 8 tokens), with no shared memory in between.  The product's k index may be permuted as long as both
// operands agree, so a thread takes 32 consecutive bytes of its two weight rows (two 16-byte loads each) and calls them
// the k it needs; the tokens' rows are read the same way, from L2.  A block of eight warps takes 16 channels; the warps
// share the row's k among them and add their integers up in shared memory.  Bound by memory: 8 tokens on 24,576 x 4,096
// 19 us (5.3 TB/s), on 4,096 x 4,096 5.8 us, where the launch and a few trips to memory are most of it (with two to four steps
// of the weight on their way instead of one no faster, and 21 to 23 us for the former, for want of warps).
//
// Some rows, or few against long channels: clusters of up to eight CTAs share a tile's k (gemm_split_kernel), so that all SMs
// fetch a weight whose tiles are fewer than they are: 32 tokens on 4,096 x 12,288 13.8 us (3.7 TB/s; 19.6 us streamed, 32 on a
// CTA a tile).
//
// Many rows: persistent kernels on the 5th-generation tensor cores (tcgen05.mma kind::i8), one CTA an SM on tiles of 128
// tokens x BNL channels, or a pair of CTAs (cta_group::2) on tiles of 256 x 256: each then fetches its own 128 token rows
// and half of the channels, a third less for the same products, and the rate at which L2 feeds the SMs bounds them: 2,048
// tokens on 24,576 x 4,096 134 us with their quantising, 3.1 Pop/s (142 us with longer waits: their instructions cost the
// epilogue its own).
// Operands by TMA (128 k a stage: rows of 128 bytes, 128-byte swizzle) through a ring of mbarrier-guarded stages, the
// accumulator twice in tensor memory, so that a tile's epilogue (integers to float32, the two scales, one rounding) runs
// under the products of the next.  Roles: warp 0 copies, warp 1 issues the products, warps 4-11 are the epilogue.
#include <cuda.h>

#include <atomic>

#include "common.cuh"

namespace {

constexpr int FEW_WARPS = 8, FEW_ROWS = 16, CHUNK = 128;     // a warp's step: 16 channels x 128 k

__device__ __forceinline__ uint4 load_stream(const signed char* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_s8(int (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                       unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A thread's 32 bytes of a row at k, zeros behind the row's end (Kp is a multiple of 16).
template <bool STREAM> __device__ __forceinline__ void load32(const signed char* row, bool in, int k, int Kp, uint4 (&v)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (in && k + 16 * i < Kp)
      v[i] = STREAM ? load_stream(row + k + 16 * i) : *reinterpret_cast<const uint4*>(row + k + 16 * i);
  }
}

// The same for rows that lie on 32 bytes (WIDE): one load, so that no sector is asked for twice.
template <bool STREAM, bool WIDE>
__device__ __forceinline__ void load_row(const signed char* row, bool in, int k, int Kp, uint4 (&v)[2]) {
  if (!WIDE) {
    load32<STREAM>(row, in, k, Kp, v);
    return;
  }
  v[0] = v[1] = make_uint4(0, 0, 0, 0);
  if (!in || k >= Kp) return;
  if (STREAM)
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w)
                 : "l"(row + k));
  else
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w)
                 : "l"(row + k));
}

// NT tiles of 8 tokens.  (Three blocks an SM with two tiles and more: 16 tokens on 6,144 x 4,096 7.1 us, with two 9.1.)
template <typename OutT, int NT, bool WIDE>
__global__ void __launch_bounds__(FEW_WARPS * 32, NT == 1 ? 4 : 3)
gemm_few_kernel(const signed char* __restrict__ x, const float* __restrict__ sx, const signed char* __restrict__ w,
                const float* __restrict__ sw, OutT* __restrict__ out, int M, int N, int Kp) {
  pdl_trigger();
  __shared__ int sums[FEW_WARPS][NT * 8][FEW_ROWS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * FEW_ROWS, m0 = blockIdx.y * (NT * 8);
  const signed char* w0 = w + (long long)(n0 + g) * Kp;
  const signed char* w1 = w0 + 8ll * Kp;
  const bool in0 = n0 + g < N, in1 = n0 + g + 8 < N;
  int acc[NT][4] = {};
  int k = warp * CHUNK + t * 32;
  uint4 a[2], b[2];
  // the weights are constants: the first step's are on their way before the wait for the kernel in front
  load_row<true, WIDE>(w0, in0, k, Kp, a);
  load_row<true, WIDE>(w1, in1, k, Kp, b);
  pdl_wait(x, sx);
  // (the tokens a step ahead too, where there are tiles enough for it to show: 16 of them on 4,096 x 4,096 6.7 -> 6.2 us, but 8
  // on 24,576 x 4,096 19.4 -> 19.9)
  constexpr bool AHEAD = NT > 1;
  uint4 c[NT][2];
  auto load_tokens = [&](int nt, int at) {
    load_row<false, WIDE>(x + (long long)(m0 + nt * 8 + g) * Kp, m0 + nt * 8 + g < M, at, Kp, c[nt]);
  };
  if (AHEAD)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) load_tokens(nt, k);
  for (; k - t * 32 < Kp; k += FEW_WARPS * CHUNK) {
    const uint4 ca[2] = {a[0], a[1]}, cb[2] = {b[0], b[1]};
    load_row<true, WIDE>(w0, in0, k + FEW_WARPS * CHUNK, Kp, a);
    load_row<true, WIDE>(w1, in1, k + FEW_WARPS * CHUNK, Kp, b);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (!AHEAD) load_tokens(nt, k);
      const uint4 cc[2] = {c[nt][0], c[nt][1]};
      if (AHEAD) load_tokens(nt, k + FEW_WARPS * CHUNK);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma_s8(acc[nt], ca[i].x, cb[i].x, ca[i].y, cb[i].y, cc[i].x, cc[i].y);
        mma_s8(acc[nt], ca[i].z, cb[i].z, ca[i].w, cb[i].w, cc[i].z, cc[i].w);
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    sums[warp][nt * 8 + 2 * t][g] = acc[nt][0];
    sums[warp][nt * 8 + 2 * t + 1][g] = acc[nt][1];
    sums[warp][nt * 8 + 2 * t][g + 8] = acc[nt][2];
    sums[warp][nt * 8 + 2 * t + 1][g + 8] = acc[nt][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 8 * FEW_ROWS; i += FEW_WARPS * 32) {
    const int m = i / FEW_ROWS, n = i % FEW_ROWS;
    if (m0 + m < M && n0 + n < N) {
      int s = 0;
#pragma unroll
      for (int v = 0; v < FEW_WARPS; ++v) s += sums[v][m][n];
      Elem<OutT>::store(out + (long long)(m0 + m) * N + n0 + n, (float)s * sx[m0 + m] * sw[n0 + n]);
    }
  }
}

template <typename OutT>
int launch_few(const void* x, const void* sx, const void* w, const void* sw, void* out, int M, int N, int Kp, cudaStream_t st) {
  const int nt = M <= 8 ? 1 : M <= 16 ? 2 : 4;
  const dim3 grid((N + FEW_ROWS - 1) / FEW_ROWS, (M + nt * 8 - 1) / (nt * 8));
  if (grid.y > 65535) return DIB_BAD_SIZE;
  auto kern = nt == 1 ? gemm_few_kernel<OutT, 1, false> : nt == 2 ? gemm_few_kernel<OutT, 2, false> : gemm_few_kernel<OutT, 4, false>;
  if (Kp % 32 == 0 && (reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(x)) % 32 == 0)
    kern = nt == 1 ? gemm_few_kernel<OutT, 1, true> : nt == 2 ? gemm_few_kernel<OutT, 2, true> : gemm_few_kernel<OutT, 4, true>;
  dib_launch(kern, grid, dim3(FEW_WARPS * 32), 0, st, reinterpret_cast<const signed char*>(x),
             reinterpret_cast<const float*>(sx), reinterpret_cast<const signed char*>(w),
             reinterpret_cast<const float*>(sw), reinterpret_cast<OutT*>(out), M, N, Kp);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// ---------------------------------------------------------------- many rows
constexpr int BM = 128, BK = 128, UMMA_K = 32;      // tokens of a tile and CTA, k of a stage, k of an instruction
constexpr int A_BYTES = BM * BK, THREADS = 384, EPI_WARP0 = 4, EPI_WARPS = 8;
constexpr int EPI_STAGE_BYTES = 32 * 128;           // a warp's 32 rows of 128 bytes
__device__ int dib_gemm_int8_error_word = 0;

template <int B_ROWS> struct Ring {                 // channels that a CTA fetches a stage
  static constexpr int STAGE = A_BYTES + B_ROWS * BK;
  static constexpr int STAGES = B_ROWS == 256 ? 4 : B_ROWS == 128 ? 6 : 8;
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + EPI_WARPS * EPI_STAGE_BYTES + (2 * STAGES + 4) * 8 + 16 + 1024;
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
template <bool PAIR>
__device__ __forceinline__ void tc_mma(unsigned elected, unsigned tmem_d, unsigned long long desc_a, unsigned long long desc_b,
                                       unsigned idesc, unsigned accum) {
  if (PAIR)
    asm volatile(
        "{\n\t"
        ".reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accum), "r"(elected)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accum), "r"(elected)
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
__device__ __forceinline__ unsigned long long smem_desc(unsigned addr) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((unsigned long long)(1024u >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// kind::i8: 32-bit integer accumulator, signed bytes, both K-major
constexpr unsigned make_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
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

__device__ __forceinline__ int cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ void store_as(float& to, float x) { to = x; }
__device__ __forceinline__ void store_as(__nv_bfloat16& to, float x) { to = __float2bfloat16_rn(x); }

struct LargeArgs {
  const float* sx;      // [M]
  const float* sw;      // [N]
  void* out;            // [M, N]
  int M, N, num_kb, m_tiles, n_tiles;
  int by_lines;         // rows of the output do not lie on 16 bytes: no TMA stores
};

// A warp's 32 token rows from row0 on and COLS columns from n0 + col0 on, in blocks of 128 bytes a row: a lane turns its row's
// integers into the output's type, stages them (swizzled) and the copy engine writes whole rows, clipped at M and N.
template <typename OutT, int COLS>
__device__ __forceinline__ void store_rows(unsigned src, const CUtensorMap* map_out, unsigned char* stage, int lane, int row0,
                                           int n0, int col0, const LargeArgs& a) {
  constexpr int PER_BLOCK = 128 / (int)sizeof(OutT);
  const float sx = row0 + lane < a.M ? a.sx[row0 + lane] : 0.f;
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
      const float* sw = a.sw + n0 + col + h;
      float4 w[8];
      if (n0 + col + h + 32 <= a.N) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const float4*>(sw + 4 * j);
      } else {
        const int left = a.N - (n0 + col + h);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[j] = make_float4(4 * j < left ? sw[4 * j] : 0.f, 4 * j + 1 < left ? sw[4 * j + 1] : 0.f,
                             4 * j + 2 < left ? sw[4 * j + 2] : 0.f, 4 * j + 3 < left ? sw[4 * j + 3] : 0.f);
      }
      tc_wait_ld();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y0 = (float)(int)v[4 * j] * sx * w[j].x, y1 = (float)(int)v[4 * j + 1] * sx * w[j].y;
        const float y2 = (float)(int)v[4 * j + 2] * sx * w[j].z, y3 = (float)(int)v[4 * j + 3] * sx * w[j].w;
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

// PAIR: two CTAs on a tile of 256 tokens x BNL channels; `full` of the first CTA counts both CTAs' copies, its commits
// signal `empty` and `acc_full` in both, `acc_empty` of the first takes an arrival of every epilogue warp of both.
template <typename OutT, int BNL, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
gemm_large_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                  const __grid_constant__ CUtensorMap map_out, const __grid_constant__ LargeArgs a) {
  constexpr int B_ROWS = PAIR ? BNL / 2 : BNL;      // channels that this CTA fetches
  using RG = Ring<B_ROWS>;
  constexpr int STAGES = RG::STAGES, STAGE = RG::STAGE, CTAS = PAIR ? 2 : 1;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* epi_stage = smem + STAGES * STAGE;
  unsigned long long* full = reinterpret_cast<unsigned long long*>(epi_stage + EPI_WARPS * EPI_STAGE_BYTES);
  unsigned long long* empty = full + STAGES;
  unsigned long long* acc_full = empty + STAGES;     // [2] a tile's accumulator is complete
  unsigned long long* acc_empty = acc_full + 2;      // [2] the epilogue has read it
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(acc_empty + 2);
  if (!PAIR) pdl_trigger();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_out);
  }
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_rank() : 0;
  const int group = blockIdx.x / CTAS, groups = gridDim.x / CTAS;
  const int tiles = a.m_tiles * a.n_tiles;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
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
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();       // both CTAs' barriers and tensor memory exist before either is used
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      // ---- copies.  The ring runs on across the tiles: load number c is k-block c % num_kb of this CTA's tile number
      // c / num_kb.  Tiles in the order of their channels, so that the CTAs side by side share them.
      const int my_tiles = tiles > group ? (tiles - group + groups - 1) / groups : 0;
      const int total = my_tiles * a.num_kb;
      const unsigned full0 = PAIR ? cluster_addr(smem_u32(full), 0) : smem_u32(full);
      auto load_w = [&](int c) {
        const int t = group + (c / a.num_kb) * groups, k = (c % a.num_kb) * BK, s = c % STAGES;
        const int n0 = (t / a.m_tiles) * BNL + rank * B_ROWS;
        unsigned char* b = smem + s * STAGE + A_BYTES;
        tma_load_2d<PAIR>(b, &map_w, k, n0, full0 + s * 8);
        if (B_ROWS == 256) tma_load_2d<PAIR>(b + 128 * BK, &map_w, k, n0 + 128, full0 + s * 8);
      };
      auto load_x = [&](int c) {
        const int t = group + (c / a.num_kb) * groups, k = (c % a.num_kb) * BK, s = c % STAGES;
        tma_load_2d<PAIR>(smem + s * STAGE, &map_x, k, (t % a.m_tiles) * CTAS * BM + rank * BM, full0 + s * 8);
      };
      const int pre = total < STAGES ? total : STAGES;
      for (int c = 0; c < pre; ++c) {      // weights are constants: the first stages' go out before the wait
        if (rank == 0) mbar_expect_tx(&full[c], CTAS * STAGE);
        load_w(c);
      }
      pdl_wait();
      for (int c = 0; c < pre; ++c) load_x(c);
      int c = pre;
      for (; c < total; ++c) {
        ok = mbar_wait_brief(&empty[c % STAGES], ((c / STAGES) - 1) & 1);
        if (!ok) break;
        if (rank == 0) mbar_expect_tx(&full[c % STAGES], CTAS * STAGE);
        load_w(c);
        load_x(c);
      }
      // given up: what was sent for arrives before this memory is another's (the pair's second CTA stays until the first, whose
      // barriers count for both, has waited)
      if (!ok && rank == 0)
        for (int s = c - STAGES; s < c; ++s) mbar_wait_brief(&full[s % STAGES], (s / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---- products
      const unsigned elected = elect_one();
      constexpr unsigned idesc = make_idesc(CTAS * BM, BNL);
      int count = 0, local = 0;
      for (int t = group; t < tiles && ok; t += groups, ++local) {
        const int buf = local & 1;
        if (local >= 2) {      // the epilogue must have read this buffer's earlier tile
          ok = __all_sync(0xffffffffu, mbar_wait_brief(&acc_empty[buf], ((local >> 1) - 1) & 1));
          if (!ok) break;
          tc_fence_after();
        }
        for (int kb = 0; kb < a.num_kb && ok; ++kb, ++count) {
          const int s = count % STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait_brief(&full[s], (count / STAGES) & 1));
          if (!ok) break;
          tc_fence_after();
          const unsigned long long da = smem_desc(smem_u32(smem + s * STAGE)), db = smem_desc(smem_u32(smem + s * STAGE) + A_BYTES);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            tc_mma<PAIR>(elected, tmem + buf * BNL, da + k * (UMMA_K >> 4), db + k * (UMMA_K >> 4), idesc, (kb > 0 || k > 0) ? 1u : 0u);
          tc_commit<PAIR>(elected, &empty[s]);
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
      constexpr int BLOCK = 128 / (int)sizeof(OutT), HALF = BNL / 2 >= BLOCK ? BNL / 2 : BNL;      // (one half: the first's)
      if (HALF == BNL / 2 || half == 0)
        store_rows<OutT, HALF>(tmem + buf * BNL + lane_base, &map_out, epi_stage + (warp - EPI_WARP0) * EPI_STAGE_BYTES, lane,
                               (t % a.m_tiles) * CTAS * BM + rank * BM + quarter * 32, (t / a.m_tiles) * BNL,
                               HALF == BNL ? 0 : half * HALF, a);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + buf * 8);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  if (!ok) atomicExch(&dib_gemm_int8_error_word, 1);
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();       // the other CTA's products and arrivals may still touch this one
  if (warp == 1) {
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Some rows (more than the streamed weight likes, fewer than fill the GPU with tiles): a cluster of S CTAs has a tile of 128
// tokens x BNL channels, each a run of the k-blocks; then each adds up the S integers of some of the columns (a thread a
// token's 8 columns) from the others' shared memory and writes them.  Only the token rows that there are, rounded up to
// a_rows, are fetched; what the products make of the rows behind them is never read.
constexpr int SPLIT_THREADS = 256, SPLIT_MAX = 8, SPLIT_RING = 192 * 1024;
struct SplitArgs {
  const float* sx;
  const float* sw;
  void* out;
  int M, N, num_kb, a_rows, stages;
  int by_lines;
};
template <int BNL> struct SplitShape {
  static constexpr int SUM_ROW = BNL * 4 + 16;      // a token's integers, 16 bytes off: no two of a warp's rows share banks
};
__device__ __forceinline__ int4 load_cluster(unsigned addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
template <typename OutT, int BNL>
__global__ void __launch_bounds__(SPLIT_THREADS)
gemm_split_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                  const __grid_constant__ SplitArgs a) {
  constexpr int SUM_ROW = SplitShape<BNL>::SUM_ROW;
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long full[16], empty[16], acc_full;
  __shared__ unsigned tmem_slot;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  pdl_trigger();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
  }
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), split = cluster_size();
  const int n0 = blockIdx.x / split * BNL, m0 = blockIdx.y * BM;
  const int kb0 = rank * a.num_kb / split, count = (rank + 1) * a.num_kb / split - kb0;
  const int b_bytes = BNL * BK, stage = b_bytes + a.a_rows * BK;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((unsigned)BNL));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      auto load_w = [&](int c) {
        const int s = c % a.stages;
        mbar_expect_tx(&full[s], stage);
        tma_load_2d<false>(smem + s * stage, &map_w, (kb0 + c) * BK, n0, smem_u32(&full[s]));
      };
      auto load_x = [&](int c) {
        const int s = c % a.stages;
        tma_load_2d<false>(smem + s * stage + b_bytes, &map_x, (kb0 + c) * BK, m0, smem_u32(&full[s]));
      };
      const int pre = count < a.stages ? count : a.stages;
      for (int c = 0; c < pre; ++c) load_w(c);      // weights are constants: the first stages' go out before the wait
      pdl_wait();
      for (int c = 0; c < pre; ++c) load_x(c);
      int c = pre;
      for (; c < count; ++c) {
        ok = mbar_wait_brief(&empty[c % a.stages], ((c / a.stages) - 1) & 1);
        if (!ok) break;
        load_w(c);
        load_x(c);
      }
      if (!ok)      // (as in the kernel above)
        for (int s = c - a.stages; s < c; ++s) mbar_wait_brief(&full[s % a.stages], (s / a.stages) & 1);
    }
  } else if (warp == 1) {
    const unsigned elected = elect_one();
    constexpr unsigned idesc = make_idesc(BM, BNL);
    for (int c = 0; c < count; ++c) {
      const int s = c % a.stages;
      ok = __all_sync(0xffffffffu, mbar_wait_brief(&full[s], (c / a.stages) & 1));
      if (!ok) break;
      tc_fence_after();
      const unsigned long long db = smem_desc(smem_u32(smem) + s * stage), da = smem_desc(smem_u32(smem) + s * stage + b_bytes);
#pragma unroll
      for (int k = 0; k < BK / UMMA_K; ++k)
        tc_mma<false>(elected, tmem, da + k * (UMMA_K >> 4), db + k * (UMMA_K >> 4), idesc, (c > 0 || k > 0) ? 1u : 0u);
      tc_commit<false>(elected, &empty[s]);
    }
    if (ok) tc_commit<false>(elected, &acc_full);
  } else if (warp >= 4) {
    // ---- integers to shared memory, over the ring: all of its copies have been read
    const int row = (warp - 4) * 32 + lane;
    if ((warp - 4) * 32 < a.a_rows) {
      ok = mbar_wait_brief(&acc_full, 0);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (ok)
#pragma unroll
        for (int c = 0; c < BNL; c += 32) {
          unsigned v[32];
          tc_ld32(tmem + ((unsigned)((warp - 4) * 32) << 16) + c, v);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(smem + row * SUM_ROW + (c + j) * 4) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
    }
  }
  if (!ok) atomicExch(&dib_gemm_int8_error_word, 1);
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  pdl_wait();
  const unsigned base = smem_u32(smem);
  const int rows = a.M - m0 < BM ? a.M - m0 : BM, groups = (BNL / 8 - rank + split - 1) / split;
  for (int e = threadIdx.x; e < rows * groups; e += SPLIT_THREADS) {
    const int group = e / rows, row = e - group * rows, col = (rank + group * split) * 8;
    if (n0 + col >= a.N) continue;
    int sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int r = 0; r < split; ++r) {
      const unsigned from = cluster_addr(base + row * SUM_ROW + col * 4, r);
      const int4 lo = load_cluster(from), hi = load_cluster(from + 16);
      sum[0] += lo.x; sum[1] += lo.y; sum[2] += lo.z; sum[3] += lo.w;
      sum[4] += hi.x; sum[5] += hi.y; sum[6] += hi.z; sum[7] += hi.w;
    }
    const float sx = a.sx[m0 + row];
    alignas(16) OutT y[8];
    const int left = a.N - (n0 + col);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) store_as(y[j], (float)sum[j] * sx * a.sw[n0 + col + j]);
    OutT* out = reinterpret_cast<OutT*>(a.out) + (long long)(m0 + row) * a.N + n0 + col;
    if (!a.by_lines && left >= 8) {
#pragma unroll
      for (int j = 0; j < 8 * (int)sizeof(OutT) / 16; ++j) reinterpret_cast<uint4*>(out)[j] = reinterpret_cast<const uint4*>(y)[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) out[j] = y[j];
    }
  }
  cluster_sync_all();       // the others may still read this one's integers
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)BNL));
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
// A row-major matrix [rows, cols] of `type`, boxes of box_rows rows of 128 bytes, 128-byte swizzle; what lies outside reads as
// zero and is not written.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, int size, const void* ptr, long long rows, long long cols, int box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)cols * size};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename OutT, int BNL, bool PAIR>
int launch_large(const void* x, const void* sx, const void* w, const void* sw, void* out, int M, int N, int Kp, int sm_count,
                 cudaStream_t st) {
  constexpr int CTAS = PAIR ? 2 : 1, B_ROWS = PAIR ? BNL / 2 : BNL;
  LargeArgs a;
  a.sx = reinterpret_cast<const float*>(sx);
  a.sw = reinterpret_cast<const float*>(sw);
  a.out = out;
  a.M = M; a.N = N;
  a.num_kb = (Kp + BK - 1) / BK;
  a.m_tiles = (M + CTAS * BM - 1) / (CTAS * BM);
  a.n_tiles = (N + BNL - 1) / BNL;
  a.by_lines = ((long long)N * sizeof(OutT)) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0;
  const long long tiles = (long long)a.m_tiles * a.n_tiles;
  if (tiles > (1ll << 24) || sm_count < CTAS) return DIB_BAD_SIZE;
  CUtensorMap mx, mw, mo;
  const CUtensorMapDataType type = sizeof(OutT) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  if (!make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, M, Kp, BM) ||
      !make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, N, Kp, B_ROWS < 128 ? B_ROWS : 128))
    return DIB_LAUNCH_FAILED;
  if (a.by_lines) mo = mx;      // (not used)
  else if (!make_map(&mo, type, sizeof(OutT), out, M, N, 32)) return DIB_LAUNCH_FAILED;
  auto kern = gemm_large_kernel<OutT, BNL, PAIR>;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Ring<B_ROWS>::SMEM) != cudaSuccess)
      return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  const int groups = (int)(tiles < sm_count / CTAS ? tiles : sm_count / CTAS);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CTAS * groups);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Ring<B_ROWS>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = dib_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, mx, mw, mo, a) != cudaSuccess) return DIB_LAUNCH_FAILED;
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// (the products read 128 token rows whatever was fetched: the last stage's lie in the memory behind it)
constexpr int SPLIT_SMEM = 1024 + SPLIT_RING + BM * BK;
// A launch of clusters of `split` CTAs.
struct SplitLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  SplitLaunch(int split, int n_tiles, int m_tiles, cudaStream_t st) {
    cfg.gridDim = dim3(split * n_tiles, m_tiles);
    cfg.blockDim = dim3(SPLIT_THREADS);
    cfg.dynamicSmemBytes = SPLIT_SMEM;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = dib_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }
};
// The CTAs that a tile's k is shared among: as many as leave all tiles running at once, two k-blocks for each at least.  A
// cluster lies within a part of the GPU, so that 148 SMs hold fewer than 49 clusters of three: the driver is asked once.
template <typename OutT, int BNL>
int split_of(int tiles, int num_kb) {
  auto kern = gemm_split_kernel<OutT, BNL>;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SPLIT_SMEM) != cudaSuccess) return 0;
    attr_set.mark();
  }
  static std::atomic<int> resident[SPLIT_MAX + 1];
  int split = num_kb / 2 < SPLIT_MAX ? num_kb / 2 : SPLIT_MAX;
  for (; split > 1; --split) {
    int n = resident[split].load(std::memory_order_relaxed);
    if (n == 0) {
      SplitLaunch launch(split, 1, 1, nullptr);
      if (cudaOccupancyMaxActiveClusters(&n, kern, &launch.cfg) != cudaSuccess) return 0;
      if (n < 1) n = 1;
      resident[split].store(n, std::memory_order_relaxed);
    }
    if (n >= tiles) break;
  }
  return split < 1 ? 1 : split;
}
template <typename OutT, int BNL>
int launch_split(const void* x, const void* sx, const void* w, const void* sw, void* out, int M, int N, int Kp, cudaStream_t st) {
  SplitArgs a;
  a.sx = reinterpret_cast<const float*>(sx);
  a.sw = reinterpret_cast<const float*>(sw);
  a.out = out;
  a.M = M; a.N = N;
  a.num_kb = (Kp + BK - 1) / BK;
  a.a_rows = M <= 32 ? 32 : M <= 64 ? 64 : BM;
  a.by_lines = ((long long)N * sizeof(OutT)) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0;
  const int m_tiles = (M + BM - 1) / BM, n_tiles = (N + BNL - 1) / BNL;
  if (m_tiles > 65535 || n_tiles > 0x7fffffff / SPLIT_MAX) return DIB_BAD_SIZE;
  const int stage = (BNL + a.a_rows) * BK;
  a.stages = SPLIT_RING / stage < 16 ? SPLIT_RING / stage : 16;
  static_assert(BM * SplitShape<BNL>::SUM_ROW <= SPLIT_RING && SPLIT_SMEM + 1024 <= 232448, "shared memory");
  CUtensorMap mx, mw;
  if (!make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, M, Kp, a.a_rows) ||
      !make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, N, Kp, BNL))
    return DIB_LAUNCH_FAILED;
  const long long tiles = (long long)m_tiles * n_tiles;
  const int split = split_of<OutT, BNL>(tiles < 0x7fffffff ? (int)tiles : 0x7fffffff, a.num_kb);
  if (split < 1) return DIB_LAUNCH_FAILED;
  SplitLaunch launch(split, n_tiles, m_tiles, st);
  if (cudaLaunchKernelEx(&launch.cfg, gemm_split_kernel<OutT, BNL>, mx, mw, a) != cudaSuccess) return DIB_LAUNCH_FAILED;
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// Form forced for measurements and tests (-1: the choice of `form`): 0 few rows, 1 tiles of 128 x 64, 2 of 128 x 128, 3 of
// 128 x 256, 4 the pair, 5 clusters on tiles of 128 x 64, 6 of 128 x 128.
int& forced_form() {
  static int v = -1;
  return v;
}
// A function of the sizes and the GPU; the form never changes a bit of the result.
int large_form(int M, int N, int sm_count) {
  const long long pair_tiles = (long long)((M + 2 * BM - 1) / (2 * BM)) * ((N + 255) / 256);
  if (sm_count >= 2 && M > BM && 3 * pair_tiles >= sm_count) return 4;
  const long long m_tiles = (M + BM - 1) / BM;
  if (m_tiles * ((N + 127) / 128) <= sm_count / 2) return 1;
  return 2 * m_tiles * ((N + 255) / 256) <= sm_count ? 2 : 3;
}
// Up to 256 rows the times of the forms are estimated, in us, from lines through measured ones (k-blocks of 128):
//   streamed weight, 8 rows     1,024 x 1,024 1.6, 4,096 x 4,096 5.8, 24,576 x 4,096 18.7, 4,096 x 12,288 12.6, 5,120 x 25,600 26;
//                               16, 24, 32 rows take some 1.15, 1.4, 1.5 times that, as a block fetches its tokens from L2
//   clusters, 128 wide          32 rows: 4,096 x 4,096 8.8, 6,144 x 4,096 9.8, 4,096 x 12,288 13.8, 5,120 x 25,600 26.5
//                               128 rows: 13.5, 14.1, 18.4, 32.3
//   clusters, 64 wide           32 rows: 2,560 x 4,096 8.0, 4,096 x 4,096 9.5; 128 rows: 10.1, 10.6
//   a tile a CTA                4,096 x 4,096 12.7, 4,096 x 12,288 32, 5,120 x 25,600 65
template <typename OutT>
int form(int M, int N, int Kp, int sm_count) {
  if (forced_form() >= 0) return forced_form();
  const int large = large_form(M, N, sm_count);
  if (M > 2 * BM) return large;
  const int num_kb = (Kp + BK - 1) / BK, m_tiles = (M + BM - 1) / BM;
  float best = 1e30f;
  int choice = large;
  auto consider = [&](int form, float us) {
    if (us < best) {
      best = us;
      choice = form;
    }
  };
  if (M <= 16 || (M <= 32 && N <= 48 * sm_count))
    consider(0, (1.2f + 0.5e-3f * Kp + (float)N * Kp / 6.8e6f) * (M <= 8 ? 1.f : M <= 16 ? 1.15f : M <= 24 ? 1.4f : 1.5f));
  if (M > 16) {
    const int width = large == 1 ? 64 : large == 2 ? 128 : 256, tiles = m_tiles * ((N + width - 1) / width);
    consider(large, 2.8f + 0.31f * num_kb * ((tiles + sm_count - 1) / sm_count));
  }
  const int tiles64 = m_tiles * ((N + 63) / 64), tiles128 = m_tiles * ((N + 127) / 128);
  const int s64 = 2 * tiles64 <= sm_count ? split_of<OutT, 64>(tiles64, num_kb) : 1;
  const int s128 = 2 * tiles128 <= sm_count ? split_of<OutT, 128>(tiles128, num_kb) : 1;
  if (s64 > 1) consider(5, 4.6f + 0.33f * ((num_kb + s64 - 1) / s64) + (M > 64 ? 1.2f : M > 32 ? 0.3f : 0.f));
  if (s128 > 1) consider(6, 5.f + 0.35f * ((num_kb + s128 - 1) / s128) + (M > 64 ? 4.5f : M > 32 ? 1.7f : 0.f));
  return choice;
}

template <typename OutT>
int launch(const void* x, const void* sx, const void* w, const void* sw, void* out, int M, int N, int Kp, int sm_count,
           cudaStream_t st) {
  switch (form<OutT>(M, N, Kp, sm_count)) {
    case 0: return launch_few<OutT>(x, sx, w, sw, out, M, N, Kp, st);
    case 1: return launch_large<OutT, 64, false>(x, sx, w, sw, out, M, N, Kp, sm_count, st);
    case 2: return launch_large<OutT, 128, false>(x, sx, w, sw, out, M, N, Kp, sm_count, st);
    case 3: return launch_large<OutT, 256, false>(x, sx, w, sw, out, M, N, Kp, sm_count, st);
    case 5: return launch_split<OutT, 64>(x, sx, w, sw, out, M, N, Kp, st);
    case 6: return launch_split<OutT, 128>(x, sx, w, sw, out, M, N, Kp, st);
    default: return launch_large<OutT, 256, true>(x, sx, w, sw, out, M, N, Kp, sm_count, st);
  }
}

}  // namespace

extern "C" {

int dib_gemm_int8_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dib_gemm_int8_error_word, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int dib_gemm_int8_status_clear() {
  const int v = 0;
  return cudaMemcpyToSymbol(dib_gemm_int8_error_word, &v, sizeof(int)) == cudaSuccess ? 0 : -1;
}
void dib_gemm_int8_force_form(int form) { forced_form() = form; }

int dib_gemm_int8(const void* x, const void* sx, const void* w, const void* sw, void* out, int M, int N, int Kp, int out_dtype,
                  int sm_count, cudaStream_t st);
// The same with x [M, K] of values (x_dtype 0 float32, 1 bfloat16; rows `stride` values apart), which `quantize`
// (dib_quantize_rows of the cache's library) first turns into codes and scales in `work` (M Kp + 4 M bytes, the scales
// behind the codes).
int dib_int8_linear(int (*quantize)(const void*, long long, void*, void*, long long, int, int, cudaStream_t),
                    const void* x, long long stride, int x_dtype, int K, void* work, const void* w, const void* sw, void* out,
                    int M, int N, int out_dtype, int sm_count, cudaStream_t st) {
  const int Kp = (K + 15) / 16 * 16;
  void* scales = reinterpret_cast<char*>(work) + (long long)M * Kp;
  const int rc = quantize(x, stride, work, scales, M, K, x_dtype, st);
  if (rc != DIB_OK) return rc;
  return dib_gemm_int8(work, scales, w, sw, out, M, N, Kp, out_dtype, sm_count, st);
}

// out[M, N] = x w^T scaled; x int8 [M, Kp], w int8 [N, Kp], Kp a multiple of 16, sx [M], sw [N] float32, out_dtype
// 0 float32, 1 bfloat16.
int dib_gemm_int8(const void* x, const void* sx, const void* w, const void* sw, void* out, int M, int N, int Kp,
                  int out_dtype, int sm_count, cudaStream_t st) {
  if (out_dtype != 0 && out_dtype != 1) return DIB_BAD_DTYPE;
  if (M < 0 || N < 0 || Kp < 16 || Kp % 16 != 0 || Kp > 133152 || sm_count < 1) return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(sw)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (M == 0 || N == 0) return DIB_OK;
  if (out_dtype == 1) return launch<__nv_bfloat16>(x, sx, w, sw, out, M, N, Kp, sm_count, st);
  return launch<float>(x, sx, w, sw, out, M, N, Kp, sm_count, st);
}

}  // extern "C"
