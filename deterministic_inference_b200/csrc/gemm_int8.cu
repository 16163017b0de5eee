// Matrix product in 8-bit integers: y[m, n] = sx[m] * sw[n] * sum_k x[m, k] * w[n, k], x and w int8 (K-major, rows of Kp
// bytes, a multiple of 16), the sum an exact 32-bit integer for K up to 133,144 (127^2 K < 2^31).  Because it is exact,
// the order in which it is added up (warps, runs of k, tile shapes) never changes a bit of the result: a row's bits
// depend on the row and the weight alone.
//
// Few rows: the weight is streamed once from memory straight into the registers of mma.sync (m16n8k32: 16 output
// channels x 8 tokens), with no shared memory in between.  The product's k index may be permuted as long as both
// operands agree, so a thread takes 32 consecutive bytes of its two weight rows (two 16-byte loads each) and calls them
// the k it needs; the tokens' rows are read the same way, from L2.  A block of eight warps takes 16 channels; the warps
// share the row's k among them and add their integers up in shared memory.
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

// NT tiles of 8 tokens
template <typename OutT, int NT>
__global__ void __launch_bounds__(FEW_WARPS * 32)
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
  load32<true>(w0, in0, k, Kp, a);
  load32<true>(w1, in1, k, Kp, b);
  pdl_wait(x, sx);
  for (; k - t * 32 < Kp; k += FEW_WARPS * CHUNK) {
    const uint4 ca[2] = {a[0], a[1]}, cb[2] = {b[0], b[1]};
    load32<true>(w0, in0, k + FEW_WARPS * CHUNK, Kp, a);
    load32<true>(w1, in1, k + FEW_WARPS * CHUNK, Kp, b);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int m = m0 + nt * 8 + g;
      uint4 c[2];
      load32<false>(x + (long long)m * Kp, m < M, k, Kp, c);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma_s8(acc[nt], ca[i].x, cb[i].x, ca[i].y, cb[i].y, c[i].x, c[i].y);
        mma_s8(acc[nt], ca[i].z, cb[i].z, ca[i].w, cb[i].w, c[i].z, c[i].w);
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
  auto kern = nt == 1 ? gemm_few_kernel<OutT, 1> : nt == 2 ? gemm_few_kernel<OutT, 2> : gemm_few_kernel<OutT, 4>;
  dib_launch(kern, grid, dim3(FEW_WARPS * 32), 0, st, reinterpret_cast<const signed char*>(x),
             reinterpret_cast<const float*>(sx), reinterpret_cast<const signed char*>(w),
             reinterpret_cast<const float*>(sw), reinterpret_cast<OutT*>(out), M, N, Kp);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

}  // namespace

extern "C" {

// out[M, N] = x w^T scaled; x int8 [M, Kp], w int8 [N, Kp], Kp a multiple of 16, sx [M], sw [N] float32, out_dtype
// 0 float32, 1 bfloat16.
int dib_gemm_int8(const void* x, const void* sx, const void* w, const void* sw, void* out, int M, int N, int Kp,
                  int out_dtype, int sm_count, cudaStream_t st) {
  if (out_dtype != 0 && out_dtype != 1) return DIB_BAD_DTYPE;
  if (M < 0 || N < 0 || Kp < 16 || Kp % 16 != 0 || Kp > 133152 || sm_count < 1) return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) != 0) return DIB_BAD_ALIGN;
  if (M == 0 || N == 0) return DIB_OK;
  if (out_dtype == 1) return launch_few<__nv_bfloat16>(x, sx, w, sw, out, M, N, Kp, st);
  return launch_few<float>(x, sx, w, sw, out, M, N, Kp, st);
}

}  // extern "C"
