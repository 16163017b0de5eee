// Rows of a matrix in 4-bit floating point (fp4.cuh has the rule): quantising activations and weights, laying out codes that were
// made elsewhere, and reading rows back.
//
// Kept: codes [M, Kp / 2] (two a byte, the first in the low half; Kp = K rounded up to 32, zeros behind K), block scales in
// tiles (fp4_scale_at; zeros behind K), units float32 [M] = 2^E.
//
// A thread has a block of 16 values: its largest is the thread's own, its scale a byte, its codes 8 bytes.  float32 rows are bound
// by memory (24,576 x 4,096: 67 us, 6.8 TB/s), bfloat16 ones by instructions, 12 a warp for 32 values (24,576 x 4,096: 49 us, 5.2 TB/s;
// 63.8 with a value divided at a time, a loop over the warps' maxima and a row a block).  Rows that do not lie on 32 bytes, or whose K is no
// multiple of 16, are read a value at a time: 24,576 x 4,095 in float32 192 us, in bfloat16 128 (2,048 of them 19 and 12, 8 2.6 and 2.1).
#include "fp4.cuh"

namespace {

template <typename T>
__device__ __forceinline__ void write_block(const Block16<T>& x, unsigned top, float down, unsigned char* codes, unsigned char* tiles,
                                            long long row, int block, int Kp, int k_tiles) {
  const unsigned scale = fp4_block_scale(top, down);
  const Fp4Scaler s = fp4_scaler(scale, down);
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = x.get(e);
  if (block * 16 < Kp)
    *reinterpret_cast<uint2*>(codes + row * (Kp / 2) + block * 8) = make_uint2(fp4_codes8(v, s), fp4_codes8(v + 8, s));
  tiles[fp4_scale_at(row, block, k_tiles)] = (unsigned char)scale;
}

// Blocks of 512 threads that an SM's registers hold.  (One value after another in flight is what counts: 24,576 x 4,096 bfloat16
// 49.3, 49.5, 48.9 us with 2, 3, 4, but 512 x 4,096 2.3, 2.7, 2.7.)
template <typename T> constexpr int rows_per_sm(int blocks) { return blocks <= 1 || (blocks == 2 && sizeof(T) == 2) ? 2 : 1; }

// A block of threads a row, and on to the row `gridDim.x` further.  BLOCKS > 0: each thread keeps that many blocks of 16 in
// registers, and (AHEAD) has the next row's on their way while it makes this one's codes; 0: the row is read twice.
template <typename T, int BLOCKS, bool AHEAD, bool WIDE>
__global__ void __launch_bounds__(512, rows_per_sm<T>(BLOCKS))
quantize_rows_kernel(const T* __restrict__ x, long long stride, unsigned char* __restrict__ codes, unsigned char* __restrict__ tiles,
                     float* __restrict__ units, unsigned M, int K, int Kp, int k_tiles) {
  pdl_prologue(x);
  __shared__ unsigned tops[2][16];
  const int blocks = k_tiles * 4;
  constexpr int KEPT = BLOCKS > 0 ? BLOCKS : 1;
  Block16<T> v[KEPT], next[AHEAD ? KEPT : 1];
  if (AHEAD) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) next[i].template load<WIDE>(x + blockIdx.x * stride, (i * blockDim.x + threadIdx.x) * 16, K);
  }
  int turn = 0;
#pragma unroll 1
  for (unsigned row = blockIdx.x; row < M; row += gridDim.x, turn ^= 1) {
    const T* src = x + row * stride;
    unsigned own[KEPT], top = 0;
    if (BLOCKS > 0) {
      if (AHEAD) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) v[i] = next[i];
        if (gridDim.x < M - row) {
#pragma unroll
          for (int i = 0; i < KEPT; ++i)
            next[i].template load<WIDE>(src + gridDim.x * stride, (i * blockDim.x + threadIdx.x) * 16, K);
        }
      } else {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) v[i].template load<WIDE>(src, (i * blockDim.x + threadIdx.x) * 16, K);
      }
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        own[i] = v[i].top();
        top = max(top, own[i]);
      }
    } else {
      for (int b = threadIdx.x; b < blocks; b += blockDim.x) {
        v[0].template load<WIDE>(src, b * 16, K);
        top = max(top, v[0].top());
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[turn][threadIdx.x >> 5] = top;
    __syncthreads();      // (a row's maxima are read before the next barrier, those of the row after next are written behind it)
    top = __reduce_max_sync(0xffffffffu, tops[turn][min(threadIdx.x & 31, blockDim.x / 32 - 1)]);
    const unsigned exponent = fp4_row_exponent(top);
    const float down = fp4_down(exponent);
    if (threadIdx.x == 0) units[row] = fp4_unit(exponent);
    if (BLOCKS > 0) {
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        const int b = i * blockDim.x + threadIdx.x;
        if (b < blocks) write_block(v[i], own[i], down, codes, tiles, row, b, Kp, k_tiles);
      }
    } else {
      for (int b = threadIdx.x; b < blocks; b += blockDim.x) {
        v[0].template load<WIDE>(src, b * 16, K);
        write_block(v[0], v[0].top(), down, codes, tiles, row, b, Kp, k_tiles);
      }
    }
  }
}

template <typename T>
int launch_rows(const void* x, long long stride, void* codes, void* tiles, void* units, long long M, int K, int sm_count,
                cudaStream_t st) {
  const int Kp = (K + 31) / 32 * 32, k_tiles = fp4_k_tiles(K), blocks = k_tiles * 4;
  const bool wide = K % 16 == 0 && (stride * sizeof(T)) % 32 == 0 && reinterpret_cast<uintptr_t>(x) % 32 == 0;
  const int per = blocks <= 512 ? 1 : blocks <= 1024 ? 2 : blocks <= 2048 ? 4 : 0;
  const int threads = per == 0 ? 512 : ((blocks + per - 1) / per + 31) / 32 * 32;
  auto kern = per == 1 ? (wide ? quantize_rows_kernel<T, 1, true, true> : quantize_rows_kernel<T, 1, true, false>)
              : per == 2 ? (wide ? quantize_rows_kernel<T, 2, true, true> : quantize_rows_kernel<T, 2, true, false>)
              : per == 4 ? (wide ? quantize_rows_kernel<T, 4, sizeof(T) == 2, true> : quantize_rows_kernel<T, 4, sizeof(T) == 2, false>)
                         : (wide ? quantize_rows_kernel<T, 0, false, true> : quantize_rows_kernel<T, 0, false, false>);
  const long long at_once = (long long)sm_count * min(32, 512 * rows_per_sm<T>(per) / threads);
  dib_launch(kern, dim3((unsigned)min(M, at_once)), dim3(threads), 0, st, reinterpret_cast<const T*>(x), stride,
             reinterpret_cast<unsigned char*>(codes), reinterpret_cast<unsigned char*>(tiles), reinterpret_cast<float*>(units),
             (unsigned)M, K, Kp, k_tiles);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// A thread a block of 16: out[row, 16 b ..] = codes * scale * unit.  Bound by memory: 24,576 x 4,096 in float32 69.9 us, 6.6 TB/s, in
// bfloat16 43.7, 5.9 TB/s.
constexpr int READ_THREADS = 256;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(READ_THREADS)
read_rows_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ tiles, const float* __restrict__ units,
                 T* __restrict__ out, long long M, int K, int Kp, int k_tiles, int blocks) {
  pdl_prologue(codes, tiles, units);
  const long long i = (long long)blockIdx.x * READ_THREADS + threadIdx.x;
  const long long row = i / blocks;
  const int b = (int)(i - row * blocks);
  if (row >= M) return;
  const uint2 w = *reinterpret_cast<const uint2*>(codes + row * (Kp / 2) + b * 8);
  const float scale = fp4_scale_value(tiles[fp4_scale_at(row, b, k_tiles)]), unit = units[row];
  float x[16];
  fp4_values8(w.x, scale, x);
  fp4_values8(w.y, scale, x + 8);
  T* dst = out + row * K + b * 16;
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] *= unit;
  if (WIDE) {
    store16(dst, x);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (b * 16 + e < K) Elem<T>::store(dst + e, x[e]);
  }
}

template <typename T>
int launch_read(const void* codes, const void* tiles, const void* units, void* out, long long M, int K, cudaStream_t st) {
  const int blocks = (K + 15) / 16;
  const long long grid = (M * blocks + READ_THREADS - 1) / READ_THREADS;
  if (grid > 0x7fffffffll) return DIB_BAD_SIZE;
  const bool wide = K % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
  dib_launch(wide ? read_rows_kernel<T, true> : read_rows_kernel<T, false>, dim3((unsigned)grid), dim3(READ_THREADS), 0, st,
             reinterpret_cast<const unsigned char*>(codes), reinterpret_cast<const unsigned char*>(tiles),
             reinterpret_cast<const float*>(units), reinterpret_cast<T*>(out), M, K, (K + 31) / 32 * 32, fp4_k_tiles(K), blocks);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// Codes, block scales and exponent bytes as rows [M, code_bytes], [M, scale_bytes], [M] -> the layout above.  A thread a block
// of 16.  (Codes behind K are dropped, a scale's sign is: a block scale is not negative.)
__global__ void __launch_bounds__(READ_THREADS)
layout_rows_kernel(const unsigned char* __restrict__ in_codes, const unsigned char* __restrict__ in_scales,
                   const unsigned char* __restrict__ in_exponents, unsigned char* __restrict__ codes, unsigned char* __restrict__ tiles,
                   float* __restrict__ units, long long M, int K, int Kp, int k_tiles) {
  pdl_prologue(in_codes, in_scales, in_exponents);
  const int blocks = k_tiles * 4, code_bytes = (K + 1) / 2, scale_bytes = (K + 15) / 16;
  const long long i = (long long)blockIdx.x * READ_THREADS + threadIdx.x;
  const long long row = i / blocks;
  const int b = (int)(i - row * blocks);
  if (row >= M) return;
  if (b * 16 < Kp) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = b * 8 + j;
      unsigned c = at < code_bytes ? in_codes[row * code_bytes + at] : 0;
      if (2 * at + 1 >= K) c &= 15;
      codes[row * (Kp / 2) + at] = (unsigned char)c;
    }
  }
  tiles[fp4_scale_at(row, b, k_tiles)] = b < scale_bytes ? in_scales[row * scale_bytes + b] & 127 : 0;
  if (b == 0) units[row] = fp4_unit(in_exponents[row]);
}

}  // namespace

extern "C" {

// codes [M, Kp / 2], tiles [ceil(M / 128), fp4_k_tiles(K), 512], units float32 [M] of x [M, K] (dtype 0 float32, 1 bfloat16),
// rows `stride` values apart.
int dib_fp4_quantize_rows(const void* x, long long stride, void* codes, void* tiles, void* units, long long M, int K, int dtype,
                          int sm_count, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (M < 0 || M > 0x7fffffffll || K < 1 || K > (1 << 30) || sm_count < 1) return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(tiles)) & 15) != 0) return DIB_BAD_ALIGN;
  if (M == 0) return DIB_OK;
  if (dtype == 1) return launch_rows<__nv_bfloat16>(x, stride, codes, tiles, units, M, K, sm_count, st);
  return launch_rows<float>(x, stride, codes, tiles, units, M, K, sm_count, st);
}

// out [M, K] (dtype 0 float32, 1 bfloat16): what the rows stand for.
int dib_fp4_read_rows(const void* codes, const void* tiles, const void* units, void* out, long long M, int K, int dtype,
                      cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (M < 0 || K < 1 || K > (1 << 30)) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) != 0) return DIB_BAD_ALIGN;
  if (M == 0) return DIB_OK;
  if (dtype == 1) return launch_read<__nv_bfloat16>(codes, tiles, units, out, M, K, st);
  return launch_read<float>(codes, tiles, units, out, M, K, st);
}

// The layout of rows that were quantised elsewhere: in_codes [M, ceil(K / 2)], in_scales [M, ceil(K / 16)] (e4m3), in_exponents [M].
int dib_fp4_layout_rows(const void* in_codes, const void* in_scales, const void* in_exponents, void* codes, void* tiles, void* units,
                        long long M, int K, cudaStream_t st) {
  if (M < 0 || K < 1 || K > (1 << 30)) return DIB_BAD_SIZE;
  if (M == 0) return DIB_OK;
  const int k_tiles = fp4_k_tiles(K);
  const long long grid = (M * k_tiles * 4 + READ_THREADS - 1) / READ_THREADS;
  if (grid > 0x7fffffffll) return DIB_BAD_SIZE;
  dib_launch(layout_rows_kernel, dim3((unsigned)grid), dim3(READ_THREADS), 0, st, reinterpret_cast<const unsigned char*>(in_codes),
             reinterpret_cast<const unsigned char*>(in_scales), reinterpret_cast<const unsigned char*>(in_exponents),
             reinterpret_cast<unsigned char*>(codes), reinterpret_cast<unsigned char*>(tiles), reinterpret_cast<float*>(units), M, K,
             (K + 31) / 32 * 32, k_tiles);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

}  // extern "C"
