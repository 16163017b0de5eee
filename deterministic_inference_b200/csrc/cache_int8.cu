// Rows in 8-bit integers: the one rule by which activations, weights, keys and values are quantised, a paged cache
// of quantised keys and values, and reading it back.
//
// A row (a token's activations, an output channel of a weight, a token's key or value of one head) of values x:
//   a = max(max |x|, 2^-100),  code = rint(x * (127 / a)) (ties to even),  scale = a / 127,  value = scale * code.
// 127 / a and a / 127 are the correctly rounded quotients and x * (127 / a) one rounded product, so the codes are the
// same on every path that makes them.  |x * (127 / a)| <= 127 (1 + 2^-23), which rounds to 127: no clamp.  The floor
// 2^-100 keeps 127 / a finite; rows below it read back as zeros, 2^-100 off at most.  A row that holds an infinity or
// a NaN has the scale NaN, so whatever reads it gets NaN and not a number that looks right.
//
// Cache: data int8 [pages, 2, Hkv, page_size, D], scales float32 [pages, 2, Hkv, page_size].
#include "common.cuh"

namespace {

constexpr float ROW_FLOOR = 7.888609052210118e-31f;      // 2^-100

struct RowScale {
  float inv, scale;
};
// bits: the largest |x| of the row as an unsigned number (infinities and NaN order above every finite one)
__device__ __forceinline__ RowScale row_scale(unsigned bits) {
  RowScale r;
  if (bits >= 0x7f800000u) {
    r.inv = 0.f;
    r.scale = __uint_as_float(0x7fc00000u);
  } else {
    const float a = fmaxf(__uint_as_float(bits), ROW_FLOOR);
    r.inv = __fdiv_rn(127.f, a);
    r.scale = __fdiv_rn(a, 127.f);
  }
  return r;
}
__device__ __forceinline__ unsigned magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// four codes in a word, x0's in the low byte (a row with scale NaN: 0 * infinity is NaN, whose integer is 0)
__device__ __forceinline__ unsigned pack4(const float* x, float inv) {
  const int c0 = __float2int_rn(__fmul_rn(x[0], inv)), c1 = __float2int_rn(__fmul_rn(x[1], inv));
  const int c2 = __float2int_rn(__fmul_rn(x[2], inv)), c3 = __float2int_rn(__fmul_rn(x[3], inv));
  return (unsigned)(c0 & 0xff) | (unsigned)(c1 & 0xff) << 8 | (unsigned)(c2 & 0xff) << 16 | (unsigned)c3 << 24;
}

template <typename T, bool ALIGNED> __device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <> __device__ __forceinline__ void load8<__nv_bfloat16, true>(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <> __device__ __forceinline__ void load8<float, true>(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16, false>(const __nv_bfloat16* p, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
}
template <> __device__ __forceinline__ void load8<float, false>(const float* p, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = p[i];
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const unsigned*>(&v);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T> __device__ __forceinline__ void load4(const T* p, float (&x)[4]);
template <> __device__ __forceinline__ void load4<float>(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
template <> __device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&x)[4]);
template <> __device__ __forceinline__ void store4<float>(float* p, const float (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <> __device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

constexpr int CACHE_THREADS = 256, ROW_LANES = 16;       // half a warp a row: 8 values a lane, twice for heads above 128

// Row r = (token, key or value, kv head).  Memory bound: a row is read once into registers.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_write_kernel(const T* __restrict__ k, const T* __restrict__ v, long long k_stride, long long v_stride,
                   signed char* __restrict__ data, float* __restrict__ scales, const int* __restrict__ slots,
                   long long rows, int Hkv, int D, int page_size, long long num_pages) {
  pdl_prologue(k, v, slots);
  const long long r = ((long long)blockIdx.x * CACHE_THREADS + threadIdx.x) / ROW_LANES;
  const int l = threadIdx.x & (ROW_LANES - 1);
  const bool in = r < rows;
  const long long token = in ? r / (2 * Hkv) : 0;
  const int rest = in ? (int)(r - token * 2 * Hkv) : 0;
  const int kv = rest >= Hkv, h = rest - kv * Hkv;
  const T* src = (kv ? v + token * v_stride : k + token * k_stride) + (long long)h * D;
  const int slot = in ? slots[token] : -1;
  float x[2][8];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = (i * ROW_LANES + l) * 8;
    if (in && d < D) {
      load8<T, ALIGNED>(src + d, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(x[i][j]));
    }
  }
#pragma unroll
  for (int o = ROW_LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (slot < 0) return;
  const long long page = slot / page_size;
  if (page >= num_pages) return;
  const long long at = ((page * 2 + kv) * Hkv + h) * page_size + (slot - page * page_size);
  const RowScale s = row_scale(top);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = (i * ROW_LANES + l) * 8;
    if (d < D) *reinterpret_cast<uint2*>(data + at * D + d) = make_uint2(pack4(x[i], s.inv), pack4(x[i] + 4, s.inv));
  }
  if (l == 0) scales[at] = s.scale;
}

template <typename T>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_read_kernel(const signed char* __restrict__ data, const float* __restrict__ scales, const int* __restrict__ slots,
                  T* __restrict__ k, T* __restrict__ v, long long rows, int Hkv, int D, int page_size,
                  long long num_pages) {
  pdl_prologue(data, scales, slots);
  const long long r = ((long long)blockIdx.x * CACHE_THREADS + threadIdx.x) / ROW_LANES;
  const int l = threadIdx.x & (ROW_LANES - 1);
  if (r >= rows) return;
  const long long token = r / (2 * Hkv);
  const int rest = (int)(r - token * 2 * Hkv);
  const int kv = rest >= Hkv, h = rest - kv * Hkv;
  const int slot = slots[token];
  const long long page = slot < 0 ? -1 : slot / page_size;
  const bool there = page >= 0 && page < num_pages;
  const long long at = there ? ((page * 2 + kv) * Hkv + h) * page_size + (slot - page * page_size) : 0;
  const float scale = there ? scales[at] : 0.f;
  T* dst = (kv ? v : k) + (token * Hkv + h) * D;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = (i * ROW_LANES + l) * 8;
    if (d >= D) break;
    const uint2 c = there ? *reinterpret_cast<const uint2*>(data + at * D + d) : make_uint2(0, 0);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = scale * (float)(signed char)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
    store8<T>(dst + d, x);
  }
}

// The step's fused projection rows [q heads | k heads | v heads]: q and k normed (RMS) and rotated, q to its output, k and v
// rounded to T, quantised and written to the token's slot; the norm's sum and the rotation are those of the kernels that
// write an unquantised cache.  A warp a (token, head), a lane 4 consecutive elements of 128 at a time; the rotation's pairs
// meet in shared memory.
constexpr int QKV_WARPS = 4;
template <typename T>
__global__ void __launch_bounds__(QKV_WARPS * 32)
qk_norm_rope_cache_int8_kernel(const T* __restrict__ qkv, T* __restrict__ q_out, signed char* __restrict__ data,
                               float* __restrict__ scales, const float* __restrict__ q_norm_w,
                               const float* __restrict__ k_norm_w, float eps, const float* __restrict__ cos_sin, int rotary_dim,
                               int max_pos, const int* __restrict__ positions, const int* __restrict__ slots, int T_tokens,
                               int Hq, int Hkv, int D, int page_size, long long num_pages) {
  pdl_prologue(qkv, q_norm_w, k_norm_w);
  __shared__ float row[QKV_WARPS][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = Hq + 2 * Hkv;
  const long long item = (long long)blockIdx.x * QKV_WARPS + warp;
  if (item >= (long long)T_tokens * heads) return;
  const int t = (int)(item / heads), head = (int)(item - (long long)t * heads);
  const bool is_q = head < Hq, is_k = !is_q && head < Hq + Hkv;
  const float* nw = is_q ? q_norm_w : is_k ? k_norm_w : nullptr;
  const int slot = is_q ? 0 : slots[t];
  const long long page = slot < 0 ? -1 : slot / page_size;
  if (!is_q && (page < 0 || page >= num_pages)) return;
  const T* src = qkv + item * D;
  float* s = row[warp];
  float x[2][4], squares[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = i * 128 + lane * 4;
    x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
    if (d < D) load4<T>(src + d, x[i]);
    squares[i] = sumsq4(x[i][0], x[i][1], x[i][2], x[i][3]);
  }
  if (nw != nullptr) {
    float total = warp_sum(squares[0]);
    if (D > 128) total = __fadd_rn(total, warp_sum(squares[1]));
    const float rstd = rms_rstd(total, D, eps);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = i * 128 + lane * 4;
      if (d < D)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = norm_scale(x[i][e], rstd, nw[d + e]);
    }
  }
  if (cos_sin != nullptr && (is_q || is_k)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = i * 128 + lane * 4;
      if (d < D) *reinterpret_cast<float4*>(s + d) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
    }
    __syncwarp();
    int pos = positions[t];
    pos = pos < 0 ? 0 : pos >= max_pos ? max_pos - 1 : pos;
    const float* tab = cos_sin + (long long)pos * rotary_dim;
    const int half = rotary_dim >> 1;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = i * 128 + lane * 4 + e;
        if (d < half) x[i][e] = rope_first(x[i][e], s[d + half], tab[d], tab[half + d]);
        else if (d < rotary_dim) x[i][e] = rope_second(s[d - half], x[i][e], tab[d - half], tab[d]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = round_to<T>(x[i][e]);
  if (is_q) {
    T* dst = q_out + ((long long)t * Hq + head) * D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = i * 128 + lane * 4;
      if (d < D) store4<T>(dst + d, x[i]);
    }
    return;
  }
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, magnitude_bits(x[i][e]));
  const RowScale scale = row_scale(__reduce_max_sync(0xffffffffu, top));
  const int kv = !is_k, h = is_k ? head - Hq : head - Hq - Hkv;
  const long long at = ((page * 2 + kv) * Hkv + h) * page_size + (slot - page * page_size);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = i * 128 + lane * 4;
    if (d < D) *reinterpret_cast<unsigned*>(data + at * D + d) = pack4(x[i], scale.inv);
  }
  if (lane == 0) scales[at] = scale.scale;
}

// ---- rows of a matrix [M, K] (row stride `stride`) -> codes [M, Kp], Kp = K rounded up to 16 with zeros, scales [M].
// A block a row; VECTORS > 0: the row stays in registers, 8 values a thread and vector; 0: it is read twice, value by
// value, for widths or strides that are no multiple of 8 or rows too long for the registers.
constexpr int ROWS_THREADS = 256;
template <typename T, int VECTORS>
__global__ void __launch_bounds__(ROWS_THREADS)
quantize_rows_kernel(const T* __restrict__ x, long long stride, signed char* __restrict__ codes,
                     float* __restrict__ scales, int K, int Kp, int early) {
  if (early) pdl_trigger();
  pdl_wait(x);
  __shared__ unsigned tops[ROWS_THREADS / 32];
  const long long row = blockIdx.x;
  const T* src = x + row * stride;
  signed char* dst = codes + row * Kp;
  float v[VECTORS > 0 ? VECTORS : 1][8];
  unsigned top = 0;
  if (VECTORS > 0) {
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const int at = (i * ROWS_THREADS + threadIdx.x) * 8;
      if (at < K) {
        load8<T, true>(src + at, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(v[i][j]));
      }
    }
  } else {
    for (int at = threadIdx.x; at < K; at += ROWS_THREADS) top = max(top, magnitude_bits(Elem<T>::load(src + at)));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ROWS_THREADS / 32; ++w) top = max(top, tops[w]);
  const RowScale s = row_scale(top);
  if (threadIdx.x == 0) scales[row] = s.scale;
  if (VECTORS > 0) {
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const int at = (i * ROWS_THREADS + threadIdx.x) * 8;
      if (at < K)
        *reinterpret_cast<uint2*>(dst + at) = make_uint2(pack4(v[i], s.inv), pack4(v[i] + 4, s.inv));
      else if (at < Kp)
        *reinterpret_cast<uint2*>(dst + at) = make_uint2(0, 0);
    }
  } else {
    for (int at = threadIdx.x; at < Kp; at += ROWS_THREADS)
      dst[at] = at < K ? (signed char)__float2int_rn(__fmul_rn(Elem<T>::load(src + at), s.inv)) : 0;
  }
}

template <typename T>
int launch_rows(const void* x, long long stride, void* codes, void* scales, long long M, int K, int Kp, int early,
                cudaStream_t st) {
  const T* p = reinterpret_cast<const T*>(x);
  signed char* c = reinterpret_cast<signed char*>(codes);
  float* s = reinterpret_cast<float*>(scales);
  const bool vec = K % 8 == 0 && stride % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int need = (Kp + ROWS_THREADS * 8 - 1) / (ROWS_THREADS * 8);
  auto kern = quantize_rows_kernel<T, 0>;
  if (vec && need <= 1) kern = quantize_rows_kernel<T, 1>;
  else if (vec && need <= 2) kern = quantize_rows_kernel<T, 2>;
  else if (vec && need <= 4) kern = quantize_rows_kernel<T, 4>;
  else if (vec && need <= 8) kern = quantize_rows_kernel<T, 8>;
  dib_launch(kern, dim3((unsigned)M), dim3(ROWS_THREADS), 0, st, p, stride, c, s, K, Kp, early);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

}  // namespace

extern "C" {

// k, v: rows [T] of Hkv * D values, `k_stride`, `v_stride` values apart (dtype 0 float32, 1 bfloat16); slots int32 [T]
// (page * page_size + offset; a negative one, or one beyond the pool, is skipped).
int dib_int8_cache_write(const void* k, const void* v, long long k_stride, long long v_stride, void* data, void* scales,
                         const void* slots, int T, int Hkv, int D, int page_size, long long num_pages, int dtype,
                         cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (T < 0 || Hkv < 1 || D < 16 || D > 256 || D % 16 != 0 || page_size < 1) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(data) & 15) != 0) return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const long long rows = (long long)T * 2 * Hkv;
  const long long blocks = (rows * ROW_LANES + CACHE_THREADS - 1) / CACHE_THREADS;
  if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
  const int per16 = dtype == 1 ? 8 : 4;
  const bool aligned = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                       k_stride % per16 == 0 && v_stride % per16 == 0;
  signed char* d = reinterpret_cast<signed char*>(data);
  float* s = reinterpret_cast<float*>(scales);
  const int* sl = reinterpret_cast<const int*>(slots);
  if (dtype == 1) {
    auto kern = aligned ? cache_write_kernel<__nv_bfloat16, true> : cache_write_kernel<__nv_bfloat16, false>;
    dib_launch(kern, dim3((unsigned)blocks), dim3(CACHE_THREADS), 0, st, reinterpret_cast<const __nv_bfloat16*>(k),
               reinterpret_cast<const __nv_bfloat16*>(v), k_stride, v_stride, d, s, sl, rows, Hkv, D, page_size, num_pages);
  } else {
    auto kern = aligned ? cache_write_kernel<float, true> : cache_write_kernel<float, false>;
    dib_launch(kern, dim3((unsigned)blocks), dim3(CACHE_THREADS), 0, st, reinterpret_cast<const float*>(k),
               reinterpret_cast<const float*>(v), k_stride, v_stride, d, s, sl, rows, Hkv, D, page_size, num_pages);
  }
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// qkv [T, (Hq + 2 Hkv) D] -> q_out [T, Hq, D] and the cache; q_norm_w, k_norm_w float32 [D] or null; cos_sin float32
// [max_pos, rotary_dim] = [cos | sin] or null; a token whose slot is none of the pool's keeps no key.
int dib_int8_qk_norm_rope_cache(const void* qkv, void* q_out, void* data, void* scales, const void* q_norm_w,
                                const void* k_norm_w, float eps, const void* cos_sin, int rotary_dim, int max_pos,
                                const void* positions, const void* slots, int T, int Hq, int Hkv, int D, int page_size,
                                long long num_pages, int dtype, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (T < 0 || Hq < 1 || Hkv < 1 || D < 16 || D > 256 || D % 16 != 0 || page_size < 1 || rotary_dim < 0 || rotary_dim > D ||
      rotary_dim % 2 != 0 || (cos_sin != nullptr && max_pos < 1))
    return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(data)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const long long blocks = ((long long)T * (Hq + 2 * Hkv) + QKV_WARPS - 1) / QKV_WARPS;
  if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
  const float *qw = reinterpret_cast<const float*>(q_norm_w), *kw = reinterpret_cast<const float*>(k_norm_w),
              *tab = reinterpret_cast<const float*>(cos_sin);
  const int *ps = reinterpret_cast<const int*>(positions), *sl = reinterpret_cast<const int*>(slots);
  signed char* d = reinterpret_cast<signed char*>(data);
  float* sc = reinterpret_cast<float*>(scales);
  if (dtype == 1)
    dib_launch(qk_norm_rope_cache_int8_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(QKV_WARPS * 32), 0, st,
               reinterpret_cast<const __nv_bfloat16*>(qkv), reinterpret_cast<__nv_bfloat16*>(q_out), d, sc, qw, kw, eps, tab,
               rotary_dim, max_pos, ps, sl, T, Hq, Hkv, D, page_size, num_pages);
  else
    dib_launch(qk_norm_rope_cache_int8_kernel<float>, dim3((unsigned)blocks), dim3(QKV_WARPS * 32), 0, st,
               reinterpret_cast<const float*>(qkv), reinterpret_cast<float*>(q_out), d, sc, qw, kw, eps, tab, rotary_dim, max_pos,
               ps, sl, T, Hq, Hkv, D, page_size, num_pages);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// k, v [T, Hkv, D] = the values that the rows in `slots` stand for; zeros for a slot that is none of the pool's.
int dib_int8_cache_read(const void* data, const void* scales, const void* slots, void* k, void* v, int T, int Hkv, int D,
                        int page_size, long long num_pages, int dtype, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (T < 0 || Hkv < 1 || D < 16 || D > 256 || D % 16 != 0 || page_size < 1) return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const long long rows = (long long)T * 2 * Hkv;
  const long long blocks = (rows * ROW_LANES + CACHE_THREADS - 1) / CACHE_THREADS;
  if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
  const signed char* d = reinterpret_cast<const signed char*>(data);
  const float* s = reinterpret_cast<const float*>(scales);
  const int* sl = reinterpret_cast<const int*>(slots);
  if (dtype == 1)
    dib_launch(cache_read_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(CACHE_THREADS), 0, st, d, s, sl,
               reinterpret_cast<__nv_bfloat16*>(k), reinterpret_cast<__nv_bfloat16*>(v), rows, Hkv, D, page_size, num_pages);
  else
    dib_launch(cache_read_kernel<float>, dim3((unsigned)blocks), dim3(CACHE_THREADS), 0, st, d, s, sl,
               reinterpret_cast<float*>(k), reinterpret_cast<float*>(v), rows, Hkv, D, page_size, num_pages);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// codes int8 [M, Kp] (Kp = K rounded up to 16, zeros behind K) and scales [M] of x [M, K], rows `stride` values apart.
// early: the kernel that follows may set itself up beside this one; 0 for a weight, which products read ahead of their
// wait for the kernel in front of them.
int dib_quantize_rows(const void* x, long long stride, void* codes, void* scales, long long M, int K, int dtype,
                      int early, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (M < 0 || M > 0x7fffffffll || K < 1 || K > (1 << 30)) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) != 0) return DIB_BAD_ALIGN;
  if (M == 0) return DIB_OK;
  const int Kp = (K + 15) / 16 * 16;
  if (dtype == 1) return launch_rows<__nv_bfloat16>(x, stride, codes, scales, M, K, Kp, early, st);
  return launch_rows<float>(x, stride, codes, scales, M, K, Kp, early, st);
}

}  // extern "C"
