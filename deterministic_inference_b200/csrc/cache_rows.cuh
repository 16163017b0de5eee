// What the kernels share that write and read a paged cache of quantised rows, whatever the rows' format: a cache's shape with divisions
// by products, and the norm and rotation of the fused projection's rows in front of their quantising.
#pragma once

#include "common.cuh"

// n / d for n < 2^31 by a product: d's reciprocal rounded up, with as many bits as make that exact
struct Divisor {
  unsigned mul, shift, d;
};
__device__ __forceinline__ unsigned quotient(unsigned n, const Divisor& v) {
  return v.mul == 0 ? n >> v.shift : __umulhi(n, v.mul) >> v.shift;
}
static inline Divisor make_divisor(unsigned d) {
  Divisor v;
  v.d = d;
  unsigned log = 0;
  while ((1ull << log) < d) ++log;
  if ((1u << log) == d) {
    v.mul = 0;
    v.shift = log;
  } else {      // n < 2^31: floor(n m / 2^(31 + log)) with m = ceil(2^(31 + log) / d) < 2^32 is exact
    v.mul = (unsigned)(((1ull << (31 + log)) + d - 1) / d);
    v.shift = log - 1;
  }
  return v;
}

struct CacheShape {
  Divisor per_token, page;      // 2 Hkv rows a token, rows a page
  unsigned rows;
  int Hkv, D;
  unsigned num_pages;
};
static inline CacheShape make_shape(long long rows, int Hkv, int D, int page_size, long long num_pages) {
  CacheShape s;
  s.per_token = make_divisor(2u * Hkv);
  s.page = make_divisor((unsigned)page_size);
  s.rows = (unsigned)rows;
  s.Hkv = Hkv; s.D = D;
  s.num_pages = (unsigned)num_pages;
  return s;
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

// The rows of the step's fused projection [q heads | k heads | v heads]: a warp has one (src, D values), a lane 4 consecutive values of
// 128 at a time.  Normed (RMS) where nw is given, rotated by the position's row of the table where `rotate`, rounded to T: the
// norm's sum and the rotation are those of the kernels that write an unquantised cache.  The rotation's pairs meet in `s`,
// 256 floats of the warp's own.
template <typename T>
__device__ __forceinline__ void norm_rope_row(const T* src, float* s, const float* nw, float eps, bool rotate, const float* cos_sin,
                                              int rotary_dim, int max_pos, const int* positions, int t, int D, float (&x)[2][4]) {
  const int lane = threadIdx.x & 31;
  float squares[2];
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
  if (rotate) {
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
}
