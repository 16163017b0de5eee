// Rows in 8-bit integers: the one rule by which activations, weights, keys and values are quantised, a paged cache
// of quantised keys and values, and reading it back.
//
// A row (a token's activations, an output channel of a weight, a token's key or value of one head) of values x:
//   a = max(max |x|, 2^-100),  code = rint(x * (127 * (1 / a))) (ties to even),  scale = a * (1 / 127),
//   value = scale * code,
// every operation rounded to float32 by itself (what a division by, or of, a plain number is in torch), so the codes are
// the same on every path that makes them.  |x * (127 * (1 / a))| <= 127 (1 + 2^-22), which rounds to 127: no clamp.  The
// floor 2^-100 keeps 127 / a finite; rows below it read back as zeros, 2^-100 off at most.  A row that holds an infinity or
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
    r.inv = __fmul_rn(__frcp_rn(a), 127.f);
    r.scale = __fmul_rn(a, 1.f / 127.f);
  }
  return r;
}
__device__ __forceinline__ unsigned magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// the larger magnitude, a NaN if either is one
__device__ __forceinline__ float larger(float top, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(x)));
  return r;
}
// The codes in the low bytes: adding 1.5 * 2^23 to the product rounds it to an integer, ties to even, and leaves that in
// the low bits (a row with scale NaN has inv 0; what 0 * infinity gives there is cleared).
__device__ __forceinline__ unsigned code_bits(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f));
}
// four codes in a word, x0's in the low byte
__device__ __forceinline__ unsigned pack4(const float* x, float inv) {
  if (inv == 0.f) return 0;
  return __byte_perm(__byte_perm(code_bits(x[0], inv), code_bits(x[1], inv), 0x0040),
                     __byte_perm(code_bits(x[2], inv), code_bits(x[3], inv), 0x0040), 0x5410);
}
// four codes as numbers: a byte with its sign turned, under the exponent of 2^23, is 2^23 + 128 + code
__device__ __forceinline__ void unpack4(unsigned w, float scale, float* x) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = __fmul_rn(__fadd_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 + i)), -8388736.f), scale);
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
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

// 32 bytes of a row at once
template <typename T> struct Piece {
  static constexpr int N = 32 / (int)sizeof(T);        // values
  unsigned w[8];
  __device__ __forceinline__ void load(const T* p) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  }
  __device__ __forceinline__ void store(T* p) const {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  }
  __device__ __forceinline__ float get(int e) const {
    if (sizeof(T) == 4) return __uint_as_float(w[e & 7]);
    return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
};
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

// A row of the cache: 128 values are LANES lanes, 32 bytes of the unquantised row each.  Memory bound: many warps of few
// registers and few instructions: 8,000 tokens of 8 heads of 128 written from bfloat16 and read back in 19.4 us, 99 MB at
// 5.1 TB/s (16 values a lane of several rows a group: 93 registers, 37 us).
constexpr int CACHE_THREADS = 256;
template <typename T> struct Rows {
  static constexpr int N = Piece<T>::N, LANES = 128 / N, GROUPS = CACHE_THREADS / LANES;
};
struct CacheShape {
  Divisor per_token, page;      // 2 Hkv rows a token, rows a page
  unsigned rows;
  int Hkv, D;
  unsigned num_pages;
};
struct CacheRow {
  long long at;      // row of the cache, or -1
  int token, kv, h;
};
// row r = (token, key or value, kv head)
__device__ __forceinline__ CacheRow cache_row(unsigned r, const CacheShape& s, const int* slots) {
  CacheRow c;
  c.at = -1;
  c.token = (int)quotient(r, s.per_token);
  const int rest = (int)(r - (unsigned)c.token * s.per_token.d);
  c.kv = rest >= s.Hkv;
  c.h = rest - c.kv * s.Hkv;
  if (r >= s.rows) return c;
  const int slot = slots[c.token];
  if (slot < 0) return c;
  const unsigned page = quotient((unsigned)slot, s.page);
  if (page < s.num_pages) c.at = ((long long)page * s.per_token.d + rest) * s.page.d + (slot - (int)(page * s.page.d));
  return c;
}

template <typename T, bool ALIGNED, int HALVES>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_write_kernel(const T* __restrict__ k, const T* __restrict__ v, long long k_stride, long long v_stride,
                   signed char* __restrict__ data, float* __restrict__ scales, const int* __restrict__ slots,
                   const __grid_constant__ CacheShape s) {
  using R = Rows<T>;
  pdl_prologue(k, v, slots);
  const int l = threadIdx.x & (R::LANES - 1);
  const CacheRow c = cache_row(blockIdx.x * R::GROUPS + threadIdx.x / R::LANES, s, slots);
  const T* src = (c.kv ? v + c.token * v_stride : k + c.token * k_stride) + c.h * s.D;
  Piece<T> x[HALVES];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < HALVES; ++i) {
    const int d = i * 128 + l * R::N;
    const bool in = c.at >= 0 && d < s.D;
    if (ALIGNED) {
      if (in) x[i].load(src + d);
    } else if (in) {
      T* to = reinterpret_cast<T*>(x[i].w);
#pragma unroll
      for (int e = 0; e < R::N; ++e) to[e] = src[d + e];
    }
    if (in)
#pragma unroll
      for (int e = 0; e < R::N; ++e) top = larger(top, x[i].get(e));
  }
#pragma unroll
  for (int o = R::LANES / 2; o > 0; o >>= 1) top = larger(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (c.at < 0) return;
  const RowScale scale = row_scale(__float_as_uint(top));
#pragma unroll
  for (int i = 0; i < HALVES; ++i) {
    const int d = i * 128 + l * R::N;
    if (d >= s.D) break;
    unsigned y[R::N / 4];
#pragma unroll
    for (int e = 0; e < R::N; e += 4) {
      const float four[4] = {x[i].get(e), x[i].get(e + 1), x[i].get(e + 2), x[i].get(e + 3)};
      y[e / 4] = pack4(four, scale.inv);
    }
    signed char* dst = data + c.at * s.D + d;
    if (R::N == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(y[0], y[1], y[R::N / 4 - 2], y[R::N / 4 - 1]);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(y[0], y[1]);
  }
  if (l == 0) scales[c.at] = scale.scale;
}

// ROWS rows a group, all asked for before the first is used: 194 MB of float32, most of it read back, in 36.0 us (5.4 TB/s) at
// 2, 42.0 at 1, 40.6 at 4.
template <typename T, int HALVES, int ROWS>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_read_kernel(const signed char* __restrict__ data, const float* __restrict__ scales, const int* __restrict__ slots,
                  T* __restrict__ k, T* __restrict__ v, const __grid_constant__ CacheShape s) {
  using R = Rows<T>;
  pdl_prologue(data, scales, slots);
  const int l = threadIdx.x & (R::LANES - 1);
  const unsigned r0 = blockIdx.x * (R::GROUPS * ROWS) + threadIdx.x / R::LANES;
  CacheRow c[ROWS];
  float scale[ROWS];
  unsigned w[ROWS][HALVES][R::N / 4];
#pragma unroll
  for (int g = 0; g < ROWS; ++g) c[g] = cache_row(r0 + g * R::GROUPS, s, slots);
#pragma unroll
  for (int g = 0; g < ROWS; ++g) {
    scale[g] = c[g].at >= 0 ? scales[c[g].at] : 0.f;
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
      const int d = i * 128 + l * R::N;
#pragma unroll
      for (int e = 0; e < R::N / 4; ++e) w[g][i][e] = 0;
      if (c[g].at >= 0 && d < s.D) {
        const signed char* src = data + c[g].at * s.D + d;
        if (R::N == 16) {
          const uint4 q = *reinterpret_cast<const uint4*>(src);
          w[g][i][0] = q.x; w[g][i][1] = q.y; w[g][i][R::N / 4 - 2] = q.z; w[g][i][R::N / 4 - 1] = q.w;
        } else {
          const uint2 q = *reinterpret_cast<const uint2*>(src);
          w[g][i][0] = q.x; w[g][i][1] = q.y;
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < ROWS; ++g) {
    if (r0 + g * R::GROUPS >= s.rows) return;
    T* dst = (c[g].kv ? v : k) + ((long long)c[g].token * s.Hkv + c[g].h) * s.D;
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
      const int d = i * 128 + l * R::N;
      if (d >= s.D) break;
      Piece<T> y;
#pragma unroll
      for (int e = 0; e < R::N / 4; ++e) {
        float x[4];
        unpack4(w[g][i][e], scale[g], x);
        if (sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < 4; ++j) y.w[(e * 4 + j) & 7] = __float_as_uint(x[j]);
        } else {
          const __nv_bfloat162 p = __floats2bfloat162_rn(x[0], x[1]), q = __floats2bfloat162_rn(x[2], x[3]);
          y.w[(e * 2) & 7] = *reinterpret_cast<const unsigned*>(&p);
          y.w[(e * 2 + 1) & 7] = *reinterpret_cast<const unsigned*>(&q);
        }
      }
      y.store(dst + d);
    }
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
template <typename T, int VECTORS, int THREADS>
__global__ void __launch_bounds__(THREADS)
quantize_rows_kernel(const T* __restrict__ x, long long stride, signed char* __restrict__ codes,
                     float* __restrict__ scales, int K, int Kp) {
  pdl_prologue(x);
  __shared__ unsigned tops[THREADS / 32];
  const long long row = blockIdx.x;
  const T* src = x + row * stride;
  signed char* dst = codes + row * Kp;
  float v[VECTORS > 0 ? VECTORS : 1][8];
  unsigned top = 0;
  if (VECTORS > 0) {
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const int at = (i * THREADS + threadIdx.x) * 8;
      if (at < K) {
        load8<T>(src + at, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(v[i][j]));
      }
    }
  } else {
    for (int at = threadIdx.x; at < K; at += THREADS) top = max(top, magnitude_bits(Elem<T>::load(src + at)));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = max(top, tops[w]);
  const RowScale s = row_scale(top);
  if (threadIdx.x == 0) scales[row] = s.scale;
  if (VECTORS > 0) {
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const int at = (i * THREADS + threadIdx.x) * 8;
      if (at < K)
        *reinterpret_cast<uint2*>(dst + at) = make_uint2(pack4(v[i], s.inv), pack4(v[i] + 4, s.inv));
      else if (at < Kp)
        *reinterpret_cast<uint2*>(dst + at) = make_uint2(0, 0);
    }
  } else {
    for (int at = threadIdx.x; at < Kp; at += THREADS)
      dst[at] = at < K ? (signed char)__float2int_rn(__fmul_rn(Elem<T>::load(src + at), s.inv)) : 0;
  }
}

CacheShape make_shape(long long rows, int Hkv, int D, int page_size, long long num_pages) {
  CacheShape s;
  s.per_token = make_divisor(2u * Hkv);
  s.page = make_divisor((unsigned)page_size);
  s.rows = (unsigned)rows;
  s.Hkv = Hkv; s.D = D;
  s.num_pages = (unsigned)num_pages;
  return s;
}
template <typename T>
int launch_write(const void* k, const void* v, long long k_stride, long long v_stride, signed char* data, float* scales,
                 const int* slots, const CacheShape& s, cudaStream_t st) {
  constexpr int GROUPS = Rows<T>::GROUPS;
  const bool wide = s.D > 128;
  const bool aligned = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 31) == 0 &&
                       (k_stride * sizeof(T)) % 32 == 0 && (v_stride * sizeof(T)) % 32 == 0 && (s.D * sizeof(T)) % 32 == 0;
  auto kern = wide ? (aligned ? cache_write_kernel<T, true, 2> : cache_write_kernel<T, false, 2>)
                   : (aligned ? cache_write_kernel<T, true, 1> : cache_write_kernel<T, false, 1>);
  dib_launch(kern, dim3((s.rows + GROUPS - 1) / GROUPS), dim3(CACHE_THREADS), 0, st, reinterpret_cast<const T*>(k),
             reinterpret_cast<const T*>(v), k_stride, v_stride, data, scales, slots, s);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}
template <typename T>
int launch_read(const signed char* data, const float* scales, const int* slots, void* k, void* v, const CacheShape& s,
                cudaStream_t st) {
  constexpr int GROUPS = Rows<T>::GROUPS;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 31) != 0) return DIB_BAD_ALIGN;
  constexpr int ROWS = 2;
  dib_launch(s.D > 128 ? cache_read_kernel<T, 2, ROWS> : cache_read_kernel<T, 1, ROWS>,
             dim3((s.rows + GROUPS * ROWS - 1) / (GROUPS * ROWS)), dim3(CACHE_THREADS), 0, st, data, scales, slots, reinterpret_cast<T*>(k), reinterpret_cast<T*>(v), s);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

template <typename T>
int launch_rows(const void* x, long long stride, void* codes, void* scales, long long M, int K, int Kp, cudaStream_t st) {
  const T* p = reinterpret_cast<const T*>(x);
  signed char* c = reinterpret_cast<signed char*>(codes);
  float* s = reinterpret_cast<float*>(scales);
  const bool vec = K % 8 == 0 && stride % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  // (256 threads a row: 2,048 rows of 4,096 6.0 us, with 512 7.4; of 12,288 24.1 and 22.5, 8 of those 2.6 and 2.0)
  const int threads = Kp > 8192 ? 512 : 256, need = (Kp + threads * 8 - 1) / (threads * 8);
  auto kern = quantize_rows_kernel<T, 0, 256>;
  bool wide = false;
  if (vec && threads == 256) {
    kern = need <= 1 ? quantize_rows_kernel<T, 1, 256> : need <= 2 ? quantize_rows_kernel<T, 2, 256> : quantize_rows_kernel<T, 4, 256>;
  } else if (vec && need <= 8) {
    kern = need <= 4 ? quantize_rows_kernel<T, 4, 512> : quantize_rows_kernel<T, 8, 512>;
    wide = true;
  }
  dib_launch(kern, dim3((unsigned)M), dim3(wide ? 512 : 256), 0, st, p, stride, c, s, K, Kp);
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
  if (rows > 0x7fffff00ll || num_pages > 0x7fffffffll) return DIB_BAD_SIZE;
  const CacheShape shape = make_shape(rows, Hkv, D, page_size, num_pages);
  signed char* d = reinterpret_cast<signed char*>(data);
  float* s = reinterpret_cast<float*>(scales);
  const int* sl = reinterpret_cast<const int*>(slots);
  if (dtype == 1)
    return launch_write<__nv_bfloat16>(k, v, k_stride, v_stride, d, s, sl, shape, st);
  return launch_write<float>(k, v, k_stride, v_stride, d, s, sl, shape, st);
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
  if (rows > 0x7fffff00ll || num_pages > 0x7fffffffll) return DIB_BAD_SIZE;
  const signed char* d = reinterpret_cast<const signed char*>(data);
  const float* s = reinterpret_cast<const float*>(scales);
  const int* sl = reinterpret_cast<const int*>(slots);
  const CacheShape shape = make_shape(rows, Hkv, D, page_size, num_pages);
  if (dtype == 1) return launch_read<__nv_bfloat16>(d, s, sl, k, v, shape, st);
  return launch_read<float>(d, s, sl, k, v, shape, st);
}

// codes int8 [M, Kp] (Kp = K rounded up to 16, zeros behind K) and scales [M] of x [M, K], rows `stride` values apart.
int dib_quantize_rows(const void* x, long long stride, void* codes, void* scales, long long M, int K, int dtype,
                      cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (M < 0 || M > 0x7fffffffll || K < 1 || K > (1 << 30)) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) != 0) return DIB_BAD_ALIGN;
  if (M == 0) return DIB_OK;
  const int Kp = (K + 15) / 16 * 16;
  if (dtype == 1) return launch_rows<__nv_bfloat16>(x, stride, codes, scales, M, K, Kp, st);
  return launch_rows<float>(x, stride, codes, scales, M, K, Kp, st);
}

}  // extern "C"
