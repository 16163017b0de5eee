// A paged cache of keys and values in 4-bit floating point (fp4.cuh has the rule; a row is a token's key or value of one head): writing
// it, from keys and values or from the step's fused projection, and reading it back, by slots or as bfloat16 pages for the
// prompt attention.
//
// Cache: data [pages, 2, Hkv, page_size, D / 2] (two codes a byte, the first in the low half), scales e4m3
// [pages, 2, Hkv, page_size, D / 16], exponents [pages, 2, Hkv, page_size] (E + 127).  128 values take 73 bytes.
//
// A lane has a block of 16 values: 32 (64) bytes of the unquantised row, 8 bytes of codes, a scale; of bfloat16 rows two such.  float32
// rows are bound by memory (8,000 tokens of 8 heads of 128 written in 14.7 us, 5.1 TB/s; read in 13.2, 5.7 TB/s; a floor of
// 11.4 at 6.55 TB/s), bfloat16 ones by what a row takes beside its values, its place, largest value and three outputs (10.1 us,
// 4.2 TB/s; read in 8.7; a floor of 6.4).
#include "cache_rows.cuh"
#include "fp4.cuh"

namespace {

constexpr int CACHE_THREADS = 256;
struct Cache4 {
  unsigned char* data;
  unsigned char* scales;
  unsigned char* exponents;
};

// A block of threads has one head's keys or values of PER consecutive tokens, so that what a page holds of them side by side is
// written and read side by side.
struct Place {
  long long at;      // row of the cache, or -1
  int token;
};
struct BlockOf {
  int kv, h, token0;
};
__device__ __forceinline__ BlockOf block_of(int per, const CacheShape& s) {
  BlockOf b;
  const unsigned t = quotient(blockIdx.x, s.per_token), rest = blockIdx.x - t * s.per_token.d;
  b.kv = rest >= (unsigned)s.Hkv;
  b.h = (int)rest - b.kv * s.Hkv;
  b.token0 = (int)t * per;
  return b;
}
__device__ __forceinline__ Place place(const BlockOf& b, int token, int tokens, const CacheShape& s, const int* slots) {
  Place c;
  c.at = -1;
  c.token = token;
  if (token >= tokens) return c;
  const int slot = slots[token];
  if (slot < 0) return c;
  const unsigned page = quotient((unsigned)slot, s.page);
  if (page < s.num_pages)
    c.at = ((long long)page * s.per_token.d + b.kv * s.Hkv + b.h) * s.page.d + (slot - (int)(page * s.page.d));
  return c;
}

// A lane has BLOCKS blocks of 16 side by side; ROWS rows a group, all asked for before the first is used.
template <typename T, bool WIDE, int LANES, int BLOCKS, int ROWS>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_write_kernel(const T* __restrict__ k, const T* __restrict__ v, long long k_stride, long long v_stride,
                   const __grid_constant__ Cache4 cache, const int* __restrict__ slots, int tokens, const __grid_constant__ CacheShape s) {
  constexpr int GROUPS = CACHE_THREADS / LANES;
  pdl_prologue(k, v, slots);
  const int d = (threadIdx.x & (LANES - 1)) * BLOCKS * 16;
  const BlockOf b = block_of(GROUPS * ROWS, s);
  const T* from = (b.kv ? v : k) + b.h * s.D;
  const long long stride = b.kv ? v_stride : k_stride;
  Place c[ROWS];
  Block16<T> x[ROWS][BLOCKS];
#pragma unroll
  for (int g = 0; g < ROWS; ++g) c[g] = place(b, b.token0 + g * GROUPS + threadIdx.x / LANES, tokens, s, slots);
#pragma unroll
  for (int g = 0; g < ROWS; ++g)
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) x[g][i].template load<WIDE>(from + c[g].token * stride, c[g].at >= 0 ? d + i * 16 : s.D, s.D);
#pragma unroll
  for (int g = 0; g < ROWS; ++g) {
    unsigned own[BLOCKS], top = 0;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      own[i] = x[g][i].top();
      top = max(top, own[i]);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (c[g].at < 0 || d >= s.D) continue;
    const unsigned exponent = fp4_row_exponent(top);
    const float down = fp4_down(exponent);
    unsigned w[2 * BLOCKS], scales = 0;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      const unsigned scale = fp4_block_scale(own[i], down);
      const Fp4Scaler q = fp4_scaler(scale, down);
      float y[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = x[g][i].get(e);
      w[2 * i] = fp4_codes8(y, q);
      w[2 * i + 1] = fp4_codes8(y + 8, q);
      scales |= scale << (8 * i);
    }
    unsigned char* codes = cache.data + c[g].at * (s.D / 2) + d / 2;
    unsigned char* tile = cache.scales + c[g].at * (s.D / 16) + d / 16;
    if (BLOCKS == 2) {
      *reinterpret_cast<uint4*>(codes) = make_uint4(w[0], w[1], w[2 * BLOCKS - 2], w[2 * BLOCKS - 1]);
      *reinterpret_cast<unsigned short*>(tile) = (unsigned short)scales;
    } else {
      *reinterpret_cast<uint2*>(codes) = make_uint2(w[0], w[1]);
      *tile = (unsigned char)scales;
    }
    if (d == 0) cache.exponents[c[g].at] = (unsigned char)exponent;
  }
}

// a block of 16 of the row at `at` as numbers; zeros for a row that is not there
struct Held16 {
  uint2 w;
  unsigned scale, exponent;
  __device__ __forceinline__ void load(const Cache4& cache, long long at, int l, int D) {
    w = make_uint2(0, 0);
    scale = exponent = 0;
    if (at >= 0 && l * 16 < D) {
      w = *reinterpret_cast<const uint2*>(cache.data + at * (D / 2) + l * 8);
      scale = cache.scales[at * (D / 16) + l];
      exponent = cache.exponents[at];
    }
  }
  __device__ __forceinline__ void values(float (&x)[16]) const {
    const float b = fp4_scale_value(scale), unit = fp4_unit(exponent);
    fp4_values8(w.x, b, x);
    fp4_values8(w.y, b, x + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= unit;
  }
};

// As above.
template <typename T, int LANES, int BLOCKS, int ROWS>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_read_kernel(const __grid_constant__ Cache4 cache, const int* __restrict__ slots, T* __restrict__ k, T* __restrict__ v,
                  int tokens, const __grid_constant__ CacheShape s) {
  constexpr int GROUPS = CACHE_THREADS / LANES;
  Cache4 held = cache;
  pdl_prologue(held.data, held.scales, held.exponents, slots);
  const int d = (threadIdx.x & (LANES - 1)) * BLOCKS * 16;
  const BlockOf b = block_of(GROUPS * ROWS, s);
  T* to = (b.kv ? v : k) + b.h * s.D + d;
  Place c[ROWS];
  Held16 x[ROWS][BLOCKS];
#pragma unroll
  for (int g = 0; g < ROWS; ++g) c[g] = place(b, b.token0 + g * GROUPS + threadIdx.x / LANES, tokens, s, slots);
#pragma unroll
  for (int g = 0; g < ROWS; ++g) {
    if (BLOCKS == 2) {
      uint4 w = make_uint4(0, 0, 0, 0);
      unsigned scales = 0, exponent = 0;
      if (c[g].at >= 0 && d < s.D) {
        w = *reinterpret_cast<const uint4*>(held.data + c[g].at * (s.D / 2) + d / 2);
        scales = *reinterpret_cast<const unsigned short*>(held.scales + c[g].at * (s.D / 16) + d / 16);
        exponent = held.exponents[c[g].at];
      }
      x[g][0] = {make_uint2(w.x, w.y), scales & 255, exponent};
      x[g][BLOCKS - 1] = {make_uint2(w.z, w.w), scales >> 8, exponent};
    } else {
      x[g][0].load(held, c[g].at, d / 16, s.D);
    }
  }
#pragma unroll
  for (int g = 0; g < ROWS; ++g) {
    if (c[g].token >= tokens || d >= s.D) return;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      float y[16];
      x[g][i].values(y);
      store16(to + (long long)c[g].token * s.Hkv * s.D + i * 16, y);
    }
  }
}

// The step's fused projection rows [q heads | k heads | v heads]: q and k normed and rotated, q to its output, k and v rounded to T,
// quantised and written to the token's slot.  A warp a (token, head), a lane 4 consecutive elements of 128 at a time: a block
// of 16 is four lanes.
// (32 / 8 heads of 128: 8 tokens 3.0 us, 2,048 tokens 41, bound by instructions.)
constexpr int QKV_WARPS = 4;
template <typename T>
__global__ void __launch_bounds__(QKV_WARPS * 32)
qk_norm_rope_cache_kernel(const T* __restrict__ qkv, T* __restrict__ q_out, const __grid_constant__ Cache4 cache,
                          const float* __restrict__ q_norm_w, const float* __restrict__ k_norm_w, float eps,
                          const float* __restrict__ cos_sin, int rotary_dim, int max_pos, const int* __restrict__ positions,
                          const int* __restrict__ slots, int T_tokens, int Hq, int Hkv, int D, int page_size, long long num_pages) {
  pdl_prologue(qkv, q_norm_w, k_norm_w);
  __shared__ float row[QKV_WARPS][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = Hq + 2 * Hkv;
  const long long item = (long long)blockIdx.x * QKV_WARPS + warp;
  if (item >= (long long)T_tokens * heads) return;
  const int t = (int)(item / heads), head = (int)(item - (long long)t * heads);
  const bool is_q = head < Hq, is_k = !is_q && head < Hq + Hkv;
  const int slot = is_q ? 0 : slots[t];
  const long long page = slot < 0 ? -1 : slot / page_size;
  if (!is_q && (page < 0 || page >= num_pages)) return;
  float x[2][4];
  norm_rope_row<T>(qkv + item * D, row[warp], is_q ? q_norm_w : is_k ? k_norm_w : nullptr, eps, cos_sin != nullptr && (is_q || is_k),
                   cos_sin, rotary_dim, max_pos, positions, t, D, x);
  if (is_q) {
    T* dst = q_out + ((long long)t * Hq + head) * D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = i * 128 + lane * 4;
      if (d < D) store4<T>(dst + d, x[i]);
    }
    return;
  }
  unsigned own[2] = {0, 0};      // of the lane's blocks
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) own[i] = max(own[i], fp4_magnitude(x[i][e]));
    own[i] = max(own[i], __shfl_xor_sync(0xffffffffu, own[i], 1));
    own[i] = max(own[i], __shfl_xor_sync(0xffffffffu, own[i], 2));
  }
  const unsigned exponent = fp4_row_exponent(__reduce_max_sync(0xffffffffu, max(own[0], own[1])));
  const float down = fp4_down(exponent);
  const int kv = !is_k, h = is_k ? head - Hq : head - Hq - Hkv;
  const long long at = ((page * 2 + kv) * Hkv + h) * page_size + (slot - page * page_size);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = i * 128 + lane * 4;
    if (d >= D) break;
    const unsigned scale = fp4_block_scale(own[i], down);
    const Fp4Scaler q = fp4_scaler(scale, down);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = fp4_quotient(x[i][e], q);
    *reinterpret_cast<unsigned short*>(cache.data + at * (D / 2) + d / 2) = (unsigned short)(q.inv == 0.f ? 0 : fp4_pack4(y));
    if ((lane & 3) == 0) cache.scales[at * (D / 16) + d / 16] = (unsigned char)scale;
  }
  if (lane == 0) cache.exponents[at] = (unsigned char)exponent;
}

// ---- the keys and values of some sequences as bfloat16 pages of their own, [pages, 2, Hkv, PAGE, D], for attention over an unquantised
// cache: what 4 bits stand for has 6 digits, so that bfloat16 holds it exactly.  Sequence number i of the launch, seq_list[i],
// has its pages from first_page[i] on, one for every PAGE keys up to the host's bound of its length.  Keys behind its real length,
// those that are on no page of the pool, and those of which the key or the value is no number, are zeros up to the page's end;
// pages wholly behind the last key, or ahead of the window of the first new token, are left as they are.  (The new block table
// follows from the bounds: the host makes it.)  Bound by memory: 32,000 tokens of 8 heads of 128 in 35 us, 4.8 TB/s; 4,096 in 8.1.
constexpr int UNPACK_PAGE = 128;      // (the host lists as many: kernels/fp4.py)
struct UnpackArgs {
  Cache4 cache;
  const int* block_table;
  const int* cu_q_lens;
  const int* seq_lens;
  const int* seq_list;      // [count]
  const int* first_page;    // [count + 1]
  __nv_bfloat16* out;
  int max_blocks, Hkv, D, page_size, window;
  long long num_pages;
};
template <int LANES>
__global__ void __launch_bounds__(CACHE_THREADS)
unpack_pages_kernel(const __grid_constant__ UnpackArgs a) {
  Cache4 held = a.cache;
  pdl_prologue(held.data, held.scales, held.exponents);
  const int seq = a.seq_list[blockIdx.z], page = blockIdx.x, rows = blockIdx.y;      // rows: (keys or values, head)
  const int first_page = a.first_page[blockIdx.z], bound = a.first_page[blockIdx.z + 1] - first_page;
  if (page >= bound) return;
  const int kv_len = (int)min((long long)a.seq_lens[seq], (long long)a.max_blocks * a.page_size);
  const int first = first_visible_key(max(kv_len - (a.cu_q_lens[seq + 1] - a.cu_q_lens[seq]), 0), a.window);
  const int key0 = page * UNPACK_PAGE;
  if (key0 >= kv_len || key0 + UNPACK_PAGE <= first) return;
  constexpr int GROUPS = CACHE_THREADS / LANES, ROWS = 2;
  const int l = threadIdx.x % LANES;
  if (l * 16 >= a.D) return;
  const int* table = a.block_table + (long long)seq * a.max_blocks;
  __nv_bfloat16* out = a.out + ((long long)(first_page + page) * 2 * a.Hkv + rows) * UNPACK_PAGE * a.D + l * 16;
#pragma unroll 1
  for (int r0 = threadIdx.x / LANES; r0 < UNPACK_PAGE; r0 += GROUPS * ROWS) {
    Held16 x[ROWS];
#pragma unroll
    for (int g = 0; g < ROWS; ++g) {
      const int key = key0 + r0 + g * GROUPS;
      long long at = -1;
      if (key < kv_len) {
        const int of = key / a.page_size, p = table[of];
        if (p >= 0 && p < a.num_pages) at = ((long long)p * 2 * a.Hkv + rows) * a.page_size + (key - of * a.page_size);
      }
      x[g].load(held, at, l, a.D);
      if (at >= 0 && max(x[g].exponent, (unsigned)held.exponents[at + (rows < a.Hkv ? a.Hkv : -a.Hkv) * a.page_size]) == FP4_NO_NUMBER)
        x[g].load(held, -1, l, a.D);
    }
#pragma unroll
    for (int g = 0; g < ROWS; ++g) {
      float y[16];
      x[g].values(y);
      store16(out + (long long)(r0 + g * GROUPS) * a.D, y);
    }
  }
}

// What the attention over the pages made above leaves open, a launch behind it (32,000 keys of 8 heads 1.7 us): the new tokens in front of the first key (a sequence
// with fewer keys than new tokens) are zeros; those that see a key whose row, or whose value's, is no number are none either.  (As such
// numbers in the pages they would reach rows that do not see them, by way of probabilities of zero.)  A block looks through the
// exponents of FINISH_KEYS keys of a kv head.
constexpr int FINISH_KEYS = 4096;
__global__ void __launch_bounds__(CACHE_THREADS)
finish_portions_kernel(const __grid_constant__ UnpackArgs a, int Hq) {
  __shared__ unsigned bits[FINISH_KEYS / 32];
  constexpr int EACH = FINISH_KEYS / (4 * CACHE_THREADS);
  pdl_trigger();
  // (the step's metadata, which no kernel of a step writes, ahead of the wait)
  const int seq = a.seq_list[blockIdx.z], q_begin = a.cu_q_lens[seq], n = a.cu_q_lens[seq + 1] - q_begin, kvh = blockIdx.y;
  const int kv_len = (int)max(min((long long)a.seq_lens[seq], (long long)a.max_blocks * a.page_size), 0ll);
  const int p0 = kv_len - n, key0 = blockIdx.x * FINISH_KEYS, G = Hq / a.Hkv;
  // four keys a thread, on one page
  const int* table = a.block_table + (long long)seq * a.max_blocks;
  long long at[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int key = key0 + (i * CACHE_THREADS + threadIdx.x) * 4, of = key / a.page_size;
    const int page = key < kv_len ? table[of] : -1;
    at[i] = page < 0 || page >= a.num_pages ? -1 : ((long long)page * 2 * a.Hkv + kvh) * a.page_size + (key - of * a.page_size);
  }
  const unsigned char* exponents = a.cache.exponents;
  __nv_bfloat16* out = a.out;
  pdl_wait(exponents, out);
  if (blockIdx.x == 0 && kvh == 0) {
    const long long pieces = (long long)max(-p0, 0) * Hq * (a.D / 8);      // of 16 bytes
    uint4* to = reinterpret_cast<uint4*>(out + (long long)q_begin * Hq * a.D);
    for (long long i = threadIdx.x; i < pieces; i += CACHE_THREADS) to[i] = make_uint4(0, 0, 0, 0);
  }
  const int first = first_visible_key(max(p0, 0), a.window);
  if (key0 >= kv_len || key0 + FINISH_KEYS <= first) return;
  if (threadIdx.x < FINISH_KEYS / 32) bits[threadIdx.x] = 0;
  __syncthreads();
  unsigned found[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    unsigned keys = 0, values = 0;
    if (at[i] >= 0) {
      keys = *reinterpret_cast<const unsigned*>(exponents + at[i]);
      values = *reinterpret_cast<const unsigned*>(exponents + at[i] + (long long)a.Hkv * a.page_size);
    }
    const unsigned both = __vcmpeq4(keys, 0xffffffffu) | __vcmpeq4(values, 0xffffffffu);
    const int left = kv_len - (key0 + (i * CACHE_THREADS + threadIdx.x) * 4);      // keys that there are
    found[i] = (both & 1) | (both >> 7 & 2) | (both >> 14 & 4) | (both >> 21 & 8);
    if (left < 4) found[i] &= left <= 0 ? 0 : (1u << left) - 1;
  }
  unsigned any = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) any |= found[i];
  if (!__syncthreads_or(any)) return;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int k = (i * CACHE_THREADS + threadIdx.x) * 4;
    if (found[i]) atomicOr(&bits[k >> 5], found[i] << (k & 31));
  }
  __syncthreads();
  // a warp a token
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n; i += CACHE_THREADS / 32) {
    const int pos = p0 + i;
    if (pos < key0) continue;
    const int lo = max(first_visible_key(pos, a.window) - key0, 0), hi = pos - key0;      // of the block's keys
    unsigned hit = 0;
#pragma unroll
    for (int w = lane; w < FINISH_KEYS / 32; w += 32) {
      const int from = lo - w * 32, to = hi - w * 32;      // bits from .. to
      if (from < 32 && to >= 0) hit |= bits[w] & (0xffffffffu << max(from, 0)) & (0xffffffffu >> max(31 - to, 0));
    }
    if (!__any_sync(0xffffffffu, hit != 0)) continue;
    uint4* row = reinterpret_cast<uint4*>(out + ((long long)(q_begin + i) * Hq + kvh * G) * a.D);
    for (int e = lane; e < G * a.D / 8; e += 32) row[e] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  }
}

// Two blocks of 16 a lane: bfloat16, rows and scales that allow it.  (8,000 tokens of 8 heads of 128 written, read: 10.1, 8.7 us, with one
// 11.3, 9.2; float32 15.8, 17.4 with two and 14.7, 13.2 with one, then two rows a lane for reading.)
template <typename T> bool two_blocks(const Cache4& cache, int D) {
  return sizeof(T) == 2 && (D & 31) == 0 && (reinterpret_cast<uintptr_t>(cache.scales) & 1) == 0;
}

template <typename T>
int launch_write(const void* k, const void* v, long long k_stride, long long v_stride, const Cache4& cache, const int* slots,
                 int tokens, const CacheShape& s, cudaStream_t st) {
  const bool wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 31) == 0 &&
                    (k_stride * sizeof(T)) % 32 == 0 && (v_stride * sizeof(T)) % 32 == 0;
  const bool two = two_blocks<T>(cache, s.D);
  const int per = CACHE_THREADS / ((s.D > 128 ? 16 : 8) >> two);
  constexpr int TWO = sizeof(T) == 2 ? 2 : 1, NARROW = 8 / TWO, BROAD = 16 / TWO;
  auto kern = two          ? s.D > 128 ? wide ? cache_write_kernel<T, true, BROAD, TWO, 1> : cache_write_kernel<T, false, BROAD, TWO, 1>
                             : wide    ? cache_write_kernel<T, true, NARROW, TWO, 1>
                                       : cache_write_kernel<T, false, NARROW, TWO, 1>
              : s.D > 128  ? wide ? cache_write_kernel<T, true, 16, 1, 1> : cache_write_kernel<T, false, 16, 1, 1>
              : wide       ? cache_write_kernel<T, true, 8, 1, 1>
                           : cache_write_kernel<T, false, 8, 1, 1>;
  dib_launch(kern, dim3((unsigned)((tokens + per - 1) / per) * 2u * s.Hkv), dim3(CACHE_THREADS), 0, st, reinterpret_cast<const T*>(k),
             reinterpret_cast<const T*>(v), k_stride, v_stride, cache, slots, tokens, s);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}
template <typename T>
int launch_read(const Cache4& cache, const int* slots, void* k, void* v, int tokens, const CacheShape& s, cudaStream_t st) {
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 31) != 0) return DIB_BAD_ALIGN;
  const bool two = two_blocks<T>(cache, s.D);
  constexpr int TWO = sizeof(T) == 2 ? 2 : 1, ROWS = sizeof(T) == 2 ? 1 : 2;
  const int per = CACHE_THREADS / ((s.D > 128 ? 16 : 8) >> two) * ROWS;
  auto kern = two ? s.D > 128 ? cache_read_kernel<T, 16 / TWO, TWO, ROWS> : cache_read_kernel<T, 8 / TWO, TWO, ROWS>
                  : s.D > 128 ? cache_read_kernel<T, 16, 1, ROWS> : cache_read_kernel<T, 8, 1, ROWS>;
  dib_launch(kern, dim3((unsigned)((tokens + per - 1) / per) * 2u * s.Hkv), dim3(CACHE_THREADS), 0, st, cache, slots,
             reinterpret_cast<T*>(k), reinterpret_cast<T*>(v), tokens, s);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}
bool shape_fits(int T, int Hkv, int D, int page_size, long long num_pages) {
  return T >= 0 && Hkv >= 1 && D >= 16 && D <= 256 && D % 16 == 0 && page_size >= 1 && (long long)T * 2 * Hkv <= 0x7fffff00ll &&
         num_pages <= 0x7fffffffll;
}
Cache4 make_cache(const void* data, const void* scales, const void* exponents) {
  Cache4 c;
  c.data = reinterpret_cast<unsigned char*>(const_cast<void*>(data));
  c.scales = reinterpret_cast<unsigned char*>(const_cast<void*>(scales));
  c.exponents = reinterpret_cast<unsigned char*>(const_cast<void*>(exponents));
  return c;
}

}  // namespace

extern "C" {

// k, v: rows [T] of Hkv * D values, `k_stride`, `v_stride` values apart (dtype 0 float32, 1 bfloat16); slots int32 [T]
// (page * page_size + offset; a negative one, or one beyond the pool, is skipped).
int dib_fp4_cache_write(const void* k, const void* v, long long k_stride, long long v_stride, void* data, void* scales, void* exponents,
                        const void* slots, int T, int Hkv, int D, int page_size, long long num_pages, int dtype, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (!shape_fits(T, Hkv, D, page_size, num_pages)) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(data) & 15) != 0) return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const CacheShape shape = make_shape((long long)T * 2 * Hkv, Hkv, D, page_size, num_pages);
  const Cache4 cache = make_cache(data, scales, exponents);
  const int* sl = reinterpret_cast<const int*>(slots);
  if (dtype == 1) return launch_write<__nv_bfloat16>(k, v, k_stride, v_stride, cache, sl, T, shape, st);
  return launch_write<float>(k, v, k_stride, v_stride, cache, sl, T, shape, st);
}

// qkv [T, (Hq + 2 Hkv) D] -> q_out [T, Hq, D] and the cache; q_norm_w, k_norm_w float32 [D] or null; cos_sin float32
// [max_pos, rotary_dim] = [cos | sin] or null; a token whose slot is none of the pool's keeps no key.
int dib_fp4_qk_norm_rope_cache(const void* qkv, void* q_out, void* data, void* scales, void* exponents, const void* q_norm_w,
                               const void* k_norm_w, float eps, const void* cos_sin, int rotary_dim, int max_pos,
                               const void* positions, const void* slots, int T, int Hq, int Hkv, int D, int page_size,
                               long long num_pages, int dtype, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (!shape_fits(T, Hkv, D, page_size, num_pages) || Hq < 1 || rotary_dim < 0 || rotary_dim > D || rotary_dim % 2 != 0 ||
      (cos_sin != nullptr && max_pos < 1))
    return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(data)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const long long blocks = ((long long)T * (Hq + 2 * Hkv) + QKV_WARPS - 1) / QKV_WARPS;
  if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
  const float *qw = reinterpret_cast<const float*>(q_norm_w), *kw = reinterpret_cast<const float*>(k_norm_w),
              *tab = reinterpret_cast<const float*>(cos_sin);
  const int *ps = reinterpret_cast<const int*>(positions), *sl = reinterpret_cast<const int*>(slots);
  const Cache4 cache = make_cache(data, scales, exponents);
  if (dtype == 1)
    dib_launch(qk_norm_rope_cache_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(QKV_WARPS * 32), 0, st,
               reinterpret_cast<const __nv_bfloat16*>(qkv), reinterpret_cast<__nv_bfloat16*>(q_out), cache, qw, kw, eps, tab,
               rotary_dim, max_pos, ps, sl, T, Hq, Hkv, D, page_size, num_pages);
  else
    dib_launch(qk_norm_rope_cache_kernel<float>, dim3((unsigned)blocks), dim3(QKV_WARPS * 32), 0, st,
               reinterpret_cast<const float*>(qkv), reinterpret_cast<float*>(q_out), cache, qw, kw, eps, tab, rotary_dim, max_pos, ps, sl,
               T, Hq, Hkv, D, page_size, num_pages);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// k, v [T, Hkv, D] = the values that the rows in `slots` stand for; zeros for a slot that is none of the pool's.
int dib_fp4_cache_read(const void* data, const void* scales, const void* exponents, const void* slots, void* k, void* v, int T, int Hkv,
                       int D, int page_size, long long num_pages, int dtype, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (!shape_fits(T, Hkv, D, page_size, num_pages)) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(data) & 15) != 0) return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const CacheShape shape = make_shape((long long)T * 2 * Hkv, Hkv, D, page_size, num_pages);
  const Cache4 cache = make_cache(data, scales, exponents);
  const int* sl = reinterpret_cast<const int*>(slots);
  if (dtype == 1) return launch_read<__nv_bfloat16>(cache, sl, k, v, T, shape, st);
  return launch_read<float>(cache, sl, k, v, T, shape, st);
}

// The keys and values of the sequences seq_list [count] as bfloat16 pages [first_page[count], 2, Hkv, 128, D] (see
// unpack_pages_kernel); first_page int32 [count + 1], max_pages the most pages of one of them.
int dib_fp4_unpack_pages(const void* data, const void* scales, const void* exponents, long long num_pages, const void* block_table,
                         int max_blocks, const void* cu_q_lens, const void* seq_lens, const void* seq_list, const void* first_page,
                         int count, int max_pages, void* out, int Hkv, int D, int page_size, int window, cudaStream_t st) {
  if (!shape_fits(0, Hkv, D, page_size, num_pages) || count < 0 || count > 65535 || max_pages < 1 || 2 * Hkv > 65535 || max_blocks < 1)
    return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(data) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 31) != 0) return DIB_BAD_ALIGN;
  if (count == 0) return DIB_OK;
  UnpackArgs a;
  a.cache = make_cache(data, scales, exponents);
  a.block_table = reinterpret_cast<const int*>(block_table);
  a.cu_q_lens = reinterpret_cast<const int*>(cu_q_lens);
  a.seq_lens = reinterpret_cast<const int*>(seq_lens);
  a.seq_list = reinterpret_cast<const int*>(seq_list);
  a.first_page = reinterpret_cast<const int*>(first_page);
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.max_blocks = max_blocks;
  a.Hkv = Hkv; a.D = D; a.page_size = page_size; a.window = window;
  a.num_pages = num_pages;
  dib_launch(D > 128 ? unpack_pages_kernel<16> : unpack_pages_kernel<8>, dim3((unsigned)max_pages, 2u * Hkv, (unsigned)count),
             dim3(CACHE_THREADS), 0, st, a);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

// out [T, Hq, D], behind the attention over the pages of dib_fp4_unpack_pages: see finish_portions_kernel.
int dib_fp4_finish_portions(const void* exponents, long long num_pages, const void* block_table, int max_blocks, const void* cu_q_lens,
                            const void* seq_lens, const void* seq_list, int count, int max_pages, void* out, int Hq, int Hkv, int D,
                            int page_size, int window, cudaStream_t st) {
  if (!shape_fits(0, Hkv, D, page_size, num_pages) || count < 0 || count > 65535 || max_pages < 1 || Hkv > 65535 || max_blocks < 1 ||
      Hq < 1 || Hq % Hkv != 0 || page_size % 4 != 0)
    return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(exponents) & 3) != 0 || (reinterpret_cast<uintptr_t>(out) & 15) != 0) return DIB_BAD_ALIGN;
  if (count == 0) return DIB_OK;
  UnpackArgs a = {};
  a.cache = make_cache(nullptr, nullptr, exponents);
  a.block_table = reinterpret_cast<const int*>(block_table);
  a.cu_q_lens = reinterpret_cast<const int*>(cu_q_lens);
  a.seq_lens = reinterpret_cast<const int*>(seq_lens);
  a.seq_list = reinterpret_cast<const int*>(seq_list);
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.max_blocks = max_blocks;
  a.Hkv = Hkv; a.D = D; a.page_size = page_size; a.window = window;
  a.num_pages = num_pages;
  const int per = FINISH_KEYS / UNPACK_PAGE;
  dib_launch(finish_portions_kernel, dim3((unsigned)((max_pages + per - 1) / per), (unsigned)Hkv, (unsigned)count), dim3(CACHE_THREADS),
             0, st, a, Hq);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

}  // extern "C"
