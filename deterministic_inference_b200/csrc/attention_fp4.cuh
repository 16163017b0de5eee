// What the forms of attention over a cache in 4-bit floating point share that cut sequences into runs of keys: how, the conversion
// of codes, and adding the runs up.
#pragma once

#include "fp4.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's references: `at` of its scores s (log 2) and D, a whole number, of its values.  A key adds 2^(s - at) to the sum of weights and
// 2^(s - at + E_v - D) v to the outputs: the value's power of two has no part in the sum, and keys whose values are zero, or next to
// it, may have all of the weight.
// As a rule D is 0, `at` LIFT below the largest s + E_v, raised when an output's weight would pass 2^(LIFT + RAISE), and a key's part of the
// sum is that weight times 2^-E_v.  Rows that see values beyond 2^TAME either way, or scores next to which E_v is lost (FAR), have both
// references found: `at` LIFT below the largest score, raised when 2^(s - at) would pass 2^HIGH, D by the largest s - at + E_v.
// Which it is follows from what the row has seen, so that its bits do.  A row that has seen no key has UNSET, 0.
constexpr float RAISE = 5.f, LIFT = 10.f, HIGH = 60.f, FAR = 1048576.f, UNSET = -3.40282347e38f;
constexpr int TAME = 40;
__device__ __forceinline__ bool is_tame(unsigned byte) { return byte - (127u - TAME) <= 2u * TAME; }      // of a value's exponent
__device__ __forceinline__ float off_value(unsigned byte) { return __uint_as_float((unsigned)max(254 - (int)byte, 0) << 23); }      // 2^-E_v
// 2^d, which may be beyond a float32, times x
__device__ __forceinline__ float times_power(float x, float d) {
  const int e = (int)d, half = e >> 1;
  return x * __uint_as_float((unsigned)(half + 127) << 23) * __uint_as_float((unsigned)(e - half + 127) << 23);
}

constexpr int SP_TILE = 128;      // keys that a CTA works on at a time

// Keys of a run.
__host__ __device__ __forceinline__ int split_keys(int kv_len, int rows) {
  const int base = kv_len <= 2048 ? 256 : 512;
  const int tiles = (rows + 15) / 16;
  return tiles <= 2 ? base : base * ((tiles + 1) / 2);
}

struct SplitArgs {
  const unsigned char* data;
  const unsigned char* scales;
  const unsigned char* exponents;
  const int* block_table;       // [B, max_blocks]
  const int* cu_q_lens;
  const int* seq_lens;
  const int* seq_list;          // the sequences of this launch, or null: seq_first ..
  int seq_first, seq_count, max_blocks;
  int Hq, Hkv, D, page_shift, window, num_pages;
  float scale;
  float* part_o;                // [seq_count, max_items, ROWS, 128]: sums, in the order of the registers
  float4* part_ml;              // [seq_count, max_items, ROWS]: references (at, D), sum of weights, nothing
  int max_items;
  int sms;                      // blocks b, b + sms, ... of the grid lie on one SM as a rule; 0: fewer blocks than would fill the GPU
};
// The place of a block among the grid's, by which it takes its share of the work: those that share an SM follow one another, so
// that their shares, each rounded to whole items, add up to about the same on every SM.
__device__ __forceinline__ int block_place(const SplitArgs& a) {
  return a.sms == 0 ? (int)blockIdx.x : (int)blockIdx.x % a.sms * ((int)gridDim.x / a.sms) + (int)blockIdx.x / a.sms;
}
// A sequence of the launch and how it is cut.
struct SplitSeq {
  int seq, q_begin, n, kv_len, tiles, split, splits;
  __device__ __forceinline__ long long items(int Hkv) const { return (long long)tiles * splits * Hkv; }
  // what an item takes, in tiles of keys, one for its beginning and end among them
  __device__ __forceinline__ int item_work() const { return (min(split, kv_len) + SP_TILE - 1) / SP_TILE + 1; }
};
// ... from its index, first token, new tokens and keys
template <int ROWS> __device__ __forceinline__ SplitSeq split_seq(const SplitArgs& a, const int4& m) {
  SplitSeq s;
  s.seq = m.x; s.q_begin = m.y; s.n = m.z; s.kv_len = m.w;
  const int rows = s.n * (a.Hq / a.Hkv);
  s.tiles = (rows + ROWS - 1) / ROWS;
  s.split = split_keys(s.kv_len, rows);
  s.splits = s.n > 0 ? max(1, (s.kv_len + s.split - 1) / s.split) : 0;
  return s;
}
__device__ __forceinline__ int4 load_seq(const SplitArgs& a, int i) {
  int4 m;
  m.x = a.seq_list != nullptr ? a.seq_list[i] : a.seq_first + i;
  m.y = a.cu_q_lens[m.x];
  m.z = a.cu_q_lens[m.x + 1] - m.y;
  m.w = max((int)min((long long)a.seq_lens[m.x], min((long long)a.max_blocks << a.page_shift, 0x7fffff00ll)), 0);
  return m;
}
template <int ROWS> __device__ __forceinline__ SplitSeq split_seq(const SplitArgs& a, int i) { return split_seq<ROWS>(a, load_seq(a, i)); }

__device__ __forceinline__ void cp_async16(unsigned to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8(unsigned to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(unsigned to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// the four bytes of a word, two codes each, as pairs of float16
__device__ __forceinline__ void codes_to_half(unsigned w, unsigned (&h)[4]) {
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ unsigned scales_to_half(unsigned two) {
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
  return r;
}
__device__ __forceinline__ unsigned mul_half(unsigned a, unsigned b) {
  unsigned r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack_half(unsigned two) {
  float2 r;
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h; }" : "=f"(r.x), "=f"(r.y) : "r"(two));
  return r;
}
__device__ __forceinline__ unsigned transposed(unsigned m) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(m));
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the dimension that place p of a row's sums in the order of the registers stands for
__device__ __forceinline__ int dim_of(int p) { return ((p & 15) >> 1) * 16 + (p >> 4) * 2 + (p & 1); }

template <typename T> __device__ __forceinline__ void store_two(T* p, float x, float y);
template <> __device__ __forceinline__ void store_two<float>(float* p, float x, float y) { *reinterpret_cast<float2*>(p) = make_float2(x, y); }
template <> __device__ __forceinline__ void store_two<__nv_bfloat16>(__nv_bfloat16* p, float x, float y) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
}

// The runs' results of a row: out = sum_r 2^(at_r + D_r - top) O_r / sum_r 2^(at_r - top) l_r, a lane 4 places of the sums.  Up to SM_RUNS runs
// are a warp's, all asked for at once; more are those of a block: warp w takes the runs w, w + 4, ... in their order, the four warps'
// sums are added in the order of the warps.  (16 sequences' 10 rows a head of some 8 runs: the attention and its merge 24.5 us with a warp a
// row, 26.2 with a block.)
constexpr int SM_WARPS = 4, SM_RUNS = 8;
template <typename T, int ROWS>
__global__ void __launch_bounds__(SM_WARPS * 32)
attention_split_merge_kernel(T* __restrict__ out, const __grid_constant__ SplitArgs a) {
  const float* part_o = a.part_o;
  const float4* part_ml = a.part_ml;
  __shared__ float4 s_o[SM_WARPS][32];
  __shared__ float s_top[SM_WARPS], s_d[SM_WARPS], s_sum[SM_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.y, G = a.Hq / a.Hkv;
  const SplitSeq s = split_seq<ROWS>(a, i);
  const bool alone = s.splits <= SM_RUNS;      // a warp a row
  const int n_rows = s.n * G;                  // of a kv head
  const long long id = alone ? (long long)blockIdx.x * SM_WARPS + warp : blockIdx.x;
  // (every warp waits, the one without work too: a grid none of whose blocks has waited ends ahead of the attention, and the
  // kernel that follows takes this one's end for the attention's)
  if (s.splits <= 1 || id >= (long long)n_rows * a.Hkv || s.items(a.Hkv) > a.max_items) {
    pdl_wait();
    pdl_trigger();
    return;
  }
  const int kvh = (int)(id / n_rows), row = (int)(id - (long long)kvh * n_rows), tile = row / ROWS, r = row % ROWS;
  const int p0 = s.kv_len - s.n;
  const int tok0 = tile * ROWS / G, tok1 = min((tile + 1) * ROWS - 1, n_rows - 1) / G;
  // the runs that hold keys which some row of the tile sees
  const int k_lo = first_visible_key(p0 + tok0, a.window), k_hi = p0 + tok1;
  const int s0 = k_lo / s.split, s1 = k_hi < k_lo ? s0 - 1 : min(k_hi / s.split, s.splits - 1);
  const long long base = ((long long)i * a.max_items + (long long)(kvh * s.tiles + tile) * s.splits) * ROWS + r;
  pdl_wait(part_o, part_ml);
  pdl_trigger();      // (not before the attention is over: the blocks of the kernel that follows would take places among its own)
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  float4 v[SM_RUNS];
  float3 ml[SM_RUNS];
  auto load = [&](int from, int step) {
#pragma unroll
    for (int u = 0; u < SM_RUNS; ++u) {
      const int run = from + u * step;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      ml[u] = make_float3(UNSET, 0.f, 0.f);
      if (run <= s1) {
        const long long at = base + (long long)run * ROWS;
        const float4 m = part_ml[at];
        ml[u] = make_float3(m.x, m.y, m.z);
        v[u] = *reinterpret_cast<const float4*>(part_o + at * 128 + lane * 4);
      }
    }
  };
  // (top_d: the largest D, relative to the highest reference, to a whole number)
  auto add = [&](float top, float top_d, bool odd) {
#pragma unroll
    for (int u = 0; u < SM_RUNS; ++u) {
      float w = fast_exp2(ml[u].x - top);
      sum = fmaf(w, ml[u].z, sum);
      if (odd) w = fast_exp2(ml[u].x - top + ml[u].y - top_d);
      o.x = fmaf(w, v[u].x, o.x); o.y = fmaf(w, v[u].y, o.y);
      o.z = fmaf(w, v[u].z, o.z); o.w = fmaf(w, v[u].w, o.w);
    }
  };
  float top = UNSET, top_d = UNSET;
  bool odd = false;      // some D is not 0
  if (alone) {
    load(s0, 1);
#pragma unroll
    for (int u = 0; u < SM_RUNS; ++u) {
      top = fmaxf(top, ml[u].x);
      odd |= ml[u].y != 0.f;
    }
    if (odd) {
#pragma unroll
      for (int u = 0; u < SM_RUNS; ++u) top_d = fmaxf(top_d, rintf(ml[u].x - top + ml[u].y));
    }
    add(top, top_d, odd);
  } else {
    load(s0 + warp, SM_WARPS);      // on their way while the references are compared
    for (int run = s0 + (int)threadIdx.x; run <= s1; run += SM_WARPS * 32) {
      const float4 m = part_ml[base + (long long)run * ROWS];
      top = fmaxf(top, m.x);
      odd |= m.y != 0.f;
    }
    top = warp_max(top);
    if (lane == 0) s_top[warp] = top;
    odd = __syncthreads_or(odd);
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    if (odd) {
      for (int run = s0 + (int)threadIdx.x; run <= s1; run += SM_WARPS * 32) {
        const float4 m = part_ml[base + (long long)run * ROWS];
        top_d = fmaxf(top_d, rintf(m.x - top + m.y));
      }
      top_d = warp_max(top_d);
      if (lane == 0) s_d[warp] = top_d;
      __syncthreads();
      top_d = fmaxf(fmaxf(s_d[0], s_d[1]), fmaxf(s_d[2], s_d[3]));
    }
    for (int from = s0 + warp; from <= s1; from += SM_RUNS * SM_WARPS) {
      if (from != s0 + warp) load(from, SM_WARPS);
      add(top, top_d, odd);
    }
    s_o[warp][lane] = o;
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp != 0) return;
    o = s_o[0][lane];
    sum = s_sum[0];
#pragma unroll
    for (int k = 1; k < SM_WARPS; ++k) {
      const float4 z = s_o[k][lane];
      o.x += z.x; o.y += z.y; o.z += z.z; o.w += z.w;
      sum += s_sum[k];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int tok = row / G, d0 = dim_of(lane * 4), d1 = dim_of(lane * 4 + 2);
  T* dst = out + ((long long)(s.q_begin + tok) * a.Hq + kvh * G + row - tok * G) * a.D;
  o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
  if (odd) {
    o.x = times_power(o.x, top_d); o.y = times_power(o.y, top_d);
    o.z = times_power(o.z, top_d); o.w = times_power(o.w, top_d);
  }
  if (d0 < a.D) store_two<T>(dst + d0, o.x, o.y);
  if (d1 < a.D) store_two<T>(dst + d1, o.z, o.w);
}
// blocks of the merge for a sequence of `rows` rows and at most `runs` runs
inline long long merge_blocks(long long rows, int runs) { return runs <= SM_RUNS ? (rows + SM_WARPS - 1) / SM_WARPS : rows; }

SplitArgs cache_args(const void* data, const void* scales, const void* exponents, long long num_pages, const void* block_table,
                     int max_blocks, const void* cu_q_lens, const void* seq_lens, int Hq, int Hkv, int D, float scale, int window) {
  SplitArgs a = {};
  a.data = reinterpret_cast<const unsigned char*>(data);
  a.scales = reinterpret_cast<const unsigned char*>(scales);
  a.exponents = reinterpret_cast<const unsigned char*>(exponents);
  a.block_table = reinterpret_cast<const int*>(block_table);
  a.cu_q_lens = reinterpret_cast<const int*>(cu_q_lens);
  a.seq_lens = reinterpret_cast<const int*>(seq_lens);
  a.max_blocks = max_blocks;
  a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.window = window;
  a.num_pages = (int)num_pages;
  a.scale = scale;
  return a;
}

}  // namespace
