// Attention of a step's new tokens over a paged cache in 8-bit integers (cache_int8.cu): query row i of head h, at
// position p, over the keys j of its sequence that it sees (j <= p, and j > p - window with a window):
//   s_j = scale * ks_j * (q . kc_j),   o = sum_j exp(s_j - m) vs_j vc_j / sum_j exp(s_j - m),
// kc, vc the codes of a key and a value, ks, vs their scales.  The scales never touch the codes: a key's joins its score,
// a value's the probability.  A row that sees no key is zeros.
//
// The form for every shape (head sizes up to 256, any page size and group ratio): a warp takes a (token, head), a lane a
// key of 32 at a time for the scores, then a lane D / 32 dimensions for the values.
#include "common.cuh"

namespace {

constexpr int ANY_WARPS = 4;
__device__ __forceinline__ float log2e() { return 1.4426950408889634f; }

template <typename T>
__global__ void __launch_bounds__(ANY_WARPS * 32)
attention_any_kernel(const T* __restrict__ q, T* __restrict__ out, const signed char* __restrict__ data,
                     const float* __restrict__ scales, const int* __restrict__ block_table, int max_blocks,
                     const int* __restrict__ token_seq, const int* __restrict__ cu_q_lens,
                     const int* __restrict__ seq_lens, int T_, int Hq, int Hkv, int D, int page_size, float scale,
                     int window) {
  pdl_prologue(q, data, scales);
  __shared__ float sq[ANY_WARPS][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * ANY_WARPS + warp;
  const bool in = item < (long long)T_ * Hq;
  const int token = in ? (int)(item / Hq) : 0, h = in ? (int)(item % Hq) : 0, kvh = h / (Hq / Hkv);
  if (in)
    for (int d = lane; d < D; d += 32) sq[warp][d] = Elem<T>::load(q + item * D + d) * scale * log2e();
  __syncwarp();
  if (!in) return;
  const int seq = token_seq[token];
  const int pos = seq_lens[seq] - (cu_q_lens[seq + 1] - token);      // a sequence's new tokens are its last ones
  const int lo = first_visible_key(pos, window), hi = (int)min((long long)pos, (long long)max_blocks * page_size - 1);
  const int* bt = block_table + (long long)seq * max_blocks;
  float m = -INFINITY, l = 0.f, o[8] = {};
  for (int k0 = lo; k0 <= hi; k0 += 32) {
    const int key = k0 + lane;
    const bool seen = key <= hi;
    const long long page = seen ? bt[key / page_size] : 0;
    const long long krow = ((page * 2) * Hkv + kvh) * page_size + (seen ? key % page_size : 0);
    const long long vrow = krow + (long long)Hkv * page_size;
    float s = -INFINITY;
    if (seen) {
      float dot = 0.f;
      const uint4* p = reinterpret_cast<const uint4*>(data + krow * D);
      for (int c = 0; c < D / 16; ++c) {
        const uint4 v = p[c];
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) dot = fmaf((float)(signed char)(w[i >> 2] >> (8 * (i & 3))), sq[warp][c * 16 + i], dot);
      }
      s = dot * scales[krow];
    }
    const float top = fmaxf(m, warp_max(s));
    const float p = seen ? exp2f(s - (top == -INFINITY ? 0.f : top)) : 0.f;
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - top);
    const float vs = seen ? scales[vrow] : 0.f;
    l = l * alpha + warp_sum(p);
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= alpha;
    const int n = min(32, hi - k0 + 1);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j) * __shfl_sync(0xffffffffu, vs, j);
      const signed char* vp = data + __shfl_sync(0xffffffffu, vrow, j) * D;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i * 32 + lane < D) o[i] = fmaf(pj, (float)vp[i * 32 + lane], o[i]);
    }
  }
  const bool none = hi < lo;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < D) Elem<T>::store(out + item * D + i * 32 + lane, none ? 0.f : o[i] / l);
}

}  // namespace

extern "C" {

int dib_int8_attention_any(const void* q, void* out, const void* data, const void* scales, const void* block_table,
                           int max_blocks, const void* token_seq, const void* cu_q_lens, const void* seq_lens, int T,
                           int Hq, int Hkv, int D, int page_size, float scale, int window, int dtype, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (T < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || D < 16 || D > 256 || D % 16 != 0 || page_size < 1) return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(data) & 15) != 0) return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const long long blocks = ((long long)T * Hq + ANY_WARPS - 1) / ANY_WARPS;
  if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
  const signed char* d = reinterpret_cast<const signed char*>(data);
  const float* s = reinterpret_cast<const float*>(scales);
  const int *bt = reinterpret_cast<const int*>(block_table), *ts = reinterpret_cast<const int*>(token_seq),
            *cu = reinterpret_cast<const int*>(cu_q_lens),
            *sl = reinterpret_cast<const int*>(seq_lens);
  if (dtype == 1)
    dib_launch(attention_any_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(ANY_WARPS * 32), 0, st,
               reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<__nv_bfloat16*>(out), d, s, bt, max_blocks, ts,
               cu, sl, T, Hq, Hkv, D, page_size, scale, window);
  else
    dib_launch(attention_any_kernel<float>, dim3((unsigned)blocks), dim3(ANY_WARPS * 32), 0, st,
               reinterpret_cast<const float*>(q), reinterpret_cast<float*>(out), d, s, bt, max_blocks, ts, cu, sl, T, Hq,
               Hkv, D, page_size, scale, window);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

}  // extern "C"
