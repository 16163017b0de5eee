// Attention of a step's new tokens over a paged cache in 4-bit floating point (cache_fp4.cu): query row i of head h, at position p, over
// the keys j of its sequence that it sees (j <= p, and j > p - window with a window):
//   s_j = scale * (q . k_j),   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),
// k_j, v_j = 2^E times (code * block scale).  A code times its block's scale has 6 digits and lies between 2^-10 and 2,688: float16
// holds it exactly, and so do the products' operands.  The powers of two join the score (a key's) and the probability (a
// value's) in float32.  A row that sees no key is zeros.  A sequence's new tokens are its last ones.
//
// Forms: split (one new token, a few drafted ones, every float32 portion: the cache is streamed once) and one for every shape.
// bfloat16 portions of prompts read the keys and values as bfloat16 pages (cache_fp4.cu) in the prompt attention of the
// unquantised cache, whose probabilities are bfloat16 numbers (outputs off by 0.0023 of the norm instead of 0.0017).
#include "attention_fp4.cuh"

namespace {

// ---------------------------------------------------------------- split form
// A sequence's rows (new token, query head of the kv group), ROWS = 8 NT at a time, against a run of its keys, by a CTA of four
// warps; a warp takes every fourth step of 32 keys, and the four are added up at the run's end.  A warp asks for its keys,
// values and their scales by itself (cp.async, three steps in a ring): nothing in a step waits for another warp.
//   S^T = K Q^T:  mma.sync m16n8k16, A = 16 keys x 16 dimensions, B = the rows' queries.  A thread's A registers want pairs of
//     dimensions of two keys; which dimensions is open as long as Q agrees: thread t of four takes the 32 from 32 t on, 16 bytes
//     of a key's codes and two block scales.  A byte is two codes and becomes two float16 numbers (one conversion), times the scale.
//   O^T = V^T P^T:  A = 16 dimensions x 16 keys, pairs of keys of a dimension: a thread has the block 16 g of four keys; the
//     nibbles of two keys are interleaved first (two instructions a word), so that a byte again is a pair.  P^T comes from
//     S^T's registers by a transposition of 8 x 8 (movmatrix).
// Keys 2 and 3, 6 and 7 of each 8 change places among the rows of the products (of scores and outputs alike), and the halves of a
// key's codes for every other four keys: then neither reading keys (two a quarter warp) nor values (four keys a half warp)
// meets a bank twice.
//
// The outputs' weights 2^(s - at + E_v - D) (the references of attention_fp4.cuh, a warp's own until the run's end) are rounded to float16 (11
// digits; two such parts of a float32 query's): at most 2^15, so that what lies 2^-29 below the largest still has all digits.  Sums are in
// float32.  Queries are scaled by a power of two to a largest element between 2^8 and 2^9, in which float16 holds bfloat16 values exactly
// down to 2^-23 of it (three parts of a float32 query's).  The products' units cut a sum's last digits off instead of rounding them: of
// float32 queries the parts' scores are added up by themselves, and the outputs' sums of 16 keys (off by 4e-7 of the norm in the root
// mean square; 1.2e-6 to 2.0e-6, by the keys, where all is left to the products: 1,000 tokens on 1,500 keys, 16 heads, 225 us
// instead of 205).
//
// Work items: (sequence, kv head, tile of rows, run of keys), a CTA takes a contiguous range of them.  The length of a run follows
// from the sequence's own lengths, so a row's bits do not depend on the rest of the step.
//
// Bound by instructions, some 700 for 32 keys: 64 requests of 2,048 keys, 16 / 4 heads: heads of 96 in bfloat16 45 us, of 128 in float32
// 54 (the stream form 31 for heads of 128 in bfloat16).
constexpr int SP_WARPS = 4, SP_THREADS = 32 * SP_WARPS, SP_STEP = 32, SP_STAGES = 3;
constexpr int SP_K = 0, SP_V = SP_STEP * 64, SP_KS = 2 * SP_V, SP_VS = SP_KS + SP_STEP * 8, SP_KE = SP_VS + SP_STEP * 8,
              SP_VE = SP_KE + SP_STEP, SP_STAGE = SP_VE + SP_STEP;      // bytes of a step: codes, block scales, exponents
constexpr int SP_ROW = 132;                                             // floats of a row's sums in shared memory: no two share banks
template <typename T> __device__ __forceinline__ float4 load_four(const T* p);
template <> __device__ __forceinline__ float4 load_four<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 load_four<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                     __uint_as_float(v.y & 0xffff0000u));
}
template <typename T, int NT> struct SplitShape {
  static constexpr int ROWS = 8 * NT, Q_PARTS = sizeof(T) == 4 ? 3 : 1, P_PARTS = sizeof(T) == 4 ? 2 : 1;
  static constexpr int CTAS = sizeof(T) == 4 ? 2 : NT == 1 ? 4 : 3;
  static constexpr int RING = SP_WARPS * SP_STAGES * SP_STAGE, ML = RING, FIRST = ML + SP_WARPS * ROWS * 16;
};

template <typename T, int NT>
__global__ void __launch_bounds__(SP_THREADS, SplitShape<T, NT>::CTAS)
attention_split_kernel(const T* __restrict__ q, T* __restrict__ out, const __grid_constant__ SplitArgs a) {
  using SH = SplitShape<T, NT>;
  constexpr int ROWS = SH::ROWS, QP = SH::Q_PARTS, PP = SH::P_PARTS;
  extern __shared__ __align__(128) unsigned char smem[];
  float4* ml = reinterpret_cast<float4*>(smem + SH::ML);      // of a warp's rows: references (at, D), sum of weights
  long long* first = reinterpret_cast<long long*>(smem + SH::FIRST);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = a.Hq / a.Hkv;
  pdl_trigger();
  // ---- the work before each sequence (metadata alone, which no kernel of a step writes)
  for (int i = threadIdx.x; i < a.seq_count; i += SP_THREADS) {
    const SplitSeq s = split_seq<ROWS>(a, i);
    first[i + 1] = s.items(a.Hkv) * s.item_work();
  }
  if (threadIdx.x == 0) first[0] = 0;
  __syncthreads();
  if (warp == 0) {
    long long base = 0;
    for (int i0 = 0; i0 < a.seq_count; i0 += 32) {
      long long v = i0 + lane < a.seq_count ? first[i0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (i0 + lane < a.seq_count) first[i0 + lane + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const long long total = first[a.seq_count];
  const int place = block_place(a);
  const long long from_work = total / gridDim.x * place + total % gridDim.x * place / gridDim.x;
  const long long to_work = total / gridDim.x * (place + 1) + total % gridDim.x * (place + 1) / gridDim.x;
  int i = 0;
  for (int hi = a.seq_count - 1; i < hi;) {      // the sequence in which the range begins
    const int mid = (i + hi + 1) >> 1;
    if (first[mid] <= from_work) i = mid; else hi = mid - 1;
  }
  pdl_wait(q);
  if (total == 0) return;
  SplitSeq s = split_seq<ROWS>(a, i);
  long long item = (from_work - first[i] + s.item_work() - 1) / s.item_work();       // the first item that begins in it

  unsigned char* ring = smem + warp * (SP_STAGES * SP_STAGE);
  const unsigned ring_at = smem_u32(ring);
  float* sums = reinterpret_cast<float*>(ring);
  const int row_bytes = a.D >> 1, row_scales = a.D >> 4, page_mask = (1 << a.page_shift) - 1;
  int old_i = -1, old_kvh = -1, old_tile = -1;
  unsigned qf[QP][NT][8][2];      // the rows' queries as B operands
  float unit[NT][2];              // of the scores, of this thread's columns (rows 2t, 2t + 1 of each eight)

  for (;; ++item) {
    while (i < a.seq_count && item >= s.items(a.Hkv)) {
      if (++i < a.seq_count) s = split_seq<ROWS>(a, i);
      item = 0;
    }
    if (i >= a.seq_count || first[i] + item * s.item_work() >= to_work) break;
    const int local = (int)item, pair = local / s.splits, run_at = (local - pair * s.splits) * s.split;
    const int kvh = pair / s.tiles, tile = pair - kvh * s.tiles;
    const int p0 = s.kv_len - s.n, row0 = tile * ROWS, rows = min(ROWS, s.n * G - row0);
    const int tok0 = row0 / G, tok1 = (row0 + rows - 1) / G;
    const int seen = max(run_at, first_visible_key(p0 + tok0, a.window)), end = min(run_at + s.split, p0 + tok1 + 1);
    if (end <= seen) {
      if (s.splits == 1)             // a sequence of one run: rows that see no key are zeros, from here
        for (int e = threadIdx.x; e < rows * a.D; e += SP_THREADS) {
          const int row = row0 + e / a.D, tok = row / G;
          Elem<T>::store(out + ((long long)(s.q_begin + tok) * a.Hq + kvh * G + row - tok * G) * a.D + e % a.D, 0.f);
        }
      continue;
    }
    const int at = seen & ~(SP_STEP - 1);
    const int steps = ((end - at + SP_STEP - 1) / SP_STEP - warp + SP_WARPS - 1) / SP_WARPS;      // of this warp
    const int lo_all = max(run_at, first_visible_key(p0 + tok1, a.window)), hi_all = min(end - 1, p0 + tok0);
    const int* table = a.block_table + (long long)s.seq * a.max_blocks;

    // lanes 0-7: the page of four keys each of step j of this warp; -1: no keys, or no page of the pool
    auto find_page = [&](int j) {
      const int key = at + (j * SP_WARPS + warp) * SP_STEP + (lane & 7) * 4;
      int page = -1;
      if (j < steps && key < end) page = table[key >> a.page_shift];
      return page >= 0 && page < a.num_pages ? page : -1;
    };
    auto copy = [&](int j, int page) {
      const int key = at + (j * SP_WARPS + warp) * SP_STEP + (lane & 7) * 4;
      // row of the cache of the first of four keys, and of their values
      const int krow = page < 0 ? -1 : ((page * 2 * a.Hkv + kvh) << a.page_shift) + (key & page_mask);
      const int vrow = krow + (a.Hkv << a.page_shift);
      const unsigned to = ring_at + j % SP_STAGES * SP_STAGE;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int four = (lane >> 4) + 2 * c, row = (lane >> 2) + 8 * c, part = lane & 3;
        const int kr = __shfl_sync(0xffffffffu, krow, four), vr = __shfl_sync(0xffffffffu, vrow, four);
        const int bytes = kr >= 0 && part * 16 < row_bytes ? 16 : 0;
        const unsigned place = row * 64 + ((part ^ (row >> 1 & 2)) << 4);
        const long long off = bytes == 0 ? 0 : part * 16;
        cp_async16(to + SP_K + place, a.data + (bytes == 0 ? 0 : (long long)(kr + (row & 3)) * row_bytes) + off, bytes);
        cp_async16(to + SP_V + place, a.data + (bytes == 0 ? 0 : (long long)(vr + (row & 3)) * row_bytes) + off, bytes);
      }
      {      // four keys' block scales lie together: D / 4 bytes
        const int four = lane >> 2, part = lane & 3;
        const int kr = __shfl_sync(0xffffffffu, krow, four), vr = __shfl_sync(0xffffffffu, vrow, four);
        const int bytes = kr >= 0 && part * 32 < a.D ? 8 : 0;
        cp_async8(to + SP_KS + four * 32 + part * 8, a.scales + (bytes == 0 ? 0 : (long long)kr * row_scales + part * 8), bytes);
        cp_async8(to + SP_VS + four * 32 + part * 8, a.scales + (bytes == 0 ? 0 : (long long)vr * row_scales + part * 8), bytes);
      }
      if (lane < 16) {
        const int row = lane < 8 ? krow : vrow;
        cp_async4(to + (lane < 8 ? SP_KE : SP_VE) + (lane & 7) * 4, a.exponents + (krow < 0 ? 0 : row), krow < 0 ? 0 : 4);
      }
    };

    int page = find_page(0);
#pragma unroll
    for (int j = 0; j < SP_STAGES - 1; ++j) {
      if (j < steps) {
        const int next = find_page(j + 1);
        copy(j, page);
        page = next;
      }
      cp_commit();
    }
    // ---- the rows' queries
    if (i != old_i || kvh != old_kvh || tile != old_tile) {
      old_i = i; old_kvh = kvh; old_tile = tile;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g, row = row0 + r, tok = row / G;
        const T* src = q + ((long long)(s.q_begin + tok) * a.Hq + kvh * G + row - tok * G) * a.D + t * 32;
        float4 x[8];
        unsigned top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < rows && t * 32 < a.D) x[k] = load_four<T>(src + 4 * k);
          top = max(max(top, fp4_magnitude(x[k].x)), max(fp4_magnitude(x[k].y), max(fp4_magnitude(x[k].z), fp4_magnitude(x[k].w))));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest element to 2^8 .. 2^9, a power of two up; a row with an infinity or a NaN: its scores are NaN
        const unsigned e = max(top >> 23, 27u);
        const float up = __uint_as_float((262u - min(e, 254u)) << 23);
        const float down = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.scale * LOG2E * __uint_as_float((e - 8u) << 23);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float y[4] = {x[k].x * up, x[k].y * up, x[k].z * up, x[k].w * up};
#pragma unroll
          for (int p = 0; p < QP; ++p) {
            const unsigned lo = pack_half(y[0], y[1]), hi = pack_half(y[2], y[3]);
            qf[p][nt][k][0] = lo;
            qf[p][nt][k][1] = hi;
            if (p + 1 < QP) {
              const float2 l2 = unpack_half(lo), h2 = unpack_half(hi);
              y[0] -= l2.x; y[1] -= l2.y; y[2] -= h2.x; y[3] -= h2.y;
            }
          }
        }
        // rows 2t and 2t + 1 of these eight are at lanes 4 (2t) and 4 (2t + 1)
        unit[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
        unit[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      }
    }
    int pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) pos[nt][c] = p0 + (row0 + nt * 8 + 2 * t + c) / G;

    float ref[NT][2], l[NT][2], o[8][NT][4];
    bool odd = false;         // some row's D is not 0 (those are in `ml`)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      ref[nt][0] = ref[nt][1] = UNSET;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d][nt][0] = o[d][nt][1] = o[d][nt][2] = o[d][nt][3] = 0.f;
    }
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      if (j + SP_STAGES - 1 < steps) {
        const int next = find_page(j + SP_STAGES);
        copy(j + SP_STAGES - 1, page);
        page = next;
      }
      cp_commit();
      cp_wait<SP_STAGES - 1>();
      __syncwarp();
      const unsigned char* st = ring + j % SP_STAGES * SP_STAGE;
      const int kb = at + (j * SP_WARPS + warp) * SP_STEP;
      const bool plain = kb >= lo_all && kb + SP_STEP - 1 <= hi_all;        // every row sees every key
      // ---- scores, in units of log 2
      float sc[2][NT][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int r0 = m * 16 + (g ^ (g >> 1 & 1)), turn = r0 >> 1 & 2;      // (r0 + 8: the same turn)
        const uint4 ka = *reinterpret_cast<const uint4*>(st + SP_K + r0 * 64 + ((t ^ turn) << 4));
        const uint4 kc = *reinterpret_cast<const uint4*>(st + SP_K + (r0 + 8) * 64 + ((t ^ turn) << 4));
        unsigned sa = 0, sb = 0;
        if (t * 32 < a.D) {
          sa = *reinterpret_cast<const unsigned short*>(st + SP_KS + (r0 >> 2) * 32 + (r0 & 3) * row_scales + 2 * t);
          sb = *reinterpret_cast<const unsigned short*>(st + SP_KS + (r0 >> 2) * 32 + 64 + (r0 & 3) * row_scales + 2 * t);
        }
        sa = scales_to_half(sa);
        sb = scales_to_half(sb);
        const unsigned wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kc.x, kc.y, kc.z, kc.w};
        float part[QP][NT][4];      // of the scores, by the queries' parts
#pragma unroll
        for (int p = 0; p < QP; ++p)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[p][nt][0] = part[p][nt][1] = part[p][nt][2] = part[p][nt][3] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const unsigned ua = __byte_perm(sa, 0, w < 2 ? 0x1010 : 0x3232), ub = __byte_perm(sb, 0, w < 2 ? 0x1010 : 0x3232);
          unsigned ha[4], hb[4];
          codes_to_half(wa[w], ha);
          codes_to_half(wb[w], hb);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            ha[x] = mul_half(ha[x], ua);
            hb[x] = mul_half(hb[x], ub);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int p = 0; p < QP; ++p) {
              mma(part[p][nt], ha[0], hb[0], ha[1], hb[1], qf[p][nt][2 * w][0], qf[p][nt][2 * w][1]);
              mma(part[p][nt], ha[2], hb[2], ha[3], hb[3], qf[p][nt][2 * w + 1][0], qf[p][nt][2 * w + 1][1]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {      // the smallest first
            sc[m][nt][e] = part[QP - 1][nt][e];
#pragma unroll
            for (int p = QP - 2; p >= 0; --p) sc[m][nt][e] += part[p][nt][e];
          }
      }
      // scores and the value's power of two.  An exponent of no number, the key's or the value's, makes those of the rows that see it NaN.
      float lv[2][2], back[2][2];      // E_v, 2^-E_v
      bool wild = false, over = odd;
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = m * 16 + h * 8 + (g ^ (g >> 1 & 1)), key = kb + r;
          const unsigned ke = st[SP_KE + r], ve = st[SP_VE + r];
          const float ks = fp4_unit(ve == FP4_NO_NUMBER ? ve : ke);
          lv[m][h] = (float)(int)ve - 127.f;
          back[m][h] = off_value(ve);
          wild |= !is_tame(ve) && (plain || (key >= seen && key < end));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float z = fmaf(sc[m][nt][2 * h + c], ks * unit[nt][c], lv[m][h]);
              if (!plain && (key < run_at || key >= end || key > pos[nt][c] || key < first_visible_key(pos[nt][c], a.window))) z = -INFINITY;
              sc[m][nt][2 * h + c] = z;
              over |= z > ref[nt][c] + (LIFT + RAISE);
            }
        }
      bool apart = false;
      if (__any_sync(0xffffffffu, over || wild)) {
        // a column's largest, by all lanes: with the values' powers of two as they are, and of the scores off `at` without them and with them
        auto column_most = [&](float (&x)[4]) {
          float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
          return top;
        };
        auto column_top = [&](int nt, int c) {
          float x[4] = {sc[0][nt][c], sc[0][nt][2 + c], sc[1][nt][c], sc[1][nt][2 + c]};
          return column_most(x);
        };
        auto column_scores = [&](int nt, int c, float at, bool values) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float value = lv[i >> 1][i & 1];
            x[i] = sc[i >> 1][nt][2 * (i & 1) + c] - value - at + (values ? value : 0.f);
          }
          return column_most(x);
        };
        auto scale_outputs = [&](int nt, int c, float f) {
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            o[d][nt][c] *= f;
            o[d][nt][2 + c] *= f;
          }
        };
        apart = __any_sync(0xffffffffu, odd || wild);
        if (!apart) {
          float to[NT][2];
          bool far = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float top = column_top(nt, c);
              to[nt][c] = top > ref[nt][c] + (LIFT + RAISE) ? top - LIFT : ref[nt][c];
              far |= to[nt][c] != UNSET && fabsf(to[nt][c]) >= FAR;
            }
          apart = __any_sync(0xffffffffu, far);
          if (!apart) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const float f = fast_exp2(ref[nt][c] - to[nt][c]);
                l[nt][c] *= f;
                scale_outputs(nt, c, f);
                ref[nt][c] = to[nt][c];
              }
          }
        }
        if (apart) {      // values or scores far from one another: the step's part of the sums of weights from here
          bool any_d = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const bool fresh = ref[nt][c] == UNSET;
              const int r = nt * 8 + 2 * t + c;
              const float was = ref[nt][c], base = fresh ? 0.f : was, old = odd ? ml[warp * ROWS + r].y : 0.f;
              const float top = column_top(nt, c);
              float to = top > was + (LIFT + RAISE) ? top - LIFT : was, d = old;
              bool wide = false;      // a value that is not tame among the keys that the row sees
#pragma unroll
              for (int i = 0; i < 4; ++i) wide |= fabsf(lv[i >> 1][i & 1]) > TAME && sc[i >> 1][nt][2 * (i & 1) + c] > -INFINITY;
              const unsigned wide_lanes = __ballot_sync(0xffffffffu, wide);
              const float top_s = column_scores(nt, c, base, false);
              const float by = top_s > (fresh ? -INFINITY : HIGH) ? rintf(top_s) - LIFT : 0.f;
              const float top_v = column_scores(nt, c, base + by, true);
              const bool both = old != 0.f || (fabsf(to) >= FAR && to != UNSET) || (wide_lanes & 0x11111111u << t) != 0;
              float f_l = fast_exp2(was - to), f_o = f_l;
              if (both) {
                to = base + by;
                d -= by;
                if (fresh || top_v - d > LIFT + RAISE) d = top_v > -INFINITY ? rintf(top_v) - LIFT : 0.f;
                f_l = fresh ? 0.f : fast_exp2(-by);
                f_o = fresh ? 0.f : fast_exp2(old - by - d);
              }
              l[nt][c] *= f_l;
              scale_outputs(nt, c, f_o);
              ref[nt][c] = to;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float& z = sc[i >> 1][nt][2 * (i & 1) + c];
                const float value = lv[i >> 1][i & 1], off = z - value - to;
                z = both ? off + (value - d) : z - to;
                l[nt][c] = d != 0.f || fabsf(value) > TAME ? l[nt][c] + fast_exp2(off) : fmaf(fast_exp2(z), back[i >> 1][i & 1], l[nt][c]);
              }
              __syncwarp();
              if (g == 0) ml[warp * ROWS + r].y = d;
              any_d |= d != 0.f;
            }
          back[0][0] = back[0][1] = back[1][0] = back[1][1] = 0.f;
          __syncwarp();
          odd = __any_sync(0xffffffffu, any_d);
        }
      }
      if (!apart) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[m][nt][i] -= ref[nt][i & 1];
      }
      // ---- weights, as B operands
      unsigned pw[PP][2][NT][2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float w[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              w[c] = fast_exp2(sc[m][nt][2 * h + c]);
              l[nt][c] = fmaf(w[c], back[m][h], l[nt][c]);
            }
            const unsigned two = pack_half(w[0], w[1]);
            pw[0][m][nt][h] = transposed(two);
            if (PP == 2) {
              const float2 held = unpack_half(two);
              pw[PP - 1][m][nt][h] = transposed(pack_half(w[0] - held.x, w[1] - held.y));
            }
          }
      // ---- outputs
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int ra = m * 16 + (2 * t ^ (t & 1)), rb = m * 16 + ((2 * t + 1) ^ (t & 1));      // and 8 keys on
        const int turn = ra >> 1 & 2, place = ((g >> 1 ^ turn) << 4) + (g & 1) * 8;
        const uint2 va = *reinterpret_cast<const uint2*>(st + SP_V + ra * 64 + place);
        const uint2 vb = *reinterpret_cast<const uint2*>(st + SP_V + rb * 64 + place);
        const uint2 vc = *reinterpret_cast<const uint2*>(st + SP_V + (ra + 8) * 64 + place);
        const uint2 vd = *reinterpret_cast<const uint2*>(st + SP_V + (rb + 8) * 64 + place);
        unsigned sab = 0, scd = 0;
        if (g * 16 < a.D) {
          const unsigned char* vs = st + SP_VS + (ra >> 2) * 32 + g;
          sab = vs[(ra & 3) * row_scales] | (unsigned)vs[(rb & 3) * row_scales] << 8;
          scd = vs[64 + (ra & 3) * row_scales] | (unsigned)vs[64 + (rb & 3) * row_scales] << 8;
        }
        if (!plain) {      // keys that no row sees: whatever is held there, nothing comes of it
          const int ka = kb + ra, kc = kb + rb;
          if (ka < seen || ka >= end) sab &= 0xff00u;
          if (kc < seen || kc >= end) sab &= 0x00ffu;
          if (ka + 8 < seen || ka + 8 >= end) scd &= 0xff00u;
          if (kc + 8 < seen || kc + 8 >= end) scd &= 0x00ffu;
        }
        sab = scales_to_half(sab);
        scd = scales_to_half(scd);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const unsigned xa = y ? va.y : va.x, xb = y ? vb.y : vb.x, xc = y ? vc.y : vc.x, xd = y ? vd.y : vd.x;
          // bytes of (this key's code, the next key's code) of the even and the odd dimensions
          unsigned e0[4], e1[4], f0[4], f1[4];
          codes_to_half((xa & 0x0f0f0f0fu) | (xb << 4 & 0xf0f0f0f0u), e0);
          codes_to_half((xa >> 4 & 0x0f0f0f0fu) | (xb & 0xf0f0f0f0u), e1);
          codes_to_half((xc & 0x0f0f0f0fu) | (xd << 4 & 0xf0f0f0f0u), f0);
          codes_to_half((xc >> 4 & 0x0f0f0f0fu) | (xd & 0xf0f0f0f0u), f1);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const unsigned a0 = mul_half(e0[x], sab), a1 = mul_half(e1[x], sab), a2 = mul_half(f0[x], scd), a3 = mul_half(f1[x], scd);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (PP == 1) {
                mma(o[4 * y + x][nt], a0, a1, a2, a3, pw[0][m][nt][0], pw[0][m][nt][1]);
              } else {
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = PP - 1; p >= 0; --p) mma(sum, a0, a1, a2, a3, pw[p][m][nt][0], pw[p][m][nt][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[4 * y + x][nt][e] += sum[e];
              }
            }
          }
        }
      }
      __syncwarp();      // the step has been read
    }
    cp_wait<0>();
    // ---- the four warps' sums of the run
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float v = l[nt][c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
        const int r = nt * 8 + 2 * t + c;
        if (g == 0) ml[warp * ROWS + r] = make_float4(ref[nt][c], odd ? ml[warp * ROWS + r].y : 0.f, v, 0.f);
#pragma unroll
        for (int d = 0; d < 8; ++d)
          *reinterpret_cast<float2*>(sums + r * SP_ROW + d * 16 + g * 2) = make_float2(o[d][nt][c], o[d][nt][2 + c]);
      }
    __syncthreads();
    {
      const int two = threadIdx.x & 63, dim = dim_of(2 * two);
#pragma unroll 2
      for (int r = threadIdx.x >> 6; r < rows; r += 2) {
        float4 w[SP_WARPS];
        float top = UNSET, top_d = 0.f;
        bool any_d = false;      // some D is not 0
#pragma unroll
        for (int x = 0; x < SP_WARPS; ++x) {
          w[x] = ml[x * ROWS + r];
          top = fmaxf(top, w[x].x);
          any_d |= w[x].y != 0.f;
        }
        if (any_d) {
          top_d = UNSET;
#pragma unroll
          for (int x = 0; x < SP_WARPS; ++x) top_d = fmaxf(top_d, rintf(w[x].x - top + w[x].y));
        }
        float sum = 0.f;
        float2 y = make_float2(0.f, 0.f);
#pragma unroll
        for (int x = 0; x < SP_WARPS; ++x) {
          float f = fast_exp2(w[x].x - top);
          const float2 v = *reinterpret_cast<const float2*>(smem + x * (SP_STAGES * SP_STAGE) + (r * SP_ROW + 2 * two) * 4);
          sum = fmaf(f, w[x].z, sum);
          if (any_d) f = fast_exp2(w[x].x - top + w[x].y - top_d);
          y.x = fmaf(f, v.x, y.x);
          y.y = fmaf(f, v.y, y.y);
        }
        if (s.splits == 1) {
          const int row = row0 + r, tok = row / G;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          y.x *= inv;
          y.y *= inv;
          if (any_d) {
            y.x = times_power(y.x, top_d);
            y.y = times_power(y.y, top_d);
          }
          if (dim < a.D) store_two<T>(out + ((long long)(s.q_begin + tok) * a.Hq + kvh * G + row - tok * G) * a.D + dim, y.x, y.y);
        } else if (local < a.max_items) {
          const long long to = ((long long)i * a.max_items + local) * ROWS + r;
          *reinterpret_cast<float2*>(a.part_o + to * 128 + 2 * two) = y;
          if (two == 0) a.part_ml[to] = make_float4(top, top_d, sum, 0.f);
        }
      }
    }
    __syncthreads();      // the sums have been read
  }
}

// ---------------------------------------------------------------- the form for every shape
// Head sizes up to 256, any page size and group ratio: a warp takes a (token, head), a lane a key of 32 at a time for
// the scores, then a lane D / 32 dimensions for the values.  Bound by a warp's chain over the keys: 2,048 of them 1.4 ms with heads of
// 128, 2.4 with 256, for one request as for sixteen.
constexpr int ANY_WARPS = 4;

template <typename T>
__global__ void __launch_bounds__(ANY_WARPS * 32)
attention_any_kernel(const T* __restrict__ q, T* __restrict__ out, const __grid_constant__ SplitArgs a, const int* __restrict__ token_seq,
                     int T_, int page_size) {
  const unsigned char *data = a.data, *scales = a.scales, *exponents = a.exponents;
  pdl_prologue(q, data, scales, exponents);
  __shared__ float sq[ANY_WARPS][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.D;
  const long long item = (long long)blockIdx.x * ANY_WARPS + warp;
  const bool in = item < (long long)T_ * a.Hq;
  const int token = in ? (int)(item / a.Hq) : 0, h = in ? (int)(item % a.Hq) : 0, kvh = h / (a.Hq / a.Hkv);
  if (in)
    for (int d = lane; d < D; d += 32) sq[warp][d] = Elem<T>::load(q + item * D + d) * a.scale * LOG2E;
  __syncwarp();
  if (!in) return;
  const int seq = token_seq[token];
  const int pos = a.seq_lens[seq] - (a.cu_q_lens[seq + 1] - token);      // a sequence's new tokens are its last ones
  const int lo = first_visible_key(pos, a.window), hi = (int)min((long long)pos, (long long)a.max_blocks * page_size - 1);
  const int* bt = a.block_table + (long long)seq * a.max_blocks;
  float m = -INFINITY, l = 0.f, o[8] = {};
  for (int k0 = lo; k0 <= hi; k0 += 32) {
    const int key = k0 + lane;
    const bool seen = key <= hi;
    const long long page = seen ? bt[key / page_size] : -1;
    const bool have = page >= 0 && page < a.num_pages;      // (a page that is none of the pool's: keys and values of zeros)
    const long long krow = (page * 2 * a.Hkv + kvh) * page_size + key % page_size;
    const long long vrow = have ? krow + (long long)a.Hkv * page_size : -1;
    float s = seen ? 0.f : -INFINITY;
    if (have) {
      float dot = 0.f;
      for (int b = 0; b < D / 16; ++b) {
        const uint2 w = *reinterpret_cast<const uint2*>(data + krow * (D / 2) + b * 8);
        const float scale = fp4_scale_value(scales[krow * (D / 16) + b]);
        float x[16];
        fp4_values8(w.x, scale, x);
        fp4_values8(w.y, scale, x + 8);
#pragma unroll
        for (int e = 0; e < 16; ++e) dot = fmaf(x[e], sq[warp][b * 16 + e], dot);
      }
      s = dot * fp4_unit(exponents[krow]);
    }
    const float top = fmaxf(m, warp_max(s));
    const float p = seen ? exp2f(s - (top == -INFINITY ? 0.f : top)) : 0.f;
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - top);
    const float unit = have ? fp4_unit(exponents[vrow]) : 0.f;
    l = l * alpha + warp_sum(p);
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= alpha;
    const int n = min(32, hi - k0 + 1);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j) * __shfl_sync(0xffffffffu, unit, j);
      const long long row = __shfl_sync(0xffffffffu, vrow, j);
      if (row < 0) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = i * 32 + lane;
        if (d < D) {
          const unsigned code = data[row * (D / 2) + d / 2] >> (4 * (d & 1)) & 15u;
          float x[8];
          fp4_values8(code, fp4_scale_value(scales[row * (D / 16) + d / 16]), x);
          o[i] = fmaf(pj, x[0], o[i]);
        }
      }
    }
  }
  const bool none = hi < lo;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < D) Elem<T>::store(out + item * D + i * 32 + lane, none ? 0.f : o[i] / l);
}

// ---------------------------------------------------------------- host side
template <typename T, int NT>
int launch_split(const void* q, void* out, SplitArgs a, int max_rows, int runs, int sm_count, cudaStream_t st) {
  using SH = SplitShape<T, NT>;
  auto kern = attention_split_kernel<T, NT>;
  const size_t smem = SH::FIRST + ((size_t)a.seq_count + 1) * 8;
  if (smem > 100 * 1024) return DIB_BAD_SIZE;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
        cudaFuncSetAttribute(attention_split_merge_kernel<T, SH::ROWS>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared) != cudaSuccess)
      return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  const int by_smem = (int)(228 * 1024 / (smem + 1024)), per_sm = by_smem < SH::CTAS ? by_smem : SH::CTAS;
  const long long most = (long long)a.max_items * a.seq_count, grid = (long long)sm_count * (per_sm < 1 ? 1 : per_sm);
  a.sms = most >= grid ? sm_count : 0;
  dib_launch(kern, dim3((unsigned)(grid < most ? grid : most)), dim3(SP_THREADS), smem, st, reinterpret_cast<const T*>(q),
             reinterpret_cast<T*>(out), a);
  DIB_CHECK_LAUNCH();
  if (runs) {
    const long long blocks = merge_blocks((long long)max_rows * a.Hkv, runs);
    if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
    dib_launch(attention_split_merge_kernel<T, SH::ROWS>, dim3((unsigned)blocks, a.seq_count), dim3(SM_WARPS * 32), 0, st,
               reinterpret_cast<T*>(out), a);
    DIB_CHECK_LAUNCH();
  }
  return DIB_OK;
}

}  // namespace

extern "C" {

// Keys of a run of the split form, for a sequence of kv_len keys and `rows` rows (new tokens x query heads of a kv head).
int dib_fp4_attention_split_keys(int kv_len, int rows) { return split_keys(kv_len, rows); }

// The split form, for the sequences seq_list[0 .. seq_count) or (null) seq_first ...: heads of 32, 64, 96 or 128, pages of a
// power of two of rows, 4 at least.  max_rows: the most rows (new tokens x query heads of a kv head) of one of them; tile_rows: 8 or
// 16 rows a tile; max_items: the most (tiles x runs x kv heads) of one; part_o float32 [seq_count, max_items, tile_rows, 128] and
// part_ml [.., 4] take partial results where `runs`, the most runs of one of them, is not 0 (1 is given as 0).
int dib_fp4_attention_split(const void* q, void* out, const void* data, const void* scales, const void* exponents, long long num_pages,
                            const void* block_table, int max_blocks, const void* cu_q_lens, const void* seq_lens,
                            const void* seq_list, int seq_first, int seq_count, int max_rows, int tile_rows, void* part_o,
                            void* part_ml, int max_items, int runs, int Hq, int Hkv, int D, int page_size, float scale,
                            int window, int dtype, int sm_count, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (seq_count < 0 || seq_count > 4096 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || D < 32 || D > 128 || D % 32 != 0 || page_size < 4 ||
      (page_size & (page_size - 1)) != 0 || num_pages * 2 * Hkv * page_size >= (1ll << 31) || max_items < 1 || sm_count < 1 ||
      (tile_rows != 8 && tile_rows != 16))
    return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) != 0 ||
      (reinterpret_cast<uintptr_t>(scales) & 7) != 0 || (reinterpret_cast<uintptr_t>(exponents) & 3) != 0)
    return DIB_BAD_ALIGN;
  if (seq_count == 0 || max_rows == 0) return DIB_OK;
  SplitArgs a = cache_args(data, scales, exponents, num_pages, block_table, max_blocks, cu_q_lens, seq_lens, Hq, Hkv, D, scale, window);
  a.seq_list = reinterpret_cast<const int*>(seq_list);
  a.seq_first = seq_first;
  a.seq_count = seq_count;
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  a.part_o = reinterpret_cast<float*>(part_o);
  a.part_ml = reinterpret_cast<float4*>(part_ml);
  a.max_items = max_items;
  using B = __nv_bfloat16;
  if (dtype == 1)
    return tile_rows == 8 ? launch_split<B, 1>(q, out, a, max_rows, runs, sm_count, st) : launch_split<B, 2>(q, out, a, max_rows, runs, sm_count, st);
  return tile_rows == 8 ? launch_split<float, 1>(q, out, a, max_rows, runs, sm_count, st)
                        : launch_split<float, 2>(q, out, a, max_rows, runs, sm_count, st);
}

int dib_fp4_attention_any(const void* q, void* out, const void* data, const void* scales, const void* exponents, const void* block_table,
                          int max_blocks, const void* token_seq, const void* cu_q_lens, const void* seq_lens, int T, int Hq, int Hkv,
                          int D, int page_size, long long num_pages, float scale, int window, int dtype, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  if (T < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || D < 16 || D > 256 || D % 16 != 0 || page_size < 1 || num_pages > 0x7fffffffll)
    return DIB_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(data) & 15) != 0) return DIB_BAD_ALIGN;
  if (T == 0) return DIB_OK;
  const long long blocks = ((long long)T * Hq + ANY_WARPS - 1) / ANY_WARPS;
  if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
  const SplitArgs a = cache_args(data, scales, exponents, num_pages, block_table, max_blocks, cu_q_lens, seq_lens, Hq, Hkv, D, scale, window);
  const int* ts = reinterpret_cast<const int*>(token_seq);
  if (dtype == 1)
    dib_launch(attention_any_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(ANY_WARPS * 32), 0, st,
               reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<__nv_bfloat16*>(out), a, ts, T, page_size);
  else
    dib_launch(attention_any_kernel<float>, dim3((unsigned)blocks), dim3(ANY_WARPS * 32), 0, st, reinterpret_cast<const float*>(q),
               reinterpret_cast<float*>(out), a, ts, T, page_size);
  DIB_CHECK_LAUNCH();
  return DIB_OK;
}

}  // extern "C"
