// Attention of a step's new tokens over a paged cache in 8-bit integers (cache_int8.cu): query row i of head h, at
// position p, over the keys j of its sequence that it sees (j <= p, and j > p - window with a window):
//   s_j = scale * ks_j * (q . kc_j),   o = sum_j exp(s_j - m) vs_j vc_j / sum_j exp(s_j - m),
// kc, vc the codes of a key and a value, ks, vs their scales.  The scales never touch the codes: a key's joins its score,
// a value's the probability.  A row that sees no key is zeros.  A sequence's new tokens are its last ones.
//
// Forms: split (one to a few new tokens: the cache is streamed once and bounds it), and one for every shape.
#include <cuda.h>

#include "common.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
__device__ int dib_attention_int8_error_word = 0;

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_2d(unsigned dst, const CUtensorMap* map, int c0, int c1, unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<unsigned long long>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- split form
// A sequence's rows (new token, query head of the kv group), 8 NT at a time, against a run of its keys, by ONE warp: no
// warp waits for another.  Per block of 32 keys a warp holds, in its own ring of shared memory, the codes of the keys and
// values (TMA, swizzled, a copy a page) and their scales (cp.async), all counted by one mbarrier a stage; the next blocks,
// of the next work item too, are under way meanwhile.
//
// Products by mma.sync, transposed so that 16 KEYS (or 16 dimensions) are the rows and 8 query rows the columns:
// S^T = K Q^T, O^T = V^T P^T.  Eight rows fill the instruction, where a decoded token of a group of 2 to 8 heads would
// leave half of it or more empty.
//   S: m16n8k32 on the keys' bytes as they are.  A query row enters as integers against its largest element, of 15 bits
//   (bfloat16) or 22 (float32), as the sum of two or three bytes: an element is off by 2^-15 (2^-22) of the row's largest
//   at most, and the dot product of the integers is exact.
//   O: m16n8k16 on float16.  Codes become float16 numbers in registers, exactly: a byte under the exponent byte 0x64 is
//   1024 + byte.  Probabilities times value scale enter as one float16 number (bfloat16 queries) or the sum of two
//   (float32), against a power of two per row that follows their largest.
// The k index of a product may be permuted as long as both operands agree: a thread takes 32 (16) consecutive bytes of a
// key as its share of S's k, and of V 16 (8) consecutive dimensions of the keys that its part of P^T belongs to, so
// nothing is shuffled but P, by movmatrix.
//
// What bounds it: the bytes of keys and values.  The row's running maximum and its power of two are touched only when a
// score has passed them by 2^8 (2^12): one vote of the warp a block, no reductions.
//
// Work items: (sequence, run of keys, kv head, tile of rows).  The length of a run follows from the sequence's own
// lengths, so a row's bits do not depend on the rest of the step, nor on NT.
constexpr int SP_WARPS = 4, SP_BLOCK = 32;

// Keys of a run: short runs where a sequence has few keys (its warps then share them), longer ones where the partial
// results would grow; with many rows a run gets longer still, as their partial results do with the rows.
__host__ __device__ __forceinline__ int split_keys(int kv_len, int rows) {
  const int base = kv_len <= 2048 ? 64 : kv_len <= 4096 ? 128 : kv_len <= 16384 ? 256 : 512;
  const int tiles = (rows + 31) / 32;
  return tiles <= 2 ? base : base * tiles;
}

__device__ __forceinline__ unsigned half2_of(unsigned w, unsigned sel) {     // two code bytes (offset by 128) -> float16 x 2
  unsigned h = __byte_perm(w, 0x64646464u, sel), r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));         // 1024 + 128
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                        unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                       unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low_of(unsigned h) {
  float f;
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, a; }" : "=f"(f) : "r"(h));
  return f;
}
__device__ __forceinline__ float high_of(unsigned h) {
  float f;
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, b; }" : "=f"(f) : "r"(h));
  return f;
}

// 1 over the power of two below w, between 2^-67 and 2^60: the quotient of two of them is finite.  (Values above 2^83 so
// leave float16's range.)
__device__ __forceinline__ float unit_of(float w) {
  const int e = min(max((int)(__float_as_uint(w) >> 23), 67), 194);
  return __uint_as_float((unsigned)(254 - e) << 23);
}

struct SplitArgs {
  const float* scales;          // [pages, 2, Hkv, page_size]
  const int* block_table;       // [B, max_blocks]
  const int* cu_q_lens;
  const int* seq_lens;
  const int* seq_list;          // the sequences of this launch, or null: seq_first ..
  int seq_first, seq_count, max_blocks;
  int Hq, Hkv, D, page_shift, window, box_rows;
  int num_pages;
  float scale;
  float* part_o;                // [seq_count, max_items, 8 NT, D]
  float2* part_ml;              // [seq_count, max_items, 8 NT]: reference maximum (log 2), sum
  int max_items;
};
// A sequence of the launch and how it is cut.
struct SplitSeq {
  int seq, q_begin, n, kv_len, tiles, split, splits;
};
template <int ROWS> __device__ __forceinline__ SplitSeq split_seq(const SplitArgs& a, int i) {
  SplitSeq s;
  s.seq = a.seq_list != nullptr ? a.seq_list[i] : a.seq_first + i;
  s.q_begin = a.cu_q_lens[s.seq];
  s.n = a.cu_q_lens[s.seq + 1] - s.q_begin;
  s.kv_len = min(a.seq_lens[s.seq], (int)min((long long)a.max_blocks << a.page_shift, 0x7fffffc0ll));
  const int rows = s.n * (a.Hq / a.Hkv);
  s.tiles = (rows + ROWS - 1) / ROWS;
  s.split = split_keys(s.kv_len, rows);
  s.splits = s.n > 0 ? max(1, (s.kv_len + s.split - 1) / s.split) : 0;
  return s;
}

template <typename T, int DP, int NT> struct SplitShape {
  static constexpr int ROWS = 8 * NT;
  static constexpr int Q_PARTS = sizeof(T) == 4 ? 3 : 2;     // bytes a query's element is the sum of
  static constexpr int P_PARTS = sizeof(T) == 4 ? 2 : 1;     // float16 numbers a probability is the sum of
  static constexpr int STAGES = 2, QUEUE = 4;
  static constexpr int TILE = SP_BLOCK * DP;                 // a block's keys, or values
  // a warp's ring: the stages' tiles (each on 1,024 bytes), then the stages' scales
  static constexpr int SCALES = STAGES * 2 * TILE;
  static constexpr int RING = (SCALES + STAGES * 256 + 1023) / 1024 * 1024;
  static constexpr size_t fixed = (size_t)SP_WARPS * (RING + STAGES * 8 + QUEUE * 32) + 1024;
};

// A work item as it is handed from the end of a warp's pipe that fetches to the one that computes.
struct __align__(16) SplitItem {
  int i, kvh, tile;             // sequence of the launch, kv head, tile of rows
  int lo;                       // first key of the run
  int at, end;                  // its keys [at, end), `at` a multiple of 32 and perhaps below the first one seen
  int out_item, unused;         // number of the item among its sequence's
};

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(SP_WARPS * 32)
attention_split_kernel(const __grid_constant__ CUtensorMap map, const T* __restrict__ q, T* __restrict__ out,
                       const __grid_constant__ SplitArgs a) {
  using SH = SplitShape<T, DP, NT>;
  constexpr int ROWS = SH::ROWS, Q_PARTS = SH::Q_PARTS, P_PARTS = SH::P_PARTS, STAGES = SH::STAGES, QUEUE = SH::QUEUE;
  constexpr int MT = DP / 16, WORDS = DP / 16;      // 32-bit words of a thread's share of a key
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + warp * SH::RING;
  SplitItem* queue = reinterpret_cast<SplitItem*>(smem + SP_WARPS * SH::RING) + warp * QUEUE;
  unsigned long long* bars =
      reinterpret_cast<unsigned long long*>(smem + SP_WARPS * (SH::RING + QUEUE * 32)) + warp * STAGES;
  int* first = reinterpret_cast<int*>(smem + SP_WARPS * (SH::RING + QUEUE * 32 + STAGES * 8));    // [seq_count + 1]
  if (threadIdx.x == 0) prefetch_tensormap(&map);
  pdl_trigger();
  // ---- the items before each sequence (metadata alone, which no kernel of a step writes)
  for (int i = threadIdx.x; i < a.seq_count; i += blockDim.x) {
    const SplitSeq s = split_seq<ROWS>(a, i);
    first[i + 1] = s.tiles * s.splits * a.Hkv;
  }
  if (threadIdx.x == 0) first[0] = 0;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&bars[s], 33);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == 0) {
    int base = 0;
    for (int i0 = 0; i0 < a.seq_count; i0 += 32) {
      int v = i0 + lane < a.seq_count ? first[i0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (i0 + lane < a.seq_count) first[i0 + lane + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const int total = first[a.seq_count];
  const int G = a.Hq / a.Hkv;
  const int stride = gridDim.x * SP_WARPS;
  const int page_mask = (1 << a.page_shift) - 1;

  // ---- the end that fetches: its item, the block of keys to be sent for next, this lane's page of it
  int f_item = warp * gridDim.x + blockIdx.x, f_at = 0, f_end = 0, f_head = 0, f_page = -1, opened = 0;
  const int* f_table = nullptr;
  // the item f_item, or the first one behind it that has keys (on this warp's list); f_item >= total: none is left
  auto open = [&]() {
    for (; f_item < total; f_item += stride) {
      int lo = 0, hi = a.seq_count - 1;          // the sequence whose items hold this one
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= f_item) lo = mid; else hi = mid - 1;
      }
      const SplitSeq s = split_seq<ROWS>(a, lo);
      const int local = f_item - first[lo];
      int r = local, tile = 0;
      if (s.tiles > 1) {
        tile = r % s.tiles;
        r /= s.tiles;
      }
      const int kvh = r / s.splits, run_at = (r - kvh * s.splits) * s.split;
      const int p0 = s.kv_len - s.n, n_rows = s.n * G;
      int tok0 = 0, tok1 = s.n - 1;
      if (s.tiles > 1) {
        tok0 = tile * ROWS / G;
        tok1 = min((tile + 1) * ROWS, n_rows) - 1;
        tok1 /= G;
      }
      const int k_lo = max(run_at, first_visible_key(p0 + tok0, a.window)), k_hi = min(run_at + s.split, p0 + tok1 + 1);
      if (k_hi > k_lo) {
        f_at = k_lo & ~(SP_BLOCK - 1);
        f_end = k_hi;
        f_table = a.block_table + (long long)s.seq * a.max_blocks;
        f_head = kvh << a.page_shift;
        __syncwarp();
        if (lane == 0) {
          SplitItem it;
          it.i = lo; it.kvh = kvh; it.tile = tile; it.lo = run_at;
          it.at = f_at; it.end = f_end; it.out_item = local; it.unused = 0;
          queue[opened % QUEUE] = it;
        }
        __syncwarp();
        ++opened;
        return;
      }
      if (s.splits == 1)                         // a sequence of one run: rows that see no key are zeros, from here
        for (int e = lane; e < min(ROWS, n_rows - tile * ROWS) * a.D; e += 32) {
          const int row = tile * ROWS + e / a.D;
          Elem<T>::store(out + ((long long)(s.q_begin + row / G) * a.Hq + kvh * G + row % G) * a.D + e % a.D, 0.f);
        }
    }
  };
  auto look_up = [&]() {                         // this lane's page of the block at f_at, or -1
    const int key = f_at + lane;
    int page = -1;
    if (key < f_end) page = f_table[key >> a.page_shift];
    f_page = page < a.num_pages ? page : -1;
  };
  // the block -> stage: lane l's key is f_at + l; the first lane of each page sends for its rows
  auto fetch = [&](int stage) {
    const unsigned tiles = smem_u32(ring) + stage * 2 * SH::TILE;
    const unsigned sc = smem_u32(ring) + SH::SCALES + stage * 256 + lane * 4;
    const int off = (f_at + lane) & page_mask;
    const bool have = f_page >= 0;
    const bool sends = have && (lane == 0 || off == 0);
    const unsigned senders = __ballot_sync(0xffffffffu, sends);
    if (lane == 0) mbar_expect_tx(&bars[stage], __popc(senders) * 2 * a.box_rows * DP);
    __syncwarp();
    const int half = a.Hkv << a.page_shift;      // rows of a page's keys
    const int row = f_page * 2 * half + f_head + off;
    if (sends) {
      tma_load_2d(tiles + lane * DP, &map, 0, row, &bars[stage]);
      tma_load_2d(tiles + SH::TILE + lane * DP, &map, 0, row + half, &bars[stage]);
    }
    if (have) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc), "l"(a.scales + row) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc + 128), "l"(a.scales + row + half) : "memory");
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bars[stage])) : "memory");
    f_at += SP_BLOCK;
    if (f_at >= f_end) {
      f_item += stride;
      open();
    }
    if (f_item < total) look_up();
  };

  pdl_wait(q);
  open();
  if (f_item < total) look_up();
  int sent = 0, used = 0;                          // blocks sent for, consumed
  for (; sent < STAGES && f_item < total; ++sent) fetch(sent);

  // where a lane finds its pieces of a tile (the copy's swizzle: bits 4.. of the address joined by bits 7..)
  constexpr int SWIZZLE = DP == 128 ? 7 : 3, LINE = DP == 128 ? 1 : 2;      // rows of 128 bytes hold LINE keys
  int k_off[WORDS / 4], v_off[2];
#pragma unroll
  for (int p = 0; p < WORDS / 4; ++p)
    k_off[p] = g * DP + (((t * (WORDS / 4) + p) ^ ((g / LINE) & SWIZZLE)) << 4);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = 2 * t + e;
    v_off[e] = DP == 128 ? r * DP + ((g ^ (r & 7)) << 4) : r * DP + (((g >> 1) ^ ((r >> 1) & 3)) << 4) + (g & 1) * 8;
  }

  bool ok = true;
  for (int taken = 0; ok && taken < opened; ++taken) {
    const SplitItem it = queue[taken % QUEUE];
    const SplitSeq s_ = split_seq<ROWS>(a, it.i);
    const int p0 = s_.kv_len - s_.n, row0 = it.tile * ROWS, rows = min(ROWS, s_.n * G - row0);
    // ---- queries: row g of tile nt as the B operand, this thread's share of the dimensions, as the sum of Q_PARTS bytes
    // of 7 bits each against the row's largest element
    unsigned qf[NT][Q_PARTS][WORDS];
    float q_unit[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const bool in = r < rows;
      const int tok = in ? (row0 + r) / G : 0, h = in ? row0 + r - tok * G : 0;
      const T* src = q + ((long long)(s_.q_begin + tok) * a.Hq + it.kvh * G + h) * a.D + t * (DP / 4);
      float x[DP / 4];
#pragma unroll
      for (int v = 0; v < DP / 4; v += 16 / (int)sizeof(T)) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (in && t * (DP / 4) + v < a.D) w = *reinterpret_cast<const uint4*>(src + v);
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (sizeof(T) == 2) {
            x[v + 2 * e] = __uint_as_float(u[e] << 16);
            x[v + 2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
          } else {
            x[v + e] = __uint_as_float(u[e]);
          }
        }
      }
      unsigned bits = 0;
#pragma unroll
      for (int d = 0; d < DP / 4; ++d) bits = max(bits, __float_as_uint(x[d]) & 0x7fffffffu);
      bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
      bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
      const float top = fmaxf(__uint_as_float(bits), 0x1p-100f);
      constexpr float MOST = Q_PARTS == 3 ? 127.f * 16384.f : 127.f * 128.f;
      const float up = MOST / top;
      // (a row that holds an infinity or a NaN: its unit is NaN, and so is all that comes of it)
      q_unit[nt] = bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.scale * LOG2E * (top / MOST);
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        int part[4][3];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          int v = __float2int_rn(x[4 * j + b] * up);
          if (Q_PARTS == 3) {
            const int above = (v + 64) >> 7;
            part[b][2] = v - above * 128;
            v = above;
          }
          part[b][0] = (v + 64) >> 7;
          part[b][1] = v - part[b][0] * 128;
        }
#pragma unroll
        for (int p = 0; p < Q_PARTS; ++p)
          qf[nt][p][j] = __byte_perm(__byte_perm(part[0][p], part[1][p], 0x0040), __byte_perm(part[2][p], part[3][p], 0x0040), 0x5410);
      }
    }
    // ---- what belongs to the rows this thread has scores of: 2t and 2t + 1 of each tile
    float unit[NT][2], m[NT][2], l[NT][2], w_unit[NT][2];
    int k_lo[NT][2], k_hi[NT][2], lo_all = it.lo, hi_all = it.end - 1;
    float o[NT][MT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + 2 * t + e;
        const bool in = r < rows;
        const int p = p0 + (in ? (row0 + r) / G : 0);
        unit[nt][e] = __shfl_sync(0xffffffffu, q_unit[nt], (2 * t + e) * 4);
        k_lo[nt][e] = max(first_visible_key(p, a.window), it.lo);
        k_hi[nt][e] = in ? min(p, it.end - 1) : -1;
        if (in) {        // (rows of the tile beyond the sequence's last one: their scores are never looked at)
          lo_all = max(lo_all, k_lo[nt][e]);
          hi_all = min(hi_all, p);
        }
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
        w_unit[nt][e] = 1.f;
      }
#pragma unroll
    for (int o_ = 1; o_ < 4; o_ <<= 1) {
      lo_all = max(lo_all, __shfl_xor_sync(0xffffffffu, lo_all, o_));
      hi_all = min(hi_all, __shfl_xor_sync(0xffffffffu, hi_all, o_));
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;

    for (int kb = it.at; kb < it.end; kb += SP_BLOCK, ++used) {
      const int stage = used % STAGES;
      ok = mbar_wait(&bars[stage], (used / STAGES) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const unsigned char* kt = ring + stage * 2 * SH::TILE;
      const unsigned char* vt = kt + SH::TILE;
      const float* sc = reinterpret_cast<const float*>(ring + SH::SCALES) + stage * 64;
      // ---- S^T, an exact integer
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint4 kw[2][WORDS / 4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int p = 0; p < WORDS / 4; ++p)
            kw[half][p] = *reinterpret_cast<const uint4*>(kt + (mt * 16 + half * 8) * DP + k_off[p]);
        int acc[NT][Q_PARTS][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int p = 0; p < Q_PARTS; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][p][e] = 0;
#pragma unroll
        for (int p4 = 0; p4 < WORDS / 4; ++p4)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int p = 0; p < Q_PARTS; ++p) {
              mma_s8(acc[nt][p], kw[0][p4].x, kw[1][p4].x, kw[0][p4].y, kw[1][p4].y, qf[nt][p][p4 * 4], qf[nt][p][p4 * 4 + 1]);
              mma_s8(acc[nt][p], kw[0][p4].z, kw[1][p4].z, kw[0][p4].w, kw[1][p4].w, qf[nt][p][p4 * 4 + 2], qf[nt][p][p4 * 4 + 3]);
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float high = (float)(acc[nt][0][e] * 128 + acc[nt][1][e]);
            s[mt][nt][e] = Q_PARTS == 3 ? fmaf(high, 128.f, (float)acc[nt][Q_PARTS - 1][e]) : high;
          }
      }
      float ks[2][2], vs[2][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ks[mt][half] = sc[mt * 16 + half * 8 + g];
          vs[mt][half] = sc[32 + mt * 16 + half * 8 + g];
        }
      const bool plain = kb >= lo_all && kb + SP_BLOCK - 1 <= hi_all;      // every row sees every key
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) s[mt][nt][2 * half + e] *= ks[mt][half] * unit[nt][e];
        }
      if (!plain) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int key = kb + mt * 16 + half * 8 + g;
                if (key < k_lo[nt][e] || key > k_hi[nt][e]) s[mt][nt][2 * half + e] = -INFINITY;
              }
      }
      bool high = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(fmaxf(s[0][nt][e], s[0][nt][2 + e]), fmaxf(s[1][nt][e], s[1][nt][2 + e]));
          high |= top[nt][e] > m[nt][e] + 8.f;
        }
      if (__any_sync(0xffffffffu, high)) {
        // some row's reference maximum rises (each row by its own scores alone)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float best = top[nt][e];
#pragma unroll
            for (int o_ = 4; o_ < 32; o_ <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o_));
            float factor = 1.f;
            if (best > m[nt][e] + 8.f) {
              factor = fast_exp2(m[nt][e] - best);     // (zero from minus infinity)
              m[nt][e] = best;
              l[nt][e] *= factor;
              // the probabilities' power of two is chosen anew: by the block's largest probability * scale
              float wt = 0.f;
#pragma unroll
              for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                  wt = fmaxf(wt, fast_exp2(s[mt][nt][2 * half + e] - best) * vs[mt][half]);
              const unsigned lanes = 0x11111111u << t;      // (every lane of a row takes this branch)
#pragma unroll
              for (int o_ = 4; o_ < 32; o_ <<= 1) wt = fmaxf(wt, __shfl_xor_sync(lanes, wt, o_));
              const float now = unit_of(wt);
              if (factor * (now / w_unit[nt][e]) <= 0x1p40f) {      // (else what O holds outweighs the block by far)
                factor *= now / w_unit[nt][e];
                w_unit[nt][e] = now;
              }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[nt][i][e] *= factor;
              o[nt][i][2 + e] *= factor;
            }
          }
      }
      // ---- probabilities, times the value's scale and the row's power of two
      bool large = false;
      float w[2][NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ref = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
          float most = 0.f;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float p = fast_exp2(s[mt][nt][2 * half + e] - ref);
              l[nt][e] += p;
              w[mt][nt][2 * half + e] = p * (vs[mt][half] * w_unit[nt][e]);
              most = fmaxf(most, w[mt][nt][2 * half + e]);
            }
          large |= most > 4096.f;
        }
      if (!plain) {        // a key that the row does not see may have a value that is no number
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (s[mt][nt][e] == -INFINITY) w[mt][nt][e] = 0.f;
      }
      if (__any_sync(0xffffffffu, large)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float wt = fmaxf(fmaxf(w[0][nt][e], w[0][nt][2 + e]), fmaxf(w[1][nt][e], w[1][nt][2 + e]));
#pragma unroll
            for (int o_ = 4; o_ < 32; o_ <<= 1) wt = fmaxf(wt, __shfl_xor_sync(0xffffffffu, wt, o_));
            float factor = 1.f;
            if (wt > 4096.f) factor = unit_of(wt);      // (of the product with the old unit)
            w_unit[nt][e] *= factor;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              w[mt][nt][e] *= factor;
              w[mt][nt][2 + e] *= factor;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[nt][i][e] *= factor;
              o[nt][i][2 + e] *= factor;
            }
          }
      }
      // ---- O^T += V^T P^T, 16 keys at a time
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        unsigned pf[NT][P_PARTS][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float w0 = w[mt][nt][2 * half], w1 = w[mt][nt][2 * half + 1];
            const unsigned hi = pack_f16(w0, w1);
            pf[nt][0][half] = transpose8(hi);
            if (P_PARTS == 2) pf[nt][P_PARTS - 1][half] = transpose8(pack_f16(w0 - low_of(hi), w1 - high_of(hi)));
          }
        // the thread's 16 (8) dimensions of the keys 2t, 2t + 1, 2t + 8, 2t + 9
        unsigned vw[4][DP / 32];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const unsigned char* src = vt + (mt * 16 + (kk >> 1) * 8) * DP + v_off[kk & 1];
          if (DP == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            vw[kk][0] = v.x ^ 0x80808080u;
            vw[kk][1] = v.y ^ 0x80808080u;
            vw[kk][DP / 32 - 2] = v.z ^ 0x80808080u;
            vw[kk][DP / 32 - 1] = v.w ^ 0x80808080u;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src);
            vw[kk][0] = v.x ^ 0x80808080u;
            vw[kk][1] = v.y ^ 0x80808080u;
          }
        }
#pragma unroll
        for (int c4 = 0; c4 < DP / 32; ++c4) {
          const unsigned x = __byte_perm(vw[0][c4], vw[1][c4], 0x5140), y = __byte_perm(vw[0][c4], vw[1][c4], 0x7362);
          const unsigned u = __byte_perm(vw[2][c4], vw[3][c4], 0x5140), z = __byte_perm(vw[2][c4], vw[3][c4], 0x7362);
          const unsigned a0 = half2_of(x, 0x4140), a1 = half2_of(x, 0x4342), a2 = half2_of(u, 0x4140), a3 = half2_of(u, 0x4342);
          const unsigned b0 = half2_of(y, 0x4140), b1 = half2_of(y, 0x4342), b2 = half2_of(z, 0x4140), b3 = half2_of(z, 0x4342);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int p = P_PARTS - 1; p >= 0; --p) {       // the small part first
              mma_f16(o[nt][2 * c4], a0, a1, a2, a3, pf[nt][p][0], pf[nt][p][1]);
              mma_f16(o[nt][2 * c4 + 1], b0, b1, b2, b3, pf[nt][p][0], pf[nt][p][1]);
            }
        }
      }
      __syncwarp();                                    // every lane has read the stage
      if (f_item < total) {
        fetch(stage);
        ++sent;
      }
    }
    if (!ok) break;
    // ---- the item's rows: finished where the sequence has one run, else partial results for the merge
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
#pragma unroll
        for (int o_ = 4; o_ < 32; o_ <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o_);
        const int r = nt * 8 + 2 * t + e;
        if (r >= rows) continue;
        const float back = 1.f / w_unit[nt][e];
        const int d0 = g * (DP / 8);
        if (d0 >= a.D) continue;
        if (s_.splits == 1) {
          const float inv = sum == 0.f ? 0.f : back / sum;
          const int tok = (row0 + r) / G;
          T* dst = out + ((long long)(s_.q_begin + tok) * a.Hq + it.kvh * G + row0 + r - tok * G) * a.D + d0;
#pragma unroll
          for (int i = 0; i < MT; i += 2) {
            if (d0 + 2 * i >= a.D) break;
            const float y0 = o[nt][i][e] * inv, y1 = o[nt][i][2 + e] * inv, y2 = o[nt][i + 1][e] * inv, y3 = o[nt][i + 1][2 + e] * inv;
            if (sizeof(T) == 2) {
              const __nv_bfloat162 lo2 = __floats2bfloat162_rn(y0, y1), hi2 = __floats2bfloat162_rn(y2, y3);
              *reinterpret_cast<uint2*>(dst + 2 * i) =
                  make_uint2(*reinterpret_cast<const unsigned*>(&lo2), *reinterpret_cast<const unsigned*>(&hi2));
            } else {
              *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(y0, y1, y2, y3);
            }
          }
        } else if (it.out_item < a.max_items) {
          const long long at = ((long long)it.i * a.max_items + it.out_item) * ROWS + r;
          float* dst = a.part_o + at * a.D + d0;
#pragma unroll
          for (int i = 0; i < MT; i += 2) {
            if (d0 + 2 * i >= a.D) break;
            *reinterpret_cast<float4*>(dst + 2 * i) =
                make_float4(o[nt][i][e] * back, o[nt][i][2 + e] * back, o[nt][i + 1][e] * back, o[nt][i + 1][2 + e] * back);
          }
          if (g == 0) a.part_ml[at] = make_float2(m[nt][e], sum);
        }
      }
  }
  if (!ok) {
    atomicExch(&dib_attention_int8_error_word, 1);
    for (int u = used + 1; u < sent; ++u) mbar_wait(&bars[u % STAGES], (u / STAGES) & 1);      // no copy outlives the warp
  }
}

// The runs' results of a row, in the order of the runs: a warp a row, a lane 4 dimensions.
constexpr int SM_WARPS = 4;
template <typename T, int NT>
__global__ void __launch_bounds__(SM_WARPS * 32)
attention_split_merge_kernel(T* __restrict__ out, const __grid_constant__ SplitArgs a) {
  constexpr int ROWS = 8 * NT;
  const float* part_o = a.part_o;
  const float2* part_ml = a.part_ml;
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.y, G = a.Hq / a.Hkv;
  const SplitSeq s = split_seq<ROWS>(a, i);
  const int n_rows = s.n * G;                      // of a kv head
  const int id = blockIdx.x * SM_WARPS + warp;
  pdl_wait(part_o, part_ml);
  if (s.splits <= 1 || id >= n_rows * a.Hkv || s.splits * s.tiles * a.Hkv > a.max_items) return;
  const int kvh = id / n_rows, row = id % n_rows, tile = row / ROWS, r = row % ROWS;
  const int p0 = s.kv_len - s.n;
  const int tok0 = tile * ROWS / G, tok1 = min((tile + 1) * ROWS - 1, n_rows - 1) / G;
  // the runs that hold keys which some row of the tile sees
  const int k_lo = first_visible_key(p0 + tok0, a.window), k_hi = p0 + tok1;
  const int s0 = k_lo / s.split, s1 = k_hi < k_lo ? s0 - 1 : min(k_hi / s.split, s.splits - 1);
  const long long base = (long long)i * a.max_items + (long long)kvh * s.splits * s.tiles + tile;
  auto at = [&](int run) { return (base + (long long)run * s.tiles) * ROWS + r; };
  float top = -INFINITY;
  for (int run = s0 + lane; run <= s1; run += 32) top = fmaxf(top, part_ml[at(run)].x);
  top = warp_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f), o2 = o;
  float sum = 0.f;
  const bool in = lane * 4 < a.D;
  for (int run0 = s0; run0 <= s1; run0 += 32) {
    float w = 0.f, ws = 0.f;
    if (run0 + lane <= s1) {
      const float2 ml = part_ml[at(run0 + lane)];
      w = fast_exp2(ml.x - ref);
      ws = w * ml.y;
    }
    sum += warp_sum(ws);
    const int n = min(32, s1 - run0 + 1);
    int j = 0;
    for (; j + 8 <= n; j += 8) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = in ? *reinterpret_cast<const float4*>(part_o + at(run0 + j + u) * a.D + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float wj = __shfl_sync(0xffffffffu, w, j + u);
        float4& d = u & 1 ? o2 : o;
        d.x = fmaf(wj, v[u].x, d.x); d.y = fmaf(wj, v[u].y, d.y);
        d.z = fmaf(wj, v[u].z, d.z); d.w = fmaf(wj, v[u].w, d.w);
      }
    }
    for (; j < n; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const float4 v = in ? *reinterpret_cast<const float4*>(part_o + at(run0 + j) * a.D + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      o.x = fmaf(wj, v.x, o.x); o.y = fmaf(wj, v.y, o.y); o.z = fmaf(wj, v.z, o.z); o.w = fmaf(wj, v.w, o.w);
    }
  }
  if (!in) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const float y[4] = {(o.x + o2.x) * inv, (o.y + o2.y) * inv, (o.z + o2.z) * inv, (o.w + o2.w) * inv};
  T* dst = out + ((long long)(s.q_begin + row / G) * a.Hq + kvh * G + row % G) * a.D + lane * 4;
#pragma unroll
  for (int e = 0; e < 4; ++e) Elem<T>::store(dst + e, y[e]);
}

// ---------------------------------------------------------------- the form for every shape
// Head sizes up to 256, any page size and group ratio: a warp takes a (token, head), a lane a key of 32 at a time for
// the scores, then a lane D / 32 dimensions for the values.
constexpr int ANY_WARPS = 4;

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
    for (int d = lane; d < D; d += 32) sq[warp][d] = Elem<T>::load(q + item * D + d) * scale * LOG2E;
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

// ---------------------------------------------------------------- host side
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
// The cache as rows of D bytes; boxes of box_rows x DP bytes (what lies beyond D reads as zero), swizzled.
bool make_cache_map(CUtensorMap* map, const void* data, long long rows, int D, int DP, int box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)D};
  const cuuint32_t box[2] = {(cuuint32_t)DP, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(data), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, DP == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, int NT>
int launch_split(const CUtensorMap& map, const void* q, void* out, const SplitArgs& a, int max_rows, int merge, int sm_count,
                 cudaStream_t st) {
  using SH = SplitShape<T, DP, NT>;
  auto kern = attention_split_kernel<T, DP, NT>;
  const size_t smem = SH::fixed + ((size_t)a.seq_count + 1) * 4;
  if (smem > 200 * 1024) return DIB_BAD_SIZE;
  static DeviceOnce attr_set;
  if (!attr_set.done()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess)
      return DIB_LAUNCH_FAILED;
    attr_set.mark();
  }
  int per_sm = 0;      // the grid is what runs at a time
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, SP_WARPS * 32, smem) != cudaSuccess || per_sm < 1)
    return DIB_LAUNCH_FAILED;
  dib_launch(kern, dim3(sm_count * per_sm), dim3(SP_WARPS * 32), smem, st, map, reinterpret_cast<const T*>(q), reinterpret_cast<T*>(out), a);
  DIB_CHECK_LAUNCH();
  if (merge) {
    const long long blocks = ((long long)max_rows * a.Hkv + SM_WARPS - 1) / SM_WARPS;
    if (blocks > 0x7fffffffll) return DIB_BAD_SIZE;
    dib_launch(attention_split_merge_kernel<T, NT>, dim3((unsigned)blocks, a.seq_count), dim3(SM_WARPS * 32), 0, st,
               reinterpret_cast<T*>(out), a);
    DIB_CHECK_LAUNCH();
  }
  return DIB_OK;
}

}  // namespace

extern "C" {

int dib_attention_int8_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dib_attention_int8_error_word, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int dib_attention_int8_status_clear() {
  const int v = 0;
  return cudaMemcpyToSymbol(dib_attention_int8_error_word, &v, sizeof(int)) == cudaSuccess ? 0 : -1;
}

// Keys of a run of the split form, for a sequence of kv_len keys and `rows` rows (new tokens x query heads of a kv head).
int dib_int8_attention_split_keys(int kv_len, int rows) { return split_keys(kv_len, rows); }

// The split form, for the sequences seq_list[0 .. seq_count) or (null) seq_first ...: heads up to 128, pages of a
// power of two of rows, 4 at least.  max_rows: the most rows (new tokens x query heads of a kv head) of one of them; tile_rows: 8
// or 16 rows a tile; max_items: the most (tiles x runs x kv heads) of one; part_o float32 [seq_count, max_items,
// tile_rows, D] and part_ml [.., 2] take partial results where merge is not 0 (some sequence may have two runs).
int dib_int8_attention_split(const void* q, void* out, const void* data, const void* scales, long long num_pages,
                             const void* block_table, int max_blocks, const void* cu_q_lens, const void* seq_lens,
                             const void* seq_list, int seq_first, int seq_count, int max_rows, int tile_rows, void* part_o,
                             void* part_ml, int max_items, int merge, int Hq, int Hkv, int D, int page_size, float scale,
                             int window, int dtype, int sm_count, cudaStream_t st) {
  if (dtype != 0 && dtype != 1) return DIB_BAD_DTYPE;
  const bool pages_fit = page_size >= 4 && (page_size & (page_size - 1)) == 0;
  if (seq_count < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || D < 16 || D > 128 || D % 16 != 0 || page_size < 1 || !pages_fit ||
      num_pages * 2 * Hkv * page_size >= (1ll << 31) || seq_count > 65535 || max_items < 1 || sm_count < 1 ||
      (tile_rows != 8 && tile_rows != 16))
    return DIB_BAD_SIZE;
  if (((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return DIB_BAD_ALIGN;
  if (seq_count == 0 || max_rows == 0) return DIB_OK;
  SplitArgs a;
  a.scales = reinterpret_cast<const float*>(scales);
  a.block_table = reinterpret_cast<const int*>(block_table);
  a.cu_q_lens = reinterpret_cast<const int*>(cu_q_lens);
  a.seq_lens = reinterpret_cast<const int*>(seq_lens);
  a.seq_list = reinterpret_cast<const int*>(seq_list);
  a.seq_first = seq_first;
  a.seq_count = seq_count;
  a.max_blocks = max_blocks;
  a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.window = window;
  a.page_shift = 0;
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  a.box_rows = page_size < SP_BLOCK ? page_size : SP_BLOCK;
  a.scale = scale;
  a.part_o = reinterpret_cast<float*>(part_o);
  a.part_ml = reinterpret_cast<float2*>(part_ml);
  a.max_items = max_items;
  a.num_pages = (int)num_pages;
  const int DP = D <= 64 ? 64 : 128;
  CUtensorMap map;
  if (!make_cache_map(&map, data, num_pages * 2 * Hkv * page_size, D, DP, a.box_rows)) return DIB_LAUNCH_FAILED;
  using B = __nv_bfloat16;
  if (dtype == 1) {
    if (DP == 128) return tile_rows == 8 ? launch_split<B, 128, 1>(map, q, out, a, max_rows, merge, sm_count, st)
                                         : launch_split<B, 128, 2>(map, q, out, a, max_rows, merge, sm_count, st);
    return tile_rows == 8 ? launch_split<B, 64, 1>(map, q, out, a, max_rows, merge, sm_count, st)
                          : launch_split<B, 64, 2>(map, q, out, a, max_rows, merge, sm_count, st);
  }
  if (DP == 128) return tile_rows == 8 ? launch_split<float, 128, 1>(map, q, out, a, max_rows, merge, sm_count, st)
                                       : launch_split<float, 128, 2>(map, q, out, a, max_rows, merge, sm_count, st);
  return tile_rows == 8 ? launch_split<float, 64, 1>(map, q, out, a, max_rows, merge, sm_count, st)
                        : launch_split<float, 64, 2>(map, q, out, a, max_rows, merge, sm_count, st);
}

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
