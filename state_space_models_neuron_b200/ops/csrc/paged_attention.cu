// Attention of one new token per sequence over a paged key-value cache.
//
//   s_t = scale q . k_t,  o = sum_t 2^(s'_t - m) v_t / sum_t 2^(s'_t - m),  s' = s log2(e), m a running maximum
//
// Bound by reading the cache once: 2 D values per token and key head for 4 D operations per query head, so a key head's queries
// (up to 8, or 16 with two column tiles) meet in one matrix product, tokens as rows and heads as columns:
//   S^T[16 tokens, 8 heads] = K Q^T,  O^T[D, 8 heads] += V^T P^T     (mma.sync m16n8k16, fp32 sums)
// The products take a fraction of the time that the bytes take, so they need no tcgen05 and its tiles of 128 tokens.  Each warp
// has a ring of its own in shared memory, which TMA fills (a step of 8 KB or more under way, boxes of 16 tokens, 128 swizzled bytes of
// a row each), so no warp waits for another one.  Fragments are read as 16-byte vectors: the channels of a product may be in any order if both
// operands agree, and so may the rows of V^T and, if P^T follows, the tokens; the orders below (sigma) are those without bank
// conflicts.  P^T is the transpose of the fragment in which S^T comes: one movmatrix per 8 tokens.
//   us, 64 x 8192 tokens of 8 heads of 128 channels, 4 queries each, bf16: one warp per query head 9071; these products with a
//   lane's copies by cp.async 503 (the warps wait for the load-store unit); TMA 331; 64 KB under way per SM instead of 128 319 (6.7 TB/s)
//
// Work is cut into steps of one key head; the steps of all sequences and key heads stand in one row, and each worker, a block or a
// warp, takes an equal share of it, however the lengths differ.  An item (a key head of a sequence) that several workers share is joined by
// the one that finishes last, in the order of the workers: (m, sum, unnormalised o) of each from the caller's workspace.
//
// 8-bit values are multiplied in fp16, which holds them exactly: queries times a power of two per head that brings their largest
// magnitude to [2^14, 2^15) (those down to 2^-31 of it stay exact, further ones are off by 2^-39 of it at most), probabilities with the scale
// of their value, as shares of a running maximum of their own (M below: scales of tokens may be any numbers).  64 x 8192 tokens
// e4m3 175 us, int8 180 (floor 169).  Where a step holds few bytes the two or three warps of a scheduler wait for their own chains of product,
// maximum, exponential, transpose and product (64 channels e4m3 58 of 44, 16 heads on one key head int8 26 of 11: 46 and 34 % of the issue
// slots while an SM is busy, 6 and 5 cycles per instruction, of which 1.8 and 1.4 are fixed latencies, 1.0 and 0.7 copies, 0.4 and 0.5 shared memory).
#include "kv_pages.cuh"
#include "gemm_scratch.h"

namespace ssm {

constexpr int PA_WARPS = 4, PA_BOX = 16, PA_COUNTERS = 2048;     // PA_BOX: tokens of a box
// Steps of a block (few items) and of a warp that make a share.  Blocks: four steps per warp (two: 200 tokens 8.3 us instead of 7.0, a join that saves
// nothing; eight: 2048 tokens 12.5 instead of 10.2).  Warps: four (one / four / twelve, us: 100 of 50 tokens bf16 12.1 / 8.4 / 17.3, 300 of 1 11.2 / 12.9 /
// 29.6, 40 of 300 int8 13.5 / 18.0 / 33.6).
constexpr int PA_BLOCK_SHARE = 4 * PA_WARPS, PA_WARP_SHARE = 4;
constexpr int FEW_ITEMS = 2, LONG_ITEM = 48;   // blocks per item and steps of an item, see the kernel
// Who takes the work of `filled` sequences with `total` steps: blocks, each of one item only; blocks, in equal shares of all steps; warps.
enum { BY_ITEM = 0, BY_BLOCK = 1, BY_WARP = 2 };
__host__ __device__ inline int paged_attn_workers(int filled, int items, int total, int most_blocks) {
  if ((long long)filled * items * FEW_ITEMS <= most_blocks) return BY_ITEM;
  return total >= (long long)filled * items * LONG_ITEM ? BY_BLOCK : BY_WARP;
}
// Steps of a worker's share; of the first guess where each item is cut by itself.
__host__ __device__ inline int paged_attn_share(int total, int workers, bool team) {
  const int even = (total + workers - 1) / workers, whole = (even + PA_WARPS - 1) / PA_WARPS * PA_WARPS;
  return team ? (whole < PA_BLOCK_SHARE ? PA_BLOCK_SHARE : whole) : (even < PA_WARP_SHARE ? PA_WARP_SHARE : even);
}
// A running maximum moves when scores pass it by 2^8: bf16 and fp16 hold larger shares as well.
// fp16 shares are at most 2^7 where M is chosen and may grow to 2^15.
constexpr float PA_GROWTH = 8.f, PA_SHARE = 32768.f;
constexpr int PA_SHARE_BITS = 7;

struct AttnArgs {
  const __nv_bfloat16* q; __nv_bfloat16* out;
  long long qb, qh;
  const uint8_t* pages[2];
  const float* scales[2];
  PageTable table;
  int B, Hq, Hk, most_blocks, groups, ratio;   // groups: of 8 or 16 query heads that share a key head; ratio: query heads per key head
  float scale;                                 // times log2(e)
  float* ws; int* counters;
};

template <int D, int T, int NT>
struct PagedAttn {
  static constexpr int BYTES = KvType<T>::BYTES, ROW = D * BYTES, HEADS = 8 * NT;
  static constexpr int SUB = ROW == 64 ? 4 : ROW == 128 ? 2 : 1, STEP = PA_BOX * SUB;        // boxes and tokens of a warp's step: 8 KB of keys and values
  static constexpr int TILE = ROW >= 128 ? 128 : 64, TILES = ROW / TILE;      // bytes of a box's rows (and of its swizzle), boxes of a row
  static constexpr int KCH = ROW / 64;                         // 16-byte pieces of a key row per lane (four lanes share a row)
  static constexpr int VB = TILE / 8, VEL = VB / BYTES;        // bytes and values of a lane's piece of a value row's tile (eight lanes share it)
  static constexpr int BOX = PA_BOX * ROW;                     // bytes of a box's keys, or values
  static constexpr int STAGE = SUB * 2 * BOX;                  // of one warp: keys and values of each box
  static constexpr int LOADED = 2 * BOX + (T == KV_BF16 ? 0 : 2 * PA_BOX * 4); // of one box, with the scales
  static constexpr int STAGES = 2;
  static constexpr int RING = PA_WARPS * STAGES * STAGE;
  static constexpr int SMEM = RING + 1024;                     // boxes begin on 1024 bytes
  // Blocks per SM.  64 KB of loads under way per SM are enough, and more of them cost bandwidth (bf16, two blocks of two stages / of three /
  // three blocks of two, us: 64 x 8192 320 / 331 / 327, one of 131072 88 / 95 / 99; 256 of 200 tokens 53.5 / 51.0 / 48.6).  Where warps
  // wait for their own chains, 8-bit values of 64 channels and int8, a third block fills the gaps (two / three: 64 channels e4m3 65 / 58, 64 x 8192 int8
  // 195 / 181, but e4m3 of 128 channels 176 / 181 and one of 131072 54 / 62).
  static constexpr int BLOCKS = SMEM > 113 * 1024 ? 1 : NT == 1 && (ROW == 64 || (ROW == 128 && T == KV_INT8)) ? 3 : 2;
  static constexpr int SLOT = HEADS * D + 3 * HEADS;           // floats of a part: o [channel][head], m, sum, M
  static constexpr int MEET = D * HEADS + D / VEL * 8;         // floats of a warp's o where the warps meet, see leave()
  static_assert(PA_WARPS * MEET * 4 <= RING && PA_COUNTERS / PA_WARPS * HEADS * 4 <= RING, "the warps' results meet in the ring");
};

// Token of row g of S^T (and of row g + 8, eight further), and 16-byte piece of a 128-byte row of V that lane group g takes: 0 4 1 5
// 2 6 3 7.  The eight lanes of one access are two neighbouring groups; their rows (of K) or pieces (of V) differ in bit 2, so that the
// swizzle, piece ^ row, sends them to eight different 16-byte columns.  Rows of 64 bytes keep their order.
template <int TILE>
__device__ __forceinline__ int sigma(int g) { return TILE == 128 ? ((g & 1) << 2) | (g >> 1) : g; }

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// a value's scale relative to M; not infinite, so that a token whose probability is 0 adds nothing, but NaN where the scale is
__device__ __forceinline__ float value_share(float scale, float G) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(scale * G), "f"(0x1p127f));
  return r;
}
// 2^(m - to), 0 for a part without tokens
__device__ __forceinline__ float part_factor(float m, float to) { return m == -INFINITY ? 0.f : exp2f(m - to); }
// What an unnormalised result is multiplied with, one after the other (8-bit values: the product alone may be below fp32's normal numbers);
// 0 where there are no tokens.
__device__ __forceinline__ float out_share(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }
__device__ __forceinline__ float out_size(float m, float M) { return m == -INFINITY ? 0.f : exp2f(M - m); }

// tokens of sequence b: not below 0, not beyond its pages
__device__ __forceinline__ int tokens_of(const AttnArgs& a, int b) {
  const int n = a.table.lengths[b];
  const long long room = (long long)a.table.width << a.table.page_shift;
  if (n <= room) return n < 0 ? 0 : n;
  report_bad_index(a.table.status);
  return (int)room;
}
// adds one to a counter; what the block wrote before its barrier is visible to whoever sees the sum, and the other way round
__device__ __forceinline__ int arrive(int* counter) {
  int before;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

template <int D, int T, int NT>
struct AttnWarp {
  using C = PagedAttn<D, T, NT>;
  static constexpr bool F16 = T != KV_BF16;
  uint32_t qf[NT][D / 8];                      // Q^T fragments; [D / 32 or D / 64 blocks of channels][4 or 8 words]
  float qs[NT][2];                             // what a sum of products of column 2c, 2c + 1 is multiplied with
  // Relative to the running maximum m, sums of 2^(s' - m); o relative to M, which is m for 16-bit values.  With 8 bits o sums
  // 2^(s' - M) times the value's scale: G = 2^(m - M), and M is at least m - 120, so that G is an fp32 number.
  float o[NT][D / 16][4], m[NT][2], l[NT][2], M[NT][2], G[NT][2];
  bool fresh;                                  // no tokens yet

  // queries of heads first .. first + HEADS - 1 of a key head; `real` of them exist
  __device__ __forceinline__ void load_queries(const AttnArgs& a, const __nv_bfloat16* q, int real) {
    const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool some = nt * 8 + g < real;
      const __nv_bfloat16* p = q + (nt * 8 + g) * a.qh;
      if (!F16) {
        #pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 u = some ? *reinterpret_cast<const uint4*>(p + i * 32 + c * 8) : make_uint4(0, 0, 0, 0);
          qf[nt][i * 4] = u.x; qf[nt][i * 4 + 1] = u.y; qf[nt][i * 4 + 2] = u.z; qf[nt][i * 4 + 3] = u.w;
        }
        qs[nt][0] = qs[nt][1] = a.scale;
      } else {
        uint32_t top = 0;
        #pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          #pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 u = some ? *reinterpret_cast<const uint4*>(p + i * 64 + c * 16 + j * 8) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
              qf[nt][i * 8 + j * 4 + k] = w[k];
              top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
            }
          }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the head's largest magnitude (not below 20, so that both factors are normal numbers); where it is not finite any will do
        const int e = max((int)(top >> 7), 20);
        const float f = __uint_as_float((uint32_t)(268 - e) << 23);                             // 2^(141 - e)
        #pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          float lo, hi;
          unpack2(mul2(bf16x2_pair(qf[nt][k]), pack2(f, f)), lo, hi);
          qf[nt][k] = pack_f16(lo, hi);
        }
        // the columns of this lane's sums are heads 2c, 2c + 1, whose exponents lanes 8c and 8c + 4 know
        #pragma unroll
        for (int j = 0; j < 2; ++j) qs[nt][j] = a.scale * __uint_as_float((uint32_t)(__shfl_sync(0xffffffffu, e, c * 8 + j * 4) - 14) << 23);
      }
    }
  }

  __device__ __forceinline__ void reset() {
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      #pragma unroll
      for (int t = 0; t < D / 16; ++t) o[nt][t][0] = o[nt][t][1] = o[nt][t][2] = o[nt][t][3] = 0.f;
      #pragma unroll
      for (int j = 0; j < 2; ++j) { m[nt][j] = l[nt][j] = M[nt][j] = 0.f; G[nt][j] = 1.f; }
    }
    fresh = true;
  }

  // largest of a lane's tokens and of the lanes with the same columns
  __device__ __forceinline__ float column_max(float x) {
    #pragma unroll
    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
  }
  __device__ __forceinline__ void scale_o(int nt, int j, float f) {
    #pragma unroll
    for (int t = 0; t < D / 16; ++t) { o[nt][t][j] *= f; o[nt][t][j + 2] *= f; }
  }

  // The boxes of a stage of this warp's ring; of the first box the first `valid & 255` tokens count, of the next as the next byte says.
  __device__ __forceinline__ void step(const uint8_t* stage, const float* scales, int valid) {
    constexpr int SUB = C::SUB, FULL = SUB == 4 ? 0x10101010 : SUB == 2 ? 0x1010 : 0x10;
    const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3, tok = sigma<C::TILE>(g);
    float s[SUB][NT][4];
    #pragma unroll
    for (int u = 0; u < SUB; ++u) {
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
      #pragma unroll
      for (int i = 0; i < C::KCH; ++i) {
        // piece c or 4 + c of the tile's row
        const int at = C::TILE == 128 ? (i >> 1) * PA_BOX * 128 + tok * 128 + ((((i & 1) * 4 + c) ^ tok) << 4) : tok * 64 + ((c ^ ((tok >> 1) & 3)) << 4);
        const uint4 x = *reinterpret_cast<const uint4*>(stage + u * 2 * C::BOX + at);
        const uint4 y = *reinterpret_cast<const uint4*>(stage + u * 2 * C::BOX + at + 8 * C::TILE);
        const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
        if (!F16) {
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<false>(s[u][nt], a[0], b[0], a[1], b[1], qf[nt][i * 4], qf[nt][i * 4 + 1]);
            mma16816<false>(s[u][nt], a[2], b[2], a[3], b[3], qf[nt][i * 4 + 2], qf[nt][i * 4 + 3]);
          }
        } else {
          #pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a0, a1, b0, b1;
            widen4<T>(a[j], a0, a1);
            widen4<T>(b[j], b0, b1);
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<true>(s[u][nt], a0, b0, a1, b1, qf[nt][i * 8 + j * 2], qf[nt][i * 8 + j * 2 + 1]);
          }
        }
      }
    }
    // lane (g, c): tokens tok and tok + 8 of each box, heads 2c and 2c + 1 of each tile: s' - m
    float vs[SUB][2];                           // scales of the values
    #pragma unroll
    for (int u = 0; u < SUB; ++u) {
      float ks[2] = {1.f, 1.f};
      if (F16) {
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          ks[i] = scales[u * 2 * PA_BOX + tok + 8 * i];
          vs[u][i] = scales[u * 2 * PA_BOX + PA_BOX + tok + 8 * i];
        }
      }
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) s[u][nt][i] = fmaf(s[u][nt][i], F16 ? qs[nt][i & 1] * ks[i >> 1] : qs[nt][i & 1], -m[nt][i & 1]);
      }
    }
    if (valid != FULL) {
      #pragma unroll
      for (int u = 0; u < SUB; ++u) {
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (tok + 8 * i < ((valid >> (8 * u)) & 255)) continue;
          vs[u][i] = 0.f;
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[u][nt][2 * i] = s[u][nt][2 * i + 1] = -INFINITY;
        }
      }
    }
    float most = s[0][0][0];
    #pragma unroll
    for (int u = 0; u < SUB; ++u) {
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) most = fmaxf(fmaxf(most, fmaxf(s[u][nt][0], s[u][nt][1])), fmaxf(s[u][nt][2], s[u][nt][3]));
    }
    const bool moves = __any_sync(0xffffffffu, most > PA_GROWTH) || fresh;
    if (moves) {
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = -INFINITY;
          #pragma unroll
          for (int u = 0; u < SUB; ++u) x = fmaxf(x, fmaxf(s[u][nt][j], s[u][nt][j + 2]));
          x = column_max(x);
          if (!fresh) x = fmaxf(x, 0.f);
          if (x == -INFINITY) x = 0.f;
          const float f = fresh ? 1.f : exp2f(-x);
          m[nt][j] += x;
          l[nt][j] *= f;
          if (!F16) scale_o(nt, j, f);
          #pragma unroll
          for (int u = 0; u < SUB; ++u) { s[u][nt][j] -= x; s[u][nt][j + 2] -= x; }
        }
      }
    }
    // 16-bit probabilities beside bf16 values come in two pieces, which have 16 bits of mantissa between them: their rounding to one would
    // add as much to the error as that of the result does (2.3e-3 instead of 1.7e-3), and the products have time (1 %).  Beside 8-bit values
    // they are one fp16 number, 11 bits: of values that were rounded to 4 or 7 bits, that adds 1 % to the result's own rounding (1.632e-3, in two
    // pieces 1.621e-3), and a second piece would cost 3 to 11 % (us, one / two: 64 x 8192 e4m3 175.5 / 184.7, 32 x 8192 int8 with 16 heads
    // on one 26.0 / 28.5, 256 channels e4m3 101 / 111).  Shares of which the largest is at least 2^6 leave fp16 its whole range: what is below 2^-20 of
    // the largest loses bits, what is below 2^-31 vanishes.
    uint32_t p[SUB][NT][2], rest[SUB][NT][2];
    most = 0.f;
    #pragma unroll
    for (int u = 0; u < SUB; ++u) {
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = exp2f(s[u][nt][i]);
          l[nt][i & 1] += e;
          s[u][nt][i] = e;
          w[i] = e * value_share(vs[u][i >> 1], G[nt][i & 1]);
        }
        if (F16) most = fmaxf(fmaxf(most, fmaxf(fabsf(w[0]), fabsf(w[1]))), fmaxf(fabsf(w[2]), fabsf(w[3])));
      }
    }
    if (F16) {
      if (__any_sync(0xffffffffu, most > PA_SHARE) || moves) {
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          #pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x = -120.f;                   // M: 2^-7 of a number above all of p times scale (2^e > scale)
            #pragma unroll
            for (int u = 0; u < SUB; ++u) {
              #pragma unroll
              for (int i = 0; i < 2; ++i)
                x = fmaxf(x, log2f(s[u][nt][2 * i + j]) + (float)(int)((__float_as_uint(vs[u][i]) >> 23) & 255) - (126.f + PA_SHARE_BITS));
            }
            x = column_max(x) + m[nt][j];
            if (!fresh) {
              x = fmaxf(x, M[nt][j]);
              scale_o(nt, j, exp2f(M[nt][j] - x));
            }
            M[nt][j] = x;
            G[nt][j] = exp2f(m[nt][j] - x);
          }
        }
      }
    }
    #pragma unroll
    for (int u = 0; u < SUB; ++u) {
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = F16 ? s[u][nt][i] * value_share(vs[u][i >> 1], G[nt][i & 1]) : s[u][nt][i];
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a = w[2 * i], b = w[2 * i + 1];
          if (F16) {
            p[u][nt][i] = transpose8x8(pack_f16(a, b));
          } else {
            // the upper piece is cut off, and the lower is never 0 or below: an infinite value stays one
            const uint32_t top = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
            p[u][nt][i] = transpose8x8(top);
            rest[u][nt][i] = transpose8x8(pack_bf16(fmaxf(a - bf16_lo(top), 0x1p-126f), fmaxf(b - bf16_hi(top), 0x1p-126f)));
          }
        }
      }
    }
    fresh = false;
    #pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const uint8_t* vst = stage + u * 2 * C::BOX + C::BOX;
      #pragma unroll
      for (int k = 0; k < C::TILES; ++k) {
        // this lane's channels of the tokens that are P^T's rows 2c, 2c + 1, 2c + 8, 2c + 9
        uint32_t x[4][C::VB / 4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (C::TILE == 128 ? c + 4 * (i & 1) : 2 * c + (i & 1)) + 8 * (i >> 1);
          const uint8_t* src = vst + k * PA_BOX * C::TILE + row * C::TILE;
          if (C::TILE == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(src + ((sigma<128>(g) ^ (row & 7)) << 4));
            x[i][0] = v.x; x[i][1] = v.y; x[i][2 % (C::VB / 4)] = v.z; x[i][3 % (C::VB / 4)] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src + (((g >> 1) ^ c) << 4) + (g & 1) * 8);
            x[i][0] = v.x; x[i][1] = v.y;
          }
        }
        if (valid != FULL) {                    // what lies behind a sequence may be NaN, which no zero share takes away
          #pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = (C::TILE == 128 ? c + 4 * (i & 1) : 2 * c + (i & 1)) + 8 * (i >> 1);
            if (row < ((valid >> (8 * u)) & 255)) continue;
            #pragma unroll
            for (int t = 0; t < C::VB / 4; ++t) x[i][t] = 0;
          }
        }
        #pragma unroll
        for (int t = 0; t < C::VB / 4; ++t) {
          if (!F16) {
            const uint32_t a0 = __byte_perm(x[0][t], x[1][t], 0x5410), a1 = __byte_perm(x[0][t], x[1][t], 0x7632);
            const uint32_t a2 = __byte_perm(x[2][t], x[3][t], 0x5410), a3 = __byte_perm(x[2][t], x[3][t], 0x7632);
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<false>(o[nt][k * (C::VEL / 2) + t], a0, a1, a2, a3, p[u][nt][0], p[u][nt][1]);
              mma16816<false>(o[nt][k * (C::VEL / 2) + t], a0, a1, a2, a3, rest[u][nt][0], rest[u][nt][1]);
            }
          } else {
            uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
            widen4<T>(__byte_perm(x[0][t], x[1][t], 0x5140), a0, a1);
            widen4<T>(__byte_perm(x[2][t], x[3][t], 0x5140), a2, a3);
            widen4<T>(__byte_perm(x[0][t], x[1][t], 0x7362), b0, b1);
            widen4<T>(__byte_perm(x[2][t], x[3][t], 0x7362), b2, b3);
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<true>(o[nt][k * (C::VEL / 2) + 2 * t], a0, a1, a2, a3, p[u][nt][0], p[u][nt][1]);
              mma16816<true>(o[nt][k * (C::VEL / 2) + 2 * t + 1], b0, b1, b2, b3, p[u][nt][0], p[u][nt][1]);
            }
          }
        }
      }
    }
  }

  __device__ __forceinline__ void add_sums() {
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      #pragma unroll
      for (int j = 0; j < 2; ++j) {
        #pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
      }
    }
  }
  // the result, for sums over the whole warp
  __device__ __forceinline__ void store(__nv_bfloat16* out, int real) {
    const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      #pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int head = nt * 8 + 2 * c + j;
        if (head >= real) continue;
        const float f = out_share(l[nt][j]), size = F16 ? out_size(m[nt][j], M[nt][j]) : 1.f;
        #pragma unroll
        for (int k = 0; k < C::TILES; ++k) {
          uint32_t w[C::VEL / 2];
          #pragma unroll
          for (int e = 0; e < C::VEL / 2; ++e) {
            const int t = k * (C::VEL / 2) + e;
            w[e] = F16 ? pack_bf16(o[nt][t][j] * f * size, o[nt][t][j + 2] * f * size) : pack_bf16(o[nt][t][j] * f, o[nt][t][j + 2] * f);
          }
          uint4* at = reinterpret_cast<uint4*>(out + head * D + (k * 8 + sigma<C::TILE>(g)) * C::VEL);
          #pragma unroll
          for (int e = 0; e < C::VEL / 8; ++e) at[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        }
      }
    }
  }
  // A part of an item: what the lanes hold, [register][lane], and (m, sum, M) of the heads.
  __device__ __forceinline__ void leave_part(float* slot) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      #pragma unroll
      for (int t = 0; t < D / 16; ++t)
        reinterpret_cast<float4*>(slot)[(nt * (D / 16) + t) * 32 + lane] = make_float4(o[nt][t][0], o[nt][t][1], o[nt][t][2], o[nt][t][3]);
      if (lane >= 4) continue;
      #pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* st = slot + C::HEADS * D + nt * 8 + 2 * c + j;
        st[0] = fresh ? -INFINITY : m[nt][j];
        st[C::HEADS] = l[nt][j];
        st[2 * C::HEADS] = fresh ? -INFINITY : F16 ? M[nt][j] : m[nt][j];
      }
    }
  }
  // the parts of an item, in their order
  template <typename Part>
  __device__ __forceinline__ void join(int parts, Part part) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    reset();
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      #pragma unroll
      for (int j = 0; j < 2; ++j) m[nt][j] = M[nt][j] = -INFINITY;
    }
    #pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float* st = part(k) + C::HEADS * D + nt * 8 + 2 * c + j;
          m[nt][j] = fmaxf(m[nt][j], st[0]);
          M[nt][j] = fmaxf(M[nt][j], st[2 * C::HEADS]);
        }
      }
    }
    for (int k = 0; k < parts; ++k) {
      const float* p = part(k);
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float* st = p + C::HEADS * D + nt * 8 + 2 * c + j;
          l[nt][j] += st[C::HEADS] * part_factor(st[0], m[nt][j]);
          f[j] = part_factor(st[2 * C::HEADS], M[nt][j]);
        }
        #pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          const float4 v = reinterpret_cast<const float4*>(p)[(nt * (D / 16) + t) * 32 + lane];
          o[nt][t][0] += f[0] * v.x; o[nt][t][1] += f[1] * v.y; o[nt][t][2] += f[0] * v.z; o[nt][t][3] += f[1] * v.w;
        }
      }
    }
  }

  // o into `to`, [channel][head] with 8 floats between the pieces of neighbouring lane groups (their banks would be the same);
  // lanes with g == 0 put (m, sum, M) of their heads into `stats`
  __device__ __forceinline__ void leave(float* to, float* stats) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + 2 * c;
      #pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const int piece = t / (C::VEL / 2) * 8 + sigma<C::TILE>(g), e = t % (C::VEL / 2);
        float* at = to + piece * (C::VEL * C::HEADS + 8) + 2 * e * C::HEADS + head;
        *reinterpret_cast<float2*>(at) = make_float2(o[nt][t][0], o[nt][t][1]);
        *reinterpret_cast<float2*>(at + C::HEADS) = make_float2(o[nt][t][2], o[nt][t][3]);
      }
      #pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (g == 0) {
          stats[head + j] = fresh ? -INFINITY : m[nt][j];
          stats[C::HEADS + head + j] = l[nt][j];
          stats[2 * C::HEADS + head + j] = fresh ? -INFINITY : F16 ? M[nt][j] : m[nt][j];
        }
      }
    }
  }
};

template <int D, int T, int NT>
__global__ void __launch_bounds__(PA_WARPS * 32, PagedAttn<D, T, NT>::BLOCKS) paged_attn_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap,
                                                                                            const __grid_constant__ CUtensorMap vmap) {
  using C = PagedAttn<D, T, NT>;
  constexpr int HEADS = C::HEADS, THREADS = PA_WARPS * 32, SUB = C::SUB, PER = 32 / SUB;       // PER: steps whose pages a warp's lanes hold
  extern __shared__ uint8_t dynamic[];
  uint8_t* ring = dynamic + (1024 - (smem_u32(dynamic) & 1023)) % 1024;
  __shared__ __align__(16) float scales[T == KV_BF16 ? 1 : PA_WARPS * C::STAGES][SUB * 2 * PA_BOX];
  __shared__ uint64_t full[PA_WARPS][C::STAGES];
  __shared__ __align__(16) float stats[PA_WARPS][3 * HEADS];
  __shared__ int arrived;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int items = a.Hk * a.groups;
  if (lane == 0) {
    #pragma unroll
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  __syncwarp();
  pdl_trigger();
  pdl_wait();

  // Where this worker's share begins.  The steps of all sequences and heads stand in a row, each sequence's heads one behind the other;
  // sequences in the order lane, lane + 32, ... of the lanes that look at them (every warp finds the same).
  // Workers cut the row at equal distances, wherever that is.  Only where there are few items is every item cut by itself, so that no worker
  // has parts of two, at the price of up to one shorter share per item (itself / row, us, bf16: 64 items of 2048 tokens 15.4 / 16.9, of 8192 47.6 /
  // 51.5, 50 of up to 4000 e4m3 14.5 / 22.8; 144 of 8192 96.9 / 95.8, of up to 8192 58 / 62;
  // 128 of 8192 with 256 channels e4m3 100.8 / 93.2, of up to 8192 56 / 65).
  // Workers are blocks, whose warps take every fourth step and meet at the end of a piece, or, where items are short, warps, which never
  // wait for each other (256 of 200 tokens, bf16 and e4m3, us: blocks 52.5 and 51.7, warps 44.6 and 33.8).  Blocks read longer stretches of
  // memory at a time (64 x 8192 bf16 319, warps 328; 64 x 2048 87 and 91, e4m3 55.0 and 55.5).
  auto steps_of = [&](int b) -> int { return (tokens_of(a, b) + C::STEP - 1) / C::STEP; };
  const int first_steps = lane < a.B ? steps_of(lane) : 0;
  int mine = first_steps * items, some = first_steps > 0;
  for (int b = lane + 32; b < a.B; b += 32) { const int n = steps_of(b); mine += n * items; some += n > 0; }
  int upto = mine;
  #pragma unroll
  for (int d = 1; d < 32; d <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += v; }
  int total = __shfl_sync(0xffffffffu, upto, 31);
  const int filled = __reduce_add_sync(0xffffffffu, some);
  if (filled < a.B) {
    // sequences without tokens
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      if (steps_of(b) > 0) continue;
      for (int i = threadIdx.x; i < a.Hq * D / 8; i += THREADS) reinterpret_cast<uint4*>(a.out + (long long)b * a.Hq * D)[i] = make_uint4(0, 0, 0, 0);
    }
  }
  const int how = paged_attn_workers(filled, items, total, a.most_blocks);
  const bool few = how == BY_ITEM, team = how != BY_WARP;
  const int workers = few ? a.most_blocks : team ? gridDim.x : gridDim.x * PA_WARPS, me = team ? blockIdx.x : blockIdx.x * PA_WARPS + warp;
  int share = paged_attn_share(total, workers, team);
  if (few) {
    // The smallest share of which there are at most most_blocks; the last guess always fits.  Counted in shares from here on.
    const int rest = workers - filled * items, fits = max(PA_BLOCK_SHARE, ((total + rest - 1) / rest + PA_WARPS - 1) / PA_WARPS * PA_WARPS);
    for (int guess = 0;; ++guess, share += (share / 8 + PA_WARPS - 1) / PA_WARPS * PA_WARPS) {
      if (guess == 6 || share > fits) share = fits;
      mine = (first_steps + share - 1) / share * items;
      for (int b = lane + 32; b < a.B; b += 32) mine += (steps_of(b) + share - 1) / share * items;
      total = __reduce_add_sync(0xffffffffu, mine);
      if (total <= workers || share == fits) break;
    }
    upto = mine;
    #pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += v; }
  }
  const int unit = few ? 1 : share;            // of the row, per worker
  if ((long long)unit * me >= total) return;
  int u = unit * me;
  const int end = total - u < unit ? total : u + unit;
  int b = lane, seq0 = upto - mine;            // first step (share) of sequence b in the row
  const bool here = seq0 <= u && u < upto;
  if (here) {
    for (;;) {
      const int n = (few ? (steps_of(b) + share - 1) / share : steps_of(b)) * items;
      if (u < seq0 + n) break;
      seq0 += n;
      b += 32;
    }
  }
  const int owner = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  b = __shfl_sync(0xffffffffu, b, owner);
  seq0 = __shfl_sync(0xffffffffu, seq0, owner);

  AttnWarp<D, T, NT> x;
  uint8_t* my_ring = ring + warp * C::STAGES * C::STAGE;
  const int page_mask = (1 << a.table.page_shift) - 1;
  int put = 0, got = 0;                        // stages of the ring: next to fill, next to read
  uint32_t parity = 0;                         // of the next to read
  bool alive = true;                           // no wait of this warp has run out

  // A piece of the share: steps of one item.
  struct Piece { int b, n, from, to, c0, parts, hk, head0, real; };
  auto take = [&](Piece& p) -> bool {
    while (u < end) {
      const int n = tokens_of(a, b), steps = (n + C::STEP - 1) / C::STEP, row = few ? (steps + share - 1) / share : steps;   // row: of an item
      if (u >= seq0 + row * items) {
        seq0 += row * items;
        b += 32;
        if (b >= a.B) b = (b & 31) + 1;
        continue;
      }
      const int item = (u - seq0) / row, at = (u - seq0) % row, item0 = seq0 + item * row, first = item % a.groups * HEADS;
      p.b = b;
      p.n = n;
      p.from = few ? at * share : at;
      p.to = min(steps, p.from + (few ? share : end - u));
      p.c0 = item0 / unit;
      p.parts = (item0 + row - 1) / unit - p.c0 + 1;             // workers that share the item
      p.hk = item / a.groups;
      p.head0 = p.hk * a.ratio + first;
      p.real = min(HEADS, a.ratio - first);
      u += few ? 1 : p.to - p.from;
      return true;
    }
    return false;
  };
  Piece cur = {};
  const int stride = team ? PA_WARPS : 1, offset = team ? warp : 0;              // steps of this warp: from + offset + stride j
  int count = 0, id = -1, valid[C::STAGES - 1];
    // Starts the copies of step j, a lane for each box; the tokens of its boxes (8 bits each), 0 where there is no page.
    auto issue = [&](int j) -> int {
      if (j >= count) return 0;
      if (j % PER == 0) {
        // the pages of the boxes of this warp's next steps, one per lane
        const int k = j + lane / SUB, t = (cur.from + offset + stride * k) * C::STEP + lane % SUB * PA_BOX;
        id = -1;
        if (k < count && t < cur.n) {
          id = a.table.ids[(long long)cur.b * a.table.width + (t >> a.table.page_shift)];
          if (id < 0 || id >= a.table.pages) { report_bad_index(a.table.status); id = -1; }
        }
      }
      const int page = __shfl_sync(0xffffffffu, id, j % PER * SUB + lane % SUB), t0 = (cur.from + offset + stride * j) * C::STEP + lane * PA_BOX;
      const bool mine = lane < SUB && page >= 0 && alive;
      const unsigned boxes = __ballot_sync(0xffffffffu, mine);
      if (boxes == 0) return 0;
      uint64_t* bar = &full[warp][put];
      if (lane == 0) mbar_expect_tx(bar, __popc(boxes) * C::LOADED);
      __syncwarp();
      if (mine) {
        const int slot = ((page * a.Hk + cur.hk) << a.table.page_shift) + (t0 & page_mask);      // below 2^31: the host sees to it
        uint8_t* dst = my_ring + put * C::STAGE + lane * 2 * C::BOX;
        #pragma unroll
        for (int k = 0; k < C::TILES; ++k) {
          tma_load_2d(dst + k * PA_BOX * C::TILE, &kmap, k * C::TILE / C::BYTES, slot, bar);
          tma_load_2d(dst + C::BOX + k * PA_BOX * C::TILE, &vmap, k * C::TILE / C::BYTES, slot, bar);
        }
        if (T != KV_BF16) {
          float* sc = scales[warp * C::STAGES + put] + lane * 2 * PA_BOX;
          bulk_load(sc, a.scales[0] + slot, PA_BOX * 4, bar);
          bulk_load(sc + PA_BOX, a.scales[1] + slot, PA_BOX * 4, bar);
        }
      }
      put = put + 1 == C::STAGES ? 0 : put + 1;
      return (int)__reduce_or_sync(0xffffffffu, mine ? (unsigned)min(PA_BOX, cur.n - t0) << (8 * lane) : 0u);
    };
  // takes the next piece and starts its first copies
  auto begin = [&]() -> bool {
    if (!take(cur)) return false;
    count = max(0, (cur.to - cur.from - offset + stride - 1) / stride);
    #pragma unroll
    for (int j = 0; j < C::STAGES - 1; ++j) valid[j] = issue(j);
    return true;
  };
  for (bool more = begin(); more;) {
    x.load_queries(a, a.q + cur.b * a.qb + cur.head0 * a.qh, cur.real);
    x.reset();
    for (int j = 0; j < count; ++j) {
      const int now = valid[0];
      #pragma unroll
      for (int i = 0; i + 1 < C::STAGES - 1; ++i) valid[i] = valid[i + 1];
      valid[C::STAGES - 2] = issue(j + C::STAGES - 1);         // into the stage that was read last
      if (now == 0) continue;
      // also a warp that has given up waits for each of its copies: none is under way when the block ends
      if (!mbar_try_wait(&full[warp][got], parity) && !mbar_wait(&full[warp][got], parity, nullptr)) {
        atomicCAS(a.table.status, 0, SSM_ERR_TIMEOUT_MBAR);
        alive = false;
      }
      alive = __all_sync(0xffffffffu, alive);
      if (alive) x.step(my_ring + got * C::STAGE, T == KV_BF16 ? nullptr : scales[warp * C::STAGES + got], now);
      got = got + 1 == C::STAGES ? 0 : got + 1;
      parity ^= got == 0;
      __syncwarp();                            // before the next copies into this stage
    }

    const Piece p = cur;
    const int real = p.real, parts = p.parts, c0 = p.c0;
    const bool whole = parts == 1;
    float* slot = whole ? nullptr : a.ws + ((long long)me * 2 + (c0 == me)) * C::SLOT;
    auto part = [&](int k) -> const float* { return a.ws + ((long long)(c0 + k) * 2 + (k == 0)) * C::SLOT; };     // the first worker's is its second
    __nv_bfloat16* out = a.out + ((long long)p.b * a.Hq + p.head0) * D;
    x.add_sums();
    if (!team) {
      more = begin();                          // under way while this one is brought to its end
      if (!whole) {
        x.leave_part(slot);
        __syncwarp();
        int before = 0;
        if (lane == 0) {
          before = arrive(a.counters + c0);
          if (before == parts - 1) a.counters[c0] = 0;
        }
        if (__shfl_sync(0xffffffffu, before, 0) != parts - 1) continue;
        __syncwarp();                          // what lane 0 has seen, all have
        x.join(parts, part);                   // all parts are there
      }
      x.store(out, real);
      continue;
    }

    // the warps of a block meet
    float* os = reinterpret_cast<float*>(ring);
    __syncthreads();
    x.leave(os + warp * C::MEET, stats[warp]);
    __syncthreads();
    // threads take a channel of four heads at a time, always the same heads
    const int fours = real <= 4 ? 1 : real <= 8 ? 2 : 4, h = threadIdx.x % fours * 4;
    {
      float f[PA_WARPS][4], mm[4], MM[4], sum[4], size[4];
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        mm[k] = MM[k] = -INFINITY;
        sum[k] = 0.f;
        #pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) { mm[k] = fmaxf(mm[k], stats[w][h + k]); MM[k] = fmaxf(MM[k], stats[w][2 * HEADS + h + k]); }
        #pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) {
          sum[k] += stats[w][HEADS + h + k] * part_factor(stats[w][h + k], mm[k]);
          f[w][k] = part_factor(stats[w][2 * HEADS + h + k], MM[k]);
        }
      }
      if (whole) {
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float o = out_share(sum[k]);
          size[k] = T == KV_BF16 ? 1.f : out_size(mm[k], MM[k]);
          #pragma unroll
          for (int w = 0; w < PA_WARPS; ++w) f[w][k] *= o;
        }
      } else if ((int)threadIdx.x < fours) {
        float* st = slot + HEADS * D + h;
        *reinterpret_cast<float4*>(st) = make_float4(mm[0], mm[1], mm[2], mm[3]);
        *reinterpret_cast<float4*>(st + HEADS) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        *reinterpret_cast<float4*>(st + 2 * HEADS) = make_float4(MM[0], MM[1], MM[2], MM[3]);
      }
      for (int d = threadIdx.x / fours; d < D; d += THREADS / fours) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(os + w * C::MEET + d * HEADS + d / C::VEL * 8 + h);
          acc[0] += v.x * f[w][0]; acc[1] += v.y * f[w][1]; acc[2] += v.z * f[w][2]; acc[3] += v.w * f[w][3];
        }
        if (whole) {
          #pragma unroll
          for (int k = 0; k < 4; ++k)
            if (h + k < real) out[(h + k) * D + d] = __float2bfloat16(T == KV_BF16 ? acc[k] : acc[k] * size[k]);
        } else {
          *reinterpret_cast<float4*>(slot + d * HEADS + h) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        }
      }
    }
    if (!whole) {
      __syncthreads();
      if (threadIdx.x == 0) {
        arrived = arrive(a.counters + c0);
        if (arrived == parts - 1) a.counters[c0] = 0;
      }
      __syncthreads();
      if (arrived == parts - 1) {
        // All parts are there: joined in the order of the blocks.  A thread looks at one head of every LOOK-th part for the largest m and M, then leaves the parts' factors in the ring.
        constexpr int LOOK = THREADS / HEADS;
        float* factors = os;                   // [part][head]
        // Up to 32 loads of a thread under way: of each of its channels from some parts.  The first come while the factors are found.
        constexpr int MANY = D * HEADS / 4 / THREADS, AT_ONCE = MANY > 2 || C::BLOCKS > 2 ? 8 : 16;
        const int d0 = threadIdx.x / fours, dd = THREADS / fours;
        float4 acc[MANY], v[AT_ONCE][MANY];
        auto load = [&](int k0) {
          #pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            #pragma unroll
            for (int i = 0; i < MANY; ++i) {
              v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (k0 + k < parts && d0 + i * dd < D) v[k][i] = *reinterpret_cast<const float4*>(part(k0 + k) + (d0 + i * dd) * HEADS + h);
            }
          }
        };
        load(0);
        #pragma unroll
        for (int i = 0; i < MANY; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int head = threadIdx.x % HEADS;
        float mm = -INFINITY, MM = -INFINITY, sum = 0.f;
        #pragma unroll 4
        for (int k = threadIdx.x / HEADS; k < parts; k += LOOK) {
          const float* st = part(k) + HEADS * D + head;
          mm = fmaxf(mm, st[0]);
          MM = fmaxf(MM, st[2 * HEADS]);
        }
        #pragma unroll
        for (int d = HEADS; d < 32; d <<= 1) {
          mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
          MM = fmaxf(MM, __shfl_xor_sync(0xffffffffu, MM, d));
        }
        if (lane < HEADS) { stats[warp][head] = mm; stats[warp][2 * HEADS + head] = MM; }
        __syncthreads();
        #pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) { mm = fmaxf(mm, stats[w][head]); MM = fmaxf(MM, stats[w][2 * HEADS + head]); }
        #pragma unroll 4
        for (int k = threadIdx.x / HEADS; k < parts; k += LOOK) {
          const float* st = part(k) + HEADS * D + head;
          sum += st[HEADS] * part_factor(st[0], mm);
          factors[k * HEADS + head] = part_factor(st[2 * HEADS], MM);
        }
        #pragma unroll
        for (int d = HEADS; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane < HEADS) stats[warp][HEADS + head] = sum;
        __syncthreads();
        if (threadIdx.x < HEADS) {
          sum = 0.f;
          #pragma unroll
          for (int w = 0; w < PA_WARPS; ++w) sum += stats[w][HEADS + head];
          stats[0][head] = out_share(sum);
          stats[1][head] = out_size(mm, MM);
        }
        __syncthreads();
        for (int k0 = 0;;) {
          #pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            if (k0 + k >= parts) break;
            const float4 f = *reinterpret_cast<const float4*>(factors + (k0 + k) * HEADS + h);
            #pragma unroll
            for (int i = 0; i < MANY; ++i) { acc[i].x += f.x * v[k][i].x; acc[i].y += f.y * v[k][i].y; acc[i].z += f.z * v[k][i].z; acc[i].w += f.w * v[k][i].w; }
          }
          k0 += AT_ONCE;
          if (k0 >= parts) break;
          load(k0);
        }
        #pragma unroll
        for (int i = 0; i < MANY; ++i) {
          const int d = d0 + i * dd;
          const float r[4] = {acc[i].x, acc[i].y, acc[i].z, acc[i].w};
          #pragma unroll
          for (int k = 0; k < 4; ++k)
            if (d < D && h + k < real)
              out[(h + k) * D + d] = __float2bfloat16(T == KV_BF16 ? r[k] * stats[0][h + k] : r[k] * stats[0][h + k] * stats[1][h + k]);
        }
      }
    }
    fence_proxy_async_smem();
    __syncthreads();                           // the ring, for TMA to write, and the statistics are free again
    more = begin();
  }
}

template <int D, int T, int NT>
static int paged_attn_launch(const AttnArgs& a, int grid, cudaStream_t st) {
  using C = PagedAttn<D, T, NT>;
  static SmemOptIn opt;
  if (int e = opt.ask(reinterpret_cast<const void*>(paged_attn_kernel<D, T, NT>), C::SMEM)) return e;
  CUtensorMap map[2];
  const uint64_t rows = ((uint64_t)a.table.pages * a.Hk) << a.table.page_shift;
  for (int i = 0; i < 2; ++i)
    if (make_tmap_2d(&map[i], C::BYTES == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, C::BYTES, a.pages[i], D, rows, C::ROW,
                     C::TILE / C::BYTES, PA_BOX, C::TILE == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
      return -SSM_ERR_BAD_ARG;
  return launch_dependent(paged_attn_kernel<D, T, NT>, dim3(grid), dim3(PA_WARPS * 32), C::SMEM, st, a, map[0], map[1]);
}

// Two column tiles for more than 8 query heads per key head, which would else be read twice (32 x 8192 tokens, 16 heads on one, two tiles / one,
// us: bf16 32 / 48, int8 25.7 / 33); 256 channels leave registers for one.
static bool two_tiles(int ratio, int D) { return ratio > 8 && D <= 128; }

template <int D, int T, int NT>
static void paged_attn_shape(int* blocks, int* slot, int* step) {
  *blocks = PagedAttn<D, T, NT>::BLOCKS;
  *slot = PagedAttn<D, T, NT>::SLOT;
  *step = PagedAttn<D, T, NT>::STEP;
}
// SMs of the current device; 0 where there is none
static int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && known[dev].load(std::memory_order_relaxed) > 0) return known[dev].load(std::memory_order_relaxed);
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}
// blocks of the launch, floats of its workspace, tokens of a step
static int paged_attn_plan(int sms, int type, int width, int page_size, int B, int Hq, int Hk, int D, int* grid, int* most_blocks, long long* floats,
                           int* tokens = nullptr) {
  int blocks = 0, slot = 0, step = 1;
  const int ratio = Hq / Hk;
  const bool two = two_tiles(ratio, D);
  #define SHAPE(DD, TT)                                                                  \
    do {                                                                                 \
      if (two) paged_attn_shape<DD, TT, (DD <= 128 ? 2 : 1)>(&blocks, &slot, &step);            \
      else paged_attn_shape<DD, TT, 1>(&blocks, &slot, &step);                                  \
    } while (0)
  KV_DISPATCH(SHAPE);
  #undef SHAPE
  if (tokens != nullptr) *tokens = step;
  const int group = two ? 16 : 8;
  // no more blocks than there can be shares
  const long long items = (long long)B * Hk * ((ratio + group - 1) / group), most = items * (((long long)width * page_size + step - 1) / step);
  if (most > 0x7fffffffll - (1 << 20)) return -SSM_ERR_BAD_ARG;                // counted in 32 bits
  const long long shares = (most + PA_BLOCK_SHARE - 1) / PA_BLOCK_SHARE + items;
  long long n = (long long)sms * blocks;
  if (n > PA_COUNTERS / PA_WARPS) n = PA_COUNTERS / PA_WARPS;
  *most_blocks = (int)n;
  if (n > shares) n = shares;
  *grid = n < 1 ? 1 : (int)n;
  *floats = (long long)*grid * PA_WARPS * 2 * slot;
  return 0;
}

}  // namespace ssm

using namespace ssm;

// floats of the workspace that ssm_paged_attn wants for these sizes on the current device; negative: an error
extern "C" long long ssm_paged_attn_workspace(int type, int width, int page_size, int B, int Hq, int Hk, int D) {
  int grid = 0, most = 0;
  long long floats = 0;
  const int sms = sm_count();
  if (sms < 1) return -(int)cudaGetLastError();
  if (Hk < 1 || Hq < Hk || Hq % Hk || B < 1) return -SSM_ERR_BAD_ARG;
  const int e = paged_attn_plan(sms, type, width, page_size, B, Hq, Hk, D, &grid, &most, &floats);
  return e ? (e < 0 ? e : -e) : floats;
}

// Who takes the work of a call with these lengths (host memory): out[4] = {0 blocks of one item each, 1 blocks, 2 warps; steps; steps of a
// share where workers take any item's; workers that may run at once}.  Host only; without a GPU for one of 148 SMs.
extern "C" int ssm_paged_attn_split(int type, int width, int page_size, int B, int Hq, int Hk, int D, const int* lengths, int* out) {
  int grid = 0, most = 0, step = 1;
  long long floats = 0, total = 0;
  int sms = sm_count();
  if (sms < 1) { cudaGetLastError(); sms = 148; }
  if (Hk < 1 || Hq < Hk || Hq % Hk || B < 1) return -SSM_ERR_BAD_ARG;
  if (const int e = paged_attn_plan(sms, type, width, page_size, B, Hq, Hk, D, &grid, &most, &floats, &step)) return e;
  const int group = two_tiles(Hq / Hk, D) ? 16 : 8, items = Hk * ((Hq / Hk + group - 1) / group);
  int filled = 0;
  for (int b = 0; b < B; ++b) {
    const long long n = lengths[b] < 0 ? 0 : lengths[b] < (long long)width * page_size ? lengths[b] : (long long)width * page_size;
    total += (n + step - 1) / step * items;
    filled += n > 0;
  }
  out[0] = paged_attn_workers(filled, items, (int)total, most);
  out[1] = (int)total;
  out[3] = out[0] == BY_WARP ? grid * PA_WARPS : out[0] == BY_BLOCK ? grid : most;
  out[2] = out[0] == BY_ITEM ? 0 : paged_attn_share((int)total, out[3], out[0] == BY_BLOCK);
  return 0;
}

struct PagedAttnCall {                         // in the order in which cuda_ops packs it
  const void* q; void* out;
  const void *kp, *vp, *ks, *vs, *table, *lengths;
  void* ws;
  int* status;
  long long qb, qh, ws_floats;                 // strides of q; floats of ws
  int type, pages, page_size, width, B, Hq, Hk, D;
  float scale;
};
extern "C" int ssm_paged_attn(const PagedAttnCall* c, cudaStream_t st) {
  AttnArgs a;
  const int D = c->D, type = c->type;
  if (!kv_table(&a.table, c->table, c->lengths, c->width, c->pages, c->page_size, c->status)) return -SSM_ERR_BAD_ARG;
  const void* all[] = {c->q, c->out, c->kp, c->vp, c->ks, c->vs, c->ws};
  for (const void* p : all) if (!kv_aligned(p)) return -SSM_ERR_BAD_ARG;
  if (c->B < 1 || c->Hk < 1 || c->Hq < c->Hk || c->Hq % c->Hk || c->qb % 8 || c->qh % 8 || c->pages < 1 ||
      (long long)c->pages * c->Hk * c->page_size > 0x7fffffffll || (type != KV_BF16 && (c->ks == nullptr || c->vs == nullptr)))
    return -SSM_ERR_BAD_ARG;
  int grid = 0;
  long long floats = 0;
  const int sms = sm_count();
  if (sms < 1) return (int)cudaGetLastError();
  if (int e = paged_attn_plan(sms, type, c->width, c->page_size, c->B, c->Hq, c->Hk, D, &grid, &a.most_blocks, &floats)) return e;
  if (c->ws_floats < floats) return -SSM_ERR_BAD_ARG;
  a.q = reinterpret_cast<const __nv_bfloat16*>(c->q);
  a.out = reinterpret_cast<__nv_bfloat16*>(c->out);
  a.qb = c->qb; a.qh = c->qh;
  a.pages[0] = reinterpret_cast<const uint8_t*>(c->kp); a.pages[1] = reinterpret_cast<const uint8_t*>(c->vp);
  a.scales[0] = reinterpret_cast<const float*>(c->ks); a.scales[1] = reinterpret_cast<const float*>(c->vs);
  a.B = c->B; a.Hq = c->Hq; a.Hk = c->Hk; a.ratio = c->Hq / c->Hk;
  const bool two = two_tiles(a.ratio, D);
  a.groups = (a.ratio + (two ? 15 : 7)) / (two ? 16 : 8);
  a.scale = c->scale * 1.4426950408889634f;
  a.ws = reinterpret_cast<float*>(c->ws);
  using Pool = ScratchPool<SCRATCH_ATTENTION>;
  Pool& pool = Pool::get();
  std::lock_guard<std::mutex> hold(pool.lock);
  Scratch s;
  if (!pool.take(st, 0, PA_COUNTERS, &s)) return (int)cudaErrorMemoryAllocation;
  a.counters = s.counters;
  #define ATTN(DD, TT)                                                                   \
    do {                                                                                 \
      if (two) return paged_attn_launch<DD, TT, (DD <= 128 ? 2 : 1)>(a, grid, st);       \
      return paged_attn_launch<DD, TT, 1>(a, grid, st);                                  \
    } while (0)
  KV_DISPATCH(ATTN);
  #undef ATTN
  return -SSM_ERR_BAD_ARG;
}
