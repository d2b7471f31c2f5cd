// Rows of queries, keys and values of one attention head: what the kernels that norm, rotate, store and differentiate them share.
//
// A head's row of D channels belongs to D / 16 neighbouring lanes, 16 channels each, as two vectors of 8.  The rotation pairs
// channel i with i + R / 2 (R = rotary dim, a multiple of 16): lane j < R / 16 holds the vectors j and j + R / 16, so that both
// halves of its pairs are in its registers; the other lanes hold such vectors of what is not rotated.  Neighbouring lanes access
// neighbouring vectors.
#pragma once
#include "common.cuh"

namespace ssm {

template <int D>
struct HeadRow {
  static constexpr int LANES = D / 16;
  int c0, c1;                                  // first channels of the two vectors
  bool turns;
  __device__ __forceinline__ HeadRow(int lane, int rot) {
    const int pairs = rot / 16;
    turns = lane < pairs;
    c0 = turns ? lane * 8 : rot + (lane - pairs) * 8;
    c1 = c0 + (turns ? rot / 2 : (D - rot) / 2);
  }
};

template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
  #pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's 16 channels as 8 pairs of neighbours: [0, 4) from c0 on, [4, 8) from c1 on.  All arithmetic is on pairs (one instruction
// for two fp32 operations): kernels that touch every value a dozen times are otherwise bound by their instructions.
using Pairs = uint64_t[8];

__device__ __forceinline__ void unpack_pairs(const uint4 a, const uint4 b, Pairs& f) {
  f[0] = bf16x2_pair(a.x); f[1] = bf16x2_pair(a.y); f[2] = bf16x2_pair(a.z); f[3] = bf16x2_pair(a.w);
  f[4] = bf16x2_pair(b.x); f[5] = bf16x2_pair(b.y); f[6] = bf16x2_pair(b.z); f[7] = bf16x2_pair(b.w);
}
__device__ __forceinline__ uint4 pack_pairs(const uint64_t* f) {
  return make_uint4(pack_bf16_pair(f[0]), pack_bf16_pair(f[1]), pack_bf16_pair(f[2]), pack_bf16_pair(f[3]));
}
__device__ __forceinline__ uint64_t both(float v) { return pack2(v, v); }
__device__ __forceinline__ float pair_sum(uint64_t v) {
  float a, b;
  unpack2(v, a, b);
  return a + b;
}
// 8 fp32 values as 4 pairs, from a 16-byte boundary
__device__ __forceinline__ void load_pairs(const float* p, uint64_t* f) {
  const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(p), b = *reinterpret_cast<const ulonglong2*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
// norm weights of the lane's channels, bf16 or fp32; nothing where there is no norm
template <int D>
__device__ __forceinline__ void load_weight(const void* w, int is32, const HeadRow<D>& at, Pairs& f) {
  if (w == nullptr) return;
  if (is32) {
    load_pairs(reinterpret_cast<const float*>(w) + at.c0, f);
    load_pairs(reinterpret_cast<const float*>(w) + at.c1, f + 4);
  } else {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(w);
    unpack_pairs(*reinterpret_cast<const uint4*>(p + at.c0), *reinterpret_cast<const uint4*>(p + at.c1), f);
  }
}
// a - b c of pairs (the paired instruction negates nothing)
__device__ __forceinline__ uint64_t fnma2(uint64_t b, uint64_t c, uint64_t a) {
  float a0, a1, b0, b1, c0, c1;
  unpack2(a, a0, a1);
  unpack2(b, b0, b1);
  unpack2(c, c0, c1);
  return pack2(fmaf(-b0, c0, a0), fmaf(-b1, c1, a1));
}
// channels i and 8 + i of the lane are turned by the angle whose cosine and sine are given, or by its negative
template <bool BACK>
__device__ __forceinline__ void turn_pairs(Pairs& y, const uint64_t (&cs)[4], const uint64_t (&sn)[4]) {
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t a = y[i], b = y[4 + i];
    if (BACK) {
      y[i] = fma2(b, sn[i], mul2(a, cs[i]));
      y[4 + i] = fnma2(a, sn[i], mul2(b, cs[i]));
    } else {
      y[i] = fnma2(b, sn[i], mul2(a, cs[i]));
      y[4 + i] = fma2(a, sn[i], mul2(b, cs[i]));
    }
  }
}
// Rows travel from global memory through slots of shared memory that only their thread uses: many loads are under way without
// registers that wait for them, and no barrier is needed.  Without `some`
// nothing is read and the slot gets zeros.
__device__ __forceinline__ void fetch16(void* slot, const void* src, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(slot)), "l"(src), "r"(some ? 16 : 0) : "memory");
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
constexpr int EACH = 8;                        // most heads that a group of lanes takes one after the other

// 1 / sqrt(mean + eps) to about a rounding: an error here moves whole rows.  One Newton step on the approximation, except where that is
// zero or infinite.
template <int D>
__device__ __forceinline__ float rms_factor(float sum_of_squares, float eps) {
  const float a = fmaf(sum_of_squares, 1.f / D, eps), r = rsqrtf(a);
  return a > 0.f && a < INFINITY ? fmaf(0.5f * r, fmaf(-a * r, r, 1.f), r) : r;
}

}  // namespace ssm
