// Rows of queries, keys and values of one attention head: what the kernels that norm, rotate, store and differentiate them share.
//
// A head's row of D channels belongs to D / 16 neighbouring lanes, 16 channels each, as two vectors of 8.  The rotation pairs
// channel i with i + R / 2 (R = rotary dim, a multiple of 16): lane j < R / 16 holds the vectors j and j + R / 16, so that both
// halves of its pairs are in its registers; the other lanes hold two neighbouring vectors of what is not rotated.
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
    c0 = turns ? lane * 8 : rot + (lane - pairs) * 16;
    c1 = turns ? c0 + rot / 2 : c0 + 8;
  }
};

template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
  #pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void unpack16(const uint4 a, const uint4 b, float (&f)[16]) {
  float lo[8], hi[8];
  unpack8(a, lo);
  unpack8(b, hi);
  #pragma unroll
  for (int i = 0; i < 8; ++i) { f[i] = lo[i]; f[8 + i] = hi[i]; }
}
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
__device__ __forceinline__ void load8(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
// 16 norm weights of the lane's channels, bf16 or fp32; ones where there is no norm
template <int D>
__device__ __forceinline__ void load_weight(const void* w, int is32, const HeadRow<D>& at, float (&f)[16]) {
  if (w == nullptr) {
    #pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = 1.f;
  } else if (is32) {
    load8(reinterpret_cast<const float*>(w) + at.c0, f);
    load8(reinterpret_cast<const float*>(w) + at.c1, f + 8);
  } else {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(w);
    unpack16(*reinterpret_cast<const uint4*>(p + at.c0), *reinterpret_cast<const uint4*>(p + at.c1), f);
  }
}
// channels i and 8 + i of the lane are a pair: turned by the angle whose cosine and sine are cs[i], sn[i]
__device__ __forceinline__ void turn16(float (&y)[16], const float (&cs)[8], const float (&sn)[8], float sign) {
  #pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = y[i], b = y[8 + i], s = sign * sn[i];
    y[i] = a * cs[i] - b * s;
    y[8 + i] = b * cs[i] + a * s;
  }
}
}  // namespace ssm
