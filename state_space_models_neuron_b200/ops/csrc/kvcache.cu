// Paged key-value cache: writing new tokens (keys normed and rotated, 8-bit values quantised in the same pass) and reading sequences
// back.  8-bit values have one fp32 scale per token and head, s = max |x| / Qmax; stored = round(x / s).
#include "head_norm.cuh"
#include "kv_pages.cuh"

namespace ssm {

__device__ __forceinline__ uint32_t e4m3x4(const float* f) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ uint32_t int8x4(const float* f) {
  uint32_t u = 0;
  #pragma unroll
  for (int i = 0; i < 4; ++i) u |= (uint32_t)(__float2int_rn(f[i]) & 0xff) << (8 * i);
  return u;
}
template <int T>
__device__ __forceinline__ float kv_value(uint32_t byte) {
  if (T == KV_INT8) return (float)(int8_t)byte;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

struct WriteArgs {
  const __nv_bfloat16* x[3];                   // queries, keys, values
  long long sb[3], sl[3], sh[3];
  const void* w[2];
  int w32[2];
  int heads[3];
  __nv_bfloat16* qo;
  void* pages[2];
  float* scales[2];
  const int* counts;
  PageTable table;
  const float* cs; const float* sn;
  int B, L, rot, table_rows;
  float eps;
};

template <int D, int T>
__global__ void __launch_bounds__(256) kv_write_kernel(const WriteArgs a) {
  constexpr int LANES = D / 16;
  const int lane = threadIdx.x % LANES, heads = a.heads[0] + a.heads[1] + a.heads[2];
  const HeadRow<D> at(lane, a.rot);
  const long long rows = (long long)a.B * a.L * heads, step = (long long)gridDim.x * (256 / LANES);
  for (long long first = (long long)blockIdx.x * (256 / LANES); first < rows; first += step) {
    const long long mine = first + threadIdx.x / LANES;
    const long long row = mine < rows ? mine : rows - 1;
    const long long token = row / heads;
    int h = (int)(row % heads), which = 0;
    if (h >= a.heads[0]) { h -= a.heads[0]; which = 1; }
    if (which == 1 && h >= a.heads[1]) { h -= a.heads[1]; which = 2; }
    const int b = (int)(token / a.L), l = (int)(token % a.L);
    const int given = a.counts == nullptr ? a.L : a.counts[b];
    const int count = given < 0 ? 0 : given > a.L ? a.L : given;
    if (count != given) report_bad_index(a.table.status);
    const int pos = a.table.lengths[b] - count + l;
    bool real = l < count && pos >= 0;
    int page = -1;
    if (real) page = page_of(a.table, b, pos);
    real = page >= 0;
    if (real && a.rot && pos >= a.table_rows) { report_bad_index(a.table.status); real = false; }
    const __nv_bfloat16* x = a.x[which] + b * a.sb[which] + l * a.sl[which] + h * a.sh[which];
    float y[16];
    unpack16(*reinterpret_cast<const uint4*>(x + at.c0), *reinterpret_cast<const uint4*>(x + at.c1), y);
    const bool normed = which < 2 && a.w[which] != nullptr;
    float ss = 0.f;
    #pragma unroll
    for (int i = 0; i < 16; ++i) ss += y[i] * y[i];
    ss = row_sum<LANES>(ss);
    if (normed) {
      float w[16];
      load_weight<D>(a.w[which], a.w32[which], at, w);
      const float r = rsqrtf(ss * (1.f / D) + a.eps);
      #pragma unroll
      for (int i = 0; i < 16; ++i) y[i] *= r * w[i];
    }
    if (which < 2 && real && at.turns) {
      float cs[8], sn[8];
      load8(a.cs + (long long)pos * (a.rot / 2) + at.c0, cs);
      load8(a.sn + (long long)pos * (a.rot / 2) + at.c0, sn);
      turn16(y, cs, sn, 1.f);
    }
    uint32_t top = 0;                            // largest magnitude as bits: NaN is above infinity, which is above all numbers
    #pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
    #pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (mine >= rows) continue;
    if (which == 0) {
      __nv_bfloat16* o = a.qo + (token * a.heads[0] + h) * D;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(o + at.c0) = real ? pack8(y) : zero;
      *reinterpret_cast<uint4*>(o + at.c1) = real ? pack8(y + 8) : zero;
      continue;
    }
    if (!real) continue;
    const long long slot = (((long long)page * a.heads[1] + h) << a.table.page_shift) + (pos & ((1 << a.table.page_shift) - 1));
    if (T == KV_BF16) {
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.pages[which - 1]) + slot * D;
      *reinterpret_cast<uint4*>(o + at.c0) = pack8(y);
      *reinterpret_cast<uint4*>(o + at.c1) = pack8(y + 8);
    } else {
      constexpr float QMAX = T == KV_E4M3 ? 448.f : 127.f;
      const bool fine = top < 0x7f800000u, some = fine && top >= (27u << 23);     // 2^-100
      const float amax = __uint_as_float(top);
      const float inv = some ? __fdiv_rn(QMAX, amax) : 0.f;
      #pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = some ? y[i] * inv : 0.f;
      uint8_t* o = reinterpret_cast<uint8_t*>(a.pages[which - 1]) + slot * D;
      uint2 lo, hi;
      if (T == KV_E4M3) {
        lo = make_uint2(e4m3x4(y), e4m3x4(y + 4)); hi = make_uint2(e4m3x4(y + 8), e4m3x4(y + 12));
      } else {
        lo = make_uint2(int8x4(y), int8x4(y + 4)); hi = make_uint2(int8x4(y + 8), int8x4(y + 12));
      }
      *reinterpret_cast<uint2*>(o + at.c0) = lo;
      *reinterpret_cast<uint2*>(o + at.c1) = hi;
      if (lane == 0) a.scales[which - 1][slot] = some ? __fdiv_rn(amax, QMAX) : fine ? 0.f : __uint_as_float(0x7fc00000u);
    }
  }
}

// 16 channels per thread
template <int D, int T, typename Out>
__global__ void __launch_bounds__(256) kv_read_kernel(const void* __restrict__ pages0, const void* __restrict__ pages1, const float* __restrict__ scale0,
                                                      const float* __restrict__ scale1, Out* __restrict__ out0, Out* __restrict__ out1,
                                                      PageTable table, int B, int most, int heads) {
  constexpr int LANES = D / 16;
  const long long total = (long long)B * most * heads * LANES, both = 2 * total;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < both; i += (long long)gridDim.x * 256) {
    const bool second = i >= total;
    const long long at = second ? i - total : i;
    const int lane = (int)(at % LANES);
    const long long row = at / LANES;
    const int h = (int)(row % heads);
    const long long tok = row / heads;
    const int b = (int)(tok / most), p = (int)(tok % most);
    float y[16];
    #pragma unroll
    for (int k = 0; k < 16; ++k) y[k] = 0.f;
    const int page = p < table.lengths[b] ? page_of(table, b, p) : -1;
    if (page >= 0) {
      const long long slot = (((long long)page * heads + h) << table.page_shift) + (p & ((1 << table.page_shift) - 1));
      const uint8_t* src = reinterpret_cast<const uint8_t*>(second ? pages1 : pages0) + (slot * D + lane * 16) * KvType<T>::BYTES;
      if (T == KV_BF16) {
        unpack16(reinterpret_cast<const uint4*>(src)[0], reinterpret_cast<const uint4*>(src)[1], y);
      } else {
        const uint4 u = *reinterpret_cast<const uint4*>(src);
        const float s = (second ? scale1 : scale0)[slot];
        const uint32_t words[4] = {u.x, u.y, u.z, u.w};
        #pragma unroll
        for (int k = 0; k < 16; ++k) y[k] = kv_value<T>((words[k / 4] >> (8 * (k % 4))) & 0xff) * s;
      }
    }
    Out* o = (second ? out1 : out0) + row * D + lane * 16;
    if (sizeof(Out) == 2) {
      reinterpret_cast<uint4*>(o)[0] = pack8(y);
      reinterpret_cast<uint4*>(o)[1] = pack8(y + 8);
    } else {
      #pragma unroll
      for (int k = 0; k < 4; ++k) reinterpret_cast<float4*>(o)[k] = make_float4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
    }
  }
}

static unsigned kv_grid(long long blocks) { return (unsigned)(blocks < 148 * 8 ? blocks : 148 * 8); }

}  // namespace ssm

using namespace ssm;

// strides: (batch, token, head) of queries, keys and values
extern "C" int ssm_kv_write(const void* q, const void* k, const void* v, const long long* strides, void* qo, const void* qw, const void* kw,
                            int qw32, int kw32, const void* cs, const void* sn, int rot, int table_rows, float eps, void* kp, void* vp,
                            void* ks, void* vs, int type, int pages, int page_size, const void* table, int width, const void* lengths,
                            const void* counts, int B, int L, int Hq, int Hk, int D, int* status, cudaStream_t st) {
  WriteArgs a;
  if (!kv_table(&a.table, table, lengths, width, pages, page_size, status)) return -SSM_ERR_BAD_ARG;
  if (B < 1 || L < 1 || Hq < 0 || Hk < 1 || rot < 0 || rot % 16 || rot > D) return -SSM_ERR_BAD_ARG;
  const void* all[] = {q, k, v, qo, qw, kw, cs, sn, kp, vp};
  for (const void* p : all) if (!kv_aligned(p)) return -SSM_ERR_BAD_ARG;
  for (int i = 0; i < 9; ++i) if (strides[i] % 8) return -SSM_ERR_BAD_ARG;
  const void* x[3] = {q, k, v};
  const int heads[3] = {Hq, Hk, Hk};
  for (int i = 0; i < 3; ++i) {
    a.x[i] = reinterpret_cast<const __nv_bfloat16*>(x[i]);
    a.sb[i] = strides[3 * i]; a.sl[i] = strides[3 * i + 1]; a.sh[i] = strides[3 * i + 2];
    a.heads[i] = heads[i];
  }
  a.w[0] = qw; a.w[1] = kw; a.w32[0] = qw32; a.w32[1] = kw32;
  a.qo = reinterpret_cast<__nv_bfloat16*>(qo);
  a.pages[0] = kp; a.pages[1] = vp;
  a.scales[0] = reinterpret_cast<float*>(ks); a.scales[1] = reinterpret_cast<float*>(vs);
  a.counts = reinterpret_cast<const int*>(counts);
  a.cs = reinterpret_cast<const float*>(cs); a.sn = reinterpret_cast<const float*>(sn);
  a.B = B; a.L = L; a.rot = rot; a.table_rows = table_rows; a.eps = eps;
  const int per = 256 / (D / 16 > 0 ? D / 16 : 1);
  const unsigned grid = kv_grid(((long long)B * L * (Hq + 2 * Hk) + per - 1) / per);
  #define WRITE(DD, TT) kv_write_kernel<DD, TT><<<grid, 256, 0, st>>>(a)
  KV_DISPATCH(WRITE);
  #undef WRITE
  return (int)cudaGetLastError();
}

extern "C" int ssm_kv_read(const void* kp, const void* vp, const void* ks, const void* vs, int type, int pages, int page_size, const void* table,
                           int width, const void* lengths, void* ko, void* vo, int out32, int B, int most, int Hk, int D, int* status,
                           cudaStream_t st) {
  PageTable t;
  if (!kv_table(&t, table, lengths, width, pages, page_size, status)) return -SSM_ERR_BAD_ARG;
  if (B < 1 || most < 1 || Hk < 1 || !kv_aligned(kp) || !kv_aligned(vp) || !kv_aligned(ko) || !kv_aligned(vo)) return -SSM_ERR_BAD_ARG;
  const unsigned grid = kv_grid((2ll * B * most * Hk * (D / 16) + 255) / 256);
  const float* s0 = reinterpret_cast<const float*>(ks);
  const float* s1 = reinterpret_cast<const float*>(vs);
  #define READ(DD, TT)                                                                                                             \
    do {                                                                                                                           \
      if (out32) kv_read_kernel<DD, TT, float><<<grid, 256, 0, st>>>(kp, vp, s0, s1, reinterpret_cast<float*>(ko),                 \
                                                                     reinterpret_cast<float*>(vo), t, B, most, Hk);                \
      else kv_read_kernel<DD, TT, __nv_bfloat16><<<grid, 256, 0, st>>>(kp, vp, s0, s1, reinterpret_cast<__nv_bfloat16*>(ko),       \
                                                                       reinterpret_cast<__nv_bfloat16*>(vo), t, B, most, Hk);      \
    } while (0)
  KV_DISPATCH(READ);
  #undef READ
  return (int)cudaGetLastError();
}
