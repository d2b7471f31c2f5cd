// Paged key-value cache: writing new tokens (keys normed and rotated, 8-bit values quantised in the same pass) and reading sequences
// back.  8-bit values have one fp32 scale per token and head, s = max |x| / Qmax; stored = round(x / s).
#include "head_norm.cuh"
#include "kv_pages.cuh"

namespace ssm {

// 16 values times inv, rounded to nearest even, as 16 bytes
__device__ __forceinline__ void quantise_e4m3(const Pairs& y, uint64_t inv, uint2& lo, uint2& hi) {
  uint32_t v[4];
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b, c, d;
    unpack2(mul2(y[2 * i], inv), a, b);
    unpack2(mul2(y[2 * i + 1], inv), c, d);
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
        : "=r"(v[i]) : "f"(a), "f"(b), "f"(c), "f"(d));
  }
  lo = make_uint2(v[0], v[1]);
  hi = make_uint2(v[2], v[3]);
}
// The sum of a number of at most 127 and 1.5 * 2^23 is rounded to an integer whose low byte is the number's.
__device__ __forceinline__ void quantise_int8(const Pairs& y, uint64_t inv, uint2& lo, uint2& hi) {
  uint32_t v[4];
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b, c, d;
    unpack2(fma2(y[2 * i], inv, both(12582912.f)), a, b);
    unpack2(fma2(y[2 * i + 1], inv, both(12582912.f)), c, d);
    v[i] = __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
  }
  lo = make_uint2(v[0], v[1]);
  hi = make_uint2(v[2], v[3]);
}
// the larger magnitude; NaN if there is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
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

constexpr int KV_THREADS = 256, KV_WARPS = KV_THREADS / 32;

// A warp takes `each` heads of one tensor for as many tokens as rows fit a warp, all asked for first, as in the norms' own kernel.
template <int D, int T>
__global__ void __launch_bounds__(KV_THREADS, 3) kv_write_kernel(const WriteArgs a, int each) {
  constexpr int LANES = D / 16, TOKENS = 32 / LANES;
  extern __shared__ uint4 slots[];             // [row][vector][thread]
  const int lane = threadIdx.x % LANES;
  const HeadRow<D> at(lane, a.rot);
  const int qu = (a.heads[0] + each - 1) / each, ku = (a.heads[1] + each - 1) / each, units = qu + 2 * ku;
  const long long warp = (long long)blockIdx.x * KV_WARPS + threadIdx.x / 32, block = warp / units;
  int part = (int)(warp - block * units);
  const int which = part < qu ? 0 : part < qu + ku ? 1 : 2;                     // the same for the whole warp
  part -= which == 0 ? 0 : which == 1 ? qu : qu + ku;
  const long long mine = block * TOKENS + threadIdx.x % 32 / LANES;
  const bool exists = mine < (long long)a.B * a.L;
  const int token = exists ? (int)mine : 0;
  const int b = token / a.L, l = token - b * a.L, h0 = part * each, h1 = exists ? min(a.heads[which], h0 + each) : 0;
  const __nv_bfloat16* x = a.x[which] + b * a.sb[which] + l * a.sl[which] + h0 * a.sh[which];
  for (int i = 0; i < each; ++i) {
    const __nv_bfloat16* src = h0 + i < h1 ? x + i * a.sh[which] : x;
    fetch16(slots + (i * 2) * KV_THREADS + threadIdx.x, src + at.c0, h0 + i < h1);
    fetch16(slots + (i * 2 + 1) * KV_THREADS + threadIdx.x, src + at.c1, h0 + i < h1);
    if (i == each / 2 - 1) fetch_commit();
  }
  fetch_commit();
  // where the token goes
  const int given = a.counts == nullptr ? a.L : a.counts[b];
  const int count = given < 0 ? 0 : given > a.L ? a.L : given;
  if (count != given) report_bad_index(a.table.status);
  const int pos = a.table.lengths[b] - count + l;
  int page = -1;
  if (l < count && pos >= 0) {
    page = page_of(a.table, b, pos);
    if (a.rot && pos >= a.table_rows) { report_bad_index(a.table.status); page = -1; }
  }
  const void* weight = which < 2 ? a.w[which] : nullptr;
  const bool turns = which < 2 && page >= 0 && at.turns;
  Pairs w;
  uint64_t cs[4], sn[4];
  load_weight<D>(weight, which < 2 ? a.w32[which] : 0, at, w);
  if (turns) {
    load_pairs(a.cs + (long long)pos * (a.rot / 2) + at.c0, cs);
    load_pairs(a.sn + (long long)pos * (a.rot / 2) + at.c0, sn);
  }
  fetch_wait<1>();                             // the first half
  for (int i = 0; i < each; ++i) {
    if (i == each / 2) fetch_wait<0>();
    Pairs y;
    unpack_pairs(slots[(i * 2) * KV_THREADS + threadIdx.x], slots[(i * 2 + 1) * KV_THREADS + threadIdx.x], y);
    if (weight != nullptr) {
      uint64_t ss = mul2(y[0], y[0]);
      #pragma unroll
      for (int k = 1; k < 8; ++k) ss = fma2(y[k], y[k], ss);
      const uint64_t r = both(rms_factor<D>(row_sum<LANES>(pair_sum(ss)), a.eps));
      #pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = mul2(mul2(y[k], r), w[k]);
    }
    if (turns) turn_pairs<false>(y, cs, sn);
    const long long slot = (((long long)page * a.heads[1] + h0 + i) << a.table.page_shift) + (pos & ((1 << a.table.page_shift) - 1));
    if (which == 0 || T == KV_BF16) {
      const bool real = page >= 0;
      if (h0 + i >= h1 || (which != 0 && !real)) continue;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      __nv_bfloat16* o = which == 0 ? a.qo + ((long long)token * a.heads[0] + h0 + i) * D : reinterpret_cast<__nv_bfloat16*>(a.pages[which - 1]) + slot * D;
      *reinterpret_cast<uint4*>(o + at.c0) = real ? pack_pairs(y) : zero;
      *reinterpret_cast<uint4*>(o + at.c1) = real ? pack_pairs(y + 4) : zero;
    } else {
      constexpr float QMAX = T == KV_E4M3 ? 448.f : 127.f;
      float top = 0.f;
      #pragma unroll
      for (int k = 0; k < 8; ++k) {
        float lo, hi;
        unpack2(y[k], lo, hi);
        top = max_nan(max_nan(top, fabsf(lo)), fabsf(hi));
      }
      #pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (h0 + i >= h1 || page < 0) continue;
      const bool some = __float_as_uint(top) - (27u << 23) < 0x7f800000u - (27u << 23);      // finite and at least 2^-100
      const uint64_t inv = both(some ? __fdiv_rn(QMAX, top) : 0.f);
      uint2 lo, hi;
      if (T == KV_E4M3) quantise_e4m3(y, inv, lo, hi); else quantise_int8(y, inv, lo, hi);
      uint8_t* o = reinterpret_cast<uint8_t*>(a.pages[which - 1]) + slot * D;
      *reinterpret_cast<uint2*>(o + at.c0) = lo;
      *reinterpret_cast<uint2*>(o + at.c1) = hi;
      // a row with a value that is not finite reads back as NaN whatever is stored
      if (lane == 0) a.scales[which - 1][slot] = some ? __fdiv_rn(top, QMAX) : top < 1.f ? 0.f : __uint_as_float(0x7fc00000u);
    }
  }
}

// A block takes rows (token, head) of one sequence, D / 16 lanes a row of keys and the same of values, two rows under way.
constexpr int READ_ROWS = 2;
template <int D, int T, typename Out>
__global__ void __launch_bounds__(KV_THREADS, 5) kv_read_kernel(const void* __restrict__ pages0, const void* __restrict__ pages1, const float* __restrict__ scale0,
                                                                const float* __restrict__ scale1, Out* __restrict__ out0, Out* __restrict__ out1,
                                                                PageTable table, int most, int heads) {
  constexpr int LANES = D / 16, GROUPS = KV_THREADS / LANES, VECS = T == KV_BF16 ? 2 : 1;
  const int lane = threadIdx.x % LANES, b = blockIdx.y, n = table.lengths[b];
  const unsigned rows = (unsigned)most * heads, first = blockIdx.x * (GROUPS * READ_ROWS) + threadIdx.x / LANES;
  uint4 u[READ_ROWS][2][VECS];
  float s[READ_ROWS][2];
  #pragma unroll
  for (int i = 0; i < READ_ROWS; ++i) {
    const unsigned row = first + i * GROUPS;
    const int p = row / heads, h = row - p * heads;
    #pragma unroll
    for (int k = 0; k < VECS; ++k) u[i][0][k] = u[i][1][k] = make_uint4(0, 0, 0, 0);
    s[i][0] = s[i][1] = 0.f;
    const int page = row < rows && p < n ? page_of(table, b, p) : -1;
    if (page < 0) continue;
    const long long slot = (((long long)page * heads + h) << table.page_shift) + (p & ((1 << table.page_shift) - 1));
    const long long at = (slot * D + lane * 16) * KvType<T>::BYTES;
    #pragma unroll
    for (int k = 0; k < VECS; ++k) {
      u[i][0][k] = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(pages0) + at)[k];
      u[i][1][k] = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(pages1) + at)[k];
    }
    if (T != KV_BF16) { s[i][0] = scale0[slot]; s[i][1] = scale1[slot]; }
  }
  #pragma unroll
  for (int i = 0; i < READ_ROWS; ++i) {
    const unsigned row = first + i * GROUPS;
    if (row >= rows) break;
    #pragma unroll
    for (int j = 0; j < 2; ++j) {
      Out* o = (j ? out1 : out0) + ((long long)b * rows + row) * D + lane * 16;
      if (T == KV_BF16 && sizeof(Out) == 2) {
        reinterpret_cast<uint4*>(o)[0] = u[i][j][0];
        reinterpret_cast<uint4*>(o)[1] = u[i][j][VECS - 1];
        continue;
      }
      Pairs y;
      if (T == KV_BF16) {
        unpack_pairs(u[i][j][0], u[i][j][VECS - 1], y);
      } else {
        const uint32_t words[4] = {u[i][j][0].x, u[i][j][0].y, u[i][j][0].z, u[i][j][0].w};
        const uint64_t s2 = both(s[i][j]);
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t lo, hi;
          widen4<T>(words[k], lo, hi);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo)), g = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          y[2 * k] = mul2(pack2(f.x, f.y), s2);
          y[2 * k + 1] = mul2(pack2(g.x, g.y), s2);
        }
      }
      if (sizeof(Out) == 2) {
        reinterpret_cast<uint4*>(o)[0] = pack_pairs(y);
        reinterpret_cast<uint4*>(o)[1] = pack_pairs(y + 4);
      } else {
        #pragma unroll
        for (int k = 0; k < 4; ++k) reinterpret_cast<ulonglong2*>(o)[k] = make_ulonglong2(y[2 * k], y[2 * k + 1]);
      }
    }
  }
}

// Heads that a warp takes one after the other: 8, or fewer where that would leave less than three blocks per SM.
static long long write_warps(long long tokens, int Hq, int Hk, int each, int D) {
  return (tokens * (D / 16) + 31) / 32 * ((Hq + each - 1) / each + 2 * ((Hk + each - 1) / each));
}
template <int D, int T>
static int kv_write_launch(const WriteArgs& a, int Hq, int Hk, cudaStream_t st) {
  const long long tokens = (long long)a.B * a.L;
  int each = EACH;
  while (each > 1 && write_warps(tokens, Hq, Hk, each, D) < 148ll * 3 * KV_WARPS) each /= 2;
  const long long grid = (write_warps(tokens, Hq, Hk, each, D) + KV_WARPS - 1) / KV_WARPS;
  if (grid > 0x7fffffffll) return -SSM_ERR_BAD_ARG;
  static SmemOptIn opt;
  if (int e = opt.ask(reinterpret_cast<const void*>(kv_write_kernel<D, T>), EACH * 2 * KV_THREADS * 16)) return e;
  kv_write_kernel<D, T><<<(unsigned)grid, KV_THREADS, each * 2 * KV_THREADS * 16, st>>>(a, each);
  return (int)cudaGetLastError();
}

}  // namespace ssm

using namespace ssm;

// strides: (batch, token, head) of queries, keys and values
extern "C" int ssm_kv_write(const void* q, const void* k, const void* v, const long long* strides, void* qo, const void* qw, const void* kw,
                            int qw32, int kw32, const void* cs, const void* sn, int rot, int table_rows, float eps, void* kp, void* vp,
                            void* ks, void* vs, int type, int pages, int page_size, const void* table, int width, const void* lengths,
                            const void* counts, int B, int L, int Hq, int Hk, int D, int* status, cudaStream_t st) {
  WriteArgs a;
  if (!kv_table(&a.table, table, lengths, width, pages, page_size, status)) return -SSM_ERR_BAD_ARG;
  if (B < 1 || L < 1 || (long long)B * L > 0x7fffffffll || Hq < 0 || Hk < 1 || rot < 0 || rot % 16 || rot > D) return -SSM_ERR_BAD_ARG;
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
  #define WRITE(DD, TT) return kv_write_launch<DD, TT>(a, Hq, Hk, st)
  KV_DISPATCH(WRITE);
  #undef WRITE
  return -SSM_ERR_BAD_ARG;
}

extern "C" int ssm_kv_read(const void* kp, const void* vp, const void* ks, const void* vs, int type, int pages, int page_size, const void* table,
                           int width, const void* lengths, void* ko, void* vo, int out32, int B, int most, int Hk, int D, int* status,
                           cudaStream_t st) {
  PageTable t;
  if (!kv_table(&t, table, lengths, width, pages, page_size, status)) return -SSM_ERR_BAD_ARG;
  if (B < 1 || most < 1 || Hk < 1 || !kv_aligned(kp) || !kv_aligned(vp) || !kv_aligned(ko) || !kv_aligned(vo)) return -SSM_ERR_BAD_ARG;
  if (B > 65535 || (long long)most * Hk > 0x7fffffffll || (D != 64 && D != 128 && D != 256)) return -SSM_ERR_BAD_ARG;
  const long long per = KV_THREADS / (D / 16) * READ_ROWS;
  const dim3 grid((unsigned)(((long long)most * Hk + per - 1) / per), B);
  const float* s0 = reinterpret_cast<const float*>(ks);
  const float* s1 = reinterpret_cast<const float*>(vs);
  #define READ(DD, TT)                                                                                                             \
    do {                                                                                                                           \
      if (out32) kv_read_kernel<DD, TT, float><<<grid, KV_THREADS, 0, st>>>(kp, vp, s0, s1, reinterpret_cast<float*>(ko),                 \
                                                                     reinterpret_cast<float*>(vo), t, most, Hk);                   \
      else kv_read_kernel<DD, TT, __nv_bfloat16><<<grid, KV_THREADS, 0, st>>>(kp, vp, s0, s1, reinterpret_cast<__nv_bfloat16*>(ko),       \
                                                                       reinterpret_cast<__nv_bfloat16*>(vo), t, most, Hk);         \
    } while (0)
  KV_DISPATCH(READ);
  #undef READ
  return (int)cudaGetLastError();
}
