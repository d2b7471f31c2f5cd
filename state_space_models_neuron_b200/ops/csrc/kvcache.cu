// Paged key-value cache: writing new tokens (keys normed and rotated, 8-bit values quantised in the same pass) and reading sequences
// back.  8-bit values have one fp32 scale per token and head, s = max |x| / Qmax; stored = round(x / s).
// Both are bound by memory where tokens are many (16 x 2048 tokens, 32 query and 8 key heads of 128 channels, int8: written, with
// norm and rotation, in 142 us, floor 113 (135 with the product x (Qmax / max) in place of the quotient x / s: other bytes at ties); read back in
// 39, floor 31), by latency for single tokens (write 3.7 us, read 2.6).
#include "head_norm.cuh"
#include "kv_pages.cuh"

namespace ssm {

// y / s of pairs rounded to nearest, from r = 1 / s rounded to nearest, by a residual step (Markstein, IBM J. Res. Dev. 34, 1990): so the
// definition's quotient is what is rounded to 8 bits, and ties (half of a row's maximum) fall where a division lets them fall.
__device__ __forceinline__ uint64_t quotient(uint64_t y, uint64_t minus_s, uint64_t r) {
  const uint64_t q = mul2(y, r);
  return fma2(fma2(q, minus_s, y), r, q);
}
// 16 values over s, rounded to nearest even, as 16 bytes
__device__ __forceinline__ void quantise_e4m3(const Pairs& y, uint64_t minus_s, uint64_t r, uint2& lo, uint2& hi) {
  uint32_t v[4];
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b, c, d;
    unpack2(quotient(y[2 * i], minus_s, r), a, b);
    unpack2(quotient(y[2 * i + 1], minus_s, r), c, d);
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
        : "=r"(v[i]) : "f"(a), "f"(b), "f"(c), "f"(d));
  }
  lo = make_uint2(v[0], v[1]);
  hi = make_uint2(v[2], v[3]);
}
// The sum of a number of at most 127 and 1.5 * 2^23 is rounded to an integer whose low byte is the number's.
__device__ __forceinline__ void quantise_int8(const Pairs& y, uint64_t minus_s, uint64_t r, uint2& lo, uint2& hi) {
  uint32_t v[4];
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b, c, d;
    unpack2(add2(quotient(y[2 * i], minus_s, r), both(12582912.f)), a, b);
    unpack2(add2(quotient(y[2 * i + 1], minus_s, r), both(12582912.f)), c, d);
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
  pdl_trigger();
  pdl_wait();
  const int qu = (a.heads[0] + each - 1) / each, ku = (a.heads[1] + each - 1) / each, units = qu + 2 * ku;
  const long long warp = (long long)blockIdx.x * KV_WARPS + threadIdx.x / 32, block = warp / units;
  int part = (int)(warp - block * units);
  const int which = part < qu ? 0 : part < qu + ku ? 1 : 2;                     // the same for the whole warp
  part -= which == 0 ? 0 : which == 1 ? qu : qu + ku;
  const long long mine = block * TOKENS + threadIdx.x % 32 / LANES;
  const bool exists = mine < (long long)a.B * a.L;
  const int token = exists ? (int)mine : 0;
  const int b = token / a.L, l = token - b * a.L, h0 = part * each, h1 = exists ? min(a.heads[which], h0 + each) : 0;
  const int given = a.counts == nullptr ? a.L : a.counts[b];
  const int count = given < 0 ? 0 : given > a.L ? a.L : given, h2 = l < count ? h1 : h0;        // padding is not read
  const __nv_bfloat16* x = a.x[which] + b * a.sb[which] + l * a.sl[which] + h0 * a.sh[which];
  for (int i = 0; i < each; ++i) {
    const __nv_bfloat16* src = h0 + i < h2 ? x + i * a.sh[which] : x;
    fetch16(slots + (i * 2) * KV_THREADS + threadIdx.x, src + at.c0, h0 + i < h2);
    fetch16(slots + (i * 2 + 1) * KV_THREADS + threadIdx.x, src + at.c1, h0 + i < h2);
    if (i == each / 2 - 1) fetch_commit();
  }
  fetch_commit();
  // where the token goes
  if (count != given) report_bad_index(a.table.status);
  const int pos = a.table.lengths[b] - count + l;
  int page = -1;
  if (l < count && pos >= 0) {
    page = page_of(a.table, b, pos);
    if (a.rot && pos >= a.table_rows) { report_bad_index(a.table.status); page = -1; }
  }
  if (!__any_sync(0xffffffffu, page >= 0)) {
    // padding: only queries leave something
    fetch_wait<0>();
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int i = h0; which == 0 && i < h1; ++i) {
      __nv_bfloat16* o = a.qo + ((long long)token * a.heads[0] + i) * D;
      *reinterpret_cast<uint4*>(o + at.c0) = zero;
      *reinterpret_cast<uint4*>(o + at.c1) = zero;
    }
    return;
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
      const float scale = some ? __fdiv_rn(top, QMAX) : top < 1.f ? 0.f : __uint_as_float(0x7fc00000u);
      float s = some ? scale : 0.f;
      if (some && top < 0x1p-40f) {            // residuals of small rows would be no normal numbers: the quotients of 2^60 times these rows are the same
        s *= 0x1p60f;
        #pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = mul2(y[k], both(0x1p60f));
      }
      const uint64_t minus_s = both(-s), r = both(some ? __frcp_rn(s) : 0.f);
      uint2 lo, hi;
      if (T == KV_E4M3) quantise_e4m3(y, minus_s, r, lo, hi); else quantise_int8(y, minus_s, r, lo, hi);
      uint8_t* o = reinterpret_cast<uint8_t*>(a.pages[which - 1]) + slot * D;
      *reinterpret_cast<uint2*>(o + at.c0) = lo;
      *reinterpret_cast<uint2*>(o + at.c1) = hi;
      // a row with a value that is not finite reads back as NaN whatever is stored
      if (lane == 0) a.scales[which - 1][slot] = scale;
    }
  }
}

// A block takes rows (token, head) of one sequence, D / 8 lanes a row of keys and the same of values, READ_ROWS rows of a thread under
// way.  A lane has 8 channels, so that what neighbours store is contiguous (16 channels each, stored as two vectors 32 bytes
// apart: 16 x 2048 int8 45.7 us).
constexpr int READ_ROWS = 4;
template <int BYTES> struct ReadVector { using Type = uint2; };
template <> struct ReadVector<2> { using Type = uint4; };
template <int D, int T, typename Out>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const uint8_t* __restrict__ pages0, const uint8_t* __restrict__ pages1, const float* __restrict__ scale0,
                                                             const float* __restrict__ scale1, Out* __restrict__ out0, Out* __restrict__ out1,
                                                             PageTable table, int most, int heads) {
  using Vector = typename ReadVector<KvType<T>::BYTES>::Type;
  constexpr int LANES = D / 8, GROUPS = KV_THREADS / LANES;
  const int lane = threadIdx.x % LANES, b = blockIdx.y, n = table.lengths[b];
  const unsigned rows = (unsigned)most * heads, first = blockIdx.x * (GROUPS * READ_ROWS) + threadIdx.x / LANES;
  Vector u[READ_ROWS][2];
  float s[READ_ROWS][2];
  #pragma unroll
  for (int i = 0; i < READ_ROWS; ++i) {
    const unsigned row = first + i * GROUPS;
    const int p = row / heads, h = row - p * heads;
    u[i][0] = u[i][1] = Vector{};
    s[i][0] = s[i][1] = 0.f;
    const int page = row < rows && p < n ? page_of(table, b, p) : -1;
    if (page < 0) continue;
    const long long slot = (((long long)page * heads + h) << table.page_shift) + (p & ((1 << table.page_shift) - 1));
    u[i][0] = reinterpret_cast<const Vector*>(pages0)[slot * LANES + lane];
    u[i][1] = reinterpret_cast<const Vector*>(pages1)[slot * LANES + lane];
    if (T != KV_BF16) { s[i][0] = scale0[slot]; s[i][1] = scale1[slot]; }
  }
  #pragma unroll
  for (int i = 0; i < READ_ROWS; ++i) {
    const unsigned row = first + i * GROUPS;
    if (row >= rows) break;
    #pragma unroll
    for (int j = 0; j < 2; ++j) {
      Out* o = (j ? out1 : out0) + ((long long)b * rows + row) * D + lane * 8;
      uint32_t words[4] = {u[i][j].x, u[i][j].y, 0, 0};
      uint64_t y[4];
      if constexpr (T == KV_BF16) {
        if (sizeof(Out) == 2) {
          *reinterpret_cast<Vector*>(o) = u[i][j];
          continue;
        }
        words[2] = u[i][j].z;
        words[3] = u[i][j].w;
        #pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = bf16x2_pair(words[k]);
      } else {
        #pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t lo, hi;
          widen4<T>(words[k], lo, hi);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo)), g = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          y[2 * k] = mul2(pack2(f.x, f.y), both(s[i][j]));
          y[2 * k + 1] = mul2(pack2(g.x, g.y), both(s[i][j]));
        }
      }
      if (sizeof(Out) == 2) {
        *reinterpret_cast<uint4*>(o) = pack_pairs(y);
      } else {
        reinterpret_cast<ulonglong2*>(o)[0] = make_ulonglong2(y[0], y[1]);
        reinterpret_cast<ulonglong2*>(o)[1] = make_ulonglong2(y[2], y[3]);
      }
    }
  }
}

// Heads that a warp takes one after the other: 8, or fewer where that would leave less than three blocks per SM (128 tokens written and read
// 6.2 us, with eight heads 9.0; 8 x 1000 written with eight, four, two heads 32.6, 31.7, 40.1).
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
  return launch_dependent(kv_write_kernel<D, T>, dim3((unsigned)grid), dim3(KV_THREADS), each * 2 * KV_THREADS * 16, st, a, each);
}

template <int D, int T, typename Out>
static int kv_read_launch(const void* kp, const void* vp, const void* ks, const void* vs, void* ko, void* vo, const PageTable& t, dim3 grid, int most, int Hk,
                          cudaStream_t st) {
  kv_read_kernel<D, T, Out><<<grid, KV_THREADS, 0, st>>>(
      reinterpret_cast<const uint8_t*>(kp), reinterpret_cast<const uint8_t*>(vp), reinterpret_cast<const float*>(ks), reinterpret_cast<const float*>(vs),
      reinterpret_cast<Out*>(ko), reinterpret_cast<Out*>(vo), t, most, Hk);
  return (int)cudaGetLastError();
}

}  // namespace ssm

using namespace ssm;

struct KvWriteCall {                           // in the order in which cuda_ops packs it
  const void *q, *k, *v;
  void* qo;
  const void *qw, *kw, *cs, *sn;
  void *kp, *vp, *ks, *vs;
  const void *table, *lengths, *counts;
  int* status;
  long long strides[9];                        // (batch, token, head) of q, k, v
  int qw32, kw32, rot, table_rows, type, pages, page_size, width, B, L, Hq, Hk, D;
  float eps;
};
extern "C" int ssm_kv_write(const KvWriteCall* c, cudaStream_t st) {
  WriteArgs a;
  const int D = c->D, type = c->type;
  if (!kv_table(&a.table, c->table, c->lengths, c->width, c->pages, c->page_size, c->status)) return -SSM_ERR_BAD_ARG;
  if (c->B < 1 || c->L < 1 || (long long)c->B * c->L > 0x7fffffffll || c->Hq < 0 || c->Hk < 1 || c->rot < 0 || c->rot % 16 || c->rot > D ||
      (c->rot && (c->cs == nullptr || c->sn == nullptr)) || (type != KV_BF16 && (c->ks == nullptr || c->vs == nullptr)))
    return -SSM_ERR_BAD_ARG;
  const void* all[] = {c->q, c->k, c->v, c->qo, c->qw, c->kw, c->cs, c->sn, c->kp, c->vp};
  for (const void* p : all) if (!kv_aligned(p)) return -SSM_ERR_BAD_ARG;
  for (int i = 0; i < 9; ++i) if (c->strides[i] % 8) return -SSM_ERR_BAD_ARG;
  const int heads[3] = {c->Hq, c->Hk, c->Hk};
  for (int i = 0; i < 3; ++i) {
    a.x[i] = reinterpret_cast<const __nv_bfloat16*>(all[i]);
    a.sb[i] = c->strides[3 * i]; a.sl[i] = c->strides[3 * i + 1]; a.sh[i] = c->strides[3 * i + 2];
    a.heads[i] = heads[i];
  }
  a.w[0] = c->qw; a.w[1] = c->kw; a.w32[0] = c->qw32; a.w32[1] = c->kw32;
  a.qo = reinterpret_cast<__nv_bfloat16*>(c->qo);
  a.pages[0] = c->kp; a.pages[1] = c->vp;
  a.scales[0] = reinterpret_cast<float*>(c->ks); a.scales[1] = reinterpret_cast<float*>(c->vs);
  a.counts = reinterpret_cast<const int*>(c->counts);
  a.cs = reinterpret_cast<const float*>(c->cs); a.sn = reinterpret_cast<const float*>(c->sn);
  a.B = c->B; a.L = c->L; a.rot = c->rot; a.table_rows = c->table_rows; a.eps = c->eps;
  #define WRITE(DD, TT) return kv_write_launch<DD, TT>(a, c->Hq, c->Hk, st)
  KV_DISPATCH(WRITE);
  #undef WRITE
  return -SSM_ERR_BAD_ARG;
}

struct KvReadCall {                            // in the order in which cuda_ops packs it
  const void *kp, *vp, *ks, *vs, *table, *lengths;
  void *ko, *vo;
  int* status;
  int type, pages, page_size, width, out32, B, most, Hk, D;
};
extern "C" int ssm_kv_read(const KvReadCall* c, cudaStream_t st) {
  PageTable t;
  const int D = c->D, type = c->type;
  if (!kv_table(&t, c->table, c->lengths, c->width, c->pages, c->page_size, c->status)) return -SSM_ERR_BAD_ARG;
  if (c->B < 1 || c->B > 65535 || c->most < 1 || c->Hk < 1 || (long long)c->most * c->Hk > 0x7fffffffll || (D != 64 && D != 128 && D != 256) ||
      !kv_aligned(c->kp) || !kv_aligned(c->vp) || !kv_aligned(c->ko) || !kv_aligned(c->vo) || (type != KV_BF16 && (c->ks == nullptr || c->vs == nullptr)))
    return -SSM_ERR_BAD_ARG;
  const long long per = KV_THREADS / (D / 8) * READ_ROWS;
  const dim3 grid((unsigned)(((long long)c->most * c->Hk + per - 1) / per), c->B);
  #define READ(DD, TT)                                                                                                                    \
    do {                                                                                                                                  \
      if (c->out32) return kv_read_launch<DD, TT, float>(c->kp, c->vp, c->ks, c->vs, c->ko, c->vo, t, grid, c->most, c->Hk, st);           \
      return kv_read_launch<DD, TT, __nv_bfloat16>(c->kp, c->vp, c->ks, c->vs, c->ko, c->vo, t, grid, c->most, c->Hk, st);                 \
    } while (0)
  KV_DISPATCH(READ);
  #undef READ
  return -SSM_ERR_BAD_ARG;
}
