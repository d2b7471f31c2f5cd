// RMS norm of every head of queries and keys with the rotary embedding in the same pass, and its backward pass.
//
//   r = 1 / sqrt(mean x^2 + eps),  n = x r w,  (y_i, y_j) = (n_i cos a - n_j sin a, n_j cos a + n_i sin a),  j = i + R / 2
//   backward: g = dy turned by -a,  h = g w,  dx = r h - x r^3 mean(h x),  dw = sum over rows of g x r
// r is computed again in the backward pass: x is read there anyway.
// Sums and the rotation are fp32; each result is rounded once.
// Bound by memory: 4 bytes per value forward, 6 backward, where the rows are many (us, 32 + 8 heads of 128 channels, forward and backward:
// 4 x 8192 tokens 108 and 183, floors 103 and 154; 2 x 4096 34 and 50, floors 26 and 38), by latency below (1 x 257 tokens 8.5 both).
// What it took: rows on their way in shared memory instead of registers (rows of both tensors in registers, two blocks per SM:
// backward 2 x 4096 69 us), arithmetic in pairs, a token's cosines and sines in registers for all its heads.
#include "head_norm.cuh"

namespace ssm {

struct HeadRows {                              // queries or keys
  const __nv_bfloat16* x; const __nv_bfloat16* dy; __nv_bfloat16* out;   // out: y, or dx in the backward pass
  const void* w;
  long long xb, xl, xh, gb, gl, gh;            // strides of x and dy; out is contiguous
  int heads, w32;
};
struct NormArgs {
  HeadRows t[2];
  const float* cs; const float* sn; const void* positions;
  int pos64, B, L, rot, table_rows;
  float eps;
  int* status;
};

// cosines and sines of the lane's pairs for token (b, l); false where the caller's position is outside the tables
__device__ __forceinline__ bool load_angles(const NormArgs& a, int token, int l, int c0, bool turns, uint64_t (&cs)[4], uint64_t (&sn)[4]) {
  long long p = l;
  if (a.positions != nullptr) p = a.pos64 ? reinterpret_cast<const long long*>(a.positions)[token] : reinterpret_cast<const int*>(a.positions)[token];
  if (p < 0 || p >= a.table_rows) {
    report_bad_index(a.status);
    return false;
  }
  if (turns) {
    load_pairs(a.cs + p * (a.rot / 2) + c0, cs);
    load_pairs(a.sn + p * (a.rot / 2) + c0, sn);
  }
  return true;
}

constexpr int NORM_THREADS = 256, NORM_WARPS = NORM_THREADS / 32;

// A warp takes `each` heads of one tensor for as many tokens as rows fit a warp (`units` such parts for them).  All its rows are asked
// for first; positions, angles and weights come while they are under way.
template <int D>
__global__ void __launch_bounds__(NORM_THREADS, 3) qk_norm_fwd_kernel(const NormArgs a, int each) {
  constexpr int LANES = D / 16, TOKENS = 32 / LANES;
  extern __shared__ uint4 slots[];             // [row][vector][thread]
  const int lane = threadIdx.x % LANES;
  const HeadRow<D> at(lane, a.rot);
  const int q_units = (a.t[0].heads + each - 1) / each, units = q_units + (a.t[1].heads + each - 1) / each;
  const long long warp = (long long)blockIdx.x * NORM_WARPS + threadIdx.x / 32;
  const long long block = warp / units;
  int part = (int)(warp - block * units);
  const int which = part >= q_units;
  if (which) part -= q_units;
  const HeadRows& t = a.t[which];
  const long long mine = block * TOKENS + threadIdx.x % 32 / LANES;
  const bool real = mine < (long long)a.B * a.L;
  const int token = real ? (int)mine : 0;
  const int b = token / a.L, l = token - b * a.L, h0 = part * each, h1 = real ? min(t.heads, h0 + each) : 0;
  const __nv_bfloat16* x = t.x + b * t.xb + l * t.xl + h0 * t.xh;
  for (int i = 0; i < each; ++i) {
    const __nv_bfloat16* src = h0 + i < h1 ? x + i * t.xh : x;
    fetch16(slots + (i * 2) * NORM_THREADS + threadIdx.x, src + at.c0, h0 + i < h1);
    fetch16(slots + (i * 2 + 1) * NORM_THREADS + threadIdx.x, src + at.c1, h0 + i < h1);
    if (i == each / 2 - 1) fetch_commit();
  }
  fetch_commit();
  __nv_bfloat16* out = t.out + ((long long)token * t.heads + h0) * D;
  Pairs w;
  uint64_t cs[4], sn[4];
  load_weight<D>(t.w, t.w32, at, w);
  bool inside = true;
  if (a.rot && real) inside = load_angles(a, token, l, at.c0, at.turns, cs, sn);
  const bool turns = a.rot && real && inside && at.turns;
  fetch_wait<1>();                             // the first half
  for (int i = 0; i < each; ++i) {             // the same number of turns for all lanes
    if (i == each / 2) fetch_wait<0>();
    Pairs y;
    unpack_pairs(slots[(i * 2) * NORM_THREADS + threadIdx.x], slots[(i * 2 + 1) * NORM_THREADS + threadIdx.x], y);
    if (t.w != nullptr) {
      uint64_t ss = mul2(y[0], y[0]);
      #pragma unroll
      for (int k = 1; k < 8; ++k) ss = fma2(y[k], y[k], ss);
      const uint64_t r = both(rms_factor<D>(row_sum<LANES>(pair_sum(ss)), a.eps));
      #pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = mul2(mul2(y[k], r), w[k]);
    }
    if (turns) turn_pairs<false>(y, cs, sn);
    if (h0 + i < h1) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(out + i * D + at.c0) = inside ? pack_pairs(y) : zero;
      *reinterpret_cast<uint4*>(out + i * D + at.c1) = inside ? pack_pairs(y + 4) : zero;
    }
  }
}

// Blocks [0, q_blocks) take the queries' rows, the others the keys'.  A warp takes `each` heads for as many tokens as rows fit a
// warp at a time, with GRAD_DEPTH rows under way, those of its next turn among them.  Each block leaves its sum of g x r in part[block][D].
constexpr int GRAD_DEPTH = 4;
template <int D>
__global__ void __launch_bounds__(NORM_THREADS, 2) qk_norm_bwd_kernel(const NormArgs a, int q_blocks, int each, float* __restrict__ part) {
  constexpr int LANES = D / 16, TOKENS = 32 / LANES;
  extern __shared__ uint4 slots[];             // [stage][vector][thread]
  pdl_trigger();
  const int which = (int)blockIdx.x >= q_blocks;
  const int block = which ? blockIdx.x - q_blocks : blockIdx.x, blocks = which ? gridDim.x - q_blocks : q_blocks;
  const HeadRows& t = a.t[which];
  const int lane = threadIdx.x % LANES;
  const HeadRow<D> at(lane, a.rot);
  const int units = (t.heads + each - 1) / each, tokens = a.B * a.L;
  const long long all = ((long long)tokens + TOKENS - 1) / TOKENS * units, warps = (long long)blocks * NORM_WARPS;      // turns of the tensor, warps that take them
  const long long mine = (long long)block * NORM_WARPS + threadIdx.x / 32;
  const int turns = mine < all ? (int)((all - mine + warps - 1) / warps) : 0, total = turns * each;

  // where a turn's rows are
  struct Place { int token, l, h0, h1; const __nv_bfloat16 *x, *g; };
  auto place = [&](int turn) -> Place {
    const long long u = mine + turn * warps, tb = u / units;
    const long long token = tb * TOKENS + threadIdx.x % 32 / LANES;
    Place p;
    const bool real = token < tokens;
    p.token = real ? (int)token : 0;
    const int b = p.token / a.L;
    p.l = p.token - b * a.L;
    p.h0 = (int)(u - tb * units) * each;
    p.h1 = real ? min(t.heads, p.h0 + each) : 0;
    p.x = t.x + b * t.xb + p.l * t.xl + p.h0 * t.xh;
    p.g = t.dy + b * t.gb + p.l * t.gl + p.h0 * t.gh;
    return p;
  };
  Place ahead;
  int ahead_turn = -1, ahead_i = each;
  auto fetch = [&](int j) {
    if (j < total) {
      if (ahead_i == each) { ahead = place(++ahead_turn); ahead_i = 0; }
      const bool some = ahead.h0 + ahead_i < ahead.h1;          // the address of a row that does not exist is not read
      uint4* to = slots + (j % GRAD_DEPTH) * 4 * NORM_THREADS + threadIdx.x;
      fetch16(to, ahead.x + at.c0, some);
      fetch16(to + NORM_THREADS, ahead.x + at.c1, some);
      fetch16(to + 2 * NORM_THREADS, ahead.g + at.c0, some);
      fetch16(to + 3 * NORM_THREADS, ahead.g + at.c1, some);
      ahead.x += t.xh;
      ahead.g += t.gh;
      ++ahead_i;
    }
    fetch_commit();
  };
  #pragma unroll
  for (int j = 0; j < GRAD_DEPTH - 1; ++j) fetch(j);
  Pairs w, dw;
  load_weight<D>(t.w, t.w32, at, w);
  #pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = 0;
  for (int turn = 0, j = 0; turn < turns; ++turn) {
    const Place p = place(turn);
    const bool real = p.h1 > 0;
    __nv_bfloat16* out = t.out + ((long long)p.token * t.heads + p.h0) * D;
    uint64_t cs[4], sn[4];
    bool inside = true;
    if (a.rot && real) inside = load_angles(a, p.token, p.l, at.c0, at.turns, cs, sn);
    const bool rotates = a.rot && real && inside && at.turns;
    for (int i = 0; i < each; ++i, ++j) {
      fetch(j + GRAD_DEPTH - 1);
      fetch_wait<GRAD_DEPTH - 1>();
      const uint4* from = slots + (j % GRAD_DEPTH) * 4 * NORM_THREADS + threadIdx.x;
      Pairs x, g;
      unpack_pairs(from[0], from[NORM_THREADS], x);
      unpack_pairs(from[2 * NORM_THREADS], from[3 * NORM_THREADS], g);
      if (!inside) {
        #pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = 0;
      }
      if (rotates) turn_pairs<true>(g, cs, sn);
      if (t.w != nullptr) {
        uint64_t ss = mul2(x[0], x[0]), hx = 0;
        #pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k) ss = fma2(x[k], x[k], ss);
          hx = fma2(mul2(g[k], x[k]), w[k], hx);
        }
        float r = rms_factor<D>(row_sum<LANES>(pair_sum(ss)), a.eps);
        if (p.h0 + i >= p.h1) r = 0.f;
        const float c = r * r * r * row_sum<LANES>(pair_sum(hx)) * (1.f / D);
        const uint64_t r2 = both(r), c2 = both(-c);
        #pragma unroll
        for (int k = 0; k < 8; ++k) {
          dw[k] = fma2(mul2(g[k], x[k]), r2, dw[k]);
          g[k] = fma2(mul2(g[k], w[k]), r2, mul2(x[k], c2));
        }
      }
      if (p.h0 + i < p.h1) {
        *reinterpret_cast<uint4*>(out + i * D + at.c0) = pack_pairs(g);
        *reinterpret_cast<uint4*>(out + i * D + at.c1) = pack_pairs(g + 4);
      }
    }
  }
  if (t.w == nullptr) return;
  __shared__ float sums[8][D];
  // the rows of a warp, then the warps one after the other: the same order at every run
  #pragma unroll
  for (int i = 0; i < 8; ++i) {
    float lo, hi;
    unpack2(dw[i], lo, hi);
    #pragma unroll
    for (int o = LANES; o < 32; o <<= 1) { lo += __shfl_xor_sync(0xffffffffu, lo, o); hi += __shfl_xor_sync(0xffffffffu, hi, o); }
    if (threadIdx.x % 32 < LANES) {
      const int c = (i < 4 ? at.c0 : at.c1 - 8) + 2 * i;
      sums[threadIdx.x / 32][c] = lo;
      sums[threadIdx.x / 32][c + 1] = hi;
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < D; c += NORM_THREADS) {
    float s = 0.f;
    #pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][c];
    part[(long long)blockIdx.x * D + c] = s;
  }
}

// dw of queries (blockIdx.y 0) and keys (1) from the blocks' sums, in their order: 32 columns, 32 groups of blocks.  Stored, or added to what is there.
struct WeightGrads { void* dst[2]; int is32[2], add[2]; };
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* part, int q_blocks, int blocks, int D, WeightGrads o) {
  __shared__ float sums[32][33];
  const int which = blockIdx.y, c = threadIdx.x % 32, g = threadIdx.x / 32, col = blockIdx.x * 32 + c;
  if (o.dst[which] == nullptr) return;
  pdl_wait();
  const int lo = which ? q_blocks : 0, hi = which ? blocks : q_blocks;
  float s = 0.f;
  #pragma unroll 4
  for (int k = lo + g; k < hi; k += 32) s += part[(long long)k * D + col];
  sums[g][c] = s;
  __syncthreads();
  if (g != 0) return;
  s = 0.f;
  #pragma unroll
  for (int k = 0; k < 32; ++k) s += sums[k][c];
  if (o.is32[which]) {
    float* p = reinterpret_cast<float*>(o.dst[which]) + col;
    *p = o.add[which] ? *p + s : s;
  } else {
    reinterpret_cast<__nv_bfloat16*>(o.dst[which])[col] = __float2bfloat16(s);
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct NormCall {                              // in the order in which cuda_ops packs it
  const void *q, *k, *dq, *dk;                 // dq, dk: gradients of the results, backward pass only
  void *qo, *ko;                               // results, or gradients of q and k
  const void *qw, *kw, *cs, *sn, *positions;
  int* status;
  void *part, *dwq, *dwk;                      // dwq, dwk: gradients of the weights, fp32 or bf16 (null: none wanted), stored or (fp32) added to
  long long strides[12];                       // (batch, token, head) of q, k, dq, dk
  int qw32, kw32, pos64, B, L, Hq, Hk, D, rot, table_rows, dq32, dk32, addq, addk;
  float eps;
};
static int norm_args(NormArgs* a, const NormCall& c, bool grads) {
  if (c.B < 1 || c.L < 1 || (long long)c.B * c.L > 0x7fffffffll || c.Hq < 1 || c.Hk < 1 || (c.D != 64 && c.D != 128 && c.D != 256) || c.rot < 0 || c.rot % 16 ||
      c.rot > c.D || (c.rot && (c.cs == nullptr || c.sn == nullptr)))
    return -SSM_ERR_BAD_ARG;
  const void* all[] = {c.q, c.k, c.qo, c.ko, c.qw, c.kw, c.cs, c.sn, grads ? c.dq : nullptr, grads ? c.dk : nullptr};
  for (const void* p : all) if (!aligned16(p)) return -SSM_ERR_BAD_ARG;
  for (int i = 0; i < (grads ? 12 : 6); ++i) if (c.strides[i] % 8) return -SSM_ERR_BAD_ARG;
  auto in = [](const void* p) { return reinterpret_cast<const __nv_bfloat16*>(p); };
  auto out = [](void* p) { return reinterpret_cast<__nv_bfloat16*>(p); };
  const long long* g = c.strides;
  a->t[0] = HeadRows{in(c.q), in(c.dq), out(c.qo), c.qw, g[0], g[1], g[2], g[6], g[7], g[8], c.Hq, c.qw32};
  a->t[1] = HeadRows{in(c.k), in(c.dk), out(c.ko), c.kw, g[3], g[4], g[5], g[9], g[10], g[11], c.Hk, c.kw32};
  a->cs = reinterpret_cast<const float*>(c.cs);
  a->sn = reinterpret_cast<const float*>(c.sn);
  a->positions = c.positions;
  a->pos64 = c.pos64;
  a->B = c.B; a->L = c.L; a->rot = c.rot; a->table_rows = c.table_rows;
  a->eps = c.eps;
  a->status = c.status;
  return 0;
}

// Heads that a warp takes one after the other: 8, or fewer where that would leave less than three blocks per SM (257 tokens with gradients
// 8.4 us, with eight heads 18; 2 x 4096 forward with eight, four, two heads 33.6, 33.2, 38.9).
static long long norm_turns(long long tokens, int heads, int each, int D) { return (tokens * (D / 16) + 31) / 32 * ((heads + each - 1) / each); }
static int heads_each(long long tokens, int Hq, int Hk, int D) {
  for (int each = EACH; each > 1; each /= 2)
    if (norm_turns(tokens, Hq, each, D) + norm_turns(tokens, Hk, each, D) >= 148ll * 3 * NORM_WARPS) return each;
  return 1;
}
struct GradPlan { int each, q_blocks, blocks; };
static GradPlan grad_plan(long long tokens, int Hq, int Hk, int D) {
  GradPlan p;
  p.each = heads_each(tokens, Hq, Hk, D);
  const long long uq = norm_turns(tokens, Hq, p.each, D), uk = norm_turns(tokens, Hk, p.each, D);
  const long long want = (uq + uk + NORM_WARPS - 1) / NORM_WARPS, most = 148 * 2;              // what runs at once
  const long long all = want < most ? want : most;
  long long q = (all * uq + (uq + uk) / 2) / (uq + uk);
  if (q < 1) q = 1;
  if (q > all - 1 && all > 1) q = all - 1;
  const long long k = all - q < 1 ? 1 : all - q;
  p.q_blocks = (int)q;
  p.blocks = (int)(q + k);
  return p;
}
template <int D>
static int norm_fwd_launch(const NormArgs& a, unsigned grid, int each, cudaStream_t st) {
  static SmemOptIn opt;
  if (int e = opt.ask(reinterpret_cast<const void*>(qk_norm_fwd_kernel<D>), EACH * 2 * NORM_THREADS * 16)) return e;
  qk_norm_fwd_kernel<D><<<grid, NORM_THREADS, each * 2 * NORM_THREADS * 16, st>>>(a, each);
  return (int)cudaGetLastError();
}
template <int D>
static int norm_bwd_launch(const NormArgs& a, const GradPlan& n, float* part, cudaStream_t st) {
  constexpr int SMEM = GRAD_DEPTH * 4 * NORM_THREADS * 16;
  static SmemOptIn opt;
  if (int e = opt.ask(reinterpret_cast<const void*>(qk_norm_bwd_kernel<D>), SMEM)) return e;
  qk_norm_bwd_kernel<D><<<n.blocks, NORM_THREADS, SMEM, st>>>(a, n.q_blocks, n.each, part);
  return (int)cudaGetLastError();
}

}  // namespace ssm

using namespace ssm;

extern "C" int ssm_qk_norm_fwd(const NormCall* c, cudaStream_t st) {
  NormArgs a;
  if (int bad = norm_args(&a, *c, false)) return bad;
  const long long tokens = (long long)c->B * c->L;
  const int each = heads_each(tokens, c->Hq, c->Hk, c->D);
  const long long grid = (norm_turns(tokens, c->Hq, each, c->D) + norm_turns(tokens, c->Hk, each, c->D) + NORM_WARPS - 1) / NORM_WARPS;
  if (grid > 0x7fffffffll) return -SSM_ERR_BAD_ARG;
  return c->D == 64 ? norm_fwd_launch<64>(a, (unsigned)grid, each, st) : c->D == 128 ? norm_fwd_launch<128>(a, (unsigned)grid, each, st)
                                                                                    : norm_fwd_launch<256>(a, (unsigned)grid, each, st);
}

// Blocks of the backward pass; `part` has that many times D floats.
extern "C" int ssm_qk_norm_bwd_blocks(long long tokens, int Hq, int Hk, int D) { return grad_plan(tokens, Hq, Hk, D).blocks; }

extern "C" int ssm_qk_norm_bwd(const NormCall* c, cudaStream_t st) {
  NormArgs a;
  if (int bad = norm_args(&a, *c, true)) return bad;
  if ((c->addq && !c->dq32) || (c->addk && !c->dk32)) return -SSM_ERR_BAD_ARG;
  const GradPlan n = grad_plan((long long)c->B * c->L, c->Hq, c->Hk, c->D);
  float* p = reinterpret_cast<float*>(c->part);
  const int e = c->D == 64 ? norm_bwd_launch<64>(a, n, p, st) : c->D == 128 ? norm_bwd_launch<128>(a, n, p, st) : norm_bwd_launch<256>(a, n, p, st);
  if (e || (c->dwq == nullptr && c->dwk == nullptr)) return e;
  return launch_dependent(qk_norm_dw_kernel, dim3(c->D / 32, 2), dim3(1024), 0, st, p, n.q_blocks, n.blocks, c->D,
                          WeightGrads{{c->dwq, c->dwk}, {c->dq32, c->dk32}, {c->addq, c->addk}});
}
