// RMS norm of every head of queries and keys with the rotary embedding in the same pass, and its backward pass.
//
//   r = 1 / sqrt(mean x^2 + eps),  n = x r w,  (y_i, y_j) = (n_i cos a - n_j sin a, n_j cos a + n_i sin a),  j = i + R / 2
//   backward: g = dy turned by -a,  h = g w,  dx = r h - x r^3 mean(h x),  dw = sum over rows of g x r
// r is computed again in the backward pass: x is read there anyway.
// Sums and the rotation are fp32; each result is rounded once.
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

// row of the tables of token (b, l); -1 where the caller's position is outside
__device__ __forceinline__ int table_row(const NormArgs& a, long long token, int l) {
  if (a.positions == nullptr) return l;
  const long long p = a.pos64 ? reinterpret_cast<const long long*>(a.positions)[token] : reinterpret_cast<const int*>(a.positions)[token];
  if (p >= 0 && p < a.table_rows) return (int)p;
  report_bad_index(a.status);
  return -1;
}

template <int D>
__global__ void __launch_bounds__(256) qk_norm_fwd_kernel(const NormArgs a) {
  constexpr int LANES = D / 16;
  const int lane = threadIdx.x % LANES, heads = a.t[0].heads + a.t[1].heads;
  const HeadRow<D> at(lane, a.rot);
  const long long rows = (long long)a.B * a.L * heads, step = (long long)gridDim.x * (256 / LANES);
  // whole warps take part in the shuffles: a row behind the last one is computed as the last and not stored
  for (long long first = (long long)blockIdx.x * (256 / LANES); first < rows; first += step) {
    const long long mine = first + threadIdx.x / LANES;
    const long long row = mine < rows ? mine : rows - 1;
    const long long token = row / heads;
    const int head = (int)(row % heads), which = head >= a.t[0].heads, h = which ? head - a.t[0].heads : head;
    const int b = (int)(token / a.L), l = (int)(token % a.L);
    const HeadRows& t = a.t[which];
    const __nv_bfloat16* x = t.x + b * t.xb + l * t.xl + h * t.xh;
    float y[16];
    unpack16(*reinterpret_cast<const uint4*>(x + at.c0), *reinterpret_cast<const uint4*>(x + at.c1), y);
    if (t.w != nullptr) {
      float w[16], ss = 0.f;
      load_weight<D>(t.w, t.w32, at, w);
      #pragma unroll
      for (int i = 0; i < 16; ++i) ss += y[i] * y[i];
      const float r = rsqrtf(row_sum<LANES>(ss) * (1.f / D) + a.eps);
      #pragma unroll
      for (int i = 0; i < 16; ++i) y[i] *= r * w[i];
    } else {
      row_sum<LANES>(0.f);
    }
    if (a.rot) {
      const int p = table_row(a, token, l);
      if (p < 0) {
        #pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = 0.f;
      } else if (at.turns) {
        float cs[8], sn[8];
        load8(a.cs + (long long)p * (a.rot / 2) + at.c0, cs);
        load8(a.sn + (long long)p * (a.rot / 2) + at.c0, sn);
        turn16(y, cs, sn, 1.f);
      }
    }
    if (mine < rows) {
      __nv_bfloat16* o = t.out + (token * t.heads + h) * D;
      *reinterpret_cast<uint4*>(o + at.c0) = pack8(y);
      *reinterpret_cast<uint4*>(o + at.c1) = pack8(y + 8);
    }
  }
}

// Blocks [0, q_blocks) take the queries' rows, the others the keys'; each leaves its sum of g x r in part[block][D].
template <int D>
__global__ void __launch_bounds__(256) qk_norm_bwd_kernel(const NormArgs a, int q_blocks, float* __restrict__ part) {
  constexpr int LANES = D / 16, ROWS = 256 / LANES;
  const int which = (int)blockIdx.x >= q_blocks;
  const int block = which ? blockIdx.x - q_blocks : blockIdx.x, blocks = which ? gridDim.x - q_blocks : q_blocks;
  const HeadRows& t = a.t[which];
  const int lane = threadIdx.x % LANES;
  const HeadRow<D> at(lane, a.rot);
  const long long rows = (long long)a.B * a.L * t.heads, step = (long long)blocks * ROWS;
  float w[16], dw[16];
  load_weight<D>(t.w, t.w32, at, w);
  #pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.f;
  for (long long first = (long long)block * ROWS; first < rows; first += step) {
    const long long mine = first + threadIdx.x / LANES;
    const bool real = mine < rows;
    const long long row = real ? mine : rows - 1;
    const long long token = row / t.heads;
    const int h = (int)(row % t.heads), b = (int)(token / a.L), l = (int)(token % a.L);
    const __nv_bfloat16* xp = t.x + b * t.xb + l * t.xl + h * t.xh;
    const __nv_bfloat16* gp = t.dy + b * t.gb + l * t.gl + h * t.gh;
    float x[16], g[16];
    unpack16(*reinterpret_cast<const uint4*>(xp + at.c0), *reinterpret_cast<const uint4*>(xp + at.c1), x);
    unpack16(*reinterpret_cast<const uint4*>(gp + at.c0), *reinterpret_cast<const uint4*>(gp + at.c1), g);
    if (a.rot) {
      const int p = table_row(a, token, l);
      if (p < 0) {
        #pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = 0.f;
      } else if (at.turns) {
        float cs[8], sn[8];
        load8(a.cs + (long long)p * (a.rot / 2) + at.c0, cs);
        load8(a.sn + (long long)p * (a.rot / 2) + at.c0, sn);
        turn16(g, cs, sn, -1.f);
      }
    }
    if (t.w != nullptr) {
      float ss = 0.f, hx = 0.f;
      #pragma unroll
      for (int i = 0; i < 16; ++i) { ss += x[i] * x[i]; hx += g[i] * w[i] * x[i]; }
      const float r = rsqrtf(row_sum<LANES>(ss) * (1.f / D) + a.eps);
      const float c = r * r * r * row_sum<LANES>(hx) * (1.f / D);
      #pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (real) dw[i] += g[i] * x[i] * r;
        g[i] = r * (g[i] * w[i]) - c * x[i];
      }
    }
    if (real) {
      __nv_bfloat16* o = t.out + row * D;
      *reinterpret_cast<uint4*>(o + at.c0) = pack8(g);
      *reinterpret_cast<uint4*>(o + at.c1) = pack8(g + 8);
    }
  }
  if (t.w == nullptr) return;
  __shared__ float sums[8][D];
  // the rows of a warp, then the warps one after the other: the same order at every run
  #pragma unroll
  for (int i = 0; i < 16; ++i) {
    #pragma unroll
    for (int o = LANES; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
  }
  if (threadIdx.x % 32 < LANES) {
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      sums[threadIdx.x / 32][at.c0 + i] = dw[i];
      sums[threadIdx.x / 32][at.c1 + i] = dw[8 + i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < D; c += 256) {
    float s = 0.f;
    #pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][c];
    part[(long long)blockIdx.x * D + c] = s;
  }
}

// dw of queries (block 0) and keys (block 1) from the blocks' sums, in the blocks' order; stored, or added to what is there.
struct WeightGrads { void* dst[2]; int is32[2], add[2]; };
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* __restrict__ part, int q_blocks, int blocks, int D, WeightGrads o) {
  __shared__ float sums[1024];
  const int which = blockIdx.x, groups = 1024 / D, c = threadIdx.x % D, g = threadIdx.x / D;
  if (o.dst[which] == nullptr) return;
  const int lo = which ? q_blocks : 0, hi = which ? blocks : q_blocks;
  float s = 0.f;
  #pragma unroll 4
  for (int k = lo + g; k < hi; k += groups) s += part[(long long)k * D + c];
  sums[threadIdx.x] = s;
  __syncthreads();
  if (g != 0) return;
  s = 0.f;
  for (int k = 0; k < groups; ++k) s += sums[k * D + c];
  if (o.is32[which]) {
    float* p = reinterpret_cast<float*>(o.dst[which]) + c;
    *p = o.add[which] ? *p + s : s;
  } else {
    reinterpret_cast<__nv_bfloat16*>(o.dst[which])[c] = __float2bfloat16(s);
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// strides: q's (batch, token, head), k's, then for the backward pass dq's and dk's
static int norm_args(NormArgs* a, const void* q, const void* k, const void* dq, const void* dk, const long long* strides, void* qo, void* ko,
                     const void* qw, const void* kw, int qw32, int kw32, const void* cs, const void* sn, const void* positions, int pos64,
                     int B, int L, int Hq, int Hk, int D, int rot, int table_rows, float eps, int* status) {
  if (B < 1 || L < 1 || Hq < 0 || Hk < 0 || Hq + Hk < 1 || (D != 64 && D != 128 && D != 256) || rot < 0 || rot % 16 || rot > D) return -SSM_ERR_BAD_ARG;
  const void* all[] = {q, k, dq, dk, qo, ko, qw, kw, cs, sn};
  for (const void* p : all) if (!aligned16(p)) return -SSM_ERR_BAD_ARG;
  for (int i = 0; i < (dq != nullptr || dk != nullptr ? 12 : 6); ++i) if (strides[i] % 8) return -SSM_ERR_BAD_ARG;
  auto in = [](const void* p) { return reinterpret_cast<const __nv_bfloat16*>(p); };
  auto out = [](void* p) { return reinterpret_cast<__nv_bfloat16*>(p); };
  const bool grads = dq != nullptr || dk != nullptr;
  const long long none[6] = {0, 0, 0, 0, 0, 0};
  const long long* g = grads ? strides + 6 : none;
  a->t[0] = HeadRows{in(q), in(dq), out(qo), qw, strides[0], strides[1], strides[2], g[0], g[1], g[2], Hq, qw32};
  a->t[1] = HeadRows{in(k), in(dk), out(ko), kw, strides[3], strides[4], strides[5], g[3], g[4], g[5], Hk, kw32};
  a->cs = reinterpret_cast<const float*>(cs);
  a->sn = reinterpret_cast<const float*>(sn);
  a->positions = positions;
  a->pos64 = pos64;
  a->B = B; a->L = L; a->rot = rot; a->table_rows = table_rows;
  a->eps = eps;
  a->status = status;
  return 0;
}

static unsigned norm_grid(long long rows, int D) {
  const long long blocks = (rows + 256 / (D / 16) - 1) / (256 / (D / 16));
  return (unsigned)(blocks < 148 * 8 ? blocks : 148 * 8);
}

}  // namespace ssm

using namespace ssm;

extern "C" int ssm_qk_norm_fwd(const void* q, const void* k, const long long* strides, void* qo, void* ko, const void* qw, const void* kw,
                               int qw32, int kw32, const void* cs, const void* sn, const void* positions, int pos64, int B, int L,
                               int Hq, int Hk, int D, int rot, int table_rows, float eps, int* status, cudaStream_t st) {
  NormArgs a;
  const int bad = norm_args(&a, q, k, nullptr, nullptr, strides, qo, ko, qw, kw, qw32, kw32, cs, sn, positions, pos64, B, L, Hq, Hk, D,
                            rot, table_rows, eps, status);
  if (bad) return bad;
  const unsigned grid = norm_grid((long long)B * L * (Hq + Hk), D);
  if (D == 64) qk_norm_fwd_kernel<64><<<grid, 256, 0, st>>>(a);
  else if (D == 128) qk_norm_fwd_kernel<128><<<grid, 256, 0, st>>>(a);
  else qk_norm_fwd_kernel<256><<<grid, 256, 0, st>>>(a);
  return (int)cudaGetLastError();
}

// Blocks of the backward pass: {queries', all}; the caller's buffer of partial sums has all * D floats.
extern "C" int ssm_qk_norm_bwd_blocks(long long tokens, int Hq, int Hk, int D, int* out2) {
  const long long all = norm_grid(tokens * (Hq + Hk), D);
  long long mine = (all * Hq + (Hq + Hk) / 2) / (Hq + Hk);
  if (Hq > 0 && mine < 1) mine = 1;
  long long theirs = all - mine;
  if (Hk > 0 && theirs < 1) theirs = 1;
  if (Hk == 0) theirs = 0;
  out2[0] = (int)mine;
  out2[1] = (int)(mine + theirs);
  return 0;
}

// dwq, dwk: gradients of the weights, fp32 or bf16 (null: none wanted), stored or (fp32) added to.
extern "C" int ssm_qk_norm_bwd(const void* q, const void* k, const void* dq, const void* dk, const long long* strides, void* dxq, void* dxk,
                               const void* qw, const void* kw, int qw32, int kw32, const void* cs, const void* sn, const void* positions,
                               int pos64, int B, int L, int Hq, int Hk, int D, int rot, int table_rows, float eps, int* status,
                               void* part, void* dwq, void* dwk, int dq32, int dk32, int addq, int addk, cudaStream_t st) {
  NormArgs a;
  const int bad = norm_args(&a, q, k, dq, dk, strides, dxq, dxk, qw, kw, qw32, kw32, cs, sn, positions, pos64, B, L, Hq, Hk, D, rot,
                            table_rows, eps, status);
  if (bad) return bad;
  if ((addq && !dq32) || (addk && !dk32)) return -SSM_ERR_BAD_ARG;
  int blocks[2];
  ssm_qk_norm_bwd_blocks((long long)B * L, Hq, Hk, D, blocks);
  float* p = reinterpret_cast<float*>(part);
  if (D == 64) qk_norm_bwd_kernel<64><<<blocks[1], 256, 0, st>>>(a, blocks[0], p);
  else if (D == 128) qk_norm_bwd_kernel<128><<<blocks[1], 256, 0, st>>>(a, blocks[0], p);
  else qk_norm_bwd_kernel<256><<<blocks[1], 256, 0, st>>>(a, blocks[0], p);
  if (dwq != nullptr || dwk != nullptr)
    qk_norm_dw_kernel<<<2, 1024, 0, st>>>(p, blocks[0], blocks[1], D, WeightGrads{{dwq, dwk}, {dq32, dk32}, {addq, addk}});
  return (int)cudaGetLastError();
}
