// Pages of a key-value cache: [page][kv head][slot][D]; a token at position p of sequence b is in slot p % page_size of page
// table[b][p / page_size].  Values are bf16, or 8 bits with one fp32 scale per token and head.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "common.cuh"

namespace ssm {

enum { KV_BF16 = 0, KV_E4M3 = 1, KV_INT8 = 2 };
template <int T> struct KvType;
template <> struct KvType<KV_BF16> { static constexpr int BYTES = 2; };
template <> struct KvType<KV_E4M3> { static constexpr int BYTES = 1; };
template <> struct KvType<KV_INT8> { static constexpr int BYTES = 1; };

struct PageTable {
  const int* ids; const int* lengths;
  int width, pages, page_shift;                // pages per sequence, pages in the pool, log2 of the page's tokens
  int* status;                                 // two words, see report_bad_index
};
// page of position p of sequence b; -1 where the caller's table has none
__device__ __forceinline__ int page_of(const PageTable& t, int b, int p) {
  const int i = p >> t.page_shift;
  int id = -1;
  if (i < t.width) id = t.ids[(long long)b * t.width + i];
  if (id >= 0 && id < t.pages) return id;
  report_bad_index(t.status);
  return -1;
}

// four 8-bit values -> two pairs of fp16, exact
template <int T>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (T == KV_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    // 1024 + (x + 128) is an fp16 number whose low byte is x + 128
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));      // 1152
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

static bool kv_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool kv_table(PageTable* t, const void* ids, const void* lengths, int width, int pages, int page_size, int* status) {
  if (width < 0 || pages < 0 || page_size < 16 || (page_size & (page_size - 1))) return false;
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  *t = PageTable{reinterpret_cast<const int*>(ids), reinterpret_cast<const int*>(lengths), width, pages, shift, status};
  return true;
}
}  // namespace ssm

#define KV_DISPATCH(KERNEL)                                        \
  do {                                                             \
    if (D == 64 && type == KV_BF16) KERNEL(64, KV_BF16);           \
    else if (D == 64 && type == KV_E4M3) KERNEL(64, KV_E4M3);      \
    else if (D == 64 && type == KV_INT8) KERNEL(64, KV_INT8);      \
    else if (D == 128 && type == KV_BF16) KERNEL(128, KV_BF16);    \
    else if (D == 128 && type == KV_E4M3) KERNEL(128, KV_E4M3);    \
    else if (D == 128 && type == KV_INT8) KERNEL(128, KV_INT8);    \
    else if (D == 256 && type == KV_BF16) KERNEL(256, KV_BF16);    \
    else if (D == 256 && type == KV_E4M3) KERNEL(256, KV_E4M3);    \
    else if (D == 256 && type == KV_INT8) KERNEL(256, KV_INT8);    \
    else return -SSM_ERR_BAD_ARG;                                  \
  } while (0)

