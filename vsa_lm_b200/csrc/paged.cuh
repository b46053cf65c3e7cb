// What the paged cache's kernels share (include/bolt3.h): where a row of a sequence lives, fast exponentials, two fp32
// values at a time.
#pragma once

#include <cuda.h>

#include "../../include/bolt3.h"
#include "kv8.cuh"

namespace paged {

using namespace b3;
using kv8::Length;

constexpr uint32_t kWaitIters = 1u << 18;   // polls of a wait; one that gives up sleeps 4 us in each, a second in all
constexpr float kLog2e = 1.4426950408889634f;

// The pages of the sequences
struct Pages {
  const int32_t* table;
  int64_t stride, width, n_pages;
  int log;                       // log2 of the rows of a page
  // the page that holds row `row` of sequence b; -1 where the table has none or names one that the pool does not have
  B3_DEV int page_of(int b, int64_t row) const {
    const int64_t i = row >> log;
    if (i >= width) return -1;
    const int pg = table[b * stride + i];
    return pg < 0 || pg >= n_pages ? -1 : pg;
  }
};

// Pages of a cache described by its pool, or false for a layout that the kernels do not take
inline bool pages_ok(int64_t n_pages, int page, int64_t width, int64_t stride, int HKV, int HD, Pages* p, const int32_t* table) {
  if (page != 16 && page != 32 && page != 64 && page != 128) return false;
  if (HD != 64 && HD != 128) return false;
  if (n_pages < 1 || width < 1 || stride < 0 || HKV < 1 || HKV > 2048) return false;
  // rows are counted in 32 bits by the tensor maps, which hold keys and values
  if (n_pages > 0x3fffffff / HKV || width > 0x7fffff00 / page) return false;
  p->table = table;
  p->stride = stride;
  p->width = width;
  p->n_pages = n_pages;
  p->log = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  return true;
}

// Tensor map of the pool's rows: (HD, page, 2 n_pages HKV), boxes of 64 columns and `rows` rows in the 128-byte swizzle
bool encode_pool(CUtensorMap* m, const void* pool, int64_t n_pages, int page, int HKV, int HD, int rows);

B3_DEV float ex2(float x) {      // 2^x, relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
B3_DEV uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
B3_DEV float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
B3_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
B3_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
B3_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
B3_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// What the two attention kernels are given
struct Attend {
  bolt3_paged_attend_args a;
  Pages pages;
  Length len;                    // len.cap: rows that a sequence may hold (the bound n + T, or the table's)
  int G, rows;
};

// many query rows (csrc/paged_prompt.cu)
size_t prompt_workspace(int B, int T, int H, int HKV, int HD, int64_t n, bool weigh);
int prompt_launch(const Attend& p, cudaStream_t s);

}  // namespace paged
