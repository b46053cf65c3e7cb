// What the 8-bit KV cache's kernels share (include/bolt3.h): the length of a sequence, the scale's floor.
#pragma once

#include "common.cuh"

namespace kv8 {

constexpr float kScaleFloor = 0x1p-40f;

// The weights of the attention kernels are 2^(u - M) in f16, whose range is 2^-24 .. 2^15. M is set 2^7 below the largest u
// seen and moves only when a weight would pass 2^15, so that the usual step has no rescaling. A weight is then rounded to
// 2^-11 of itself or to within 2^-32 of the largest one, whichever is more. (With M at the largest, what lies below 2^-25 of
// it was lost from the numerator: many thousand such keys are a visible share of the output.)
constexpr float kHeadroom = 7.f, kMostWeight = 15.f;

// Rows sequence b holds before the call, or -1 for an idle one. `bad` is set for a length that is
// neither idle nor leaves room for T rows.
struct Length {
  const int32_t* lens;
  const int64_t* pos_dev;
  int64_t n, pos_ref, pos_span, cap, T;
  B3_DEV int64_t rows(int b, bool& bad) const {
    int64_t s = n;
    if (lens != nullptr) {
      s = lens[b];
      if (s == -1) return -1;
    } else if (pos_dev != nullptr) {
      const int64_t d = *pos_dev - pos_ref;
      if (d < 0 || d >= pos_span) {
        bad = true;
        return -1;
      }
      s += d;
    }
    if (s < 0 || s > cap - T) {
      bad = true;
      return -1;
    }
    return s;
  }
};

// max that keeps a NaN
B3_DEV float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// four int8 of a word as two f16 pairs, exactly: x + 128 in the low bits of 1024's mantissa, minus 1152
B3_DEV void s8x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  lo = __byte_perm(u, 0x64646464u, 0x4140);
  hi = __byte_perm(u, 0x64646464u, 0x4342);
  asm("sub.f16x2 %0, %0, %1;\n" : "+r"(lo) : "r"(0x64806480u));
  asm("sub.f16x2 %0, %0, %1;\n" : "+r"(hi) : "r"(0x64806480u));
}

// as two bf16 pairs, exactly: 128 + the low seven bits, minus 128, or minus 256 for a negative one
B3_DEV void s8x4_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t x = __byte_perm(w, 0x43434343u, 0x4140), y = __byte_perm(w, 0x43434343u, 0x4342);
  asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(lo) : "r"(x & 0xff7fff7fu), "r"(x & 0xff80ff80u));
  asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(hi) : "r"(y & 0xff7fff7fu), "r"(y & 0xff80ff80u));
}

}  // namespace kv8
