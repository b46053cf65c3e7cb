// Softmax attention of new tokens over the 8-bit KV cache, for few query rows per KV head.
//
// For a query row and the keys j it sees, with t_j = sm_scale * scale_k[j] * (q . k8_j):
//   y = sum_j e^t_j scale_v[j] v8_j / sum_j e^t_j.
// The value scale goes into the exponent: u_j = t_j log2(e) + log2 scale_v[j], w_j = 2^(u_j - M) with M a
// bound on the u_j seen so far, numerator sum w_j v8_j, denominator sum w_j / scale_v[j]. So the f16 weights
// of the product are relative to the largest weighted value, however far the scales of two tokens lie apart.
// A weight more than 2^126 below the bound is zero in both sums; that matters only where two tokens' value scales
// lie more than 2^100 apart. Sums and the outputs are fp32. Roundings: w_j to f16 (2^-11 relative, or 2^-32 of the
// largest weighted value: kHeadroom) for the product with the int8 values, which f16 holds exactly; a query row to
// 16-bit integers, relative to its largest value (2^-16 of it; bf16 has already rounded that value to 2^-9), as
// q = 256 hi + lo, so that q . k8 is two int8 products summed exactly.
//
// Bound by HBM: 2 (HD + 4) bytes per key and KV head. The cache is read in blocks of 32 keys, for 8 or 16 query
// rows at once (T * G of them, token-major; more rows: more passes). All blocks of all (sequence, KV head)s are
// one list, and every warp of the machine takes an equal run of it, whatever the lengths of the sequences: within
// a run each head's stretch is a softmax of its own, finished there if it is the whole cache of that head, else
// left in the workspace for a second kernel that joins the runs. A call with little to read takes a CTA per head
// instead, whose warps take its blocks in turn and join in shared memory: one launch.
// A warp works on its own: its lane 0 brings the next block's keys and values by TMA (4 KB boxes; 16-byte copies by
// every lane reached 4.5 TB/s where boxes reach 6.4) into a ring of the warp's own, swizzled so that the fragment
// loads below are free of bank conflicts, and the warp waits on an mbarrier of its own. Both products have the keys or
// dimensions in M and the query rows in N (no padding for up to 8 rows): S^T = K Q^T by mma.sync m16n8k32 on the int8
// keys as they are, with the dimensions permuted so that a lane's 16 bytes feed two products; O^T = V^T P^T by
// m16n8k16 on f16, output dimensions permuted likewise, P^T being S^T transposed by movmatrix.
//
// Measured on a B200, 32 heads on 8 of 128, one token: 131072 keys 57.7 us (4.8 TB/s; 49 of it streaming, the rest the
// join of 1776 runs), 64 sequences of up to 2304 keys 51 us (4.6 TB/s).
#include "../../include/bolt3.h"
#include "kv8.cuh"
#include "kv8_prompt.cuh"
#include "tc5.cuh"
#include "trace.h"

#include <cudaTypedefs.h>

#include <mutex>

namespace {

using namespace b3;
using namespace kv8;

constexpr uint32_t kWaitIters = 1u << 24;
constexpr int kBlock = 32;      // keys of a block: two 16-key halves of the products
constexpr float kLog2e = 1.4426950408889634f;

template <int NT>
constexpr int kWarps = NT == 1 ? 12 : 8;        // one CTA per SM; 168 or 255 registers a thread

struct Params {
  CUtensorMap map;              // the cache's rows: (HD, cap, 2 B HKV), box (HD, kBlock, 1)
  bolt3_kv8_attend_args a;
  Length len;
  int G, rows;
  int n_runs;                   // warps that share the blocks of a column tile; 0: a CTA per head
  float* part;                  // [column tile][run][2][NC][HD] sums: a run's first stretch, its last
  float2* part_ml;              // [..][NC] (bound, sum of weights)
  int2* span;                   // [column tile][head]: where its first partial sum is, its last run; -1: no partial sums
};

B3_DEV void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
B3_DEV uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
B3_DEV uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
B3_DEV float lds4(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
  return v;
}
B3_DEV float ex2(float x) {      // 2^x, relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
B3_DEV float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
B3_DEV float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
B3_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
B3_DEV void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
B3_DEV uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
B3_DEV uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// the four f16 pairs (row A, row B) of two words' bytes: pairs of byte 0, 1, 2, 3. `lo` and `hi` are the byte
// selections that interleave the words (0x5140, 0x7362), or that do so with the words the other way round
B3_DEV void s8x4_pairs(uint32_t wa, uint32_t wb, uint32_t lo, uint32_t hi, uint32_t (&p)[4]) {
  const uint32_t ua = wa ^ 0x80808080u, ub = wb ^ 0x80808080u;
  const uint32_t l = __byte_perm(ua, ub, lo), h = __byte_perm(ua, ub, hi);
  p[0] = __byte_perm(l, 0x64646464u, 0x4140);
  p[1] = __byte_perm(l, 0x64646464u, 0x4342);
  p[2] = __byte_perm(h, 0x64646464u, 0x4140);
  p[3] = __byte_perm(h, 0x64646464u, 0x4342);
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("sub.f16x2 %0, %0, %1;\n" : "+r"(p[i]) : "r"(0x64806480u));
}

// A warp's ring: stages of a block, keys then values, as TMA writes them: rows of HD bytes whose 16-byte pieces are
// permuted within 8 rows (HD 128: piece ^ row % 8; HD 64: piece ^ row / 2 % 4).
template <int HD>
struct Ring {
  static constexpr int KC = HD / 64;      // 16-byte pieces of a key row per lane
  static constexpr int VW = HD / 32;      // words of a value row per lane
  static constexpr int kSide = kBlock * HD;
  static constexpr int kStage = 2 * kSide;
  static constexpr int kDepth = 256 / HD;
  static constexpr int kWarp = kDepth * kStage;
  static constexpr int kScale = kDepth * 2 * kBlock * 4;   // scales, beside the ring
  // cache row (of 8) that stands at place `slot` of the products: so that the eight lanes of a phase of a load
  // fall on different banks
  static B3_DEV int row_of(int slot) { return HD == 128 ? (slot >> 1) | (slot & 1) << 2 : slot; }
  // byte offset of piece c of row r
  static B3_DEV uint32_t at(int r, int c) { return r * HD + ((c ^ (HD == 128 ? r & 7 : r >> 1 & 3)) << 4); }
};

// Where a warp stands in its ring
struct RingState {
  uint32_t ring, scale, bars;   // shared addresses
  uint32_t phase = 0;           // parity of each stage's next wait
  int stage = 0;
  bool dead = false;            // a wait ran out
};

template <int HD, int NT>
constexpr size_t stream_smem() {
  const size_t ring = (size_t)kWarps<NT> * (Ring<HD>::kWarp + Ring<HD>::kScale), join = (size_t)kWarps<NT> * 8 * NT * (HD * 4 + 8);
  return (ring > join ? ring : join) + 1024;
}

// Running softmax of a warp over a stretch of one head's keys, for 8 NT query rows.
template <int HD, int NT>
struct Softmax {
  static constexpr int MT = HD / 16;            // 16-dimension tiles of the output
  float o[MT][NT][4];                           // row grp: dimension 4 VW grp + 2 m, row grp + 8: the one after it
  float M0[NT], M1[NT], l0[NT], l1[NT];         // of query rows 2 tig and 2 tig + 1 of each tile of 8
};

// Blocks 0, step, .. < n_blk, counted from blk0, of head (b, kvh), of whose keys query row r of this tile sees the
// first s + token + 1.
template <int HD, int NT>
B3_DEV void walk(const Params& p, RingState& rs, int b, int kvh, int64_t s, int col0, int64_t blk0, int n_blk, int step,
                 Softmax<HD, NT>& f) {
  using R = Ring<HD>;
  constexpr int KC = R::KC, VW = R::VW, MT = HD / 16, kDepth = R::kDepth;
  const bolt3_kv8_attend_args& a = p.a;
  const int lane = threadIdx.x & 31, grp = lane >> 2, tig = lane & 3;
  const int head = b * a.HKV + kvh, heads = a.B * a.HKV;
  const int64_t row0 = blk0 * kBlock;                                           // the stretch's first row of the head
  const float* sc = a.scale + (int64_t)head * a.cap;
  if (rs.dead) n_blk = 0;
  auto load = [&](int blk, int stage) {
    const int64_t row = row0 + (int64_t)blk * kBlock;
    if (lane == 0) {                            // rows at or past cap come as zeros
      uint64_t* bar = reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(rs.bars + 8 * stage));
      void* dst = reinterpret_cast<void*>(__cvta_shared_to_generic(rs.ring + stage * R::kStage));
      tc5::mbar_expect_tx(bar, R::kStage);
      tc5::tma_load_3d(dst, &p.map, 0, (int)row, head, bar);
      tc5::tma_load_3d(reinterpret_cast<char*>(dst) + R::kSide, &p.map, 0, (int)row, heads + head, bar);
    }
    const float* z = sc + min(row + lane, a.cap - 1);
    cp4(rs.scale + stage * (2 * kBlock * 4) + lane * 4, z);
    cp4(rs.scale + stage * (2 * kBlock * 4) + kBlock * 4 + lane * 4, z + (int64_t)heads * a.cap);
  };
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) {
    if (i * step < n_blk) {
      int st = rs.stage + i;
      load(i * step, st >= kDepth ? st - kDepth : st);
    }
    cp_async_commit();
  }

  // queries as B fragments: a lane holds row grp of each n8 tile, dimensions 16 (tig + 4 c) .. + 15, as the high and
  // the low bytes of 16-bit integers. Row r of the tile is head kvh * G + r % G of token r / G
  uint32_t qh[NT][KC][4], ql[NT][KC][4];
  float c0[NT], c1[NT];                        // sm_scale log2(e) times the unit of rows 2 tig and 2 tig + 1
  int see0[NT], see1[NT];                      // keys of the stretch these rows see (any number for a row past the last)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = col0 + 8 * n + grp;
    float x[KC][16], m = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      uint4 r0 = make_uint4(0, 0, 0, 0), r1 = r0;
      if (r < p.rows) {
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + b * a.q_sb + (r / p.G) * a.q_st +
                                                          (int64_t)(kvh * p.G + r % p.G) * HD + 16 * (tig + 4 * c));
        r0 = src[0];
        r1 = src[1];
      }
      const uint32_t w[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 v = unpack_bf16(w[i]);
        x[c][2 * i] = v.x;
        x[c][2 * i + 1] = v.y;
        m = max_nan(m, max_nan(fabsf(v.x), fabsf(v.y)));
      }
    }
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = max_nan(m, 1e-30f);
    const float to_int = 32512.f / m;           // 127 * 256: the high byte stays within -127 .. 127
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t hw = 0, lw = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int v = __float2int_rn(x[c][4 * i + j] * to_int);
          hw |= ((uint32_t)((v + 128) >> 8) & 255u) << (8 * j);
          lw |= ((uint32_t)v & 255u) << (8 * j);
        }
        qh[n][c][i] = hw;
        ql[n][c][i] = lw;
      }
    const float up = a.sm_scale * kLog2e * (m * (1.f / 32512.f));
    c0[n] = __shfl_sync(0xffffffffu, up, 8 * tig);
    c1[n] = __shfl_sync(0xffffffffu, up, 8 * tig + 4);
    const int r0 = col0 + 8 * n + 2 * tig;
    const int64_t first = s + 1 - row0;
    see0[n] = (int)min(max(first + r0 / p.G, (int64_t)0), (int64_t)0x7ffffff0);
    see1[n] = (int)min(max(first + (r0 + 1) / p.G, (int64_t)0), (int64_t)0x7ffffff0);
  }
  const int see_all = (int)min(max(s + 1 + col0 / p.G - row0, (int64_t)0), (int64_t)0x7ffffff0);   // what every row sees
  const int kg = R::row_of(grp);               // this lane's keys of a block: kg + 8 h
  uint32_t k_at[KC], v_at[2];                  // this lane's pieces of key row kg, of the value rows of slots 2 tig, 2 tig + 1
#pragma unroll
  for (int c = 0; c < KC; ++c) k_at[c] = R::at(kg, tig + 4 * c);
  // every other lane takes the two value rows in the other order, to keep off each other's banks
  const bool swap = HD == 128 ? grp & 1 : tig & 1;
  const uint32_t sel_lo = swap ? 0x1504 : 0x5140, sel_hi = swap ? 0x3726 : 0x7362;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = R::row_of(2 * tig + (j ^ (int)swap));
    v_at[j] = R::kSide + (VW == 4 ? R::at(r, grp) : R::at(r, grp >> 1) + (grp & 1) * 8);
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    f.M0[n] = f.M1[n] = neg_inf();
    f.l0[n] = f.l1[n] = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) f.o[m][n][0] = f.o[m][n][1] = f.o[m][n][2] = f.o[m][n][3] = 0.f;
  }
  for (int blk = 0; blk < n_blk; blk += step) {
    __syncwarp();                               // every lane has read the stage that is refilled now
    const int ahead = blk + (kDepth - 1) * step, stage = rs.stage;
    if (ahead < n_blk) load(ahead, stage == 0 ? kDepth - 1 : stage - 1);
    cp_async_commit();
    cp_async_wait<kDepth - 1>();
    const bool ok = tc5::mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(rs.bars + 8 * stage)),
                                   rs.phase >> stage & 1, kWaitIters);
    if (!__all_sync(0xffffffffu, ok)) {         // also: the scales come from other lanes' copies
      rs.dead = true;
      break;
    }
    rs.phase ^= 1u << stage;
    rs.stage = stage == kDepth - 1 ? 0 : stage + 1;
    const uint32_t at = rs.ring + stage * R::kStage, at_s = rs.scale + stage * (2 * kBlock * 4);
    float ks[4], lg[4], iv[4];                  // of keys kg + 8 h: key scale, log2 and reciprocal of the value scale
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      ks[h] = lds4(at_s + (kg + 8 * h) * 4);
      lg[h] = lds4(at_s + (kBlock + kg + 8 * h) * 4);
    }
    // S^T = K Q^T; half i holds keys 16 i + kg and 16 i + kg + 8
    float t[2][NT][4];
    {
      uint4 k[4][KC];
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int c = 0; c < KC; ++c) k[h][c] = lds16(at + k_at[c] + 8 * h * HD);
      int acc[2][NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[0][n][i] = acc[1][n][i] = 0;
#pragma unroll
      for (int part = 0; part < 2; ++part) {    // the high bytes, times 256, then the low bytes
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 x = k[2 * i][c], y = k[2 * i + 1][c];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint32_t(&q)[4] = part == 0 ? qh[n][c] : ql[n][c];
              mma_s8(acc[i][n], x.x, y.x, x.y, y.y, q[0], q[1]);
              mma_s8(acc[i][n], x.z, y.z, x.w, y.w, q[2], q[3]);
            }
          }
        if (part == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][n][e] <<= 8;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) t[i][n][e] = (float)acc[i][n][e];
    }
    uint32_t vw[8][VW];                         // [4 i + 2 h + j]: value row of slot 2 tig + (j ^ swap) + 8 h + 16 i
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t from = at + v_at[j & 1] + 8 * (j >> 1) * HD;
      if constexpr (VW == 4) {
        const uint4 x = lds16(from);
        vw[j][0] = x.x; vw[j][1] = x.y; vw[j][2] = x.z; vw[j][3] = x.w;
      } else {
        const uint2 x = lds8(from);
        vw[j][0] = x.x; vw[j][1] = x.y;
      }
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      iv[h] = rcp(lg[h]);
      lg[h] = lg2(lg[h]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        t[i][n][0] = fmaf(t[i][n][0], ks[2 * i] * c0[n], lg[2 * i]);
        t[i][n][1] = fmaf(t[i][n][1], ks[2 * i] * c1[n], lg[2 * i]);
        t[i][n][2] = fmaf(t[i][n][2], ks[2 * i + 1] * c0[n], lg[2 * i + 1]);
        t[i][n][3] = fmaf(t[i][n][3], ks[2 * i + 1] * c1[n], lg[2 * i + 1]);
      }
    const bool masked = blk * kBlock + kBlock > see_all;
    if (masked) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = blk * kBlock + 16 * i + kg;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (key >= see0[n]) t[i][n][0] = neg_inf();
          if (key >= see1[n]) t[i][n][1] = neg_inf();
          if (key + 8 >= see0[n]) t[i][n][2] = neg_inf();
          if (key + 8 >= see1[n]) t[i][n][3] = neg_inf();
        }
      }
    }
    // the bounds move only when a weight would pass 2^15 (and at the first key a row sees)
    bool over = false;
    float m0[NT], m1[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m0[n] = fmaxf(fmaxf(t[0][n][0], t[0][n][2]), fmaxf(t[1][n][0], t[1][n][2]));
      m1[n] = fmaxf(fmaxf(t[0][n][1], t[0][n][3]), fmaxf(t[1][n][1], t[1][n][3]));
      over |= m0[n] > f.M0[n] + kMostWeight || m1[n] > f.M1[n] + kMostWeight;
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          m0[n] = fmaxf(m0[n], __shfl_xor_sync(0xffffffffu, m0[n], x));
          m1[n] = fmaxf(m1[n], __shfl_xor_sync(0xffffffffu, m1[n], x));
        }
        m0[n] = fmaxf(f.M0[n], m0[n] - kHeadroom);
        m1[n] = fmaxf(f.M1[n], m1[n] - kHeadroom);
        const float f0 = f.M0[n] == neg_inf() ? 0.f : ex2(f.M0[n] - m0[n]), f1 = f.M1[n] == neg_inf() ? 0.f : ex2(f.M1[n] - m1[n]);
        f.M0[n] = m0[n];
        f.M1[n] = m1[n];
        f.l0[n] *= f0;
        f.l1[n] *= f1;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          f.o[m][n][0] *= f0; f.o[m][n][2] *= f0;
          f.o[m][n][1] *= f1; f.o[m][n][3] *= f1;
        }
      }
    }
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float r0 = f.M0[n] == neg_inf() ? 0.f : f.M0[n], r1 = f.M1[n] == neg_inf() ? 0.f : f.M1[n];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float w0 = ex2(t[i][n][0] - r0), w1 = ex2(t[i][n][1] - r1), w2 = ex2(t[i][n][2] - r0), w3 = ex2(t[i][n][3] - r1);
        if (masked) {                           // a key that a row does not see has weight 0, whatever its scale holds
          f.l0[n] += (w0 == 0.f ? 0.f : w0 * iv[2 * i]) + (w2 == 0.f ? 0.f : w2 * iv[2 * i + 1]);
          f.l1[n] += (w1 == 0.f ? 0.f : w1 * iv[2 * i]) + (w3 == 0.f ? 0.f : w3 * iv[2 * i + 1]);
        } else {
          f.l0[n] = fmaf(w0, iv[2 * i], fmaf(w2, iv[2 * i + 1], f.l0[n]));
          f.l1[n] = fmaf(w1, iv[2 * i], fmaf(w3, iv[2 * i + 1], f.l1[n]));
        }
        pb[i][n][0] = transpose8(pack_f16(w0, w1));
        pb[i][n][1] = transpose8(pack_f16(w2, w3));
      }
    }
    // O^T += V^T P^T: tile 2 w + j holds dimensions 4 VW grp + 4 w + 2 j (rows grp) and + 1 (rows grp + 8)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t u[4], v[4];
        s8x4_pairs(vw[4 * i][w], vw[4 * i + 1][w], sel_lo, sel_hi, u);
        s8x4_pairs(vw[4 * i + 2][w], vw[4 * i + 3][w], sel_lo, sel_hi, v);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma_f16(f.o[2 * w + j][n], u[2 * j], u[2 * j + 1], v[2 * j], v[2 * j + 1], pb[i][n][0], pb[i][n][1]);
      }
  }
  cp_async_wait<0>();
  __syncwarp();
  if (rs.dead && n_blk > 0) {                   // give copies in flight one more bounded wait each before leaving
    for (int st = 0; st < kDepth; ++st)
      tc5::mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(rs.bars + 8 * st)), rs.phase >> st & 1, kWaitIters);
    if (lane == 0 && a.status) atomicOr(a.status, 2);
  }
  // the lanes' sums of weights (the bounds are the same in all lanes of a row)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      f.l0[n] += __shfl_xor_sync(0xffffffffu, f.l0[n], x);
      f.l1[n] += __shfl_xor_sync(0xffffffffu, f.l1[n], x);
    }
}

// element (row r, first dimension) of head (b, kvh)'s output
template <int HD>
B3_DEV bf16* out_row(const Params& p, int b, int kvh, int row) {
  return reinterpret_cast<bf16*>(p.a.y) + (((int64_t)b * p.a.T + row / p.G) * p.a.H + kvh * p.G + row % p.G) * HD;
}

// blocks that a head of a sequence with s rows has for a tile whose last row is of token `last`
B3_DEV int64_t blocks_of(int64_t s, int last) { return s < 0 ? 0 : (s + last + kBlock) / kBlock; }

template <int HD, int NT>
__global__ void __launch_bounds__(32 * kWarps<NT>) kv8_stream_kernel(const __grid_constant__ Params p) {
  using R = Ring<HD>;
  constexpr int NC = 8 * NT, MT = HD / 16, VW = R::VW, kW = kWarps<NT>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t s_bars[kW][R::kDepth];
  const bolt3_kv8_attend_args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, tig = lane & 3;
  const int tile = blockIdx.y, col0 = tile * NC;
  const int last = (min(col0 + NC, p.rows) - 1) / p.G;          // token of the tile's last row
  unsigned char* smem = smem_raw + ((1024 - (tc5::smem_u32(smem_raw) & 1023)) & 1023);
  RingState rs;
  rs.ring = tc5::smem_u32(smem) + warp * R::kWarp;
  rs.scale = tc5::smem_u32(smem) + kW * R::kWarp + warp * R::kScale;
  rs.bars = tc5::smem_u32(s_bars[warp]);
  if (lane == 0) {
    for (int i = 0; i < R::kDepth; ++i) tc5::mbar_init(&s_bars[warp][i], 1);
    tc5::mbar_fence_init();
  }
  __syncwarp();
  Softmax<HD, NT> f;
  grid_dep_launch();
  grid_dep_wait();
  bool bad = false;

  if (p.n_runs == 0) {
    const int b = blockIdx.x / a.HKV, kvh = blockIdx.x % a.HKV;
    const int64_t s = p.len.rows(b, bad);
    if (bad && tid == 0 && tile == 0 && a.status) atomicOr(a.status, 8);
    const int64_t nb = blocks_of(s, last);
    walk<HD, NT>(p, rs, b, kvh, s, col0, warp, (int)max(nb - warp, (int64_t)0), kW, f);
    __syncthreads();                                            // the rings are read: their memory is free
    float* so = reinterpret_cast<float*>(smem);                 // [kW][NC][HD]
    float2* sml = reinterpret_cast<float2*>(so + kW * NC * HD);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + 2 * tig;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float* at = so + (warp * NC + r) * HD + 4 * VW * grp + 2 * m;
        *reinterpret_cast<float2*>(at) = make_float2(f.o[m][n][0], f.o[m][n][2]);
        *reinterpret_cast<float2*>(at + HD) = make_float2(f.o[m][n][1], f.o[m][n][3]);
      }
      if (grp == 0) {
        sml[warp * NC + r] = make_float2(f.M0[n], f.l0[n]);
        sml[warp * NC + r + 1] = make_float2(f.M1[n], f.l1[n]);
      }
    }
    __syncthreads();
    const int rows = min(NC, p.rows - col0);
    for (int i = tid; i < rows * HD; i += 32 * kW) {
      const int r = i / HD, d = i % HD;
      float m = neg_inf();
#pragma unroll
      for (int w = 0; w < kW; ++w) m = fmaxf(m, sml[w * NC + r].x);
      float acc = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        const float2 ml = sml[w * NC + r];
        const float g = ml.x == neg_inf() ? 0.f : exp2f(ml.x - m);
        acc = fmaf(so[(w * NC + r) * HD + d], g, acc);
        l = fmaf(ml.y, g, l);
      }
      out_row<HD>(p, b, kvh, col0 + r)[d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
    }
    return;
  }

  // this warp's run of the list of all blocks, ordered by sequence, head, key
  const int run = blockIdx.x * kW + warp;
  if (run >= p.n_runs) return;
  int b = 0;
  int64_t total = 0, lo, hi, start = 0;                         // start: of sequence b's blocks in the list
  int64_t s, nb;
  if (a.lens == nullptr) {
    s = p.len.rows(0, bad);
    nb = blocks_of(s, last);
    total = nb * a.B * a.HKV;
    if (bad && run == 0 && lane == 0 && tile == 0 && a.status) atomicOr(a.status, 8);
    const int64_t runs = min((int64_t)p.n_runs, total);         // none is empty: the join takes all from first to last
    if (run >= runs) return;
    lo = total * run / runs;
    hi = total * (run + 1) / runs;
    b = (int)(lo / (nb * a.HKV));
    start = b * nb * a.HKV;
  } else {
    for (int i = lane; i < a.B; i += 32) total += blocks_of(p.len.rows(i, bad), last);
    if (bad && run == 0 && tile == 0 && a.status) atomicOr(a.status, 8);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    total *= a.HKV;
    const int64_t runs = min((int64_t)p.n_runs, total);         // none is empty: the join takes all from first to last
    if (run >= runs) return;
    lo = total * run / runs;
    hi = total * (run + 1) / runs;
    // the sequence that block lo belongs to
    for (int i0 = 0;; i0 += 32) {
      const int64_t mine = i0 + lane < a.B ? blocks_of(p.len.rows(i0 + lane, bad), last) * a.HKV : 0;
      int64_t upto = mine;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, start + upto > lo);
      if (past) {
        const int at = __ffs(past) - 1;
        b = i0 + at;
        start += __shfl_sync(0xffffffffu, upto - mine, at);
        break;
      }
      start += __shfl_sync(0xffffffffu, upto, 31);
      if (i0 + 32 >= a.B) return;                               // not reached: lo < total
    }
    s = p.len.rows(b, bad);
    nb = blocks_of(s, last);
  }
  int kvh = (int)((lo - start) / nb);
  bool first = true;
  while (lo < hi) {
    const int64_t head = start + kvh * nb;                      // this head's first block in the list
    const int64_t b0 = lo - head, b1 = min(hi - head, nb);
    walk<HD, NT>(p, rs, b, kvh, s, col0, b0, (int)(b1 - b0), 1, f);
    const bool whole = b0 == 0 && b1 == nb;
    int2* span = p.span + (int64_t)tile * a.B * a.HKV + b * a.HKV + kvh;
    const int64_t slot = ((int64_t)tile * p.n_runs + run) * 2 + (first ? 0 : 1);
    if (lane == 0) {
      if (whole) {
        *span = make_int2(-1, -1);
      } else {
        if (b0 == 0) span->x = run * 2 + (first ? 0 : 1);
        if (b1 == nb) span->y = run;
      }
    }
    if (whole) {                                         // the head's whole cache: done
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = col0 + 8 * n + 2 * tig;
        const float i0 = f.l0[n] == 0.f ? 0.f : 1.f / f.l0[n], i1 = f.l1[n] == 0.f ? 0.f : 1.f / f.l1[n];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int d = 4 * VW * grp + 2 * m;
          if (r < p.rows)
            *reinterpret_cast<uint32_t*>(out_row<HD>(p, b, kvh, r) + d) = pack_bf16(f.o[m][n][0] * i0, f.o[m][n][2] * i0);
          if (r + 1 < p.rows)
            *reinterpret_cast<uint32_t*>(out_row<HD>(p, b, kvh, r + 1) + d) = pack_bf16(f.o[m][n][1] * i1, f.o[m][n][3] * i1);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = 8 * n + 2 * tig;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float* at = p.part + (slot * NC + r) * HD + 4 * VW * grp + 2 * m;
          if (col0 + r < p.rows) *reinterpret_cast<float2*>(at) = make_float2(f.o[m][n][0], f.o[m][n][2]);
          if (col0 + r + 1 < p.rows) *reinterpret_cast<float2*>(at + HD) = make_float2(f.o[m][n][1], f.o[m][n][3]);
        }
        if (grp == 0) {
          p.part_ml[slot * NC + r] = make_float2(f.M0[n], f.l0[n]);
          p.part_ml[slot * NC + r + 1] = make_float2(f.M1[n], f.l1[n]);
        }
      }
    }
    first = false;
    lo = head + b1;
    if (b1 == nb && ++kvh == a.HKV && lo < hi) {                // on to the next sequence that has keys
      kvh = 0;
      start += nb * a.HKV;
      do {
        ++b;
        if (a.lens != nullptr) {
          s = p.len.rows(b, bad);
          nb = blocks_of(s, last);
        }
      } while (nb == 0);
    }
  }
}

// The runs' partial sums of a (head, query row) joined: by one warp where a head has few of them (ROWS = 4 rows a block),
// else by all warps of a block (ROWS = 1)
constexpr int kMaxJoinWarps = 16;

template <int HD, int NC, int ROWS>
__global__ void __launch_bounds__(ROWS == 1 ? 32 * kMaxJoinWarps : 32 * ROWS) kv8_join_kernel(const __grid_constant__ Params p) {
  constexpr int EPL = HD / 32;                                  // dimensions of a lane
  __shared__ float s_acc[ROWS == 1 ? kMaxJoinWarps : 1][HD], s_m[kMaxJoinWarps], s_l[kMaxJoinWarps];
  const bolt3_kv8_attend_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = ROWS == 1 ? blockDim.x >> 5 : 1;
  const int head = blockIdx.x, b = head / a.HKV, kvh = head % a.HKV, row = blockIdx.y * ROWS + (ROWS == 1 ? 0 : warp);
  const int tile = row / NC, r = row % NC;
  grid_dep_launch();
  grid_dep_wait();
  if (row >= p.rows) return;
  bool bad = false;
  const bool idle = p.len.rows(b, bad) < 0;
  const int2 span = p.span[(int64_t)tile * gridDim.x + head];
  bf16* y = out_row<HD>(p, b, kvh, row);
  const int r0 = span.x >> 1;
  if (idle || (span.x >= 0 && (span.x >= 2 * p.n_runs || span.y < r0 || span.y >= p.n_runs))) {   // (the latter: a run gave up)
    if (warp == 0 || ROWS > 1)
      for (int i = lane; i < HD; i += 32) y[i] = __float2bfloat16_rn(0.f);
    return;
  }
  if (span.x < 0) return;                                       // the run wrote the output itself
  const int64_t base = (int64_t)tile * p.n_runs * 2;
  const int n = span.y - r0 + 1;
  float m = neg_inf(), l = 0.f, acc[EPL] = {};
  constexpr int kBatch = 4;
  for (int i0 = ROWS == 1 ? warp : 0; i0 < n; i0 += kBatch * n_warps) {
    float2 ml[kBatch];
    float x[kBatch][EPL];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * n_warps;
      const int64_t at = (base + (i == 0 ? span.x : 2 * (r0 + min(i, n - 1)))) * NC + r;   // a later run's first stretch
      ml[j] = i < n ? p.part_ml[at] : make_float2(neg_inf(), 0.f);
#pragma unroll
      for (int e = 0; e < EPL; ++e) x[j][e] = i < n ? p.part[at * HD + 32 * e + lane] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float to = fmaxf(m, ml[j].x), ref = to == neg_inf() ? 0.f : to;
      const float f0 = exp2f(m - ref), f1 = exp2f(ml[j].x - ref);   // exp2f(-inf) = 0
      m = to;
      l = fmaf(l, f0, ml[j].y * f1);
#pragma unroll
      for (int e = 0; e < EPL; ++e) acc[e] = fmaf(acc[e], f0, x[j][e] * f1);
    }
  }
  if constexpr (ROWS > 1) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) y[32 * e + lane] = __float2bfloat16_rn(l == 0.f ? 0.f : acc[e] / l);
  } else {
#pragma unroll
    for (int e = 0; e < EPL; ++e) s_acc[warp][32 * e + lane] = acc[e];
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < HD; i += blockDim.x) {
      m = neg_inf();
      for (int w = 0; w < n_warps; ++w) m = fmaxf(m, s_m[w]);
      float sum = 0.f;
      l = 0.f;
      for (int w = 0; w < n_warps; ++w) {
        const float g = s_m[w] == neg_inf() ? 0.f : exp2f(s_m[w] - m);
        sum = fmaf(s_acc[w][i], g, sum);
        l = fmaf(s_l[w], g, l);
      }
      y[i] = __float2bfloat16_rn(l == 0.f ? 0.f : sum / l);
    }
  }
}

// how a call is cut: columns of a CTA (in 8), column tiles, runs
struct Plan {
  int nt, tiles, runs;
  size_t bytes;
};

Plan plan_of(int B, int T, int H, int HKV, int HD, int64_t n) {
  Plan pl;
  const int64_t rows = (int64_t)T * (H / HKV), heads = (int64_t)B * HKV;
  pl.nt = rows <= 8 ? 1 : 2;
  pl.tiles = (int)((rows + 8 * pl.nt - 1) / (8 * pl.nt));
  const int64_t warps = pl.nt == 1 ? kWarps<1> : kWarps<2>;
  const int64_t per_head = (n + T + kBlock - 1) / kBlock, blocks = heads * per_head;
  // A CTA per head where all are on the machine at once and a warp gets five blocks at most (32 query heads on 8, HD 128:
  // one sequence of 1000 tokens 9.0 us against 10.7 in runs, of 2000 13.4 against 12.4, of 4000 21.1 against 13.1; with
  // 16 rows a head, of 800 13.3 against 14.3, of 1200 15.6 against 14.5; 64 sequences of 200 tokens, 512 heads, 25.3
  // against 16.0). Else every warp a run, of two blocks or more
  int64_t runs = 0;
  if (heads * pl.tiles > 148 || per_head > 5 * warps) runs = blocks / 2 < 148 * warps ? blocks / 2 : 148 * warps;
  if (runs < 1 && heads * pl.tiles > 148) runs = 1;
  pl.runs = (int)runs;
  pl.bytes = 0;
  if (runs > 0)
    pl.bytes = (size_t)pl.tiles * ((size_t)runs * 2 * (size_t)(8 * pl.nt) * ((size_t)HD * 4 + 8) + (size_t)heads * 8);
  return pl;
}

template <int HD, int NT>
int launch_stream(Params p, const Plan& pl, cudaStream_t s) {
  constexpr int NC = 8 * NT;
  constexpr size_t smem = stream_smem<HD, NT>();
  if (cudaFuncSetAttribute(kv8_stream_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  p.n_runs = pl.runs;
  p.part = reinterpret_cast<float*>(p.a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part + (size_t)pl.tiles * pl.runs * 2 * NC * HD);
  p.span = reinterpret_cast<int2*>(p.part_ml + (size_t)pl.tiles * pl.runs * 2 * NC);
  const unsigned heads = (unsigned)(p.a.B * p.a.HKV), ctas = pl.runs == 0 ? heads : (unsigned)((pl.runs + kWarps<NT> - 1) / kWarps<NT>);
  if (launch_overlapped(kv8_stream_kernel<HD, NT>, dim3(ctas, (unsigned)pl.tiles), dim3(32 * kWarps<NT>), smem, s, p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  if (pl.runs == 0) return BOLT3_OK;
  const int per_head = pl.runs / (int)heads + 2;                // partial sums that a head has on average, about
  const cudaError_t e = per_head <= 8
      ? launch_overlapped(kv8_join_kernel<HD, NC, 4>, dim3(heads, (unsigned)((p.rows + 3) / 4)), dim3(128), 0, s, p)
      : launch_overlapped(kv8_join_kernel<HD, NC, 1>, dim3(heads, (unsigned)p.rows), dim3(per_head >= 32 ? 512 : 256), 0, s, p);
  if (e != cudaSuccess) return BOLT3_ERR_CUDA;
  return BOLT3_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// the cache's int8 rows (HD, cap, 2 B HKV), boxes of kBlock rows, swizzled over the row's bytes
bool encode_cache(CUtensorMap* m, const bolt3_kv8_attend_args* a) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a->HD, (cuuint64_t)a->cap, (cuuint64_t)2 * a->B * a->HKV};
  const cuuint64_t strides[2] = {(cuuint64_t)a->HD, (cuuint64_t)a->cap * a->HD};
  const cuuint32_t box[3] = {(cuuint32_t)a->HD, kBlock, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(a->data), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, a->HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether a call's rows go to the kernel for many rows, which works on tiles of 128. Measured at 32 heads on 8, HD 128, 32 and
// 48 rows of a head: 64 sequences of 2304 tokens 143 and 214 us here, 198 and 199 there; of 300 tokens 48 and 70, 51 and 51;
// one sequence of 2304 18 and 22, 19 and 20. Not everywhere the better one: 16 sequences take 31 us here at 32 rows and 300
// tokens, 13 there, 65 at 2304 tokens, 51 there
bool many_rows(int T, int H, int HKV) { return (int64_t)T * (H / HKV) > 32; }

bool shape_ok(int B, int T, int H, int HKV, int HD) {
  return B > 0 && T > 0 && HKV > 0 && H > 0 && H % HKV == 0 && H / HKV <= 16 && (HD == 64 || HD == 128) &&
         T <= (1 << 24) / (H / HKV) && (int64_t)B * HKV <= 0x3fffffff;
}

}  // namespace

extern "C" size_t bolt3_kv8_attend_workspace(int B, int T, int H, int HKV, int HD, int64_t n) {
  if (!shape_ok(B, T, H, HKV, HD) || n < 0 || n > 0x7fffffff) return 0;
  return many_rows(T, H, HKV) ? kv8_prompt_workspace(B, T, H, HKV, HD, n) : plan_of(B, T, H, HKV, HD, n).bytes;
}

extern "C" int bolt3_kv8_attend(const bolt3_kv8_attend_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_kv8_attend");
  if (!a || !a->q || !a->data || !a->scale || !a->y) return BOLT3_ERR_ARG;
  if (a->lens != nullptr && a->pos_dev != nullptr) return BOLT3_ERR_ARG;
  if (a->pos_dev != nullptr && a->pos_span < 1) return BOLT3_ERR_ARG;
  if (!shape_ok(a->B, a->T, a->H, a->HKV, a->HD)) return BOLT3_ERR_SHAPE;
  const int64_t dmax = a->pos_dev != nullptr ? a->pos_span - 1 : 0;
  if (a->n < 0 || a->n > a->cap || a->cap < a->T || a->cap > 0x7fffffff || (a->lens == nullptr && a->n > a->cap - a->T - dmax)) return BOLT3_ERR_CAPACITY;
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->data | (uintptr_t)a->scale | (uintptr_t)a->y | (uintptr_t)a->workspace;
  if ((al & 15) || ((a->q_sb | a->q_st) & 7)) return BOLT3_ERR_ALIGN;
  const Length len{a->lens, a->pos_dev, a->n, a->pos_ref, a->pos_span, a->cap, a->T};
  if (many_rows(a->T, a->H, a->HKV)) return kv8_prompt_launch(a, len, (cudaStream_t)stream);
  const Plan pl = plan_of(a->B, a->T, a->H, a->HKV, a->HD, a->n);
  if (pl.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < pl.bytes)) return BOLT3_ERR_CAPACITY;
  Params p;
  if (!encode_cache(&p.map, a)) return BOLT3_ERR_CUDA;
  p.a = *a;
  p.len = len;
  p.G = a->H / a->HKV;
  p.rows = a->T * p.G;
  cudaStream_t s = (cudaStream_t)stream;
  if (a->HD == 128) return pl.nt == 1 ? launch_stream<128, 1>(p, pl, s) : launch_stream<128, 2>(p, pl, s);
  return pl.nt == 1 ? launch_stream<64, 1>(p, pl, s) : launch_stream<64, 2>(p, pl, s);
}
