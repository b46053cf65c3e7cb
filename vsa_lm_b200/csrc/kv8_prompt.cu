// Softmax attention of many query rows (prompt slices) over the 8-bit KV cache, on the tensor cores' TMEM path.
//
// The mathematics and its roundings are those of kv8_attend.cu: with t_j the score of key j in log2 units and
// u_j = t_j + log2 scale_v[j], weights w_j = 2^(u_j - M) in f16, y = sum w_j v8_j / sum (w_j / scale_v[j]). The int8 keys
// are exact in bf16, so the scores are products of the queries as they are; the int8 values are exact in f16.
//
// Bound by arithmetic: 4 HD operations per (query row, key), and one exponential. A CTA holds two tiles of 128 query
// rows (T * G rows of one KV head, token-major) and walks the keys in blocks of 128, so that a block is widened from
// int8 once for 256 rows. Roles, which meet only at mbarriers:
// - warps 16-19 widen keys, 20-23 values: global int8 -> registers (a block ahead) -> operand tiles in shared memory
//   (two stages each); the latter also prepare the block's scales;
// - one lane of warp 24 issues tcgen05.mma: S = Q K^T into TMEM, O += P V with P as the TMEM operand;
// - warps 0-7 and 8-15 are the softmax of a tile, 64 keys at a time: scores out of TMEM, weights back over them, fp32
//   arithmetic in packed pairs. A warp takes 16 TMEM lanes in the 16x256b layout, a thread 16 of the 64 keys of two rows:
//   what belongs to a key (its scales) is then read from shared memory once for two rows, where a thread per row, all
//   lanes reading the same address, took twice the shared-memory time of the MMAs; and with four such warps on a
//   scheduler one's latencies are filled by the others. The bound M moves only when a weight would pass 2^15; only then
//   are the sums in TMEM rescaled.
// While one tile's softmax runs, the tensor cores work on the other tile. With few heads the keys are split over CTAs,
// whose partial sums a second kernel joins.
//
// Measured on a B200: 64 x 128 tokens after 2048, 32 heads on 8 of 128, 370 to 385 us by the clock under load (0.77 to
// 0.74 PFLOP/s; 173 us at the machine's bf16 rate). A CTA is ready for its first scores after 6000 cycles, takes 5100 for a block of 128 keys (the MMAs of its
// two tiles 2048, their exponentials 2048) and 3700 for its output. The softmax warps bound it: 64 keys take them about
// 1900 cycles, the four of a scheduler issuing half of the time, at 72 to 80 registers with little to overlap within a
// warp. (Scores are waited for 900 cycles of a block, but bringing them earlier, 64 keys at a time into the columns that
// the other 64 have left, took 380 us.)
#include "../../include/bolt3.h"
#include "kv8.cuh"
#include "kv8_prompt.cuh"
#include "tc5.cuh"
#include "trace.h"

namespace {

using namespace b3;
using namespace kv8;

constexpr int kKeys = 128;                       // of a block
constexpr int kThreads = 896;                    // 16 softmax warps, 4 + 4 widening warps, 1 issuing warp (of 4)
// registers of a thread by role, out of the 72 that each of the 896 is launched with: 4 * 80 + 64 + 64 + 56 = 7 * 72
constexpr int kRegsSoftmax = 80, kRegsWiden = 64, kRegsIssue = 56;
template <int N>
B3_DEV void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
B3_DEV void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }
constexpr uint32_t kWaitIters = 1u << 24;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  bolt3_kv8_attend_args a;
  Length len;
  int G, rows, tiles, splits;                    // tiles: pairs of 128 rows of a head
  uint32_t per_G;                                // ceil(2^32 / G), 0 for G = 1
  float* part;                                   // [head][row][split][HD] sums, then [..] (bound, sum of weights)
  float2* part_ml;
};

template <int HD>
struct Smem {
  unsigned char q[2][kKeys * HD * 2];            // K-major operand tiles: HD / 64 blocks of [128 rows][64 columns]
  unsigned char k[2][kKeys * HD * 2];
  unsigned char v[2][kKeys * HD * 2];
  float scale[2][3][kKeys];                      // key scale (times sm_scale log2(e)), log2 and
                                                 // reciprocal of the value scale
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2][2], pv_half[2], o_full[2];
  uint32_t tbase;
  int err;
};

// the token of a query row (exact for rows below 2^28)
B3_DEV int token_of(const Params& p, int row) { return p.per_G == 0 ? row : (int)__umulhi((uint32_t)row, p.per_G); }

B3_DEV float ex2(float x) {
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
B3_DEV uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// two fp32 at a time
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

// 64 columns of 16 TMEM lanes: a thread gets columns 8 n + 2 (lane % 4) and the next one of lanes lane / 4 (registers
// 4 n, 4 n + 1) and lane / 4 + 8 (4 n + 2, 4 n + 3)
B3_DEV void ld_16x64(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// 32 columns of 16 TMEM lanes: column 4 n + lane % 4 of lanes lane / 4 (register 2 n) and lane / 4 + 8 (2 n + 1)
B3_DEV void st_16x32(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}

// the layout of ld_16x64, 32 columns
B3_DEV void ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
B3_DEV void st_16x32f(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}

// 16 int8, keys as bf16, values as f16, to a row's 16-byte chunks 2 c and 2 c + 1 (the address of the first, swizzled; the
// other one is beside it)
template <bool KEYS>
B3_DEV void widen16(unsigned char* at, const uint4& x) {
  auto widen = [](uint32_t w, uint32_t& lo, uint32_t& hi) { KEYS ? s8x4_to_bf16(w, lo, hi) : s8x4_to_f16(w, lo, hi); };
  uint4 lo, hi;
  widen(x.x, lo.x, lo.y);
  widen(x.y, lo.z, lo.w);
  widen(x.z, hi.x, hi.y);
  widen(x.w, hi.z, hi.w);
  *reinterpret_cast<uint4*>(at) = lo;
  *reinterpret_cast<uint4*>((uintptr_t)at ^ 16) = hi;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>(smem_raw + ((1024 - (tc5::smem_u32(smem_raw) & 1023)) & 1023));
  const bolt3_kv8_attend_args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x / p.tiles, b = head / a.HKV, kvh = head % a.HKV;
  const int row0 = (blockIdx.x % p.tiles) * 256, n_tile = min(2, (p.rows - row0 + 127) / 128);
  const int split = blockIdx.y;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(&sm.k_full[i], 128);
      tc5::mbar_init(&sm.k_empty[i], 1);
      tc5::mbar_init(&sm.v_full[i], 128);
      tc5::mbar_init(&sm.v_empty[i], 1);
      tc5::mbar_init(&sm.s_full[i], 1);
      tc5::mbar_init(&sm.p_full[i][0], 256);
      tc5::mbar_init(&sm.p_full[i][1], 256);
      tc5::mbar_init(&sm.pv_half[i], 1);
      tc5::mbar_init(&sm.o_full[i], 1);
    }
    tc5::mbar_fence_init();
    sm.err = 0;
  }
  grid_dep_launch();
  grid_dep_wait();
  bool bad = false;
  const int64_t s = p.len.rows(b, bad);
  if (bad && tid == 0 && blockIdx.x % p.tiles == 0 && split == 0 && a.status) atomicOr(a.status, 8);
  auto out_row = [&](int row) {
    const int t = token_of(p, row), g = row - t * p.G;
    return reinterpret_cast<bf16*>(a.y) + ((int64_t)b * a.T * a.H + kvh * p.G) * HD + (int64_t)t * (a.H * HD) + g * HD;
  };
  // blocks of keys that the last row of this CTA sees, and this split's share of them
  const int last = token_of(p, min(row0 + 256, p.rows) - 1);
  const int64_t all = s < 0 ? 0 : (s + last + kKeys) / kKeys;
  const int64_t lo = all * split / p.splits, hi = all * (split + 1) / p.splits;
  const int n_blk = (int)(hi - lo);
  if (n_blk == 0) {                              // the same for all threads: nothing has been allocated
    if (tid < 256 && row0 + tid < p.rows) {
      if (p.splits > 1) {
        const int64_t at = ((int64_t)head * p.rows + row0 + tid) * p.splits + split;
        p.part_ml[at] = make_float2(neg_inf(), 0.f);
      } else {
        uint4* y = reinterpret_cast<uint4*>(out_row(row0 + tid));
        for (int i = 0; i < HD / 8; ++i) y[i] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }

  // the query rows into their operand tiles; the other warps are at their first loads meanwhile
  if (warp < 16) {
    constexpr int CPR = HD / 8, RPW = 32 / CPR;                   // 16-byte chunks of a row, rows of a warp's instruction
    const int c = lane % CPR;
    const bf16* q = reinterpret_cast<const bf16*>(a.q) + b * a.q_sb + (int64_t)(kvh * p.G) * HD + 8 * c;
#pragma unroll
    for (int i = 0; i < 16 / RPW; ++i) {
      const int r = warp * 16 + lane / CPR + i * RPW, t = token_of(p, row0 + r), g = row0 + r - t * p.G;
      const bool in = row0 + r < p.rows;
      cp_async16(sm.q[0] + (r >> 7) * sizeof(sm.q[0]) + (c >> 3) * (kKeys * 128) + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
                 in ? q + t * a.q_st + g * HD : q, in);
    }
    asm volatile("cp.async.wait_all;\nfence.proxy.async.shared::cta;\n" ::: "memory");
  }
  if (warp == 24) {
    tc5::tmem_alloc(&sm.tbase, 512);
    tc5::tmem_relinquish();
  }
  // every warp comes here once: the queries are in place, the barriers and the TMEM are there
  auto all_ready = [&] {
    tc5::fence_before_sync();
    asm volatile("bar.sync 0;\n" ::: "memory");
    tc5::fence_after_sync();
    return sm.tbase;                             // S / P of tile i: columns 128 i; O of tile i: 256 + 128 i
  };
  auto wait = [&](uint64_t* bar, int phase) {
    if (tc5::mbar_wait(bar, (uint32_t)phase & 1, kWaitIters)) return true;
    sm.err = 1;
    return false;
  };

  if (warp >= 16 && warp < 24) {
    // ---- widening: keys, or values and scales
    fewer_regs<kRegsWiden>();
    // piece i of thread t: 16 bytes t % 4 (+ 4 for odd i at HD 128) of row t / 4 + 32 (i / KC). The eight lanes of a phase
    // of a store then hold two neighbouring rows' chunks of one column block: all banks differ
    constexpr int KC = HD / 64, NP = 4 * KC;
    const bool values = warp >= 20;
    const int t = tid & 127, r0 = t >> 2;
    const int64_t side = (int64_t)a.B * a.HKV * a.cap;
    const int8_t* base = a.data + ((int64_t)head * a.cap + (values ? side : 0) + lo * kKeys) * HD + 16 * (t & 3);
    const float* ks = a.scale + (int64_t)head * a.cap + lo * kKeys + t;
    const int end = (int)min(a.cap - 1 - lo * kKeys, (int64_t)0x7fffff00);   // the buffer's last row
    uint64_t *full = values ? sm.v_full : sm.k_full, *empty = values ? sm.v_empty : sm.k_empty;
    unsigned char* out = (values ? sm.v[0] : sm.k[0]) + r0 * 128 + (((2 * (t & 3)) ^ (r0 & 7)) << 4);
    uint4 x[NP];
    float k_sc = 0.f, v_sc = 0.f;
    auto fetch = [&](int j) {
      if (j * kKeys + kKeys - 1 <= end) {
        const int8_t* src = base + ((int64_t)j * kKeys + r0) * HD;
#pragma unroll
        for (int i = 0; i < NP; ++i) x[i] = __ldg(reinterpret_cast<const uint4*>(src + 32 * (i / KC) * HD + 64 * (i % KC)));
        if (values) {
          k_sc = __ldg(ks + j * kKeys);
          v_sc = __ldg(ks + side + j * kKeys);
        }
      } else {                                                    // rows past the buffer are read as its last one and masked
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int row = min(j * kKeys + r0 + 32 * (i / KC), end);
          x[i] = __ldg(reinterpret_cast<const uint4*>(base + (int64_t)row * HD + 64 * (i % KC)));
        }
        if (values) {
          const int row = min(j * kKeys + t, end) - t;
          k_sc = __ldg(ks + row);
          v_sc = __ldg(ks + side + row);
        }
      }
    };
    fetch(0);
    all_ready();
    const float c_all = a.sm_scale * kLog2e;                      // into the key scales
    for (int j = 0; j < n_blk; ++j) {
      const int st = j & 1;
      if (j >= 2 && !wait(&empty[st], (j >> 1) - 1)) break;
      unsigned char* to = out + st * sizeof(sm.k[0]);
      auto at = [&](int i) { return to + (i % KC) * (kKeys * 128) + 32 * (i / KC) * 128; };
      if (!values) {
#pragma unroll
        for (int i = 0; i < NP; ++i) widen16<true>(at(i), x[i]);
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) widen16<false>(at(i), x[i]);
        sm.scale[st][0][t] = k_sc * c_all;
        sm.scale[st][1][t] = lg2(v_sc);
        sm.scale[st][2][t] = rcp(v_sc);
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      tc5::mbar_arrive(&full[st]);
      if (j + 1 < n_blk) fetch(j + 1);
    }
  } else if (warp >= 24) {
    // ---- issue. The whole warp runs the loop, so that addresses and descriptors are uniform over it (a lone thread in a
    // branch of its own needed 170 cycles an MMA for moving them to where the instruction takes them); one lane issues
    fewer_regs<kRegsIssue>();
    const uint32_t tb = all_ready();
    if (warp == 24) {
      uint32_t one;
      asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
      constexpr uint32_t kIdS = tc5::idesc_bf16(128, kKeys, false, false), kIdO = tc5::idesc_f16(128, HD, false, true);
      constexpr uint64_t kTile = sizeof(sm.q[0]) >> 4;            // from one tile's descriptor to the next one's
      const uint32_t tu = __shfl_sync(0xffffffffu, tb, 0);
      const uint64_t q_desc = tc5::sdesc(tc5::smem_u32(sm.q[0]), 16, 1024), k_desc = tc5::sdesc(tc5::smem_u32(sm.k[0]), 16, 1024);
      const uint64_t v_desc = tc5::sdesc(tc5::smem_u32(sm.v[0]), kKeys * 128, 1024);
      auto scores = [&](int i, int st) {
        const uint64_t qd = q_desc + i * kTile, kd = k_desc + st * kTile;
        if (one) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            constexpr uint64_t kBlock = (kKeys * 128) >> 4;       // a block of 64 columns
            tc5::mma_ss(tu + i * 128, qd + (ks >> 2) * kBlock + (ks & 3) * 2, kd + (ks >> 2) * kBlock + (ks & 3) * 2, kIdS, ks > 0);
          }
          tc5::commit(&sm.s_full[i]);
        }
      };
      auto product = [&](int i, int st, int h, bool first) {
        const uint64_t vd = v_desc + st * kTile + 4 * h * 128;
        const uint32_t d = tu + 256 + i * 128, pa = tu + i * 128 + 32 * h;
        if (one) {
          tc5::mma_ts(d, pa, vd, kIdO, !first);
          tc5::mma_ts(d, pa + 8, vd + 128, kIdO, 1);
          tc5::mma_ts(d, pa + 16, vd + 256, kIdO, 1);
          tc5::mma_ts(d, pa + 24, vd + 384, kIdO, 1);
        }
      };
      auto wait_all = [&](uint64_t* bar, int phase) { return __all_sync(0xffffffffu, wait(bar, phase)) != 0; };
      bool ok = wait_all(&sm.k_full[0], 0);
      if (ok) {
        tc5::fence_after_sync();
        for (int i = 0; i < n_tile; ++i) scores(i, 0);
        if (one) tc5::commit(&sm.k_empty[0]);
      }
      for (int j = 0; ok && j < n_blk; ++j) {
        const int st = j & 1;
        ok = wait_all(&sm.v_full[st], j >> 1);
        for (int i = 0; ok && i < n_tile; ++i) {
          ok = wait_all(&sm.p_full[i][0], j);
          if (!ok) break;
          tc5::fence_after_sync();
          product(i, st, 0, j == 0);
          if (one) tc5::commit(&sm.pv_half[i]);
          ok = wait_all(&sm.p_full[i][1], j);
          if (!ok) break;
          tc5::fence_after_sync();
          product(i, st, 1, false);
          if (j + 1 == n_blk) {
            if (one) tc5::commit(&sm.o_full[i]);
          } else {
            if (i == 0) ok = wait_all(&sm.k_full[st ^ 1], (j + 1) >> 1);
            if (!ok) break;
            tc5::fence_after_sync();
            scores(i, st ^ 1);
          }
        }
        if (ok && one) {
          tc5::commit(&sm.v_empty[st]);
          if (j + 1 < n_blk) tc5::commit(&sm.k_empty[st ^ 1]);
        }
      }
    }
  } else {
    const uint32_t tb = all_ready();
    more_regs<kRegsSoftmax>();
    if ((warp >> 3) < n_tile) {
    // ---- softmax of tile i: this thread's two rows are those of TMEM lanes first_lane + grp and + grp + 8
    const int i = warp >> 3, grp = lane >> 2, tig = lane & 3;
    const int first_lane = 32 * (warp & 3) + 16 * (warp >> 2 & 1), first_row = row0 + 128 * i + first_lane + grp;
    const uint32_t lanes = (uint32_t)first_lane << 16, ts = tb + i * 128 + lanes, to = tb + 256 + i * 128 + lanes;
    const int seen = (int)min(s + 1 - lo * kKeys, (int64_t)0x7fffff00);           // keys of this split that token 0 sees
    const int see_all = seen + token_of(p, row0 + i * 128);                          // that every row of the tile sees
    float M[2] = {neg_inf(), neg_inf()};
    uint64_t l[2] = {0, 0};                                       // sums of weights over this thread's keys, in pairs
    bool ok = true;
    for (int j = 0; ok && j < n_blk; ++j) {
      const int st = j & 1;
      ok = wait(&sm.v_full[st], j >> 1);                          // the scales
      ok = ok && wait(&sm.s_full[i], j);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc5::fence_after_sync();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t sc[32];
        ld_16x64(ts + 64 * h, sc);
        const float* ks = sm.scale[st][0] + 64 * h + 2 * tig;
        const float* lg = sm.scale[st][1] + 64 * h + 2 * tig;
        const float* iv = sm.scale[st][2] + 64 * h + 2 * tig;
        const int key = j * kKeys + 64 * h;
        float2 t[2][8];                                           // row q, keys 8 n + 2 tig and the next
        tc5::ld_wait();
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const uint64_t k2 = *reinterpret_cast<const uint64_t*>(ks + 8 * n), g2 = *reinterpret_cast<const uint64_t*>(lg + 8 * n);
#pragma unroll
          for (int q = 0; q < 2; ++q)
            t[q][n] = unpair(fma2(pair(__uint_as_float(sc[4 * n + 2 * q]), __uint_as_float(sc[4 * n + 2 * q + 1])), k2, g2));
        }
        const bool masked = key + 64 > see_all;                   // the same for the whole tile
        if (masked) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int r = min(first_row + 8 * q, p.rows - 1);
            const int left = seen + token_of(p, r) - key - 2 * tig;   // seen, from this thread's first
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              if (8 * n >= left) t[q][n].x = neg_inf();
              if (8 * n + 1 >= left) t[q][n].y = neg_inf();
            }
          }
        }
        // the bounds move only when a weight would pass 2^15 (and at the first key)
        float m[2];
        bool over = false;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          m[q] = fmaxf(t[q][0].x, t[q][0].y);
#pragma unroll
          for (int n = 1; n < 8; ++n) m[q] = max3(m[q], t[q][n].x, t[q][n].y);
          over |= m[q] > M[q] + kMostWeight;
        }
        if (__any_sync(0xffffffffu, over)) {
          float f[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            m[q] = quad_max(m[q]);
            const float to_M = m[q] > M[q] + kMostWeight ? m[q] - kHeadroom : M[q];
            f[q] = M[q] == neg_inf() ? 0.f : ex2(M[q] - to_M);    // 1 where the bound stays
            M[q] = to_M;
            l[q] = mul2(l[q], pair(f[q], f[q]));
          }
          if (j > 0 || h > 0) {
            if (h > 0) {                                          // the first half's product may still be under way
              ok = __all_sync(0xffffffffu, wait(&sm.pv_half[i], j));
              tc5::fence_after_sync();
            }
            if (ok) {
#pragma unroll 1
              for (int d = 0; d < HD; d += 32) {
                uint32_t o[16];
                ld_16x32(to + d, o);
                tc5::ld_wait();
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f[x >> 1 & 1]);
                st_16x32f(to + d, o);
              }
              tc5::st_wait();
            }
          }
        }
        uint32_t w[16];
        if (masked) {                                             // an unseen key has weight 0, whatever its scale holds
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float ref = M[q] == neg_inf() ? 0.f : M[q];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const float e0 = ex2(t[q][n].x - ref), e1 = ex2(t[q][n].y - ref);
              l[q] = add2(l[q], pair(e0 == 0.f ? 0.f : e0 * iv[8 * n], e1 == 0.f ? 0.f : e1 * iv[8 * n + 1]));
              w[2 * n + q] = pack_f16(e0, e1);
            }
          }
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const uint64_t i2 = *reinterpret_cast<const uint64_t*>(iv + 8 * n);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const float2 u = unpair(add2(pair(t[q][n].x, t[q][n].y), pair(-M[q], -M[q])));
              const float e0 = ex2(u.x), e1 = ex2(u.y);
              l[q] = fma2(pair(e0, e1), i2, l[q]);
              w[2 * n + q] = pack_f16(e0, e1);
            }
          }
        }
        st_16x32(ts + 32 * h, w);
        tc5::st_wait();
        tc5::fence_before_sync();
        tc5::mbar_arrive(&sm.p_full[i][h]);
      }
    }
    float sum[2], inv[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float2 x = unpair(l[q]);
      sum[q] = quad_sum(x.x + x.y);
      inv[q] = sum[q] == 0.f ? 0.f : 1.f / sum[q];
    }
    ok = ok && wait(&sm.o_full[i], 0);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc5::fence_after_sync();
      // bf16 rows by way of this warp's sixteen rows of the query tile, whose products are done: whole rows to a store (4 bytes
      // of 8 rows to a store took 5000 cycles)
      unsigned char* out = sm.q[i] + first_lane * HD * 2;
#pragma unroll 1
      for (int d = 0; d < HD; d += 32) {
        uint32_t o[16];
        ld_16x32(to + d, o);
        tc5::ld_wait();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (p.splits > 1) {
            const int row = first_row + 8 * q;
            float* dst = p.part + (((int64_t)head * p.rows + row) * p.splits + split) * HD + d + 2 * tig;
#pragma unroll
            for (int n = 0; n < 4; ++n)
              if (row < p.rows) *reinterpret_cast<uint2*>(dst + 8 * n) = make_uint2(o[4 * n + 2 * q], o[4 * n + 2 * q + 1]);
          } else {
#pragma unroll
            for (int n = 0; n < 4; ++n)
              *reinterpret_cast<uint32_t*>(out + (grp + 8 * q) * HD * 2 + (((d / 8 + n) ^ grp) << 4) + 4 * tig) =
                  pack_bf16(__uint_as_float(o[4 * n + 2 * q]) * inv[q], __uint_as_float(o[4 * n + 2 * q + 1]) * inv[q]);
          }
        }
      }
      if (p.splits == 1) {
        constexpr int CPR = HD / 8, RPW = 32 / CPR;
        const int c = lane % CPR;
        __syncwarp();
#pragma unroll
        for (int r = lane / CPR; r < 16; r += RPW) {
          const int row = row0 + 128 * i + first_lane + r;
          if (row < p.rows) reinterpret_cast<uint4*>(out_row(row))[c] = *reinterpret_cast<uint4*>(out + r * HD * 2 + ((c ^ (r & 7)) << 4));
        }
      }
      if (p.splits > 1 && tig == 0) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (first_row + 8 * q < p.rows)
            p.part_ml[((int64_t)head * p.rows + first_row + 8 * q) * p.splits + split] = make_float2(M[q], sum[q]);
      }
    }
    }
  }
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  if (warp == 24) tc5::tmem_dealloc(sm.tbase, 512);
  if (tid == 0 && sm.err && a.status) atomicOr(a.status, 2);
}

// one warp per (head, query row): the splits' partial sums joined
template <int HD>
__global__ void __launch_bounds__(128) kv8_prompt_join_kernel(const __grid_constant__ Params p) {
  constexpr int EPL = HD / 32;
  const bolt3_kv8_attend_args& a = p.a;
  const int lane = threadIdx.x & 31;
  grid_dep_launch();
  grid_dep_wait();
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (int64_t)a.B * a.HKV * p.rows) return;
  const int head = (int)(item / p.rows), row = (int)(item % p.rows), b = head / a.HKV, kvh = head % a.HKV;
  const int64_t at = item * p.splits;
  float m = neg_inf(), l = 0.f, acc[EPL] = {};
  for (int i = 0; i < p.splits; ++i) m = fmaxf(m, p.part_ml[at + i].x);
  for (int i = 0; i < p.splits; ++i) {
    const float2 ml = p.part_ml[at + i];
    if (ml.x == neg_inf() && ml.y == 0.f) continue;               // no keys: its sums were not written
    const float f = ml.x == neg_inf() ? 0.f : exp2f(ml.x - m);
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = fmaf(p.part[(at + i) * HD + 32 * e + lane], f, acc[e]);
  }
  bf16* y = reinterpret_cast<bf16*>(a.y) + (((int64_t)b * a.T + row / p.G) * a.H + kvh * p.G + row % p.G) * HD;
#pragma unroll
  for (int e = 0; e < EPL; ++e) y[32 * e + lane] = __float2bfloat16_rn(l == 0.f ? 0.f : acc[e] / l);
}

struct Plan {
  int tiles, splits;
  size_t bytes;
};

Plan plan_of(int B, int T, int H, int HKV, int HD, int64_t n) {
  Plan pl;
  const int64_t rows = (int64_t)T * (H / HKV), heads = (int64_t)B * HKV;
  pl.tiles = (int)((rows + 255) / 256);
  // as many splits as fill the machine, of four blocks or more
  int64_t splits = 148 / (heads * pl.tiles);
  const int64_t most = (n + T + kKeys - 1) / kKeys / 4;
  if (splits > most) splits = most;
  pl.splits = splits < 1 ? 1 : (int)splits;
  pl.bytes = pl.splits > 1 ? (size_t)heads * (size_t)rows * (size_t)pl.splits * ((size_t)HD * 4 + 8) : 0;
  return pl;
}

template <int HD>
int launch(Params& p, const Plan& pl, cudaStream_t s) {
  const size_t smem = sizeof(Smem<HD>) + 1024;
  if (cudaFuncSetAttribute(kv8_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  const int64_t heads = (int64_t)p.a.B * p.a.HKV;
  p.part = reinterpret_cast<float*>(p.a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part + (size_t)heads * p.rows * pl.splits * HD);
  if (launch_overlapped(kv8_prompt_kernel<HD>, dim3((unsigned)(heads * pl.tiles), (unsigned)pl.splits), dim3(kThreads), smem, s,
                        p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  if (pl.splits > 1 && launch_overlapped(kv8_prompt_join_kernel<HD>, dim3((unsigned)((heads * p.rows + 3) / 4)), dim3(128), 0, s,
                                         p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  return BOLT3_OK;
}

}  // namespace

size_t kv8_prompt_workspace(int B, int T, int H, int HKV, int HD, int64_t n) { return plan_of(B, T, H, HKV, HD, n).bytes; }

int kv8_prompt_launch(const bolt3_kv8_attend_args* a, const Length& len, cudaStream_t s) {
  const Plan pl = plan_of(a->B, a->T, a->H, a->HKV, a->HD, a->n);
  if (pl.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < pl.bytes)) return BOLT3_ERR_CAPACITY;
  if ((int64_t)a->B * a->HKV * pl.tiles > 0x7fffffff) return BOLT3_ERR_SHAPE;
  Params p;
  p.a = *a;
  p.len = len;
  p.G = a->H / a->HKV;
  p.per_G = p.G == 1 ? 0 : 0xffffffffu / p.G + 1;
  p.rows = a->T * p.G;
  p.tiles = pl.tiles;
  p.splits = pl.splits;
  return a->HD == 128 ? launch<128>(p, pl, s) : launch<64>(p, pl, s);
}
