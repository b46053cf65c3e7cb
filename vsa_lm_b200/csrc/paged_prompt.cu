// Softmax attention of many query rows (prompt slices) over the pages of a bf16 KV cache, on the tensor cores' TMEM path,
// and the record of the weights that the cached rows got.
//
// The mathematics is that of paged_attend.cu, with weights rounded to bf16 for the product with the values.
//
// attend. Bound by arithmetic: 4 HD operations per (query row, key), and one exponential; at HD 128 the MMAs of a block of 128
// keys by 256 rows take 2048 cycles of an SM, its exponentials 2048. A CTA holds two tiles of 128 query rows (T * G rows of one
// KV head, token-major) and walks the keys in blocks of 128. Roles, which meet only at mbarriers:
// - warp 16 brings keys and values by TMA, a box for each page that a block touches, two stages each;
// - one lane of warps 17 and 18 issues a tile's tcgen05.mma: S = Q K^T into TMEM, O += P V with P as the TMEM operand, 64 keys
//   at a time: once a half's weights have been used, the next block's scores of that half are on their way, while the softmax is
//   at the other half;
// - warp 19 clears the value rows of the last block that no query row of the CTA sees (a page's unused rows may hold
//   anything, and 0 times a NaN is one);
// - warps 0-7 and 8-15 are the softmax of a tile, 64 keys at a time: scores out of TMEM, weights back over them. A warp takes
//   16 TMEM lanes in the 16x256b layout, so that a row's reference is shared by a quad of lanes alone. The reference moves only
//   when a weight would pass 2^kMost; only then are the sums in TMEM rescaled.
// With few heads the keys are split over CTAs, whose
// partial sums a second kernel joins.
//
// record. A key's weight needs the rows' sums over all keys, so the scores are computed again once these are known, this time
// with the keys in the TMEM lanes: S^T = K Q^T, a thread per key, which sums 2^(t - lse) over the query columns in registers; no
// two threads add to one record, whatever the split. A CTA holds up to 512 query rows of a head and walks a range of its keys.
// Bound by the exponentials: 4096 cycles of an SM for 128 keys by 512 rows, against 2048 of its MMAs; a quarter of them are
// polynomials on the FMA pipes (16 sequences of 128 tokens after 2048, 8 heads, with the attention: 132 us, with none 137, with three
// eighths 134, half 140).
#include <type_traits>

#include "paged.cuh"
#include "tc5.cuh"
#include "trace.h"

namespace {

using namespace paged;

constexpr int kKeys = 128;                       // of a block
constexpr float kMost = 20.f;                    // log2 of the largest weight relative to the reference
constexpr int kThreads = 640;                    // 16 softmax warps, loads, MMAs of either tile, clearing
constexpr int kRows = 512;                       // query rows of a CTA of the record kernel
constexpr int kRecordThreads = 576;              // 16 summing warps, loads, MMAs

struct Params {
  CUtensorMap map;                               // the pool's rows, boxes of 64 columns and a page
  Attend c;
  int tiles, splits;                             // tiles: pairs of 128 rows of a head
  uint32_t per_G;                                // ceil(2^32 / G), 0 for G = 1
  float* part;                                   // [head][row][split][HD] sums, then [..] (reference, sum of weights)
  float2* part_ml;
  float* lse;                                    // [head][row] log2 of the sum of 2^t, +inf for an idle sequence; null: no record
  int ranges;                                    // of keys of a head, each a CTA of the record kernel
};

template <int HD>
struct Smem {
  unsigned char q[2][kKeys * HD * 2];            // K-major operand tiles: HD / 64 blocks of [128 rows][64 columns]
  unsigned char k[2][kKeys * HD * 2];
  unsigned char v[2][kKeys * HD * 2];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], v_last, v_clean;
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], o_full[2];    // of a tile, of a half of its keys
  uint32_t tbase;
  int err;
};

template <int HD>
struct RecordSmem {
  unsigned char q[kRows / kKeys][kKeys * HD * 2];
  unsigned char k[2][kKeys * HD * 2];
  float lse[2][kRows];                           // of even groups of rows, of odd ones
  int token[2][kRows];
  float sum[4][kRows / kKeys][kKeys];            // of a block's keys, of each tile's rows
  uint64_t k_full[2], k_empty[2], s_full[kRows / kKeys], s_empty[kRows / kKeys], sum_full[4][kRows / kKeys];
  uint32_t tbase;
  int err;
};

// the token of a query row (exact for rows below 2^28)
B3_DEV int token_of(const Params& p, int row) { return p.per_G == 0 ? row : (int)__umulhi((uint32_t)row, p.per_G); }

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
// All threads of the CTA meet. bar.sync in a string is the aligned form, which takes a warp's first lanes to arrive for the
// whole warp, and the compiler does not bring a warp together for it that parted before (a page looked up by some lanes): the
// others then went on before the tensor memory was there
B3_DEV void meet_all() {
  __syncwarp();
  asm volatile("barrier.sync 0;\n" ::: "memory");
  __syncwarp();
}
// 2^x of two numbers without the MUFU, relative error 2^-22.6: the nearest integer by adding 1.5 2^23, in whose low bits it then
// stands, and a polynomial for the rest, in [-1/2, 1/2] (degree 5 with 1 at 0, its largest relative error the
// smallest, fitted anew for every coefficient after those before it were rounded to fp32: 2^-23.3). From -127 down, and so for a
// row past the last, 0, as by the MUFU: the exponent bits of 2^-127 are those of 0; a NaN stays one
B3_DEV float2 ex2_fma(float2 x) {
  asm("max.NaN.f32 %0, %0, %1;\n" : "+f"(x.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;\n" : "+f"(x.y) : "f"(-127.f));
  const uint64_t v = pair(x.x, x.y), r = add2(v, pair(12582912.f, 12582912.f));
  const uint64_t f = fma2(add2(r, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), v);
  uint64_t y = pair(0.00132695551f, 0.00132695551f);
  y = fma2(y, f, pair(0.0096712932f, 0.0096712932f));
  y = fma2(y, f, pair(0.0555071086f, 0.0555071086f));
  y = fma2(y, f, pair(0.240222469f, 0.240222469f));
  y = fma2(y, f, pair(0.693147004f, 0.693147004f));
  y = fma2(y, f, pair(1.f, 1.f));
  const float2 n = unpair(r);
  return unpair(mul2(y, pair(__int_as_float((__float_as_int(n.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(n.y) << 23) + 0x3f800000))));
}
B3_DEV bool elected() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

// query rows row0 + r0 .. of head (b, kvh) into K-major operand tiles, 16 rows by each of the calling warps (r0 = 16 warp)
template <int HD>
B3_DEV void copy_queries(const Params& p, unsigned char* tiles, int b, int kvh, int row0, int r0, int lane) {
  constexpr int CPR = HD / 8, RPW = 32 / CPR;                     // 16-byte chunks of a row, rows of a warp's instruction
  const bolt3_paged_attend_args& a = p.c.a;
  const int c = lane % CPR;
  const bf16* q = reinterpret_cast<const bf16*>(a.q) + b * a.q_sb + (int64_t)(kvh * p.c.G) * HD + 8 * c;
#pragma unroll
  for (int i = 0; i < 16 / RPW; ++i) {
    const int r = r0 + lane / CPR + i * RPW, t = token_of(p, row0 + r), g = row0 + r - t * p.c.G;
    const bool in = row0 + r < p.c.rows;
    cp_async16(tiles + (r >> 7) * (kKeys * HD * 2) + (c >> 3) * (kKeys * 128) + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
               in ? q + t * a.q_st + (int64_t)g * HD : q, in);
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>(smem_raw + ((1024 - (tc5::smem_u32(smem_raw) & 1023)) & 1023));
  const bolt3_paged_attend_args& a = p.c.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x / p.tiles, b = head / a.HKV, kvh = head % a.HKV;
  const int row0 = (blockIdx.x % p.tiles) * 256, n_tile = min(2, (p.c.rows - row0 + 127) / 128);
  const int split = blockIdx.y;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(&sm.k_full[i], 1);
      tc5::mbar_init(&sm.k_empty[i], n_tile);
      tc5::mbar_init(&sm.v_full[i], 1);
      tc5::mbar_init(&sm.v_empty[i], n_tile);
      for (int h = 0; h < 2; ++h) {
        tc5::mbar_init(&sm.s_full[i][h], 1);
        tc5::mbar_init(&sm.p_full[i][h], 256);
        tc5::mbar_init(&sm.pv_done[i][h], 1);
      }
      tc5::mbar_init(&sm.o_full[i], 1);
    }
    tc5::mbar_init(&sm.v_last, 1);
    tc5::mbar_init(&sm.v_clean, 32);
    tc5::mbar_fence_init();
    sm.err = 0;
  }
  meet_all();                                    // the barriers are there: loads may begin
  grid_dep_wait();
  bool bad = false;
  const int64_t s = p.c.len.rows(b, bad);
  if (bad && tid == 0 && blockIdx.x % p.tiles == 0 && split == 0 && a.status) atomicOr(a.status, 8);
  auto out_row = [&](int row) {
    const int t = token_of(p, row), g = row - t * p.c.G;
    return reinterpret_cast<bf16*>(a.y) + ((int64_t)b * a.T * a.H + kvh * p.c.G) * HD + (int64_t)t * (a.H * HD) + g * HD;
  };
  // blocks of keys that the last row of this CTA sees, and this split's share of them
  const int last = token_of(p, min(row0 + 256, p.c.rows) - 1);
  const int64_t all = s < 0 ? 0 : (s + last + kKeys) / kKeys;
  const int64_t lo = all * split / p.splits, hi = all * (split + 1) / p.splits;
  const int n_blk = (int)(hi - lo);
  if (n_blk == 0) {                              // the same for all threads: nothing has been allocated
    if (tid < 256 && row0 + tid < p.c.rows) {
      const int64_t row = (int64_t)head * p.c.rows + row0 + tid;
      if (p.splits > 1) {
        p.part_ml[row * p.splits + split] = make_float2(neg_inf(), 0.f);
      } else {
        uint4* y = reinterpret_cast<uint4*>(out_row(row0 + tid));
        for (int i = 0; i < HD / 8; ++i) y[i] = make_uint4(0, 0, 0, 0);
        if (p.lse != nullptr) p.lse[row] = -neg_inf();
      }
    }
    return;
  }
  const int seen = (int)min(s + 1 - lo * kKeys, (int64_t)0x7fffff00);             // keys of this split that token 0 sees
  const int seen_last = (int)min(s + 1 + last - lo * kKeys, (int64_t)0x7fffff00);   // that the CTA's last row sees
  const bool ragged = seen_last < n_blk * kKeys;  // the last block ends with rows that no row sees

  // the query rows into their operand tiles; the first loads are under way meanwhile
  if (warp < 16) {
    copy_queries<HD>(p, sm.q[0], b, kvh, row0, warp * 16, lane);
    asm volatile("cp.async.wait_all;\nfence.proxy.async.shared::cta;\n" ::: "memory");
  }
  if (warp == 17) {
    tc5::tmem_alloc(&sm.tbase, 512);
    tc5::tmem_relinquish();
    grid_dep_launch();                           // here alone, for the whole CTA (common.cuh)
  }
  // every warp comes here once: the queries are in place, the TMEM is there
  auto all_ready = [&] {
    tc5::fence_before_sync();
    meet_all();
    tc5::fence_after_sync();
    return sm.tbase;                             // S of tile i: columns 128 i, weights of a half over its first 32; O of tile i: 256 + 128 i
  };
  auto wait = [&](uint64_t* bar, int phase) {
    if (tc5::mbar_wait(bar, (uint32_t)phase & 1, kWaitIters)) return true;
    sm.err = 1;
    return false;
  };
  auto wait_all = [&](uint64_t* bar, int phase) {
    const bool ok = __all_sync(0xffffffffu, wait(bar, phase)) != 0;
    __syncwarp();                                // what follows is for a whole warp (tcgen05.ld, barriers)
    return ok;
  };

  if (warp == 16) {
    // ---- loads: lane l < CB boxes brings columns 64 (l % CB) of box l / CB
    constexpr int CB = HD / 64;
    const Pages& pages = p.c.pages;
    const int log = 7 - pages.log;               // log2 of the boxes of a block, a page each
    const bool issues = lane < CB << log;
    const int cb = lane % CB, unit = lane / CB;
    const uint32_t to = cb * (kKeys * 128) + (unit << (pages.log + 7));
    // the first row of the pool that this lane's box of block j is, of its head's keys. Without a page (behind the last row, or
    // a bad entry) that is the pool's first: no row of it counts
    const int first = ((int)lo << log) + unit, end = issues ? min((int)hi << log, (int)((s + a.T - 1) >> pages.log) + 1) : 0;   // pages
    auto lookup = [&](int j) {
      const int i = first + (j << log);
      if (i >= end) return kvh;
      const int pg = pages.page_of(b, (int64_t)i << pages.log);
      if (pg < 0 && a.status) atomicOr(a.status, 8);
      return max(pg, 0) * a.HKV + kvh;
    };
    int next = lookup(0);
    int done = 0;                                // blocks whose loads were issued
    bool ok = true;
    for (int j = 0; ok && j < n_blk; ++j) {
      if (j == 2) all_ready();                   // the first two blocks come while the queries do
      const int st = j & 1, z = next;
      next = lookup(j + 1);
      ok = j < 2 || wait_all(&sm.k_empty[st], (j >> 1) - 1);
      if (!ok) break;
      if (lane == 0) tc5::mbar_expect_tx(&sm.k_full[st], kKeys * HD * 2);
      __syncwarp();
      if (issues) tc5::tma_load_3d(sm.k[st] + to, &p.map, 64 * cb, 0, z, &sm.k_full[st]);
      ok = j < 2 || wait_all(&sm.v_empty[st], (j >> 1) - 1);
      if (!ok) {                                 // give the keys' copies one more bounded wait before leaving
        wait(&sm.k_full[st], j >> 1);
        break;
      }
      // the values that are cleared have a barrier of their own: who waits for it has not followed the others' phases
      uint64_t* bar = ragged && j + 1 == n_blk ? &sm.v_last : &sm.v_full[st];
      if (lane == 0) tc5::mbar_expect_tx(bar, kKeys * HD * 2);
      __syncwarp();
      if (issues) tc5::tma_load_3d(sm.v[st] + to, &p.map, 64 * cb, 0, z + (int)(pages.n_pages * a.HKV), bar);
      done = j + 1;
    }
    if (n_blk <= 2) all_ready();
    for (int j = max(0, done - 2); j < done; ++j) {   // no copy is in flight when the CTA ends
      wait(&sm.k_full[j & 1], j >> 1);
      if (ragged && j + 1 == n_blk) wait(&sm.v_last, 0);
      else wait(&sm.v_full[j & 1], j >> 1);
    }
  } else if (warp == 17 || warp == 18) {
    // ---- issue, tile i. The whole warp runs the loop, and what it counts with comes from one lane, so that addresses and
    // descriptors are uniform over it (moving them to where the instruction takes them cost more than the MMAs); one lane issues.
    // Step after step: the product of a half of block j, then the same half's scores of block j + 1 (j = -1: scores alone). One
    // place in the code for either: with the first scores before the loop, in a copy of their own, the loop's were issued twice
    // at HD 64
    const uint32_t tb = all_ready();
    const int i = __shfl_sync(0xffffffffu, warp, 0) - 17, blocks = __shfl_sync(0xffffffffu, i < n_tile ? n_blk : -1, 0);
    const bool tail = __shfl_sync(0xffffffffu, (int)ragged, 0) != 0, one = elected();
    constexpr uint32_t kIdS = tc5::idesc_bf16(128, kKeys / 2, false, false), kIdO = tc5::idesc_bf16(128, HD, false, true);
    constexpr uint64_t kTile = sizeof(sm.q[0]) >> 4;              // from one tile's descriptor to the next one's
    const uint32_t tu = __shfl_sync(0xffffffffu, tb, 0) + i * 128;
    const uint64_t qd = tc5::sdesc(tc5::smem_u32(sm.q[0]), 16, 1024) + i * kTile, k_desc = tc5::sdesc(tc5::smem_u32(sm.k[0]), 16, 1024);
    const uint64_t v_desc = tc5::sdesc(tc5::smem_u32(sm.v[0]), kKeys * 128, 1024);
    bool ok = true;
#pragma unroll 1
    for (int j = -1; ok && j < blocks; ++j) {
      const int st = j & 1;
#pragma unroll 1
      for (int h = 0; ok && h < 2; ++h) {
        if (j >= 0) {
          if (h == 0) ok = tail && j + 1 == blocks ? wait_all(&sm.v_clean, 0) : wait_all(&sm.v_full[st], j >> 1);
          ok = ok && wait_all(&sm.p_full[i][h], j);
          if (!ok) break;
          tc5::fence_after_sync();
          const uint64_t vd = v_desc + st * kTile + 4 * h * 128;
          const uint32_t d = tu + 256, pa = tu + 64 * h;
          if (one) {
            tc5::mma_ts(d, pa, vd, kIdO, j > 0 || h > 0);
            tc5::mma_ts(d, pa + 8, vd + 128, kIdO, 1);
            tc5::mma_ts(d, pa + 16, vd + 256, kIdO, 1);
            tc5::mma_ts(d, pa + 24, vd + 384, kIdO, 1);
            tc5::commit(&sm.pv_done[i][h]);
            if (h == 1) tc5::commit(j + 1 == blocks ? &sm.o_full[i] : &sm.v_empty[st]);
          }
        }
        if (j + 1 < blocks) {
          if (h == 0) ok = wait_all(&sm.k_full[st ^ 1], (j + 1) >> 1);
          if (!ok) break;
          tc5::fence_after_sync();
          const uint64_t kd = k_desc + (st ^ 1) * kTile + 4 * h * 128;
          if (one) {
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
              constexpr uint64_t kBlock = (kKeys * 128) >> 4;     // a block of 64 columns
              tc5::mma_ss(tu + 64 * h, qd + (ks >> 2) * kBlock + (ks & 3) * 2, kd + (ks >> 2) * kBlock + (ks & 3) * 2, kIdS, ks > 0);
            }
            tc5::commit(&sm.s_full[i][h]);
            if (h == 1) tc5::commit(&sm.k_empty[st ^ 1]);
          }
        }
      }
    }
    // no arrival is under way when the CTA ends
    if (ok && blocks > 0) wait_all(&sm.k_empty[(blocks - 1) & 1], (blocks - 1) >> 1);
    if (ok && blocks > 0) wait_all(&sm.o_full[i], 0);
  } else if (warp == 19) {
    all_ready();
    if (ragged) {
      const int j = n_blk - 1, st = j & 1, first = seen_last - j * kKeys;
      // also where a wait ran out: the arrival must come, or the issuing warp waits for it in vain
      if (wait(&sm.v_last, 0)) {
        for (int i = lane; i < (kKeys - first) * (HD / 8); i += 32) {
          const int r = first + i / (HD / 8), c = i % (HD / 8);
          *reinterpret_cast<uint4*>(sm.v[st] + (c >> 3) * (kKeys * 128) + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      tc5::mbar_arrive(&sm.v_clean);
    }
  } else {
    const uint32_t tb = all_ready();
    if ((warp >> 3) < n_tile) {
      // ---- softmax of tile i: this thread's two rows are those of TMEM lanes first_lane + grp and + grp + 8
      const int i = warp >> 3, grp = lane >> 2, tig = lane & 3;
      const int first_lane = 32 * (warp & 3) + 16 * (warp >> 2 & 1), first_row = row0 + 128 * i + first_lane + grp;
      const uint32_t lanes = (uint32_t)first_lane << 16, ts = tb + i * 128 + lanes, to = tb + 256 + i * 128 + lanes;
      const int see_all = seen + token_of(p, row0 + i * 128);       // that every row of the tile sees
      const float scale = a.sm_scale * kLog2e;
      float M[2] = {neg_inf(), neg_inf()};
      uint64_t l[2] = {0, 0};                                       // sums of weights over this thread's keys, in pairs
      bool ok = true;
      for (int j = 0; ok && j < n_blk; ++j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ok = ok && wait_all(&sm.s_full[i][h], j);
          if (!ok) break;
          tc5::fence_after_sync();
          uint32_t sc[32];
          ld_16x64(ts + 64 * h, sc);
          const int key = j * kKeys + 64 * h;
          tc5::ld_wait();
          if (key + 64 > see_all) {                                 // the same for the whole tile
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int left = seen + token_of(p, min(first_row + 8 * q, p.c.rows - 1)) - key - 2 * tig;   // seen, from this thread's first
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                if (8 * n >= left) sc[4 * n + 2 * q] = 0xff800000u;
                if (8 * n + 1 >= left) sc[4 * n + 2 * q + 1] = 0xff800000u;
              }
            }
          }
          // the references move only when a weight would pass 2^kMost (and at the first key)
          float m[2];
          bool over = false;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            m[q] = fmaxf(__uint_as_float(sc[2 * q]), __uint_as_float(sc[2 * q + 1]));
#pragma unroll
            for (int n = 1; n < 8; ++n) m[q] = max3(m[q], __uint_as_float(sc[4 * n + 2 * q]), __uint_as_float(sc[4 * n + 2 * q + 1]));
            m[q] *= scale;
            over |= m[q] > M[q] + kMost;
          }
          if (__any_sync(0xffffffffu, over)) {
            float f[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              m[q] = quad_max(m[q]);
              const float to_M = m[q] > M[q] + kMost ? m[q] : M[q];
              f[q] = M[q] == neg_inf() ? 0.f : ex2(M[q] - to_M);    // 1 where the reference stays
              M[q] = to_M;
              l[q] = mul2(l[q], pair(f[q], f[q]));
            }
            if (j > 0 || h > 0) {
              ok = h > 0 ? wait_all(&sm.pv_done[i][0], j) : wait_all(&sm.pv_done[i][1], j - 1);   // the last product
              tc5::fence_after_sync();
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
          const float r0 = M[0] == neg_inf() ? 0.f : -M[0], r1 = M[1] == neg_inf() ? 0.f : -M[1];
          const uint64_t ref[2] = {pair(r0, r0), pair(r1, r1)};
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const float2 u = unpair(fma2(pair(__uint_as_float(sc[4 * n + 2 * q]), __uint_as_float(sc[4 * n + 2 * q + 1])), pair(scale, scale), ref[q]));
              const float e0 = ex2(u.x), e1 = ex2(u.y);
              l[q] = add2(l[q], pair(e0, e1));
              w[2 * n + q] = pack_bf16(e0, e1);
            }
          st_16x32(ts + 64 * h, w);
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
      __syncwarp();
      if (ok) {
        tc5::fence_after_sync();
        // bf16 rows by way of this warp's sixteen rows of the query tile, whose products are done: whole rows to a store
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
              float* dst = p.part + (((int64_t)head * p.c.rows + row) * p.splits + split) * HD + d + 2 * tig;
#pragma unroll
              for (int n = 0; n < 4; ++n)
                if (row < p.c.rows) *reinterpret_cast<uint2*>(dst + 8 * n) = make_uint2(o[4 * n + 2 * q], o[4 * n + 2 * q + 1]);
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
            if (row < p.c.rows) reinterpret_cast<uint4*>(out_row(row))[c] = *reinterpret_cast<uint4*>(out + r * HD * 2 + ((c ^ (r & 7)) << 4));
          }
        }
        if (tig == 0) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (first_row + 8 * q >= p.c.rows) continue;
            const int64_t row = (int64_t)head * p.c.rows + first_row + 8 * q;
            if (p.splits > 1) p.part_ml[row * p.splits + split] = make_float2(M[q], sum[q]);
            else if (p.lse != nullptr) p.lse[row] = sum[q] == 0.f ? -neg_inf() : M[q] + log2f(sum[q]);
          }
        }
      }
    }
  }
  tc5::fence_before_sync();
  meet_all();
  tc5::fence_after_sync();
  if (warp == 17) tc5::tmem_dealloc(sm.tbase, 512);
  if (tid == 0 && sm.err && a.status) atomicOr(a.status, 2);
}

// one warp per (head, query row): the splits' partial sums joined. A lane holds the factors of splits lane, lane + 32, .., kOf of them;
// four splits' sums are on their way at once, of more than 32 splits eight (1 head of 20030 keys, 480 rows: 26.9 us in 53
// splits; one after another, in 39, 33.5)
constexpr int kMostSplits = 148;

template <int HD, int kOf>
__global__ void __launch_bounds__(128) paged_prompt_join_kernel(const __grid_constant__ Params p) {
  constexpr int EPL = HD / 32, kBatch = kOf == 1 ? 4 : 8;
  const bolt3_paged_attend_args& a = p.c.a;
  const int lane = threadIdx.x & 31;
  grid_dep_launch();
  grid_dep_wait();
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (int64_t)a.B * a.HKV * p.c.rows) return;
  const int head = (int)(item / p.c.rows), row = (int)(item % p.c.rows), b = head / a.HKV, kvh = head % a.HKV;
  const int64_t at = item * p.splits;
  float2 ml[kOf];
  float m = neg_inf(), l = 0.f, f[kOf], acc[EPL] = {};
#pragma unroll
  for (int c = 0; c < kOf; ++c) {
    const int i = 32 * c + lane;
    ml[c] = i < p.splits ? p.part_ml[at + i] : make_float2(neg_inf(), 0.f);
    m = fmaxf(m, ml[c].x);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
#pragma unroll
  for (int c = 0; c < kOf; ++c) {
    f[c] = ml[c].x == neg_inf() ? 0.f : exp2f(ml[c].x - m);
    l = fmaf(ml[c].y, f[c], l);
    if (ml[c].x == neg_inf() && ml[c].y == 0.f) f[c] = -1.f;      // no keys: its sums were not written
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
  for (int c = 0; c < kOf; ++c) {
    const int n = min(p.splits - 32 * c, 32);
    for (int j0 = 0; j0 < n; j0 += kBatch) {                      // the same for the whole warp
      float x[kBatch][EPL];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) x[j][e] = p.part[(at + 32 * c + min(j0 + j, n - 1)) * HD + 32 * e + lane];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float g = __shfl_sync(0xffffffffu, f[c], j0 + j & 31);
        if (j0 + j >= n || g == -1.f) continue;
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] = fmaf(x[j][e], g, acc[e]);
      }
    }
  }
  bf16* y = reinterpret_cast<bf16*>(a.y) + (((int64_t)b * a.T + row / p.c.G) * a.H + kvh * p.c.G + row % p.c.G) * HD;
#pragma unroll
  for (int e = 0; e < EPL; ++e) y[32 * e + lane] = __float2bfloat16_rn(l == 0.f ? 0.f : acc[e] / l);
  if (lane == 0 && p.lse != nullptr) p.lse[item] = l == 0.f ? -neg_inf() : m + log2f(l);
}

// the weights of a range of a head's keys, summed over its query rows, into their records
template <int HD>
__global__ void __launch_bounds__(kRecordThreads, 1) paged_prompt_record_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  RecordSmem<HD>& sm = *reinterpret_cast<RecordSmem<HD>*>(smem_raw + ((1024 - (tc5::smem_u32(smem_raw) & 1023)) & 1023));
  constexpr int NQ = kRows / kKeys;
  const bolt3_paged_attend_args& a = p.c.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x / p.ranges, range = blockIdx.x % p.ranges, b = head / a.HKV, kvh = head % a.HKV;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(&sm.k_full[i], 1);
      tc5::mbar_init(&sm.k_empty[i], 1);
    }
    for (int i = 0; i < NQ; ++i) {
      tc5::mbar_init(&sm.s_full[i], 1);
      tc5::mbar_init(&sm.s_empty[i], 128);
      for (int x = 0; x < 4; ++x) tc5::mbar_init(&sm.sum_full[x][i], 4);
    }
    tc5::mbar_fence_init();
    sm.err = 0;
  }
  meet_all();                                    // the barriers are there: loads may begin
  // Queries, keys, table and lengths come from kernels before the attention, but only this wait makes their writes visible here: read
  // before it, while the attention still runs, they saved 2 us and rested on an order that is promised nowhere
  grid_dep_wait();
  bool bad = false;
  const int64_t s = p.c.len.rows(b, bad);
  const int64_t all = s < 0 ? 0 : (s + a.T + kKeys - 1) / kKeys, lo = all * range / p.ranges, hi = all * (range + 1) / p.ranges;
  const int n_blk = (int)(hi - lo), groups = (p.c.rows + kRows - 1) / kRows;
  if (n_blk == 0) return;                        // the same for all threads: nothing has been allocated
  if (warp == 17) {
    tc5::tmem_alloc(&sm.tbase, 512);
    tc5::tmem_relinquish();
    grid_dep_launch();                           // here alone, for the whole CTA (common.cuh)
  }
  auto wait = [&](uint64_t* bar, int phase) {
    if (tc5::mbar_wait(bar, (uint32_t)phase & 1, kWaitIters)) return true;
    sm.err = 1;
    return false;
  };
  auto wait_all = [&](uint64_t* bar, int phase) {
    const bool ok = __all_sync(0xffffffffu, wait(bar, phase)) != 0;
    __syncwarp();                                // what follows is for a whole warp (tcgen05.ld, barriers)
    return ok;
  };
  const int total = groups * n_blk;              // blocks of keys that come, group after group
  // all warps come here before a group (its queries are in place) and after the last
  auto meet = [&] {
    tc5::fence_before_sync();
    meet_all();
    tc5::fence_after_sync();
  };
  // the first and the last block of group g that one of its rows sees: all of them up to that of its last row
  auto tiles_of = [&](int g) { return min(NQ, (p.c.rows - g * kRows + kKeys - 1) / kKeys); };

  if (warp == 16) {
    constexpr int CB = HD / 64;
    const Pages& pages = p.c.pages;
    const int log = 7 - pages.log;
    const bool issues = lane < CB << log;
    const int cb = lane % CB, unit = lane / CB;
    const int first = ((int)lo << log) + unit, end = issues ? min((int)hi << log, (int)((s + a.T - 1) >> pages.log) + 1) : 0;   // pages
    auto lookup = [&](int j) {
      const int i = first + (j << log);
      return i >= end ? kvh : max(pages.page_of(b, (int64_t)i << pages.log), 0) * a.HKV + kvh;
    };
    int done = 0;
    bool ok = true;
    for (int g = 0; g < groups; ++g) {
      int next = lookup(0);
      bool met = false;
      for (int j = 0; ok && j < n_blk; ++j) {
        if (j == 2) {                            // the first two blocks come while the queries do
          meet();
          met = true;
        }
        const int it = g * n_blk + j, st = it & 1, z = next;
        next = lookup(j + 1);
        ok = it < 2 || wait_all(&sm.k_empty[st], (it >> 1) - 1);
        if (!ok) break;
        if (lane == 0) tc5::mbar_expect_tx(&sm.k_full[st], kKeys * HD * 2);
        __syncwarp();
        if (issues)
          tc5::tma_load_3d(sm.k[st] + cb * (kKeys * 128) + (unit << (pages.log + 7)), &p.map, 64 * cb, 0, z, &sm.k_full[st]);
        done = it + 1;
      }
      if (!met) meet();
      // no copy is in flight when the CTA ends
      if (g + 1 == groups || !ok)
        for (int it = max(0, done - 2); it < done; ++it) wait(&sm.k_full[it & 1], it >> 1);
    }
  } else if (warp == 17) {
    const bool one = elected();
    constexpr uint32_t kId = tc5::idesc_bf16(128, kKeys, false, false);
    constexpr uint64_t kTile = (kKeys * HD * 2) >> 4;
    const uint64_t q_desc = tc5::sdesc(tc5::smem_u32(sm.q[0]), 16, 1024), k_desc = tc5::sdesc(tc5::smem_u32(sm.k[0]), 16, 1024);
    uint32_t used = 0;                           // parity of each tile's next wait for its columns; a first use does not wait
    uint32_t first = (1u << NQ) - 1;
    bool ok = true;
    for (int g = 0; g < groups; ++g) {
      meet();
      const uint32_t tu = __shfl_sync(0xffffffffu, sm.tbase, 0);
      const int nq = tiles_of(g);
      for (int j = 0; ok && j < n_blk; ++j) {
        const int it = g * n_blk + j, st = it & 1;
        ok = wait_all(&sm.k_full[st], it >> 1);
        for (int i = 0; ok && i < nq; ++i) {
          if (first >> i & 1) {
            first &= ~(1u << i);
          } else {
            ok = wait_all(&sm.s_empty[i], (int)(used >> i & 1));
            used ^= 1u << i;
          }
          if (!ok) break;
          tc5::fence_after_sync();
          if (one) {
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
              constexpr uint64_t kBlock = (kKeys * 128) >> 4;
              const uint64_t at = (ks >> 2) * kBlock + (ks & 3) * 2;
              tc5::mma_ss(tu + i * 128, k_desc + st * kTile + at, q_desc + i * kTile + at, kId, ks > 0);
            }
            tc5::commit(&sm.s_full[i]);
          }
        }
        if (ok && one) tc5::commit(&sm.k_empty[st]);
      }
    }
    if (ok) wait_all(&sm.k_empty[(total - 1) & 1], (total - 1) >> 1);   // no arrival is under way when the CTA ends
  } else {
    // ---- a thread is key 32 (warp % 4) + lane of a block, for the rows of tile warp / 4
    const int i = warp >> 2, key = 32 * (warp & 3) + lane;
    const float scale = a.sm_scale * kLog2e;
    const uint64_t scale2 = pair(scale, scale);
    const int64_t cap = a.width * a.page;
    float* record = a.weight + (int64_t)head * cap;
    bool ok = true;
    for (int g = 0; g < groups; ++g) {
      const int row0 = g * kRows, nq = tiles_of(g);
      // This group's queries, sums and tokens. The tile's MMAs of the group before are done: this warp has read their scores. The
      // tile's other warps may still be turning theirs into weights, by that group's sums and tokens: those of this one go beside
      // them, where nobody has read since the meeting at the start of the group before
      float* lse_of = sm.lse[g & 1];
      int* tokens = sm.token[g & 1];
      copy_queries<HD>(p, sm.q[0], b, kvh, row0, warp * 32, lane);
      copy_queries<HD>(p, sm.q[0], b, kvh, row0, warp * 32 + 16, lane);
      const int r = row0 + tid;
      lse_of[tid] = r < p.c.rows ? -p.lse[(int64_t)head * p.c.rows + r] : neg_inf();   // negated
      tokens[tid] = token_of(p, min(r, p.c.rows - 1));
      asm volatile("cp.async.wait_all;\nfence.proxy.async.shared::cta;\n" ::: "memory");
      meet();
      const uint32_t ts = sm.tbase + i * 128 + ((uint32_t)(32 * (warp & 3)) << 16);
      const int first_token = token_of(p, row0);
      if (i >= nq) continue;
      // The tiles' sums of a block's keys meet two blocks later, in the order of the tiles, at one tile's threads: no tile waits
      // for another at every block. The four slots suffice: a tile comes to block j + 4 once the MMAs of block j + 3 were issued
      // for all tiles, and so after each of them let go of the scores of block j + 2, which the one at which the sums of block j
      // meet does after it has read them
      float was = 0.f;                           // the record of this thread's key of the block before the last
      auto meets_here = [&](int j) { return j >= 0 && i == min(j & 3, nq - 1); };
      auto at = [&](int j) { return (lo + j) * kKeys + key; };
      auto fetch = [&](int j) {
        if (meets_here(j) && at(j) < s + a.T) was = record[at(j)];
      };
      auto add = [&](int j) {
        if (!meets_here(j)) return;
        const int it = g * n_blk + j;
        float w = 0.f;
        for (int x = 0; x < nq; ++x) {
          ok = ok && wait(&sm.sum_full[it & 3][x], it >> 2);
          w += sm.sum[it & 3][x][key];
        }
        if (ok && at(j) < s + a.T) record[at(j)] = was + w;
      };
      for (int j = 0; j < n_blk; ++j) {
        const int it = g * n_blk + j;
        const int64_t key0 = (lo + j) * kKeys;
        add(j - 2);
        float sum = 0.f;
        ok = ok && wait(&sm.s_full[i], it);
        ok = __all_sync(0xffffffffu, ok);
        __syncwarp();
        if (ok) {
          tc5::fence_after_sync();
          const bool masked = key0 + kKeys > s + 1 + first_token;     // the same for all threads
          const int rel = (int)max(min(key0 + key - s, (int64_t)0x7fffffff), (int64_t)-1);   // the first token that sees this key
          uint64_t acc = 0;
          // the next 32 scores are on their way while these are used; once the last have come, the next block's may overwrite them
          auto run = [&](auto cut) {
            uint32_t x[2][32];
            tc5::ld32(ts, x[0]);
            tc5::ld_wait();
#pragma unroll
            for (int c = 0; c < kKeys; c += 32) {
              const uint32_t(&y)[32] = x[c / 32 & 1];
              if (c + 32 < kKeys) tc5::ld32(ts + c + 32, x[c / 32 + 1 & 1]);
              const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(lse_of + i * kKeys + c);
              const int4* token = reinterpret_cast<const int4*>(tokens + i * kKeys + c);
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const ulonglong2 z = lse[u];
                const float2 a0 = unpair(fma2(pair(__uint_as_float(y[4 * u]), __uint_as_float(y[4 * u + 1])), scale2, z.x));
                const float2 a1 = unpair(fma2(pair(__uint_as_float(y[4 * u + 2]), __uint_as_float(y[4 * u + 3])), scale2, z.y));
                float e0, e1, e2, e3;
                if (u % 4 == 3) {                            // a quarter off the MUFU
                  const float2 b0 = ex2_fma(a0), b1 = ex2_fma(a1);
                  e0 = b0.x; e1 = b0.y; e2 = b1.x; e3 = b1.y;
                } else {
                  e0 = ex2(a0.x); e1 = ex2(a0.y); e2 = ex2(a1.x); e3 = ex2(a1.y);
                }
                if constexpr (cut) {
                  const int4 t = token[u];
                  e0 = t.x >= rel ? e0 : 0.f;
                  e1 = t.y >= rel ? e1 : 0.f;
                  e2 = t.z >= rel ? e2 : 0.f;
                  e3 = t.w >= rel ? e3 : 0.f;
                }
                acc = add2(acc, add2(pair(e0, e1), pair(e2, e3)));
              }
              if (c + 32 < kKeys) tc5::ld_wait();
              if (c + 64 == kKeys) {
                tc5::fence_before_sync();
                tc5::mbar_arrive(&sm.s_empty[i]);
              }
            }
          };
          if (masked) run(std::true_type{});
          else run(std::false_type{});
          const float2 x = unpair(acc);
          sum = x.x + x.y;
        } else {
          tc5::mbar_arrive(&sm.s_empty[i]);
        }
        sm.sum[it & 3][i][key] = sum;
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(&sm.sum_full[it & 3][i]);
        fetch(j - 1);
      }
      add(n_blk - 2);
      fetch(n_blk - 1);
      add(n_blk - 1);
    }
  }
  meet();
  if (warp == 17) tc5::tmem_dealloc(sm.tbase, 512);
  if (tid == 0 && sm.err && a.status) atomicOr(a.status, 2);
}

struct Plan {
  int tiles, splits, ranges;
  size_t part, ml, lse, bytes;                   // offsets
};

Plan plan_of(int B, int T, int H, int HKV, int HD, int64_t n, bool weigh) {
  Plan pl;
  const int64_t rows = (int64_t)T * (H / HKV), heads = (int64_t)B * HKV, blocks = (n + T + kKeys - 1) / kKeys;
  pl.tiles = (int)((rows + 255) / 256);
  // Splits of the keys, as many as fit the machine with the rows' tiles: of a few numbers the one with the shortest time, a block
  // taking 1.65 us, a join 3.3 and its sums, written and read, their bytes at 10 TB/s. 5 heads of 396 keys, 192 rows: 4 splits
  // 9.9 us, 1 13.0; 2 of 1700 keys, 1200 rows: 7 splits 17.2, 3 or 14 20.2. An estimate: near its border it takes the slower side (8 of
  // 428 keys, 512 rows: 6.60 for 1 split against 6.63 for 4, measured 15.1 and 14.3 us)
  pl.splits = 1;
  double best = (double)blocks * 1.65;
  for (int64_t room = min(148 / (heads * pl.tiles), blocks); room > 1; room = room * 3 / 4) {
    const int64_t longest = (blocks + room - 1) / room, of = (blocks + longest - 1) / longest;
    const double cost = (double)longest * 1.65 + 3.3 + (double)(of * heads * rows * HD) * 8e-7;
    if (cost < best) {
      best = cost;
      pl.splits = (int)of;
    }
  }
  // ranges of keys: as many as give the shortest longest SM, a CTA costing a block and a half beside its own (its queries).
  // 16 sequences of 17 blocks, 8 heads: with the attention 136 us, 2 ranges 143
  pl.ranges = 1;
  double least = 0;
  for (int64_t r = 1; r <= 32 && r <= blocks; ++r) {
    const double waves = (double)((heads * r + 147) / 148), cost = waves * ((double)((blocks + r - 1) / r) + 1.5);
    if (r == 1 || cost < least) {
      least = cost;
      pl.ranges = (int)r;
    }
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 15) & ~(size_t)15;
    return was;
  };
  const size_t parts = pl.splits > 1 ? (size_t)heads * (size_t)rows * (size_t)pl.splits : 0;
  pl.part = take(parts * (size_t)HD * 4);
  pl.ml = take(parts * 8);
  pl.lse = take(weigh ? (size_t)heads * (size_t)rows * 4 : 0);
  pl.bytes = at;
  return pl;
}

template <int HD>
int launch(Params& p, const Plan& pl, cudaStream_t s) {
  const size_t smem = sizeof(Smem<HD>) + 1024, rsmem = sizeof(RecordSmem<HD>) + 1024;
  if (cudaFuncSetAttribute(paged_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      cudaFuncSetAttribute(paged_prompt_record_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rsmem) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  const int64_t heads = (int64_t)p.c.a.B * p.c.a.HKV;
  if (launch_overlapped(paged_prompt_kernel<HD>, dim3((unsigned)(heads * pl.tiles), (unsigned)pl.splits), dim3(kThreads), smem, s,
                        p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  if (pl.splits > 1 && launch_overlapped(pl.splits <= 32 ? paged_prompt_join_kernel<HD, 1> : paged_prompt_join_kernel<HD, (kMostSplits + 31) / 32>,
                                         dim3((unsigned)((heads * p.c.rows + 3) / 4)), dim3(128), 0, s, p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  if (p.lse != nullptr && launch_overlapped(paged_prompt_record_kernel<HD>, dim3((unsigned)(heads * pl.ranges)), dim3(kRecordThreads),
                                            rsmem, s, p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  return BOLT3_OK;
}

}  // namespace

namespace paged {

size_t prompt_workspace(int B, int T, int H, int HKV, int HD, int64_t n, bool weigh) {
  return plan_of(B, T, H, HKV, HD, n, weigh).bytes;
}

int prompt_launch(const Attend& c, cudaStream_t s) {
  const bolt3_paged_attend_args& a = c.a;
  const Plan pl = plan_of(a.B, a.T, a.H, a.HKV, a.HD, c.len.cap - a.T, a.weight != nullptr);
  const int64_t heads = (int64_t)a.B * a.HKV;
  if (heads * pl.tiles > 0x7fffffff || heads * pl.ranges > 0x7fffffff || (heads * c.rows + 3) / 4 > 0x7fffffff) return BOLT3_ERR_SHAPE;
  Params p;
  if (!encode_pool(&p.map, a.pages, a.n_pages, a.page, a.HKV, a.HD, a.page)) return BOLT3_ERR_CUDA;
  p.c = c;
  p.per_G = c.G == 1 ? 0 : 0xffffffffu / c.G + 1;
  p.tiles = pl.tiles;
  p.splits = pl.splits;
  p.ranges = pl.ranges;
  char* ws = reinterpret_cast<char*>(a.workspace);
  p.part = reinterpret_cast<float*>(ws + pl.part);
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
  p.lse = a.weight != nullptr ? reinterpret_cast<float*>(ws + pl.lse) : nullptr;
  return a.HD == 128 ? launch<128>(p, pl, s) : launch<64>(p, pl, s);
}

}  // namespace paged
