// Softmax attention of new tokens over the pages of a bf16 KV cache, for few query rows per KV head, and the record of
// the weights that the cached rows got.
//
// For a query row and the keys j it sees, with t_j = sm_scale log2(e) (q . k_j):
//   w_j = 2^(t_j - M), y = sum_j w_j v_j / sum_j w_j, and the record of key j gains w_j / sum w summed over the query rows.
// M is a running reference, not the maximum: it is set to the largest t when that would pass it by more than 2^kMost, so
// that the usual block has no rescaling and no reduction across lanes (a vote); bf16 and fp32 hold such weights as well as
// smaller ones. Scores, weights and sums are fp32. In the product with the values a weight is two bf16 terms (its rounding
// and the rest, 2^-17 of it): the kernel waits for memory, and with one term the error would be that of the output's own
// rounding once more.
//
// Bound by HBM: 4 HD bytes per key and KV head. The cache is read in blocks of 32 keys, for 8 or 16 query rows at once
// (T * G of them, token-major). All blocks of all (sequence, KV head)s are one list, and every warp of the machine takes an
// equal run of it, whatever the lengths of the sequences: within a run each head's stretch is a softmax of its own, finished
// there if it is the whole cache of that head, else left in the workspace for a second kernel that joins the runs. Where the
// heads fit the machine at once, a CTA takes one instead (plan_of), and its warps the head's blocks in turn, joined in shared
// memory. 64 sequences of 2176 keys, 8 heads of 128: 92 us, 6.2 TB/s; one of 131072 keys: 88 us, 6.1 TB/s.
// A warp works on its own: lanes bring the next block's keys and values by TMA, a box for each page that the block touches,
// into a ring of the warp's own, in the 128-byte swizzle, whose ldmatrix reads are free of bank conflicts; the page numbers
// of the next 32 boxes stand in the warp's registers, those after them are on their way. Both products have the keys or
// dimensions in M and the query rows in N (no padding for up to 8 rows): S^T = K Q^T and O^T = V^T P^T by mma.sync m16n8k16,
// P^T being S^T transposed by movmatrix. Value rows that no query row sees are cleared in the fragments: a page's
// unused rows may hold anything.
//
// The record needs the sum over all keys, which is known after the last one: the scores are left in the workspace (4 bytes
// per key and query row, against 4 HD of the cache) and turned into weights afterwards, a key by one thread, so that no two
// add to one record. 64 sequences of 2176 keys, 8 heads of 128, 4 rows each: 101 us with records.
#include "paged.cuh"
#include "tc5.cuh"
#include "trace.h"

namespace {

using namespace paged;

constexpr int kBlock = 32;      // keys of a block: two 16-key halves of the products
constexpr int kWarps = 7;       // of a CTA, one CTA per SM: rings of 32 KB
constexpr float kMost = 20.f;   // log2 of the largest weight relative to the reference

struct Params {
  CUtensorMap map;              // the pool's rows, boxes of 64 columns and min(page, kBlock) rows
  Attend c;
  int n_runs;                   // warps that share all blocks; 0: a CTA per head
  int apart;                    // the records are made by a kernel of their own
  float* part;                  // [run][2][NC][HD] sums: a run's first stretch, its last
  float2* part_ml;              // [..][NC] (reference, sum of weights)
  int2* span;                   // [head]: where its first partial sum is, its last run; -1: no partial sums
  float* lse;                   // [head][rows] log2 of the sum of 2^t over the keys, +inf for an idle sequence
  float* score;                 // [head][most keys][score_row] t
  int64_t most;                 // keys that a head can have
  int score_row;                // rows, rounded up to even
};

template <int HD>
struct Ring {
  static constexpr int kSide = kBlock * HD * 2;            // bytes of a block's keys: HD / 64 tiles of [32 rows][128 bytes]
  static constexpr int kStage = 2 * kSide;
  static constexpr int kDepth = 32768 / kStage;
};

// Where a warp stands in its ring
struct RingState {
  uint32_t ring, bars;          // shared addresses
  uint32_t phase = 0;           // parity of each stage's next wait
  int stage = 0;
  bool dead = false;            // a wait ran out
};

// Running softmax of a warp over a stretch of one head's keys, for 8 NT query rows
template <int HD, int NT>
struct Softmax {
  static constexpr int MT = HD / 16;            // 16-dimension tiles of the output
  float o[MT][NT][4];                           // dimension 16 m + grp of rows 2 tig, 2 tig + 1, then dimension + 8
  float M0[NT], M1[NT], l0[NT], l1[NT];         // of query rows 2 tig and 2 tig + 1 of each tile of 8
};

B3_DEV void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
B3_DEV void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
B3_DEV uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

// Blocks blk0, blk0 + step, .. (n_it of them) of head (b, kvh), of whose keys query row r sees the first s + token + 1.
template <int HD, int NT>
B3_DEV void walk(const Params& p, RingState& rs, int b, int kvh, int64_t s, int64_t blk0, int n_it, int step,
                 Softmax<HD, NT>& f) {
  using R = Ring<HD>;
  constexpr int KS = HD / 16, MT = HD / 16, CB = HD / 64, kDepth = R::kDepth;
  const bolt3_paged_attend_args& a = p.c.a;
  const Pages& pages = p.c.pages;
  const int lane = threadIdx.x & 31, grp = lane >> 2, tig = lane & 3;
  const int head = b * a.HKV + kvh;
  if (rs.dead) n_it = 0;
  // a block is `units` boxes of rows (two for pages of 16 rows); lane l looks up the page of box l of the next 32
  const int units_log = pages.log == 4 ? 1 : 0, per_log = 5 - units_log, rows_log = 5 - units_log;
  const int64_t end_row = s + a.T;
  auto lookup = [&](int it0) {
    const int64_t row = (blk0 + (int64_t)(it0 + (lane >> units_log)) * step) * kBlock + ((lane & ((1 << units_log) - 1)) << rows_log);
    if (it0 + (lane >> units_log) >= n_it || row >= end_row) return -1;
    const int pg = pages.page_of(b, row);
    if (pg < 0 && a.status) atomicOr(a.status, 8);
    return pg;
  };
  int win = lookup(0), win_next = lookup(1 << per_log);
  // lane l < 2 CB units brings box l: keys or values (bit 0), columns 64 c, unit u
  const int side = lane & 1, cb = (lane >> 1) % CB, unit = (lane >> 1) / CB;
  const bool issues = lane < 2 * CB << units_log;
  // rows are read once: what else the call keeps in L2 (scores, partial sums) stays there. 64 sequences of 2176 keys, 8 heads: 95 -> 92 us,
  // with records 110 -> 103
  const uint64_t once = tc5::policy_evict_first();
  auto load = [&](int it, int stage) {
    const int at = it & ((1 << per_log) - 1);
    if (at == 0 && it > 0) {
      win = win_next;
      win_next = lookup(it + (1 << per_log));
    }
    const int pg = __shfl_sync(0xffffffffu, win, (at << units_log) + (issues ? unit : 0));
    uint64_t* bar = reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(rs.bars + 8 * stage));
    if (lane == 0) tc5::mbar_expect_tx(bar, R::kStage);
    __syncwarp();
    if (issues) {
      const int64_t row = (blk0 + (int64_t)it * step) * kBlock + (unit << rows_log);
      // without a page (behind the last row, or a bad entry) the box is read from the pool's first: no row of it counts
      const int z = (int)((side * pages.n_pages + max(pg, 0)) * a.HKV + kvh);
      void* dst = reinterpret_cast<void*>(
          __cvta_shared_to_generic(rs.ring + stage * R::kStage + side * R::kSide + cb * (kBlock * 128) + (unit << (rows_log + 7))));
      tc5::tma_load_3d(dst, &p.map, 64 * cb, (int)(row & ((1 << pages.log) - 1)), z, bar, once);
    }
  };
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i)
    if (i < n_it) {
      const int st = rs.stage + i;
      load(i, st >= kDepth ? st - kDepth : st);
    }

  // queries as B fragments: a lane holds row grp of each n8 tile, dimensions 16 k + 2 tig, + 1, + 8, + 9. Row r is head
  // kvh * G + r % G of token r / G
  uint32_t q[NT][KS][2];
  int see0[NT], see1[NT];                      // keys from blk0 on that rows 2 tig, 2 tig + 1 see (any number for a row past the last)
  const int64_t row0 = blk0 * kBlock;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + grp;
    const bool live = r < p.c.rows;
    const bf16* src = reinterpret_cast<const bf16*>(a.q) + (live ? b * a.q_sb + (r / p.c.G) * a.q_st + (int64_t)(kvh * p.c.G + r % p.c.G) * HD : 0);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        q[n][k][j] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 2 * tig + 8 * j) : 0u;
    const int r0 = 8 * n + 2 * tig;
    const int64_t first = s + 1 - row0;
    see0[n] = (int)min(max(first + r0 / p.c.G, (int64_t)0), (int64_t)0x7ffffff0);
    see1[n] = (int)min(max(first + (r0 + 1) / p.c.G, (int64_t)0), (int64_t)0x7ffffff0);
  }
  const int see_all = (int)min(max(s + 1 - row0, (int64_t)0), (int64_t)0x7ffffff0);      // what every row sees
  const int see_any = (int)min(max(s + a.T - row0, (int64_t)0), (int64_t)0x7ffffff0);    // what some row sees
  const float scale = a.sm_scale * kLog2e;
  // ldmatrix addresses within a tile: keys: row lane % 16, 16-byte chunk lane / 16; values: row lane % 8 + 8 (lane / 16),
  // chunk lane / 8 % 2. Chunk c of row r stands at c ^ r % 8
  const uint32_t k_row = (lane & 15) * 128, v_row = ((lane & 7) + (lane >> 4) * 8) * 128, sw = lane & 7;
  const uint32_t k_c = lane >> 4, v_c = lane >> 3 & 1;

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    f.M0[n] = f.M1[n] = neg_inf();
    f.l0[n] = f.l1[n] = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) f.o[m][n][0] = f.o[m][n][1] = f.o[m][n][2] = f.o[m][n][3] = 0.f;
  }
  for (int it = 0; it < n_it; ++it) {
    __syncwarp();                               // every lane has read the stage that is refilled now
    const int ahead = it + kDepth - 1, stage = rs.stage;
    if (ahead < n_it) load(ahead, stage == 0 ? kDepth - 1 : stage - 1);
    const bool ok = tc5::mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(rs.bars + 8 * stage)),
                                   rs.phase >> stage & 1, kWaitIters);
    if (!__all_sync(0xffffffffu, ok)) {
      rs.dead = true;
      break;
    }
    __syncwarp();                               // the matrix instructions below are for a whole warp
    rs.phase ^= 1u << stage;
    rs.stage = stage == kDepth - 1 ? 0 : stage + 1;
    const uint32_t at = rs.ring + stage * R::kStage;
    const int key0 = it * step * kBlock;        // of the block, from blk0 on
    // S^T = K Q^T; half i holds keys 16 i + grp and 16 i + grp + 8
    float t[2][NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int n = 0; n < NT; ++n) t[i][n][0] = t[i][n][1] = t[i][n][2] = t[i][n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t x[4];
        ldsm4(x, at + (k >> 2) * (kBlock * 128) + i * (16 * 128) + k_row + ((((k & 3) * 2 + k_c) ^ sw) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(t[i][n], x, q[n][k][0], q[n][k][1]);
      }
    }
    const bool masked = key0 + kBlock > see_all;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[i][n][e] *= scale;
        if (masked) {
          const int key = key0 + 16 * i + grp;
          if (key >= see0[n]) t[i][n][0] = neg_inf();
          if (key >= see1[n]) t[i][n][1] = neg_inf();
          if (key + 8 >= see0[n]) t[i][n][2] = neg_inf();
          if (key + 8 >= see1[n]) t[i][n][3] = neg_inf();
        }
      }
    if (p.score != nullptr) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int r = 8 * n + 2 * tig, key = key0 + 16 * i + grp;
          if (r >= p.score_row) continue;
          float* to = p.score + ((int64_t)head * p.most + row0 + key) * p.score_row + r;
          if (key < see_any) *reinterpret_cast<float2*>(to) = make_float2(t[i][n][0], t[i][n][1]);
          if (key + 8 < see_any) *reinterpret_cast<float2*>(to + 8 * p.score_row) = make_float2(t[i][n][2], t[i][n][3]);
        }
      __syncwarp();
    }
    // the references move only when a weight would pass 2^kMost (and at the first key a row sees)
    bool over = false;
    float m0[NT], m1[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m0[n] = fmaxf(fmaxf(t[0][n][0], t[0][n][2]), fmaxf(t[1][n][0], t[1][n][2]));
      m1[n] = fmaxf(fmaxf(t[0][n][1], t[0][n][3]), fmaxf(t[1][n][1], t[1][n][3]));
      over |= m0[n] > f.M0[n] + kMost || m1[n] > f.M1[n] + kMost;
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          m0[n] = fmaxf(m0[n], __shfl_xor_sync(0xffffffffu, m0[n], x));
          m1[n] = fmaxf(m1[n], __shfl_xor_sync(0xffffffffu, m1[n], x));
        }
        m0[n] = fmaxf(f.M0[n], m0[n]);
        m1[n] = fmaxf(f.M1[n], m1[n]);
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
    uint32_t hi[2][NT][2], lo[2][NT][2];        // P^T as B fragments, two terms
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float r0 = f.M0[n] == neg_inf() ? 0.f : f.M0[n], r1 = f.M1[n] == neg_inf() ? 0.f : f.M1[n];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float w0 = ex2(t[i][n][0] - r0), w1 = ex2(t[i][n][1] - r1), w2 = ex2(t[i][n][2] - r0), w3 = ex2(t[i][n][3] - r1);
        f.l0[n] += w0 + w2;
        f.l1[n] += w1 + w3;
        uint32_t a0, a1;
        const float2 h0 = rbf2(w0, w1, a0), h1 = rbf2(w2, w3, a1);
        hi[i][n][0] = transpose8(a0);
        hi[i][n][1] = transpose8(a1);
        lo[i][n][0] = transpose8(pack_bf16(w0 - h0.x, w1 - h0.y));
        lo[i][n][1] = transpose8(pack_bf16(w2 - h1.x, w3 - h1.y));
      }
    }
    // O^T += V^T P^T: tile m holds dimensions 16 m + grp and + 8
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // keys 2 tig, 2 tig + 1 (and + 8) of this half that some row sees
      uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
      if (masked) {
        const int key = key0 + 16 * i + 2 * tig;
        keep0 = (key < see_any ? 0xffffu : 0u) | (key + 1 < see_any ? 0xffff0000u : 0u);
        keep1 = (key + 8 < see_any ? 0xffffu : 0u) | (key + 9 < see_any ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t x[4];
        ldsm4_t(x, at + R::kSide + (m >> 2) * (kBlock * 128) + i * (16 * 128) + v_row + ((((m & 3) * 2 + v_c) ^ sw) << 4));
        if (masked) {
          x[0] &= keep0;
          x[1] &= keep0;
          x[2] &= keep1;
          x[3] &= keep1;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816(f.o[m][n], x, hi[i][n][0], hi[i][n][1]);
          mma16816(f.o[m][n], x, lo[i][n][0], lo[i][n][1]);
        }
      }
    }
  }
  __syncwarp();
  if (rs.dead && n_it > 0) {                    // give copies in flight one more bounded wait each before leaving
    for (int st = 0; st < kDepth; ++st)
      tc5::mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(rs.bars + 8 * st)), rs.phase >> st & 1, kWaitIters);
    if (lane == 0 && a.status) atomicOr(a.status, 2);
  }
  // the lanes' sums of weights (the references are the same in all lanes of a row)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      f.l0[n] += __shfl_xor_sync(0xffffffffu, f.l0[n], x);
      f.l1[n] += __shfl_xor_sync(0xffffffffu, f.l1[n], x);
    }
}

// query row `row` of head (b, kvh)'s output
template <int HD>
B3_DEV bf16* out_row(const Attend& c, int b, int kvh, int row) {
  return reinterpret_cast<bf16*>(c.a.y) + (((int64_t)b * c.a.T + row / c.G) * c.a.H + kvh * c.G + row % c.G) * HD;
}

// blocks of a head of a sequence with s rows before the call
B3_DEV int64_t blocks_of(int64_t s, int T) { return s < 0 ? 0 : (s + T + kBlock - 1) / kBlock; }

// log2 of the sum of 2^t, from a reference and the sum relative to it
B3_DEV float lse_of(float m, float l) { return l == 0.f ? -neg_inf() : m + log2f(l); }

// the records of keys key0, key0 + step, .. (kKeysAt of them, those below `end`) of a sequence with s rows before the call: their
// weights over the rows of a head that see them. `lse` of the head's rows
constexpr int kKeysAt = 4;
B3_DEV void record(const Params& p, int head, int64_t cap, int64_t s, int64_t key0, int step, int64_t end, const float* lse) {
  const float* t = p.score + ((int64_t)head * p.most + key0) * p.score_row;
  float* weight = p.c.a.weight + head * cap + key0;
  float sum[kKeysAt], was[kKeysAt];
  int first[kKeysAt];                                           // row that sees the key first
#pragma unroll
  for (int u = 0; u < kKeysAt; ++u) {
    const int64_t key = key0 + u * step;
    first[u] = key >= end ? 0x7fffffff : key > s ? (int)(key - s) * p.c.G : 0;
    was[u] = key < end ? weight[u * step] : 0.f;
    sum[u] = 0.f;
  }
#pragma unroll 2
  for (int r = 0; r < p.c.rows; r += 2) {
    float2 x[kKeysAt];
#pragma unroll
    for (int u = 0; u < kKeysAt; ++u)
      if (r + 1 >= first[u]) x[u] = *reinterpret_cast<const float2*>(t + (int64_t)u * step * p.score_row + r);
#pragma unroll
    for (int u = 0; u < kKeysAt; ++u) {
      if (r >= first[u]) sum[u] += ex2(x[u].x - lse[r]);
      if (r + 1 >= first[u] && r + 1 < p.c.rows) sum[u] += ex2(x[u].y - lse[r + 1]);
    }
  }
#pragma unroll
  for (int u = 0; u < kKeysAt; ++u)
    if (key0 + u * step < end) weight[u * step] = was[u] + sum[u];
}

template <int HD, int NT>
__global__ void __launch_bounds__(32 * kWarps) paged_stream_kernel(const __grid_constant__ Params p) {
  using R = Ring<HD>;
  constexpr int NC = 8 * NT, MT = HD / 16;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t s_bars[kWarps][R::kDepth];
  __shared__ float s_lse[NC];
  const bolt3_paged_attend_args& a = p.c.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, tig = lane & 3;
  unsigned char* smem = smem_raw + ((1024 - (tc5::smem_u32(smem_raw) & 1023)) & 1023);
  RingState rs;
  rs.ring = tc5::smem_u32(smem) + warp * R::kDepth * R::kStage;
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
    const int b = blockIdx.x / a.HKV, kvh = blockIdx.x % a.HKV, head = blockIdx.x;
    const int64_t s = p.c.len.rows(b, bad);
    if (bad && tid == 0 && a.status) atomicOr(a.status, 8);
    const int64_t nb = blocks_of(s, a.T);
    walk<HD, NT>(p, rs, b, kvh, s, warp, nb > warp ? (int)((nb - warp + kWarps - 1) / kWarps) : 0, kWarps, f);
    __syncthreads();                                            // the rings are read: their memory is free
    float* so = reinterpret_cast<float*>(smem);                 // [kWarps][NC][HD]
    float2* sml = reinterpret_cast<float2*>(so + kWarps * NC * HD);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + 2 * tig;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float* at = so + (warp * NC + r) * HD + 16 * m + grp;
        at[0] = f.o[m][n][0];
        at[HD] = f.o[m][n][1];
        at[8] = f.o[m][n][2];
        at[HD + 8] = f.o[m][n][3];
      }
      if (grp == 0) {
        sml[warp * NC + r] = make_float2(f.M0[n], f.l0[n]);
        sml[warp * NC + r + 1] = make_float2(f.M1[n], f.l1[n]);
      }
    }
    __syncthreads();
    for (int i = tid; i < p.c.rows * HD; i += 32 * kWarps) {
      const int r = i / HD, d = i % HD;
      float m = neg_inf();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sml[w * NC + r].x);
      float acc = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = sml[w * NC + r];
        const float g = ml.x == neg_inf() ? 0.f : exp2f(ml.x - m);
        acc = fmaf(so[(w * NC + r) * HD + d], g, acc);
        l = fmaf(ml.y, g, l);
      }
      out_row<HD>(p.c, b, kvh, r)[d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
      if (d == 0) {
        if (p.apart) p.lse[(int64_t)head * p.c.rows + r] = lse_of(m, l);
        else s_lse[r] = lse_of(m, l);
      }
    }
    if (p.score != nullptr && !p.apart) {
      __syncthreads();
      const int64_t cap = a.width * a.page;
      if (s >= 0)
        for (int64_t key = tid; key < s + a.T; key += kKeysAt * 32 * kWarps) record(p, head, cap, s, key, 32 * kWarps, s + a.T, s_lse);
    }
    return;
  }

  // this warp's run of the list of all blocks, ordered by sequence, head, key
  const int run = blockIdx.x * kWarps + warp;
  if (run >= p.n_runs) return;
  int b = 0;
  int64_t total = 0, lo, hi, start = 0;                         // start: of sequence b's blocks in the list
  int64_t s, nb;
  if (a.lens == nullptr) {
    s = p.c.len.rows(0, bad);
    nb = blocks_of(s, a.T);
    total = nb * a.B * a.HKV;
    if (bad && run == 0 && lane == 0 && a.status) atomicOr(a.status, 8);
    const int64_t runs = min((int64_t)p.n_runs, total);         // none is empty: the join takes all from first to last
    if (run >= runs) return;
    lo = total * run / runs;
    hi = total * (run + 1) / runs;
    b = (int)(lo / (nb * a.HKV));
    start = b * nb * a.HKV;
  } else {
    for (int i = lane; i < a.B; i += 32) total += blocks_of(p.c.len.rows(i, bad), a.T);
    if (bad && run == 0 && a.status) atomicOr(a.status, 8);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    total *= a.HKV;
    const int64_t runs = min((int64_t)p.n_runs, total);
    if (run >= runs) return;
    lo = total * run / runs;
    hi = total * (run + 1) / runs;
    // the sequence that block lo belongs to
    for (int i0 = 0;; i0 += 32) {
      const int64_t mine = i0 + lane < a.B ? blocks_of(p.c.len.rows(i0 + lane, bad), a.T) * a.HKV : 0;
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
    s = p.c.len.rows(b, bad);
    nb = blocks_of(s, a.T);
  }
  int kvh = (int)((lo - start) / nb);
  bool first = true;
  while (lo < hi) {
    const int64_t at0 = start + kvh * nb;                       // this head's first block in the list
    const int64_t b0 = lo - at0, b1 = min(hi - at0, nb);
    const int head = b * a.HKV + kvh;
    walk<HD, NT>(p, rs, b, kvh, s, b0, (int)(b1 - b0), 1, f);
    const bool whole = b0 == 0 && b1 == nb;
    int2* span = p.span + head;
    const int64_t slot = (int64_t)run * 2 + (first ? 0 : 1);
    if (lane == 0) {
      if (whole) {
        *span = make_int2(-1, -1);
      } else {
        if (b0 == 0) span->x = run * 2 + (first ? 0 : 1);
        if (b1 == nb) span->y = run;
      }
    }
    if (whole) {                                                // the head's whole cache: done
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = 8 * n + 2 * tig;
        const float i0 = f.l0[n] == 0.f ? 0.f : 1.f / f.l0[n], i1 = f.l1[n] == 0.f ? 0.f : 1.f / f.l1[n];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (r < p.c.rows) {
            bf16* y = out_row<HD>(p.c, b, kvh, r) + 16 * m + grp;
            y[0] = __float2bfloat16_rn(f.o[m][n][0] * i0);
            y[8] = __float2bfloat16_rn(f.o[m][n][2] * i0);
          }
          if (r + 1 < p.c.rows) {
            bf16* y = out_row<HD>(p.c, b, kvh, r + 1) + 16 * m + grp;
            y[0] = __float2bfloat16_rn(f.o[m][n][1] * i1);
            y[8] = __float2bfloat16_rn(f.o[m][n][3] * i1);
          }
        }
        if (grp == 0 && p.score != nullptr) {
          float* lse = p.lse + (int64_t)head * p.c.rows;
          if (r < p.c.rows) lse[r] = lse_of(f.M0[n], f.l0[n]);
          if (r + 1 < p.c.rows) lse[r + 1] = lse_of(f.M1[n], f.l1[n]);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = 8 * n + 2 * tig;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float* at = p.part + (slot * NC + r) * HD + 16 * m + grp;
          if (r < p.c.rows) {
            at[0] = f.o[m][n][0];
            at[8] = f.o[m][n][2];
          }
          if (r + 1 < p.c.rows) {
            at[HD] = f.o[m][n][1];
            at[HD + 8] = f.o[m][n][3];
          }
        }
        if (grp == 0) {
          p.part_ml[slot * NC + r] = make_float2(f.M0[n], f.l0[n]);
          p.part_ml[slot * NC + r + 1] = make_float2(f.M1[n], f.l1[n]);
        }
      }
    }
    first = false;
    lo = at0 + b1;
    if (b1 == nb && ++kvh == a.HKV && lo < hi) {                // on to the next sequence that has keys
      kvh = 0;
      start += nb * a.HKV;
      do {
        if (++b >= a.B) return;                                 // not reached while the lengths stand
        if (a.lens != nullptr) {
          s = p.c.len.rows(b, bad);
          nb = blocks_of(s, a.T);
        }
      } while (nb == 0);
    }
  }
}

// Where the partial sums of a head are: the first one's slot, the first run, their number. false: there are none, and the row's
// output has been written (done) or is 0 (an idle sequence, or a run gave up)
struct Parts {
  int x, r0, n;
  bool done;
};
B3_DEV bool parts_of(const Params& p, int head, Parts& f) {
  bool bad = false;
  const int2 span = p.span[head];
  f.x = span.x;
  f.r0 = span.x >> 1;
  f.n = span.y - f.r0 + 1;
  f.done = span.x < 0;
  if (p.c.len.rows(head / p.c.a.HKV, bad) < 0 || (span.x >= 0 && (span.x >= 2 * p.n_runs || span.y < f.r0 || span.y >= p.n_runs))) {
    f.done = false;
    return false;
  }
  return !f.done;
}
// slot of the i-th of them: a later run's first stretch
B3_DEV int64_t slot_of(const Parts& f, int i) { return i == 0 ? f.x : 2 * (int64_t)(f.r0 + i); }

// The sums i0, i0 + step, .. of query row r joined, by a warp: the reference, the sum of weights, the outputs'
// dimensions 32 e + lane
template <int HD, int NC>
B3_DEV void join(const Params& p, const Parts& f, int r, int i0, int step, float& m, float& l, float (&acc)[HD / 32]) {
  const int lane = threadIdx.x & 31;
  m = neg_inf();
  l = 0.f;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) acc[e] = 0.f;
  constexpr int kBatch = 4;
  for (; i0 < f.n; i0 += kBatch * step) {
    float2 ml[kBatch];
    float x[kBatch][HD / 32];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * step;
      const int64_t at = slot_of(f, min(i, f.n - 1)) * NC + r;
      ml[j] = i < f.n ? p.part_ml[at] : make_float2(neg_inf(), 0.f);
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) x[j][e] = i < f.n ? p.part[at * HD + 32 * e + lane] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float to = fmaxf(m, ml[j].x), ref = to == neg_inf() ? 0.f : to;
      const float f0 = exp2f(m - ref), f1 = exp2f(ml[j].x - ref);   // exp2f(-inf) = 0
      m = to;
      l = fmaf(l, f0, ml[j].y * f1);
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) acc[e] = fmaf(acc[e], f0, x[j][e] * f1);
    }
  }
}

// The same for many: 32 sums' references first, a lane each, so that kBatch of the sums are on their way at once
template <int HD, int NC>
B3_DEV void join_many(const Params& p, const Parts& f, int r, int i0, int step, float& m, float& l, float (&acc)[HD / 32]) {
  constexpr int kBatch = 16;
  const int lane = threadIdx.x & 31;
  m = neg_inf();
  l = 0.f;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) acc[e] = 0.f;
  for (; i0 < f.n; i0 += 32 * step) {
    const int i = i0 + lane * step, n = min((f.n - i0 + step - 1) / step, 32);
    const float2 ml = i < f.n ? p.part_ml[slot_of(f, i) * NC + r] : make_float2(neg_inf(), 0.f);
    float to = ml.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, x));
    to = fmaxf(m, to);
    const float ref = to == neg_inf() ? 0.f : to, f0 = exp2f(m - ref), f1 = exp2f(ml.x - ref);   // exp2f(-inf) = 0
    float sum = ml.y * f1;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    m = to;
    l = fmaf(l, f0, sum);
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) acc[e] *= f0;
    for (int j0 = 0; j0 < n; j0 += kBatch) {
      float x[kBatch][HD / 32];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int64_t at = (slot_of(f, i0 + min(j0 + j, n - 1) * step) * NC + r) * HD + lane;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) x[j][e] = p.part[at + 32 * e];
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float g = __shfl_sync(0xffffffffu, f1, (j0 + j) & 31);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e)
          if (j0 + j < n) acc[e] = fmaf(x[j][e], g, acc[e]);
      }
    }
  }
}

// A head's output row where there are no sums to join
template <int HD>
B3_DEV void zero_row(const Params& p, int head, int row) {
  bf16* y = out_row<HD>(p.c, head / p.c.a.HKV, head % p.c.a.HKV, row);
  for (int i = threadIdx.x & 31; i < HD; i += 32) y[i] = __float2bfloat16_rn(0.f);
}

// The runs' partial sums of a (head, query row) where a head has few of them, joined by a warp (64 heads with 18 each: 157 us, by a block
// 151; 256 heads with 6: the same); with records, blocks from
// `joins` on turn the scores of kKeysAt * kJoinThreads keys of a head into weights at the same time (a launch less, and
// neither waits for the other: 64 sequences of 2176 keys, 8 heads, 112 -> 110 us), for which they join the rows' sums of weights
constexpr int kJoinThreads = 256;

template <int HD, int NC>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ Params p, int joins, int chunks) {
  constexpr int kJoinWarps = kJoinThreads / 32;
  __shared__ float s_lse[16];
  const bolt3_paged_attend_args& a = p.c.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.B * a.HKV;
  grid_dep_launch();
  grid_dep_wait();
  Parts f;
  if ((int)blockIdx.x < joins) {
    const int64_t item = (int64_t)blockIdx.x * kJoinWarps + warp;
    if (item >= (int64_t)heads * p.c.rows) return;
    const int head = (int)(item / p.c.rows), row = (int)(item - (int64_t)head * p.c.rows);
    if (!parts_of(p, head, f)) {
      if (!f.done) zero_row<HD>(p, head, row);
      return;
    }
    float m, l, acc[HD / 32];
    join<HD, NC>(p, f, row, 0, 1, m, l, acc);
    bf16* y = out_row<HD>(p.c, head / a.HKV, head % a.HKV, row);
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) y[32 * e + lane] = __float2bfloat16_rn(l == 0.f ? 0.f : acc[e] / l);
    return;
  }
  const int at = blockIdx.x - joins, head = at / chunks, b = head / a.HKV;
  bool bad = false;
  const int64_t s = p.c.len.rows(b, bad), key = (int64_t)(at % chunks) * (kKeysAt * kJoinThreads) + threadIdx.x;
  if (s < 0 || key - threadIdx.x >= s + a.T) return;            // the same for the whole block
  if (threadIdx.x < p.c.rows) {
    const int row = threadIdx.x;
    float m = neg_inf(), l = 0.f;
    if (parts_of(p, head, f)) {
#pragma unroll 4
      for (int i = 0; i < f.n; ++i) {
        const float2 ml = p.part_ml[slot_of(f, i) * NC + row];
        const float to = fmaxf(m, ml.x), ref = to == neg_inf() ? 0.f : to;
        l = fmaf(l, exp2f(m - ref), ml.y * exp2f(ml.x - ref));
        m = to;
      }
      s_lse[row] = lse_of(m, l);
    } else {
      s_lse[row] = f.done ? p.lse[(int64_t)head * p.c.rows + row] : -neg_inf();
    }
  }
  __syncthreads();
  record(p, head, a.width * a.page, s, key, kJoinThreads, s + a.T, s_lse);
}

// The same for heads with more partial sums: a block for each query row. From eight to a warp on (kMany) 16 at once: 1 head of
// 102400 keys 17.9 us, otherwise 38; 4 heads of 3239 keys 9.2, otherwise 8.6
constexpr int kMaxJoinWarps = 16;

template <int HD, int NC, bool kMany>
__global__ void __launch_bounds__(32 * kMaxJoinWarps) paged_join_long_kernel(const __grid_constant__ Params p) {
  __shared__ float s_acc[kMaxJoinWarps][HD], s_m[kMaxJoinWarps], s_l[kMaxJoinWarps];
  const bolt3_paged_attend_args& a = p.c.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
  const int head = blockIdx.x, row = blockIdx.y;
  grid_dep_launch();
  grid_dep_wait();
  float* lse = p.score != nullptr ? p.lse + (int64_t)head * p.c.rows + row : nullptr;
  Parts f;
  if (!parts_of(p, head, f)) {             // the same for the whole block
    if (!f.done && warp == 0) {
      zero_row<HD>(p, head, row);
      if (lse != nullptr && lane == 0) *lse = -neg_inf();
    }
    return;
  }
  float m, l, acc[HD / 32];
  if constexpr (kMany) join_many<HD, NC>(p, f, row, warp, n_warps, m, l, acc);
  else join<HD, NC>(p, f, row, warp, n_warps, m, l, acc);
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) s_acc[warp][32 * e + lane] = acc[e];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  bf16* y = out_row<HD>(p.c, head / a.HKV, head % a.HKV, row);
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
    if (i == 0 && lse != nullptr) *lse = lse_of(m, l);
  }
}

// The scores of a head's keys turned into weights and added to their records, once the rows' sums over all keys are known
constexpr int kRecordThreads = 256;

__global__ void __launch_bounds__(kRecordThreads) paged_record_kernel(const __grid_constant__ Params p, int chunks) {
  __shared__ float s_lse[16];
  const bolt3_paged_attend_args& a = p.c.a;
  const int head = blockIdx.x / chunks, b = head / a.HKV;
  const int64_t key = (int64_t)(blockIdx.x % chunks) * (kKeysAt * kRecordThreads) + threadIdx.x;
  grid_dep_launch();
  grid_dep_wait();
  bool bad = false;
  const int64_t s = p.c.len.rows(b, bad);
  if (s < 0) return;
  if (threadIdx.x < p.c.rows) s_lse[threadIdx.x] = p.lse[(int64_t)head * p.c.rows + threadIdx.x];
  __syncthreads();
  record(p, head, a.width * a.page, s, key, kRecordThreads, s + a.T, s_lse);
}

// how a call is cut: query rows (in 8), runs
struct Plan {
  int nt, runs, apart, score_row;
  size_t part, ml, span, lse, score, bytes;                     // offsets
};

Plan plan_of(int B, int T, int H, int HKV, int HD, int64_t n, bool ragged, bool weigh) {
  Plan pl;
  const int64_t rows = (int64_t)T * (H / HKV), heads = (int64_t)B * HKV;
  pl.nt = rows <= 8 ? 1 : 2;
  const int64_t per_head = (n + T + kBlock - 1) / kBlock, blocks = heads * per_head;
  // A CTA per head, which needs no join (4 us), where all are on the machine at once and none works for much longer than the
  // machine would: a CTA streams at 1 / 58 of the machine's bandwidth, a block of each warp in 1 us. Of a ragged batch one
  // sequence may be all there is. Else every warp a run, of two blocks or more. 3 heads of 701 keys with records 9.6 us, in runs
  // 10.3; of 1701 15.4, in runs 10.6; 128 heads of 3001 keys 33.7, in runs 37.6
  pl.runs = 0;
  if (heads > 148 || per_head * (58 - min(ragged ? (int64_t)HKV : heads, (int64_t)58)) > (int64_t)(3.5 * kWarps * 58)) {
    const int64_t runs = blocks / 2 < 148 * kWarps ? blocks / 2 : 148 * kWarps;
    pl.runs = runs < 1 ? 1 : (int)runs;
  }
  // A CTA per head makes its records itself, up to 4096 keys: 24 heads of 701 keys 9.9 us in all, with a kernel apart 10.9; 64 heads of
  // 3001 keys 25.0, apart 24.4; of 12001 keys 82, apart 75
  pl.apart = weigh && (pl.runs > 0 || per_head > 128);
  pl.score_row = (int)((rows + 1) & ~1);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 15) & ~(size_t)15;
    return was;
  };
  const size_t slots = (size_t)pl.runs * 2 * (size_t)(8 * pl.nt);
  pl.part = take(slots * (size_t)HD * 4);
  pl.ml = take(slots * 8);
  pl.span = take(pl.runs > 0 ? (size_t)heads * 8 : 0);
  pl.lse = take(weigh ? (size_t)heads * (size_t)rows * 4 : 0);
  pl.score = take(weigh ? (size_t)heads * (size_t)(n + T) * (size_t)pl.score_row * 4 : 0);
  pl.bytes = at;
  return pl;
}

template <int HD, int NT>
int launch_stream(Params& p, const Plan& pl, cudaStream_t s) {
  constexpr int NC = 8 * NT;
  constexpr size_t smem = (size_t)kWarps * 32768 + 1024;
  static_assert(smem >= (size_t)kWarps * NC * (HD * 4 + 8) + 1024, "the join's sums fit the rings");
  if (cudaFuncSetAttribute(paged_stream_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  const unsigned heads = (unsigned)(p.c.a.B * p.c.a.HKV), ctas = pl.runs == 0 ? heads : (unsigned)((pl.runs + kWarps - 1) / kWarps);
  if (launch_overlapped(paged_stream_kernel<HD, NT>, dim3(ctas), dim3(32 * kWarps), smem, s, p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  static_assert(kJoinThreads == kRecordThreads, "of a block of records");
  const int chunks = (int)((p.most + kKeysAt * kRecordThreads - 1) / (kKeysAt * kRecordThreads));
  const int per_head = pl.runs / (int)heads + 2;                // partial sums that a head has on average, about
  if (pl.runs > 0 && per_head <= 8) {
    const unsigned joins = (unsigned)(((int64_t)heads * p.c.rows + kJoinThreads / 32 - 1) / (kJoinThreads / 32));
    return launch_overlapped(paged_join_kernel<HD, NC>, dim3(joins + (p.score != nullptr ? heads * (unsigned)chunks : 0u)),
                             dim3(kJoinThreads), 0, s, p, (int)joins, chunks) == cudaSuccess ? BOLT3_OK : BOLT3_ERR_CUDA;
  }
  if (pl.runs > 0 && launch_overlapped(per_head >= 8 * kMaxJoinWarps ? paged_join_long_kernel<HD, NC, true> : paged_join_long_kernel<HD, NC, false>,
                                       dim3(heads, (unsigned)p.c.rows), dim3(per_head >= 32 ? 512 : 256), 0, s, p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  if (p.apart &&
      launch_overlapped(paged_record_kernel, dim3(heads * (unsigned)chunks), dim3(kRecordThreads), 0, s, p, chunks) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  return BOLT3_OK;
}

// Whether a call's rows go to the kernel for many rows, which works on tiles of 128: from 17 rows on, where this one's products
// pass its loads. 8 sequences of 2048 keys, 8 heads: 16 rows 22.7 us, there 23.5; 32 rows (two passes over the keys) 39.1, there 24.7
bool many_rows(int T, int H, int HKV) { return (int64_t)T * (H / HKV) > 16; }

bool shape_ok(int B, int T, int H, int HKV, int HD) {
  return B > 0 && T > 0 && HKV > 0 && H > 0 && H % HKV == 0 && H / HKV <= 16 && (HD == 64 || HD == 128) &&
         T <= (1 << 24) / (H / HKV) && (int64_t)B * HKV <= 0x3fffffff;
}

// Whether outputs would be written over queries that are still to be read. Outputs in the place of their own queries are not: a
// query row's output is written by who has read it, after all of the row's keys, or by the join. But the records of many rows read
// the queries again once the outputs are written
bool overwrites(const bolt3_paged_attend_args& a) {
  const int64_t row = (int64_t)a.H * a.HD, sb = (a.B - 1) * a.q_sb, st = (a.T - 1) * a.q_st;
  const bf16* q = reinterpret_cast<const bf16*>(a.q);
  const bf16* y = reinterpret_cast<const bf16*>(a.y);
  const bool apart = y >= q + (sb > 0 ? sb : 0) + (st > 0 ? st : 0) + row || q + (sb < 0 ? sb : 0) + (st < 0 ? st : 0) >= y + (int64_t)a.B * a.T * row;
  const bool own = y == q && (a.T == 1 || a.q_st == row) && (a.B == 1 || a.q_sb == a.T * row);
  return !apart && !(own && (a.weight == nullptr || !many_rows(a.T, a.H, a.HKV)));
}

}  // namespace

extern "C" size_t bolt3_paged_attend_workspace(int B, int T, int H, int HKV, int HD, int64_t n, int weigh) {
  if (!shape_ok(B, T, H, HKV, HD) || n < 0 || n > 0x7fffffff) return 0;
  if (many_rows(T, H, HKV)) return prompt_workspace(B, T, H, HKV, HD, n, weigh != 0);
  return max(plan_of(B, T, H, HKV, HD, n, false, weigh != 0).bytes, plan_of(B, T, H, HKV, HD, n, true, weigh != 0).bytes);
}

extern "C" int bolt3_paged_attend(const bolt3_paged_attend_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_paged_attend");
  if (!a || !a->q || !a->pages || !a->table || !a->y) return BOLT3_ERR_ARG;
  if (a->lens != nullptr && a->pos_dev != nullptr) return BOLT3_ERR_ARG;
  if (a->pos_dev != nullptr && a->pos_span < 1) return BOLT3_ERR_ARG;
  if (!shape_ok(a->B, a->T, a->H, a->HKV, a->HD)) return BOLT3_ERR_SHAPE;
  Params p;
  if (!pages_ok(a->n_pages, a->page, a->width, a->table_stride, a->HKV, a->HD, &p.c.pages, a->table)) return BOLT3_ERR_SHAPE;
  const int64_t cap = a->width * a->page, dmax = a->pos_dev != nullptr ? a->pos_span - 1 : 0;
  if (a->n < 0 || a->n > cap - a->T - dmax) return BOLT3_ERR_CAPACITY;
  if (!(a->sm_scale > 0.f && a->sm_scale <= 3.4e38f)) return BOLT3_ERR_ARG;
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->pages | (uintptr_t)a->y | (uintptr_t)a->workspace;
  if ((al & 15) || ((a->q_sb | a->q_st) & 7)) return BOLT3_ERR_ALIGN;
  if (overwrites(*a)) return BOLT3_ERR_ARG;
  const int64_t n = a->n + dmax;                                // no sequence holds more before the call
  if (bolt3_paged_attend_workspace(a->B, a->T, a->H, a->HKV, a->HD, n, a->weight != nullptr) >
      (a->workspace != nullptr ? a->workspace_bytes : 0))
    return BOLT3_ERR_CAPACITY;
  p.c.a = *a;
  p.c.len = Length{a->lens, a->pos_dev, a->n, a->pos_ref, a->pos_span, n + a->T, a->T};
  p.c.G = a->H / a->HKV;
  p.c.rows = a->T * p.c.G;
  cudaStream_t s = (cudaStream_t)stream;
  if (many_rows(a->T, a->H, a->HKV)) return prompt_launch(p.c, s);
  if (!encode_pool(&p.map, a->pages, a->n_pages, a->page, a->HKV, a->HD, a->page < kBlock ? a->page : kBlock)) return BOLT3_ERR_CUDA;
  // blocks of the joins (a warp for each query row) and of the records
  if ((int64_t)a->B * a->HKV * (p.c.rows + (n + a->T + kRecordThreads - 1) / kRecordThreads) > 0x7fffffff) return BOLT3_ERR_SHAPE;
  const Plan pl = plan_of(a->B, a->T, a->H, a->HKV, a->HD, n, a->lens != nullptr, a->weight != nullptr);
  char* ws = reinterpret_cast<char*>(a->workspace);
  p.n_runs = pl.runs;
  p.apart = pl.apart;
  p.part = reinterpret_cast<float*>(ws + pl.part);
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
  p.span = reinterpret_cast<int2*>(ws + pl.span);
  p.lse = reinterpret_cast<float*>(ws + pl.lse);
  p.score = a->weight != nullptr ? reinterpret_cast<float*>(ws + pl.score) : nullptr;
  p.score_row = pl.score_row;
  p.most = n + a->T;
  if (a->HD == 128) return pl.nt == 1 ? launch_stream<128, 1>(p, pl, s) : launch_stream<128, 2>(p, pl, s);
  return pl.nt == 1 ? launch_stream<64, 1>(p, pl, s) : launch_stream<64, 2>(p, pl, s);
}
