// Softmax attention of new tokens over the 8-bit KV cache, for few query rows per KV head.
//
// For a query row and the keys j it sees, with t_j = sm_scale * scale_k[j] * (q . k8_j):
//   y = sum_j e^t_j scale_v[j] v8_j / sum_j e^t_j.
// The value scale goes into the exponent: u_j = t_j log2(e) + log2 scale_v[j], w_j = 2^(u_j - M) with M a
// bound on the u_j seen so far, numerator sum w_j v8_j, denominator sum w_j / scale_v[j]. So the f16 weights
// of the product are relative to the largest weighted value, however far the scales of two tokens lie apart.
// Sums and the outputs are fp32; w_j is rounded to f16 (2^-11 relative) for the product, the int8 operands
// are exact in f16, and a query row is brought to f16 by a power of two of its own (exact down to 2^-25 of
// its largest value).
//
// Bound by HBM: 2 (HD + 4) bytes per key and KV head. A CTA takes one (sequence, KV head), a share of its
// keys and 8 or 16 query rows (T * G of them, token-major). Each warp walks blocks of 16 keys on its own:
// K goes from global memory into the fragments of mma.sync m16n8k16 (S^T = K Q^T, keys in M, query rows in
// N: no padding for up to 8 rows) with the dimensions permuted so that a lane's 16 bytes feed four products;
// V likewise for O^T = V^T P^T with the output dimensions permuted. P^T is S^T transposed by movmatrix. No
// shared memory before the end, where the warps' partial sums are joined; the CTAs' partial sums of a split
// cache go through the workspace to a second kernel.
#include "../../include/bolt3.h"
#include "kv8.cuh"
#include "trace.h"

namespace {

using namespace b3;
using namespace kv8;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;   // a weight may exceed its bound by 2^8 before the bound moves: f16 holds 2^15

struct Params {
  bolt3_kv8_attend_args a;
  Length len;
  int G, rows, n_splits;
  float* part;                  // [column tile][chain][split][NC][HD] sums, then [..][NC] (M, l)
  float2* part_ml;
};

B3_DEV uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
B3_DEV uint2 ldg8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
B3_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
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
// the four f16 pairs (row A, row B) of two words' bytes: pairs of byte 0, 1, 2, 3
B3_DEV void s8x4_pairs(uint32_t wa, uint32_t wb, uint32_t (&p)[4]) {
  const uint32_t ua = wa ^ 0x80808080u, ub = wb ^ 0x80808080u;
  const uint32_t lo = __byte_perm(ua, ub, 0x5140), hi = __byte_perm(ua, ub, 0x7362);
  p[0] = __byte_perm(lo, 0x64646464u, 0x4140);
  p[1] = __byte_perm(lo, 0x64646464u, 0x4342);
  p[2] = __byte_perm(hi, 0x64646464u, 0x4140);
  p[3] = __byte_perm(hi, 0x64646464u, 0x4342);
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("sub.f16x2 %0, %0, %1;\n" : "+r"(p[i]) : "r"(0x64806480u));
}

// the bytes of one block of 16 keys that a lane holds
template <int HD>
struct KeyBlock {
  static constexpr int KC = HD / 64;      // 16-byte pieces of a key row per lane
  static constexpr int VW = HD / 32;      // words of a value row per lane
  uint4 k[2][KC];
  uint32_t v[4][VW];
  float ks[2], vs[2];
};

template <int HD, int NT>
__global__ void __launch_bounds__(kThreads) kv8_stream_kernel(const Params p) {
  constexpr int NC = 8 * NT;                                   // query rows of this CTA
  constexpr int KC = KeyBlock<HD>::KC, VW = KeyBlock<HD>::VW;
  constexpr int MT = HD / 16;                                  // 16-dimension tiles of the output
  extern __shared__ __align__(16) unsigned char smem[];
  const bolt3_kv8_attend_args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, tig = lane & 3;
  const int chain = blockIdx.x, split = blockIdx.y, tile = blockIdx.z;
  const int b = chain / a.HKV, kvh = chain % a.HKV;
  const int col0 = tile * NC;
  bool bad = false;
  const int64_t s = p.len.rows(b, bad);
  if (bad && tid == 0 && split == 0 && tile == 0 && a.status) atomicOr(a.status, 8);
  // keys that any row of this tile sees, in whole blocks of 16 shared among the splits
  const int last_row = min(col0 + NC, p.rows) - 1;
  const int64_t L = s < 0 ? 0 : s + last_row / p.G + 1;
  const int64_t blocks = (L + 15) / 16;
  const int64_t share = (blocks + p.n_splits - 1) / p.n_splits;
  const int64_t blk_lo = split * share, blk_hi = min(blocks, blk_lo + share);

  const int8_t* kd = a.data + (int64_t)chain * a.cap * HD;
  const int8_t* vd = kd + (int64_t)a.B * a.HKV * a.cap * HD;
  const float* ksc = a.scale + (int64_t)chain * a.cap;
  const float* vsc = ksc + (int64_t)a.B * a.HKV * a.cap;

  // row r of the tile is head kvh * G + r % G of token r / G
  auto q_row = [&](int r) {
    return reinterpret_cast<const bf16*>(a.q) + b * a.q_sb + (r / p.G) * a.q_st + (int64_t)(kvh * p.G + r % p.G) * HD;
  };
  // queries as B fragments: a lane holds row grp of each n8 tile, dimensions 16 (tig + 4 c) .. + 15
  uint32_t qf[NT][KC][8];
  float c0[NT], c1[NT];                        // sm_scale log2(e) 2^e of rows 2 tig and 2 tig + 1
  int64_t see0[NT], see1[NT];                  // keys these rows see
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = col0 + 8 * n + grp;
    float x[KC][16], m = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      uint4 r0 = make_uint4(0, 0, 0, 0), r1 = r0;
      if (r < p.rows && s >= 0) {
        const uint4* src = reinterpret_cast<const uint4*>(q_row(r) + 16 * (tig + 4 * c));
        r0 = src[0];
        r1 = src[1];
      }
      const uint32_t w[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = unpack_bf16(w[i]);
        x[c][2 * i] = f.x;
        x[c][2 * i + 1] = f.y;
        m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
    m = quad_max(m);
    // 2^-e brings the row's largest value into [1, 2): f16 keeps all of a bf16's bits down to 2^-17 of it
    const int e = m > 0.f && m < 3e38f ? max(ilogbf(m), -100) : 0;
    const float down = exp2f((float)-e);
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) qf[n][c][i] = pack_f16(x[c][2 * i] * down, x[c][2 * i + 1] * down);
    const float up = a.sm_scale * kLog2e * exp2f((float)e);
    c0[n] = __shfl_sync(0xffffffffu, up, 8 * tig);
    c1[n] = __shfl_sync(0xffffffffu, up, 8 * tig + 4);
    const int r0 = col0 + 8 * n + 2 * tig;
    see0[n] = s < 0 || r0 >= p.rows ? 0 : s + r0 / p.G + 1;
    see1[n] = s < 0 || r0 + 1 >= p.rows ? 0 : s + (r0 + 1) / p.G + 1;
  }

  auto load = [&](int64_t blk, KeyBlock<HD>& kb) {
    const int64_t key = blk * 16;
    const int64_t end = L - 1;                                 // rows past it are read as the last one and masked
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t row = min(key + grp + 8 * h, end);
#pragma unroll
      for (int c = 0; c < KC; ++c) kb.k[h][c] = ldg16(kd + row * HD + 16 * (tig + 4 * c));
      kb.ks[h] = __ldg(ksc + row);
      kb.vs[h] = __ldg(vsc + row);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t row = min(key + 2 * tig + (j & 1) + 8 * (j >> 1), end);
      if constexpr (VW == 4) {
        const uint4 x = ldg16(vd + row * HD + 16 * grp);
        kb.v[j][0] = x.x; kb.v[j][1] = x.y; kb.v[j][2] = x.z; kb.v[j][3] = x.w;
      } else {
        const uint2 x = ldg8(vd + row * HD + 8 * grp);
        kb.v[j][0] = x.x; kb.v[j][1] = x.y;
      }
    }
  };

  float o[MT][NT][4];
  float M0[NT], M1[NT], l0[NT], l1[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    M0[n] = M1[n] = neg_inf();
    l0[n] = l1[n] = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
  }

  KeyBlock<HD> next;
  int64_t blk = blk_lo + warp;
  if (blk < blk_hi) load(blk, next);
  for (; blk < blk_hi; blk += kWarps) {
    KeyBlock<HD> kb = next;
    if (blk + kWarps < blk_hi) load(blk + kWarps, next);
    // S^T = K Q^T for keys grp and grp + 8
    float st[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) st[n][0] = st[n][1] = st[n][2] = st[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const uint32_t wa[4] = {kb.k[0][c].x, kb.k[0][c].y, kb.k[0][c].z, kb.k[0][c].w};
      const uint32_t wb[4] = {kb.k[1][c].x, kb.k[1][c].y, kb.k[1][c].z, kb.k[1][c].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a0, a1, a2, a3;
        s8x4_to_f16(wa[w], a0, a2);
        s8x4_to_f16(wb[w], a1, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(st[n], a0, a1, a2, a3, qf[n][c][2 * w], qf[n][c][2 * w + 1]);
      }
    }
    const int64_t key = blk * 16 + grp;
    const float lga = log2f(kb.vs[0]), lgb = log2f(kb.vs[1]);
    const float iva = __frcp_rn(kb.vs[0]), ivb = __frcp_rn(kb.vs[1]);
    bool over = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      st[n][0] = key < see0[n] ? fmaf(st[n][0], kb.ks[0] * c0[n], lga) : neg_inf();
      st[n][1] = key < see1[n] ? fmaf(st[n][1], kb.ks[0] * c1[n], lga) : neg_inf();
      st[n][2] = key + 8 < see0[n] ? fmaf(st[n][2], kb.ks[1] * c0[n], lgb) : neg_inf();
      st[n][3] = key + 8 < see1[n] ? fmaf(st[n][3], kb.ks[1] * c1[n], lgb) : neg_inf();
      over |= fmaxf(st[n][0], st[n][2]) > M0[n] + kSlack || fmaxf(st[n][1], st[n][3]) > M1[n] + kSlack;
    }
    // the bounds move only when a weight would pass 2^8 (and at the first key a row sees)
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float m0 = fmaxf(st[n][0], st[n][2]), m1 = fmaxf(st[n][1], st[n][3]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
          m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
        }
        m0 = fmaxf(M0[n], m0);
        m1 = fmaxf(M1[n], m1);
        const float f0 = M0[n] == neg_inf() ? 0.f : exp2f(M0[n] - m0), f1 = M1[n] == neg_inf() ? 0.f : exp2f(M1[n] - m1);
        M0[n] = m0;
        M1[n] = m1;
        l0[n] *= f0;
        l1[n] *= f1;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          o[m][n][0] *= f0; o[m][n][2] *= f0;
          o[m][n][1] *= f1; o[m][n][3] *= f1;
        }
      }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float r0 = M0[n] == neg_inf() ? 0.f : M0[n], r1 = M1[n] == neg_inf() ? 0.f : M1[n];
      const float w0 = exp2f(st[n][0] - r0), w1 = exp2f(st[n][1] - r1), w2 = exp2f(st[n][2] - r0), w3 = exp2f(st[n][3] - r1);
      // a key that a row does not see has weight 0, whatever its scale holds
      l0[n] += (w0 == 0.f ? 0.f : w0 * iva) + (w2 == 0.f ? 0.f : w2 * ivb);
      l1[n] += (w1 == 0.f ? 0.f : w1 * iva) + (w3 == 0.f ? 0.f : w3 * ivb);
      pb[n][0] = transpose8(pack_f16(w0, w1));
      pb[n][1] = transpose8(pack_f16(w2, w3));
    }
    // O^T += V^T P^T: tile 2 w + i holds dimensions 16 grp + 4 w + 2 i (rows grp) and + 1 (rows grp + 8)
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      uint32_t u[4], v[4];
      s8x4_pairs(kb.v[0][w], kb.v[1][w], u);
      s8x4_pairs(kb.v[2][w], kb.v[3][w], v);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma_f16(o[2 * w + i][n], u[2 * i], u[2 * i + 1], v[2 * i], v[2 * i + 1], pb[n][0], pb[n][1]);
    }
  }

  // join the lanes' sums of weights (the bounds are the same in all lanes of a row), then the warps
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0[n] += __shfl_xor_sync(0xffffffffu, l0[n], x);
      l1[n] += __shfl_xor_sync(0xffffffffu, l1[n], x);
    }
  float* so = reinterpret_cast<float*>(smem);                  // [kWarps][NC][HD]
  float2* sml = reinterpret_cast<float2*>(so + kWarps * NC * HD);   // [kWarps][NC]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + 2 * tig;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int d = 4 * VW * grp + 2 * m;
      float* at = so + (warp * NC + r) * HD + d;
      *reinterpret_cast<float2*>(at) = make_float2(o[m][n][0], o[m][n][2]);
      *reinterpret_cast<float2*>(at + HD) = make_float2(o[m][n][1], o[m][n][3]);
    }
    if (grp == 0) {
      sml[warp * NC + r] = make_float2(M0[n], l0[n]);
      sml[warp * NC + r + 1] = make_float2(M1[n], l1[n]);
    }
  }
  __syncthreads();
  const int rows = min(NC, p.rows - col0);
  const int64_t slot = ((int64_t)tile * gridDim.x + chain) * p.n_splits + split;
  for (int i = tid; i < rows * HD; i += kThreads) {
    const int r = i / HD, d = i % HD;
    float m = neg_inf();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sml[w * NC + r].x);
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = sml[w * NC + r];
      const float f = ml.x == neg_inf() ? 0.f : exp2f(ml.x - m);
      acc = fmaf(so[(w * NC + r) * HD + d], f, acc);
      l = fmaf(ml.y, f, l);
    }
    if (p.n_splits == 1) {
      const int row = col0 + r;
      bf16* y = reinterpret_cast<bf16*>(a.y) + (((int64_t)b * a.T + row / p.G) * a.H + kvh * p.G + row % p.G) * HD;
      y[d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
    } else {
      p.part[(slot * NC + r) * HD + d] = acc;
      if (d == 0) p.part_ml[slot * NC + r] = make_float2(m, l);
    }
  }
}

// one block of HD threads per (chain, query row): the splits' partial sums joined
template <int HD, int NC>
__global__ void __launch_bounds__(HD) kv8_join_kernel(const Params p, int n_chains) {
  const bolt3_kv8_attend_args& a = p.a;
  const int chain = blockIdx.x, row = blockIdx.y, d = threadIdx.x;
  const int tile = row / NC, r = row % NC;
  const int64_t slot = ((int64_t)tile * n_chains + chain) * p.n_splits;
  float m = neg_inf();
  for (int i = 0; i < p.n_splits; ++i) m = fmaxf(m, p.part_ml[(slot + i) * NC + r].x);
  float acc = 0.f, l = 0.f;
  for (int i = 0; i < p.n_splits; ++i) {
    const float2 ml = p.part_ml[(slot + i) * NC + r];
    if (ml.x == neg_inf() && ml.y == 0.f) continue;
    const float f = ml.x == neg_inf() ? 0.f : exp2f(ml.x - m);
    acc = fmaf(p.part[((slot + i) * NC + r) * HD + d], f, acc);
    l = fmaf(ml.y, f, l);
  }
  const int b = chain / a.HKV, kvh = chain % a.HKV;
  bf16* y = reinterpret_cast<bf16*>(a.y) + (((int64_t)b * a.T + row / p.G) * a.H + kvh * p.G + row % p.G) * HD;
  y[d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
}

// columns of a CTA, column tiles and splits of a call
struct Plan {
  int nt, tiles, splits;
  size_t bytes;
};

Plan plan_of(int B, int T, int H, int HKV, int HD, int64_t n) {
  Plan pl;
  const int64_t rows = (int64_t)T * (H / HKV), chains = (int64_t)B * HKV;
  pl.nt = rows <= 8 ? 1 : 2;
  pl.tiles = (int)((rows + 8 * pl.nt - 1) / (8 * pl.nt));
  // as many splits as fill 148 SMs with four CTAs each, none under 64 keys per CTA
  const int64_t want = (148 * 4 + chains * pl.tiles - 1) / (chains * pl.tiles);
  const int64_t most = (n + T + 63) / 64;
  int64_t sp = want < most ? want : most;
  pl.splits = (int)(sp < 1 ? 1 : sp);
  pl.bytes = 0;
  if (pl.splits > 1)
    pl.bytes = (size_t)pl.tiles * (size_t)chains * (size_t)pl.splits * (size_t)(8 * pl.nt) * ((size_t)HD * 4 + 8);
  return pl;
}

template <int HD, int NT>
int launch_stream(Params& p, const Plan& pl, cudaStream_t s) {
  constexpr int NC = 8 * NT;
  constexpr size_t smem = (size_t)kWarps * NC * (HD * 4 + 8);
  const int chains = p.a.B * p.a.HKV;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kv8_stream_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  p.part = reinterpret_cast<float*>(p.a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part + (size_t)pl.tiles * chains * pl.splits * NC * HD);
  kv8_stream_kernel<HD, NT><<<dim3((unsigned)chains, (unsigned)pl.splits, (unsigned)pl.tiles), kThreads, smem, s>>>(p);
  if (cudaGetLastError() != cudaSuccess) return BOLT3_ERR_CUDA;
  if (pl.splits > 1) {
    kv8_join_kernel<HD, NC><<<dim3((unsigned)chains, (unsigned)p.rows), HD, 0, s>>>(p, chains);
    if (cudaGetLastError() != cudaSuccess) return BOLT3_ERR_CUDA;
  }
  return BOLT3_OK;
}

bool shape_ok(int B, int T, int H, int HKV, int HD) {
  return B > 0 && T > 0 && HKV > 0 && H > 0 && H % HKV == 0 && H / HKV <= 16 && (HD == 64 || HD == 128) &&
         T <= 65535 / (H / HKV) && (int64_t)B * HKV <= 0x7fffffff;
}

}  // namespace

extern "C" size_t bolt3_kv8_attend_workspace(int B, int T, int H, int HKV, int HD, int64_t n) {
  if (!shape_ok(B, T, H, HKV, HD) || n < 0) return 0;
  return plan_of(B, T, H, HKV, HD, n).bytes;
}

extern "C" int bolt3_kv8_attend(const bolt3_kv8_attend_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_kv8_attend");
  if (!a || !a->q || !a->data || !a->scale || !a->y) return BOLT3_ERR_ARG;
  if (a->lens != nullptr && a->pos_dev != nullptr) return BOLT3_ERR_ARG;
  if (a->pos_dev != nullptr && a->pos_span < 1) return BOLT3_ERR_ARG;
  if (!shape_ok(a->B, a->T, a->H, a->HKV, a->HD)) return BOLT3_ERR_SHAPE;
  const int64_t dmax = a->pos_dev != nullptr ? a->pos_span - 1 : 0;
  if (a->n < 0 || a->cap < a->T || (a->lens == nullptr && a->n > a->cap - a->T - dmax)) return BOLT3_ERR_CAPACITY;
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->data | (uintptr_t)a->scale | (uintptr_t)a->y | (uintptr_t)a->workspace;
  if ((al & 15) || ((a->q_sb | a->q_st) & 7)) return BOLT3_ERR_ALIGN;
  const Plan pl = plan_of(a->B, a->T, a->H, a->HKV, a->HD, a->n);
  if (pl.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < pl.bytes)) return BOLT3_ERR_CAPACITY;
  Params p;
  p.a = *a;
  p.len = Length{a->lens, a->pos_dev, a->n, a->pos_ref, a->pos_span, a->cap, a->T};
  p.G = a->H / a->HKV;
  p.rows = a->T * p.G;
  p.n_splits = pl.splits;
  cudaStream_t s = (cudaStream_t)stream;
  if (a->HD == 128) return pl.nt == 1 ? launch_stream<128, 1>(p, pl, s) : launch_stream<128, 2>(p, pl, s);
  return pl.nt == 1 ? launch_stream<64, 1>(p, pl, s) : launch_stream<64, 2>(p, pl, s);
}
