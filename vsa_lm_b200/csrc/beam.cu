// Beam search on the device: the selection over beams and vocabulary, and the reordering of decode states.
//
// select. With lse_k = log sum_v e^x_kv, continuation (k, v) scores s_k + (x_kv - lse_k); the K best of a
// group's K * V survive. Bound by HBM: the logits are read once. Within a beam the order is the logits',
// so the pass that sums the exponentials also finds each chunk's K best logits:
// - select_chunk_kernel: a block holds a chunk of 8192 logits of one row in registers. Maximum and sum of exponentials,
//   then a threshold: the K-th largest of the maxima of 16 columns of threads is no larger than the chunk's K-th largest
//   logit, so the few logits at or above it contain the K best; they are ranked by counting. Chunks with many equal
//   logits (more than the list holds) take K rounds of a block maximum instead.
// - select_group_kernel: a block per group merges the chunks' sums and lists, a warp per beam, and then the beams' lists:
//   both are sorted, so a lane stands at the head of a list and the best head of the warp is next (8 x 16 beams of 34000
//   fp32 logits: 31 us; with all K^2 continuations ranked by counting 38).
// Measured on a B200: 64 x 4 beams of 151936 bf16 logits, a fifth finished, 24 us (2.6 TB/s; see below what it is busy
// with); 64 x 16 beams of 34000 fp32 logits 57 us (2.5 TB/s); 1 x 4 of 32000 fp32 8 us (two launches and their latency).
// reorder. Bound by HBM: the bytes of every beam that is not its own parent are read from the parent and
// written, in place for any map: where a parent is moved itself, a thread holds its bytes of all parents of the
// group before it writes any; where none is (the maps that select gives), beams are copied one by one, eight
// 16-byte loads ahead. Blocks cover the items' bytes flattened, so that many small arrays are one launch. Measured:
// 16 x 4 beams, a Bolt-3 layer's state and 256 tokens of an anchor cache in one launch, 23 us (6.0 TB/s).
#include "../../include/bolt3.h"
#include "common.cuh"
#include "trace.h"

namespace {

using namespace b3;

constexpr int kMaxK = 16;
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------------------------------- select

// Blocks of four warps, ten on an SM (blocks of eight with chunks of 16384, five on an SM, take the same time). At 256 rows
// of 151936 bf16 logits, a fifth of them finished, the kernel is busy for 14.5 us: exponentials 7.3, instructions 7.7, DRAM
// 9.5 of them
constexpr int kSelThreads = 128;
constexpr int kPerThread = 64;
constexpr int kChunk = kSelThreads * kPerThread;      // logits of a block
template <bool FP32>
constexpr int kSelBlocks = FP32 ? 5 : 10;             // of an SM
constexpr int kListCap = 256;                         // candidates at or above the threshold
constexpr int64_t kMaxV = 64 * kChunk;
constexpr int kMaxChunks = 65;                        // of a row, which may begin after a 16-byte boundary

struct Cand {
  float x;
  int32_t v;
};
// a before b in the order of a row: larger logit, then lower index
B3_DEV bool before(Cand a, Cand b) { return a.x > b.x || (a.x == b.x && a.v < b.v); }

// the number of candidates of the list before c
B3_DEV int rank_of(Cand c, const Cand* list, int count) {
  int rank = 0;
#pragma unroll 4
  for (int i = 0; i < count; ++i) rank += before(list[i], c);
  return rank;
}

struct SelParams {
  bolt3_beam_select_args a;
  int n_chunks;
  float2* sums;       // [B * K][n_chunks] (maximum, sum of e^(x - maximum))
  Cand* cands;        // [B * K][n_chunks][K], best first, v = -1 where there are fewer
};

// the row has continuations of its own (its logits count)
B3_DEV bool row_live(const bolt3_beam_select_args& a, int64_t r) {
  return !(a.finished != nullptr && a.finished[r]) && a.scores[r] > neg_inf();
}

B3_DEV float ex2(float x) {      // 2^x, relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
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
B3_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// the larger of two bf16 pairs, a number before a NaN
B3_DEV uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A thread's logits as they were loaded: words of one fp32 or two bf16
template <bool FP32>
struct Logits {
  static constexpr int EPL = FP32 ? 4 : 8;            // logits of a 16-byte load
  static constexpr int NW = FP32 ? 64 : 32;
  static constexpr uint32_t kNone = FP32 ? 0xff800000u : 0xff80ff80u;   // -infinity in every place
  uint32_t w[NW];
  B3_DEV float largest() const {                      // NaNs left out
    if constexpr (FP32) {
      float m = neg_inf();
#pragma unroll
      for (int i = 0; i < NW; ++i) m = fmaxf(m, __uint_as_float(w[i]));
      return m;
    } else {
      uint32_t m = kNone;
#pragma unroll
      for (int i = 0; i < NW; ++i) m = max_bf16x2(m, w[i]);
      const float2 f = unpack_bf16(m);
      return fmaxf(f.x, f.y);
    }
  }
  B3_DEV float x(int i) const {
    if constexpr (FP32) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  // of logits 32 h .. 32 h + 31: a bit for every one at or above t, a bf16 value where they are
  B3_DEV uint32_t at_least(float t, int h) const {
    uint32_t mask = 0;
    if constexpr (FP32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) mask |= __uint_as_float(w[32 * h + i]) >= t ? 1u << i : 0u;
    } else {
      const __nv_bfloat162 tt = __float2bfloat162_rn(t);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        mask |= __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w[16 * h + i]), tt) & (0x10001u << i);
    }
    return mask;
  }
  static B3_DEV int of_bit(int bit, int h) { return 32 * h + (FP32 ? bit : (bit & 15) * 2 + (bit >> 4)); }
};

template <bool FP32>
__global__ void __launch_bounds__(kSelThreads, kSelBlocks<FP32>) select_chunk_kernel(const __grid_constant__ SelParams p) {
  using L = Logits<FP32>;
  constexpr int EPL = L::EPL, kBytes = FP32 ? 4 : 2, kPer = kPerThread;
  __shared__ float s_max[kSelThreads / 2], s_sum[kSelThreads / 32];
  __shared__ int s_count;
  __shared__ Cand s_list[kListCap];
  const bolt3_beam_select_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x, item = r * p.n_chunks + blockIdx.y;
  // Chunks are cut at 16-byte boundaries whatever the row's alignment: logit e of the chunk is logit lo + e of the row,
  // lo < 0 where the row begins within the chunk's first 16 bytes
  const char* row = reinterpret_cast<const char*>(a.logits) + r * a.row_stride * kBytes;
  const int lo = (int)blockIdx.y * kChunk - (int)(reinterpret_cast<uintptr_t>(row) & 15) / kBytes;
  row += (int64_t)lo * kBytes;
  const int from = max(0, -lo), n = min(kChunk, (int)a.V - lo);   // logits of the chunk: [from, n)
  grid_dep_launch();
  grid_dep_wait();
  if (!row_live(a, r)) return;
  auto bits = [&](int e) {
    if constexpr (FP32) return reinterpret_cast<const uint32_t*>(row)[e];
    else return (uint32_t) reinterpret_cast<const uint16_t*>(row)[e];
  };
  auto value = [&](int e) { return __uint_as_float(FP32 ? bits(e) : bits(e) << 16); };
  auto place = [&](int i) { return ((i / EPL) * kSelThreads + tid) * EPL + i % EPL; };   // of a thread's logit i in the chunk
  L l;
#pragma unroll
  for (int i = 0; i < L::NW / 4; ++i) {
    const int e = (i * kSelThreads + tid) * EPL;
    uint4 q = make_uint4(L::kNone, L::kNone, L::kNone, L::kNone);
    if (e >= from && e + EPL <= n) {
      q = __ldcs(reinterpret_cast<const uint4*>(row + (int64_t)e * kBytes));
    } else if (e + EPL > from && e < n) {             // the row's first or last 16 bytes
      uint32_t w[4] = {L::kNone, L::kNone, L::kNone, L::kNone};
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (e + j >= from && e + j < n) {
          if constexpr (FP32) w[j] = bits(e + j);
          else w[j / 2] = j & 1 ? (w[j / 2] & 0xffffu) | bits(e + j) << 16 : (w[j / 2] & 0xffff0000u) | bits(e + j);
        }
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    l.w[4 * i] = q.x; l.w[4 * i + 1] = q.y; l.w[4 * i + 2] = q.z; l.w[4 * i + 3] = q.w;
  }
  // every thread sums against its own maximum: nothing here waits for another warp. The exponents are x log2(e) - off with
  // off = m log2(e) rounded, whose remainder (up to 64 at the bound) is the same for all of them and taken out of the sum.
  // From 2^30 on, fp32 neighbours are 64 apart: what is below m adds nothing, and the sum is the number of logits equal to m
  const float m = l.largest();
  float sum = 0.f;
  if (fabsf(m) >= 0x1p30f) {
    if (m > neg_inf()) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum += l.x(i) == m ? 1.f : 0.f;
    }
  } else {
    const float off = m * kLog2e;
    const uint64_t l2e = pair(kLog2e, kLog2e), minus = pair(-off, -off);
    uint64_t s0 = 0, s1 = 0;
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const float2 u = unpair(fma2(pair(l.x(i), l.x(i + 1)), l2e, minus));
      const float2 v = unpair(fma2(pair(l.x(i + 2), l.x(i + 3)), l2e, minus));
      s0 = add2(s0, pair(ex2(u.x), ex2(u.y)));
      s1 = add2(s1, pair(ex2(v.x), ex2(v.y)));
    }
    const float2 u = unpair(add2(s0, s1));
    sum = u.x + u.y;
    if (sum != sum) {                                 // NaNs among the logits count as -infinity
      sum = 0.f;
#pragma unroll 1
      for (int i = 0; i < kPer; ++i)
        if (place(i) >= from && place(i) < n) sum += ex2(fmaf(fmaxf(value(place(i)), neg_inf()), kLog2e, -off));
    }
    sum *= ex2(-fmaf(m, kLog2e, -off));
  }
  // column c: the threads tid = c mod 16, all of them with logits once 16 threads have some
  const float col = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
  if (lane < 16) s_max[warp * 16 + lane] = col;
  if (tid == 0) s_count = 0;
  __syncthreads();
  // tau: the K-th largest of the 16 columns' maxima, found by lane i as the one that K - 1 others are ahead of
  float own = neg_inf();
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) own = fmaxf(own, s_max[i * 16 + (lane & 15)]);
  int rank = 0;
  float top = own;
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    const float o = __shfl_xor_sync(0xffffffffu, own, i);
    rank += o > own || (o == own && ((lane ^ i) & 15) < (lane & 15));
    top = fmaxf(top, o);
  }
  const float tau = __shfl_sync(0xffffffffu, own, __ffs(__ballot_sync(0xffffffffu, rank == a.K - 1)) - 1);
  sum = warp_sum(m > neg_inf() ? sum * ex2((m - top) * kLog2e) : 0.f);
  if (lane == 0) s_sum[warp] = sum;
  const bool any = m >= tau && m > neg_inf();
  const unsigned some = __ballot_sync(0xffffffffu, any);
  if (some != 0) {                                    // the list's order does not matter: it is ranked below
    int at = 0;
    if (lane == 0) at = atomicAdd(&s_count, __popc(some));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(some & ((1u << lane) - 1));
    if (any) {
      // tau is one of the logits, or -infinity: then any logit above that counts
      const float t = tau > neg_inf() ? tau : FP32 ? -3.4028235e38f : -3.3895314e38f;
      uint32_t mask[2] = {l.at_least(t, 0), l.at_least(t, 1)};
      const bool one = __popc(mask[0]) + __popc(mask[1]) == 1;       // then it is the largest
#pragma unroll
      for (int h = 0; h < 2; ++h)
        for (; mask[h]; mask[h] &= mask[h] - 1) {
          const int e = place(L::of_bit(__ffs(mask[h]) - 1, h));
          if (at < 0) at = atomicAdd(&s_count, 1);    // the place of a thread's first is taken above
          if (at < kListCap) s_list[at] = Cand{one ? m : value(e), lo + e};
          at = -1;
        }
    }
  }
  __syncthreads();
  const int count = s_count;
  Cand* out = p.cands + item * a.K;
  if (tid == 0) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kSelThreads / 32; ++i) t += s_sum[i];
    p.sums[item] = make_float2(top, t);
  }
  if (count <= kListCap) {
    for (int j = tid; j < count; j += kSelThreads) {
      const Cand c = s_list[j];
      const int better = rank_of(c, s_list, count);
      if (better < a.K) out[better] = c;
    }
    if (tid >= count && tid < a.K) out[tid] = Cand{neg_inf(), -1};
    return;
  }
  // many equal logits: K rounds, each the best candidate after the last one
  Cand last{__int_as_float(0x7f800000), -1};
#pragma unroll 1
  for (int k = 0; k < a.K; ++k) {
    Cand best{neg_inf(), 0x7fffffff};
#pragma unroll 1
    for (int i = 0; i < kPer; ++i) {
      if (place(i) < from || place(i) >= n) continue;
      const Cand c{value(place(i)), lo + place(i)};
      if (c.x > neg_inf() && before(last, c) && before(c, best)) best = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Cand c{__shfl_xor_sync(0xffffffffu, best.x, o), __shfl_xor_sync(0xffffffffu, best.v, o)};
      if (before(c, best)) best = c;
    }
    __syncthreads();
    if (lane == 0) s_list[warp] = best;
    __syncthreads();
    best = s_list[0];
    for (int i = 1; i < kSelThreads / 32; ++i)
      if (before(s_list[i], best)) best = s_list[i];
    last = best;
    if (tid == 0) out[k] = best;                      // more than kListCap are above -infinity: all K exist
  }
}

// a block per group, a warp per beam for the merge of its chunks
__global__ void __launch_bounds__(32 * kMaxK) select_group_kernel(const __grid_constant__ SelParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float c_score[kMaxK * kMaxK];
  __shared__ int32_t c_token[kMaxK * kMaxK];
  __shared__ bool s_done[kMaxK];
  const bolt3_beam_select_args& a = p.a;
  const int K = a.K, tid = threadIdx.x, lane = tid & 31, k = tid >> 5;
  const int64_t b = blockIdx.x, r = b * K + k;
  const int per_row = p.n_chunks * K;
  Cand* all = reinterpret_cast<Cand*>(smem) + (size_t)k * per_row;
  grid_dep_launch();
  grid_dep_wait();
  const bool done = a.finished != nullptr && a.finished[r];
  const float own = a.scores[r];
  if (lane == 0) s_done[k] = done;       // the outputs may be the inputs: nothing of these is read later
  if (!done && own > neg_inf()) {
    for (int i = lane; i < per_row; i += 32) all[i] = p.cands[r * per_row + i];
    float m = neg_inf();
    for (int i = lane; i < p.n_chunks; i += 32) m = fmaxf(m, p.sums[r * p.n_chunks + i].x);
    m = warp_max(m);
    float s = 0.f;
    for (int i = lane; i < p.n_chunks; i += 32) {
      const float2 c = p.sums[r * p.n_chunks + i];
      if (c.x > neg_inf()) s += c.y * exp2f((c.x - m) * kLog2e);
    }
    s = warp_sum(s);
    // The log-sum-exp m + log s is rounded to 2^-18 or better for logits below 64, which also takes up in which order the
    // sum was made (it goes by the row's alignment); larger ones would round log s away and are measured from m
    const float log_s = logf(s), lse = m + log_s;
    const bool from_m = !(fabsf(m) < 64.f);
    __syncwarp();
    // each lane walks the sorted lists of three chunks (at most 65 in all), their heads in registers; the order is (logit,
    // lowest index) as a pair of integers (x + 0 makes one of the two zeros; key 0 is the end of a list)
    int at[3];
    uint32_t key[3];
    Cand head[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      at[j] = (lane + 32 * j) * K;
      head[j] = lane + 32 * j < p.n_chunks ? all[at[j]] : Cand{neg_inf(), -1};
      key[j] = head[j].v >= 0 ? fkey(head[j].x + 0.f) : 0;
    }
    int n = 0;
    for (; n < K; ++n) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(key[0], key[1]), key[2]));
      if (top == 0) break;
      uint32_t low = 0xffffffffu;
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (key[j] == top) low = min(low, (uint32_t)head[j].v);
      const uint32_t win = __reduce_min_sync(0xffffffffu, low);
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (key[j] == top && (uint32_t)head[j].v == win) {
          const float sc = own + (from_m ? (head[j].x - m) - log_s : head[j].x - lse);
          c_score[k * K + n] = sc != sc ? neg_inf() : sc;
          c_token[k * K + n] = (int32_t)win;
          head[j] = ++at[j] < (lane + 32 * j + 1) * K ? all[at[j]] : Cand{neg_inf(), -1};
          key[j] = head[j].v >= 0 ? fkey(head[j].x + 0.f) : 0;
        }
    }
    if (lane >= n && lane < K) c_score[k * K + lane] = neg_inf();
  } else if (lane < K) {
    const float sc = done && lane == 0 ? own : neg_inf();
    c_score[k * K + lane] = sc != sc ? neg_inf() : sc;
    c_token[k * K + lane] = (int32_t)a.eos_ids[0];
  }
  __syncthreads();
  if (tid >= 32) return;
  // the K best of the beams' sorted lists: lane k stands at beam k's list; the order is score, then beam, then place in it
  int at = lane * K, c = -1;             // lane i gets the candidate of rank i
  auto head = [&] {
    const float x = lane < K && at < (lane + 1) * K ? c_score[at] : neg_inf();
    return x > neg_inf() ? fkey(x + 0.f) : 0;
  };
  uint32_t key = head();
  for (int i = 0; i < K; ++i) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, key);
    if (best == 0) break;
    const int from = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
    const int pick = __shfl_sync(0xffffffffu, at, from);
    if (lane == i) c = pick;
    if (lane == from) {
      ++at;
      key = head();
    }
  }
  // lane i: the continuation of rank i. The first child of a parent takes the parent's slot, the others what is left
  const int par = c < 0 ? 32 + lane : c / K;
  const unsigned same = __match_any_sync(0xffffffffu, par);
  const bool first = c >= 0 && __ffs(same) - 1 == lane;
  const unsigned held = __reduce_or_sync(0xffffffffu, first ? 1u << par : 0u);
  const unsigned later = __ballot_sync(0xffffffffu, c >= 0 && !first);
  int slot = par;
  if (c >= 0 && !first) {
    unsigned left = ~held;
    for (int i = __popc(later & ((1u << lane) - 1)); i > 0; --i) left &= left - 1;
    slot = __ffs(left) - 1;
  }
  const unsigned used = __reduce_or_sync(0xffffffffu, c >= 0 ? 1u << slot : 0u);
  if (lane < K && !(used >> lane & 1)) {
    a.out_scores[b * K + lane] = neg_inf();
    a.out_parent[b * K + lane] = lane;
    a.out_token[b * K + lane] = a.n_eos > 0 ? a.eos_ids[0] : 0;
    a.out_finished[b * K + lane] = 1;
  }
  if (c >= 0) {
    const int64_t o = b * K + slot, tok = c_token[c];
    bool fin = s_done[par];
    for (int e = 0; e < a.n_eos; ++e) fin |= tok == a.eos_ids[e];
    a.out_scores[o] = c_score[c];
    a.out_parent[o] = par;
    a.out_token[o] = tok;
    a.out_finished[o] = fin;
  }
}

size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }

// ------------------------------------------------------------------------------------------- reorder

constexpr int kMoveThreads = 256;
constexpr int kMaxItems = 128;

struct MoveItem {
  unsigned char* base;
  int64_t outer_stride, beam_stride, row_stride;
  int64_t lo;                         // first byte of a row
  int64_t units;                      // n_row * units_per_row
  uint32_t row_units;                 // units of a row
  int32_t unit;
  uint32_t first_block, blocks;       // of one (outer, group)
};

struct MoveParams {
  const int32_t* parent;
  int32_t* status;
  int K, B, n_items;
  MoveItem item[kMaxItems];
};

constexpr int kMoveAhead = 8;         // units of a thread

// off: byte offset of a thread's unit u within a beam, -1 past the end
template <typename V, int KM>
B3_DEV void move_units(const MoveItem& it, unsigned char* group, uint32_t blk, const int (&par)[KM], unsigned moved, bool chained) {
  int64_t off[kMoveAhead];
#pragma unroll
  for (int u = 0; u < kMoveAhead; ++u) {
    const int64_t i = (int64_t)blk * (kMoveThreads * kMoveAhead) + u * kMoveThreads + threadIdx.x;
    if (it.units == it.row_units) {
      off[u] = i < it.units ? it.lo + i * (int64_t)sizeof(V) : -1;
    } else {
      const int64_t r = i / it.row_units;
      off[u] = i < it.units ? r * it.row_stride + it.lo + (i - r * it.row_units) * (int64_t)sizeof(V) : -1;
    }
  }
  if (chained) {
#pragma unroll 1
    for (int u = 0; u < kMoveAhead; ++u) {
      int64_t at = -1;
#pragma unroll
      for (int x = 0; x < kMoveAhead; ++x)
        if (x == u) at = off[x];
      if (at < 0) continue;
      V v[KM];
#pragma unroll
      for (int j = 0; j < KM; ++j)
        if (moved >> j & 1) v[j] = *reinterpret_cast<const V*>(group + par[j] * it.beam_stride + at);
#pragma unroll
      for (int j = 0; j < KM; ++j)
        if (moved >> j & 1) *reinterpret_cast<V*>(group + j * it.beam_stride + at) = v[j];
    }
    return;
  }
#pragma unroll 1
  for (int j = 0; j < KM; ++j) {
    if (!(moved >> j & 1)) continue;
    int from = 0;
#pragma unroll
    for (int x = 0; x < KM; ++x)
      if (x == j) from = par[x];
    const unsigned char* src = group + from * it.beam_stride;
    unsigned char* dst = group + j * it.beam_stride;
    V v[kMoveAhead];
#pragma unroll
    for (int u = 0; u < kMoveAhead; ++u)
      if (off[u] >= 0) v[u] = *reinterpret_cast<const V*>(src + off[u]);
#pragma unroll
    for (int u = 0; u < kMoveAhead; ++u)
      if (off[u] >= 0) *reinterpret_cast<V*>(dst + off[u]) = v[u];
  }
}

template <int KM>
__global__ void __launch_bounds__(kMoveThreads) reorder_kernel(const __grid_constant__ MoveParams p) {
  grid_dep_launch();
  grid_dep_wait();
  // the item of this block: the last one that starts at or before it
  int lo = 0, hi = p.n_items - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.item[mid].first_block <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const MoveItem& it = p.item[lo];
  const uint32_t local = blockIdx.x - it.first_block;
  const uint32_t blk = local % it.blocks, og = local / it.blocks;
  const int g = (int)(og % p.B), outer = (int)(og / p.B);
  int par[KM];
  unsigned moved = 0;
#pragma unroll
  for (int j = 0; j < KM; ++j) {
    par[j] = j;
    if (j < p.K) {
      const int q = p.parent[(int64_t)g * p.K + j];
      if (q < 0 || q >= p.K) {
        if (threadIdx.x == 0 && p.status) atomicOr(p.status, 8);
      } else if (q != j) {
        par[j] = q;
        moved |= 1u << j;
      }
    }
  }
  if (moved == 0) return;
  unsigned char* group = it.base + outer * it.outer_stride + (int64_t)g * p.K * it.beam_stride;
  bool chained = false;                 // whether a parent is moved itself
#pragma unroll
  for (int j = 0; j < KM; ++j) chained |= (moved >> par[j] & 1) && (moved >> j & 1);
  if (it.unit == 16) move_units<uint4, KM>(it, group, blk, par, moved, chained);
  else if (it.unit == 4) move_units<uint32_t, KM>(it, group, blk, par, moved, chained);
  else move_units<unsigned char, KM>(it, group, blk, par, moved, chained);
}

template <int KM>
int launch_reorder(const MoveParams& p, uint32_t blocks, cudaStream_t s) {
  return launch_overlapped(reorder_kernel<KM>, dim3(blocks), dim3(kMoveThreads), 0, s, p) == cudaSuccess ? BOLT3_OK : BOLT3_ERR_CUDA;
}

}  // namespace

extern "C" size_t bolt3_beam_select_workspace(int B, int K, int64_t V) {
  if (B <= 0 || K <= 0 || K > kMaxK || V <= 0 || V > kMaxV) return 0;
  const size_t rows = (size_t)B * K, nc = (size_t)((V + 7 + kChunk - 1) / kChunk);
  return align16(rows * nc * sizeof(float2)) + align16(rows * nc * K * sizeof(Cand));
}

extern "C" int bolt3_beam_select(const bolt3_beam_select_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_beam_select");
  if (!a || !a->logits || !a->scores || !a->out_scores || !a->out_parent || !a->out_token || !a->out_finished)
    return BOLT3_ERR_ARG;
  if (a->n_eos < 0 || a->n_eos > 8) return BOLT3_ERR_ARG;
  if (a->finished != nullptr && a->n_eos == 0) return BOLT3_ERR_ARG;   // a finished beam goes on with eos_ids[0]
  if (a->B <= 0 || a->K <= 0 || a->K > kMaxK || a->V <= 0 || a->V > kMaxV || (int64_t)a->B * a->K > 0x1ffffff)
    return BOLT3_ERR_SHAPE;
  if (a->row_stride < a->V) return BOLT3_ERR_CAPACITY;
  const uintptr_t el = a->logits_fp32 ? 3 : 1;
  if (((uintptr_t)a->logits & el) || ((uintptr_t)a->workspace & 15)) return BOLT3_ERR_ALIGN;
  if (!a->workspace || a->workspace_bytes < bolt3_beam_select_workspace(a->B, a->K, a->V)) return BOLT3_ERR_CAPACITY;
  for (int i = 0; i < a->n_eos; ++i)
    if (a->eos_ids[i] < 0 || a->eos_ids[i] >= a->V) return BOLT3_ERR_ARG;
  SelParams p;
  p.a = *a;
  const int slip = a->logits_fp32 ? 3 : 7;            // logits by which a row may begin after a 16-byte boundary
  p.n_chunks = (int)((a->V + slip + kChunk - 1) / kChunk);
  const size_t rows = (size_t)a->B * a->K;
  p.sums = reinterpret_cast<float2*>(a->workspace);
  p.cands = reinterpret_cast<Cand*>(reinterpret_cast<char*>(a->workspace) + align16(rows * p.n_chunks * sizeof(float2)));
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid((unsigned)rows, (unsigned)p.n_chunks);
  if (launch_overlapped(a->logits_fp32 ? select_chunk_kernel<true> : select_chunk_kernel<false>, grid, dim3(kSelThreads), 0,
                        s, p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  // the limit is the largest call's, not this one's: it is the kernel's, and another thread may set it before this launch
  const size_t smem = (size_t)a->K * p.n_chunks * a->K * sizeof(Cand);
  if (smem > 40 * 1024 &&
      cudaFuncSetAttribute(select_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)(kMaxK * kMaxK * kMaxChunks * sizeof(Cand))) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  return launch_overlapped(select_group_kernel, dim3((unsigned)a->B), dim3(32 * a->K), smem, s, p) == cudaSuccess
             ? BOLT3_OK : BOLT3_ERR_CUDA;
}

extern "C" int bolt3_beam_reorder(const bolt3_beam_reorder_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_beam_reorder");
  if (!a || !a->parent || (a->n_items > 0 && !a->items) || a->n_items < 0) return BOLT3_ERR_ARG;
  if (a->B <= 0 || a->K <= 0 || a->K > kMaxK) return BOLT3_ERR_SHAPE;
  if (a->t0 < 0 || a->t1 < a->t0) return BOLT3_ERR_ARG;
  for (int i = 0; i < a->n_items; ++i) {
    const bolt3_beam_item& it = a->items[i];
    if (!it.base || it.n_outer <= 0 || it.n_row <= 0 || it.row_bytes <= 0 || it.token_bytes < 0) return BOLT3_ERR_ARG;
    if (it.unit != 1 && it.unit != 4 && it.unit != 16) return BOLT3_ERR_ARG;
    if (it.token_bytes > 0 && a->t1 > it.row_bytes / it.token_bytes) return BOLT3_ERR_CAPACITY;
    const int64_t m = it.outer_stride | it.beam_stride | it.row_stride | it.token_bytes |
                      (it.token_bytes > 0 ? 0 : it.row_bytes) | (int64_t)(uintptr_t)it.base;
    if (m & (it.unit - 1)) return BOLT3_ERR_ALIGN;
  }
  const int km = a->K <= 4 ? 4 : a->K <= 8 ? 8 : 16;
  const int per_block = kMoveThreads * kMoveAhead;
  cudaStream_t s = (cudaStream_t)stream;
  MoveParams p;
  p.parent = a->parent;
  p.status = a->status;
  p.K = a->K;
  p.B = a->B;
  int i = 0;
  while (i < a->n_items) {
    uint64_t blocks = 0;
    p.n_items = 0;
    for (; i < a->n_items && p.n_items < kMaxItems; ++i) {
      const bolt3_beam_item& it = a->items[i];
      const int64_t lo = it.token_bytes > 0 ? a->t0 * it.token_bytes : 0;
      const int64_t bytes = it.token_bytes > 0 ? (a->t1 - a->t0) * it.token_bytes : it.row_bytes;
      if (bytes == 0) continue;
      MoveItem m;
      m.base = reinterpret_cast<unsigned char*>(it.base);
      m.outer_stride = it.outer_stride; m.beam_stride = it.beam_stride; m.row_stride = it.row_stride;
      m.lo = lo;
      m.unit = it.unit;
      if (bytes / it.unit > 0x7fffffff) return BOLT3_ERR_SHAPE;
      m.row_units = (uint32_t)(bytes / it.unit);
      m.units = (int64_t)m.row_units * it.n_row;
      const uint64_t nb = (uint64_t)((m.units + per_block - 1) / per_block);
      const uint64_t total = nb * (uint64_t)it.n_outer * (uint64_t)a->B;
      if (nb > 0x7fffffff || total > 0x7fffffff) return BOLT3_ERR_SHAPE;
      if (blocks + total > 0x7fffffff) break;            // the rest goes into another launch
      m.blocks = (uint32_t)nb;
      m.first_block = (uint32_t)blocks;
      blocks += total;
      p.item[p.n_items++] = m;
    }
    if (p.n_items == 0) continue;
    const int rc = km == 4 ? launch_reorder<4>(p, (uint32_t)blocks, s)
                 : km == 8 ? launch_reorder<8>(p, (uint32_t)blocks, s)
                           : launch_reorder<16>(p, (uint32_t)blocks, s);
    if (rc != BOLT3_OK) return rc;
  }
  return BOLT3_OK;
}
