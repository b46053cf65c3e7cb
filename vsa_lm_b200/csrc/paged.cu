// The paged bf16 cache of a softmax anchor: new tokens into the pages (per-head RMSNorm, rotation, one rounding), and
// the eviction of rows by recorded attention weight.
//
// append, per head row x of HD values: x <- x * rsqrt(mean(x^2) + eps) * w, then the rotation of the pairs (i, i + HD/2)
// by pos * inv_freq[i], in fp32, one rounding to bf16; values are copied. The angle's product is taken in fp64 and reduced
// to one turn before the fp32 sine: at position 100000 an fp32 product is off by 0.004 of a radian, more than a bf16 step.
// Bound by HBM: (2 H + 4 HKV) HD bf16 per token. A row is HD / 8 lanes, a lane holding four neighbouring values of each
// half, so that a rotation's pair is in one lane; a block takes four tokens (few tokens: a share of one token's rows).
//
// evict: a CTA per (sequence, KV head). The threshold weight comes from a radix selection over the weights as ordered 32-bit
// keys (digits of 11, 11 and 10 bits, counted in shared memory); then every thread walks a stretch of rows of its own, so that
// one block-wide sum gives the ranks of equal weights, and one those of dropped rows below `keep` and of kept rows behind it,
// which are paired by rank. Only those rows move. Bound by HBM: 8 bytes per row, and 8 HD + 16 per moved row.
#include <cudaTypedefs.h>

#include <mutex>

#include "paged.cuh"
#include "tc5.cuh"
#include "trace.h"

namespace paged {

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
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

bool encode_pool(CUtensorMap* m, const void* pool, int64_t n_pages, int page, int HKV, int HD, int rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)page, (cuuint64_t)(2 * n_pages * HKV)};
  const cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)page * HD * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(pool), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace paged

namespace {

using namespace paged;

// ------------------------------------------------------------------------------------------- append

constexpr int kThreads = 256;
constexpr int kAhead = 4;                            // rows that a thread has in flight

template <int LPR>
B3_DEV float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// blockIdx.x = TPB tokens, blockIdx.y = share of their rows
template <int HD, int TPB>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ bolt3_paged_append_args a,
                                                                const __grid_constant__ Length len,
                                                                const __grid_constant__ Pages pages, int rows_per_block) {
  constexpr int LPR = HD / 8;                        // lanes of a row
  constexpr int RPI = kThreads / LPR;                // rows of one iteration
  __shared__ float4 trig[TPB][HD / 4];               // cos, sin of a pair of dimensions, cos, sin of the next
  // of each token: its cache row (-1: idle), its position, its first q, k and v element, the pool row of its first head's key
  // (-1: no page), the record of its first head
  __shared__ int64_t s_row[TPB], s_pos[TPB], s_src[TPB][3], s_out[TPB], s_rec[TPB];
  const int tid = threadIdx.x, part = tid % LPR;
  const int64_t tok0 = (int64_t)blockIdx.x * TPB, tokens = (int64_t)a.B * a.T;
  const int n_rows = a.H + 2 * a.HKV;
  const int first = TPB == 1 ? blockIdx.y * rows_per_block : 0;
  const int end = TPB == 1 ? min(n_rows, first + rows_per_block) : (int)min((int64_t)TPB, tokens - tok0) * n_rows;
  const int64_t cap = a.width * a.page;
  grid_dep_launch();
  grid_dep_wait();
  if (tid < TPB && tok0 + tid < tokens) {
    bool bad = false;
    const int b = (int)((tok0 + tid) / a.T), t = (int)((tok0 + tid) % a.T);
    const int64_t s = len.rows(b, bad);
    int pg = -1;
    if (s >= 0) {
      pg = pages.page_of(b, s + t);
      bad |= pg < 0;
    }
    if (bad && a.status) atomicOr(a.status, 8);
    s_row[tid] = s < 0 ? -1 : s + t;
    s_pos[tid] = a.pos != nullptr ? (int64_t)a.pos[b] + t : a.pos0 + (s + t - a.n);
    s_src[tid][0] = b * a.q_sb + t * a.q_st;
    s_src[tid][1] = b * a.k_sb + t * a.k_st;
    s_src[tid][2] = b * a.v_sb + t * a.v_st;
    s_out[tid] = pg < 0 ? -1 : (int64_t)pg * a.HKV * a.page + ((s + t) & (a.page - 1));
    s_rec[tid] = (int64_t)b * a.HKV * cap + s + t;
  }
  __syncthreads();
  for (int i = tid; a.inv_freq != nullptr && i < TPB * (HD / 2); i += kThreads) {
    const int k = i / (HD / 2), f = i % (HD / 2);
    if (tok0 + k < tokens && s_row[k] >= 0) {
      const double turn = (double)s_pos[k] * (double)a.inv_freq[f] * 0.15915494309189533577;   // 1 / (2 pi)
      float sn, cs;
      sincosf((float)((turn - rint(turn)) * 6.28318530717958647693), &sn, &cs);
      reinterpret_cast<float2*>(trig[k])[f] = make_float2(cs, sn);
    }
  }
  const bool norms = a.q_norm_w != nullptr || a.k_norm_w != nullptr;
  // whole groups of LPR lanes share a row, but the shuffles name the warp: rows past the end compute on zeros
  // and store nothing
  int item_r = first + tid / LPR, item_t = 0;        // row and token of this thread's next item
  if (TPB > 1) {
    item_t = item_r / n_rows;
    item_r -= item_t * n_rows;
  }
  for (int r0 = first; r0 < end; r0 += kAhead * RPI) {
    uint2 raw[kAhead][2];
    int row[kAhead], tk[kAhead];                     // row of its token (-1: past the end), token of the block
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool live = r0 + u * RPI + tid / LPR < end;
      tk[u] = live ? item_t : 0;
      const int r = live ? item_r : 0;
      row[u] = live ? r : -1;
      const bool is_q = r < a.H, is_k = !is_q && r < a.H + a.HKV;
      const int h = is_q ? r : is_k ? r - a.H : r - a.H - a.HKV;
      const bf16* src = reinterpret_cast<const bf16*>(is_q ? a.q : is_k ? a.k : a.v) + s_src[tk[u]][is_q ? 0 : is_k ? 1 : 2] + h * HD;
      raw[u][0] = raw[u][1] = make_uint2(0, 0);
      if (live && s_row[tk[u]] >= 0) {
        raw[u][0] = __ldg(reinterpret_cast<const uint2*>(src) + part);
        raw[u][1] = __ldg(reinterpret_cast<const uint2*>(src + HD / 2) + part);
      }
      item_r += RPI;
      if (TPB > 1)
        while (item_r >= n_rows) {
          item_r -= n_rows;
          ++item_t;
        }
    }
    if (r0 == first) __syncthreads();                // the sines and cosines
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (r0 + u * RPI >= end) break;                // the same for all threads
      const int r = row[u];
      const bool is_q = r < a.H, is_k = !is_q && r < a.H + a.HKV;
      uint2 o0 = raw[u][0], o1 = raw[u][1];
      if (is_q || is_k || norms) {                   // (norms: the shuffles need whole warps)
        float x[8];                                  // values 4 part .., HD / 2 + 4 part ..
        const float2 p0 = unpack_bf16(o0.x), p1 = unpack_bf16(o0.y), p2 = unpack_bf16(o1.x), p3 = unpack_bf16(o1.y);
        x[0] = p0.x; x[1] = p0.y; x[2] = p1.x; x[3] = p1.y; x[4] = p2.x; x[5] = p2.y; x[6] = p3.x; x[7] = p3.y;
        if (norms) {
          const float* w = is_q ? a.q_norm_w : is_k ? a.k_norm_w : nullptr;
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
          ss = row_sum<LPR>(ss);
          if (w != nullptr) {
            const float inv = rsqrtf(ss * (1.f / HD) + a.eps);
            const float4 w0 = reinterpret_cast<const float4*>(w)[part], w1 = reinterpret_cast<const float4*>(w + HD / 2)[part];
            const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * ww[i];
          }
        }
        if (is_q || is_k) {
          if (a.inv_freq != nullptr) {
            const float4* cs = trig[tk[u]] + 2 * part;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float4 z = cs[i / 2];            // of pairs i and i + 1
              const float a0 = x[i], b0 = x[4 + i], a1 = x[i + 1], b1 = x[5 + i];
              x[i] = fmaf(a0, z.x, -b0 * z.y);
              x[4 + i] = fmaf(b0, z.x, a0 * z.y);
              x[i + 1] = fmaf(a1, z.z, -b1 * z.w);
              x[5 + i] = fmaf(b1, z.z, a1 * z.w);
            }
          }
          o0 = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
          o1 = make_uint2(pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
        }
      }
      if (r < 0) continue;
      const int h = is_q ? r : is_k ? r - a.H : r - a.H - a.HKV;
      bf16* out;
      if (is_q) {
        if (s_row[tk[u]] < 0) o0 = o1 = make_uint2(0, 0);
        out = reinterpret_cast<bf16*>(a.q_out) + ((tok0 + tk[u]) * a.H + h) * HD;
      } else {
        if (s_out[tk[u]] < 0) continue;
        out = reinterpret_cast<bf16*>(a.pages) + (s_out[tk[u]] + ((is_k ? 0 : a.n_pages * a.HKV) + h) * a.page) * HD;
      }
      reinterpret_cast<uint2*>(out)[part] = o0;
      reinterpret_cast<uint2*>(out + HD / 2)[part] = o1;
      if (is_k && part == 0 && a.weight != nullptr) {
        const int64_t at = s_rec[tk[u]] + h * cap;
        a.weight[at] = 0.f;
        a.order[at] = (int32_t)s_pos[tk[u]];
      }
    }
  }
}

// -------------------------------------------------------------------------------------------- evict

constexpr int kEvictThreads = 512;
constexpr int kBins = 2048;
constexpr int kCached = 16384;                       // rows whose keys are kept in shared memory
constexpr int kInline = 512;                         // moves of a head that its own CTA makes, whatever the number of heads

struct Evict {
  bolt3_paged_evict_args a;
  Pages pages;
  int64_t most;                                      // moves that a head can have
  int2* moves;                                       // [head][most] (to, from)
  int32_t* count;                                    // [head]
  int split;                                         // a second kernel moves the rows
};

// sum over the block's earlier threads, and over all
B3_DEV uint64_t block_before(uint64_t v, uint64_t* s_warp, uint64_t& total) {
  constexpr int W = kEvictThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += x;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = up;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const uint64_t x = s_warp[w];
    if (w < warp) before += x;
    total += x;
  }
  return before + up - v;
}

// rows `to` of a head become rows `from`: lanes [0, HD / 8) a key row, the next HD / 8 its value row
template <int HD>
B3_DEV void move_rows(const Evict& p, int b, int h, const int2* moves, int first, int end, int step, int lane) {
  constexpr int LPR = HD / 8, RPW = 16 / LPR;        // lanes of a row; moves of a warp's instruction
  const bolt3_paged_evict_args& a = p.a;
  const int sub = lane / (2 * LPR), side = lane / LPR % 2, part = lane % LPR;
  uint4* pool = reinterpret_cast<uint4*>(a.pages) + (side ? a.n_pages * a.HKV * a.page * LPR : 0) + part;
  const int64_t rec = ((int64_t)b * a.HKV + h) * a.width * a.page;
  auto at = [&](int row) { return (((int64_t)p.pages.page_of(b, row) * a.HKV + h) * a.page + (row & (a.page - 1))) * LPR; };
  constexpr int kBatch = 4;
  for (int i0 = first * RPW; i0 < end; i0 += step * RPW * kBatch) {
    uint4 x[kBatch];
    int2 m[kBatch];
    float w[kBatch];
    int32_t o[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * step * RPW + sub;
      m[u] = i < end ? moves[i] : make_int2(-1, -1);
      if (m[u].x >= 0) {
        x[u] = pool[at(m[u].y)];
        if (side == 0 && part == 0) {
          w[u] = a.weight[rec + m[u].y];
          o[u] = a.order[rec + m[u].y];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (m[u].x < 0) continue;
      pool[at(m[u].x)] = x[u];
      if (side == 0 && part == 0) {
        a.weight[rec + m[u].x] = w[u];
        a.order[rec + m[u].x] = o[u];
      }
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(kEvictThreads) paged_evict_kernel(const __grid_constant__ Evict p) {
  extern __shared__ uint32_t s_key[];                // keys of the first rows, then a bit per row: new enough to stay
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint64_t s_warp[kEvictThreads / 32];
  __shared__ uint32_t s_digit;
  __shared__ int s_left, s_bad;
  const bolt3_paged_evict_args& a = p.a;
  const int tid = threadIdx.x, head = blockIdx.x, b = head / a.HKV, h = head % a.HKV;
  const int64_t cap = a.width * a.page;
  grid_dep_launch();
  grid_dep_wait();
  const int64_t held = a.lens != nullptr ? (int64_t)a.lens[b] : a.n;
  const bool bad = held < -1 || held > a.n;          // (n <= cap is the host's check)
  if (tid == 0) {
    if (bad && h == 0 && a.status) atomicOr(a.status, 8);
    if (h == 0 && a.lens_out != nullptr) a.lens_out[b] = bad ? -1 : (int32_t)min(held, a.keep);
    p.count[head] = 0;
    s_bad = 0;
  }
  if (bad || held <= a.keep) return;                 // the same for all threads
  const int n = (int)held, keep = (int)a.keep;
  const float* weight = a.weight + ((int64_t)b * a.HKV + h) * cap;
  const int32_t* order = a.order + ((int64_t)b * a.HKV + h) * cap;
  const int cached = min(n, kCached);
  __syncthreads();

  // every page that a row may leave or reach is in the pool
  for (int i = tid; i <= (n - 1) >> p.pages.log; i += kEvictThreads)
    if (p.pages.page_of(b, (int64_t)i << p.pages.log) < 0) s_bad = 1;
  // the newest position, then how many rows are new enough to stay
  int newest = (int)0x80000000;
  for (int i = tid; i < n; i += kEvictThreads) newest = max(newest, order[i]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if ((tid & 31) == 0) s_warp[tid >> 5] = (uint64_t)(uint32_t)newest;
  __syncthreads();
  if (s_bad) {
    if (tid == 0 && a.status) atomicOr(a.status, 8);
    return;
  }
#pragma unroll
  for (int w = 0; w < kEvictThreads / 32; ++w) newest = max(newest, (int)(uint32_t)s_warp[w]);
  const int64_t above = (int64_t)newest - a.recent;
  // NaN as +infinity; no key is 0
  auto key_of = [&](float w) { return w != w ? 0xff800000u : fkey(w); };
  int fresh = 0;
  for (int i = tid; i < n; i += kEvictThreads) {
    fresh += order[i] > above;
    if (i < cached) s_key[i] = key_of(weight[i]);
  }
  uint64_t total;
  block_before((uint64_t)fresh, s_warp, total);
  const bool all_fresh_stay = (int64_t)total <= keep;
  // New rows rank before all others. Where they all stay, they need no order among themselves; where they do not, the
  // other rows are out
  auto rank_key = [&](int i, uint32_t k) {
    const bool f = order[i] > above;
    return all_fresh_stay ? (f ? 0xffffffffu : k) : (f ? k : 0u);
  };
  for (int i = tid; i < cached; i += kEvictThreads) s_key[i] = rank_key(i, s_key[i]);
  auto get = [&](int i) { return i < cached ? s_key[i] : rank_key(i, key_of(weight[i])); };

  // the keep-th largest key, digit by digit: rows of the digits so far are candidates, `left` of them stay
  uint32_t prefix = 0;
  int left = keep;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const uint32_t mask = (1u << bits) - 1;
    for (int i = tid; i < kBins; i += kEvictThreads) s_hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kEvictThreads) {
      const uint32_t k = get(i);
      if (pass == 0 || k >> (shift + bits) == prefix >> (shift + bits)) atomicAdd(&s_hist[(k >> shift) & mask], 1u);
    }
    __syncthreads();
    // bins from the largest digit on, four to a thread
    constexpr int PER = kBins / kEvictThreads;
    uint32_t c[PER], sum = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) sum += c[u] = s_hist[kBins - 1 - (tid * PER + u)];
    uint64_t before = block_before((uint64_t)sum, s_warp, total);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if ((int64_t)before < left && (int64_t)(before + c[u]) >= left) {
        s_digit = kBins - 1 - (tid * PER + u);
        s_left = left - (int)before;
      }
      before += c[u];
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
  }
  // rows above `prefix` stay, and the first `left` of those equal to it
  const int per = (n + kEvictThreads - 1) / kEvictThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
  int equal = 0;
  for (int i = i0; i < i1; ++i) equal += get(i) == prefix;
  int rank = (int)block_before((uint64_t)equal, s_warp, total);
  const int rank0 = rank;
  uint64_t mine = 0;                                 // dropped rows below keep, kept rows from it on
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = get(i);
    const bool stays = k > prefix || (k == prefix && rank++ < left);
    if (i < keep) mine += !stays;
    else mine += (uint64_t)stays << 32;
  }
  const uint64_t before = block_before(mine, s_warp, total);
  int hole = (int)(uint32_t)before, mover = (int)(before >> 32);
  int2* moves = p.moves + (int64_t)head * p.most;
  rank = rank0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = get(i);
    const bool stays = k > prefix || (k == prefix && rank++ < left);
    if (i < keep && !stays) moves[hole++].x = i;
    if (i >= keep && stays) moves[mover++].y = i;
  }
  const int n_moves = (int)(uint32_t)total;
  if (tid == 0) p.count[head] = n_moves;
  if (p.split) return;
  __syncthreads();
  move_rows<HD>(p, b, h, moves, tid >> 5, n_moves, kEvictThreads / 32, tid & 31);
}

// the moves of a head, shared by gridDim.y blocks
template <int HD>
__global__ void __launch_bounds__(kThreads) paged_move_kernel(const __grid_constant__ Evict p) {
  grid_dep_launch();
  grid_dep_wait();
  const int head = blockIdx.x, warps = kThreads / 32;
  move_rows<HD>(p, head / p.a.HKV, head % p.a.HKV, p.moves + (int64_t)head * p.most, blockIdx.y * warps + (threadIdx.x >> 5),
                p.count[head], gridDim.y * warps, threadIdx.x & 31);
}

int64_t most_moves(int64_t n, int64_t keep) { return n <= keep ? 0 : n - keep < keep ? n - keep : keep; }

template <int HD>
int launch_evict(const Evict& p, cudaStream_t s) {
  const int64_t heads = (int64_t)p.a.B * p.a.HKV;
  const size_t smem = (size_t)(p.a.n < kCached ? p.a.n : kCached) * 4;
  if (cudaFuncSetAttribute(paged_evict_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCached * 4) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  if (launch_overlapped(paged_evict_kernel<HD>, dim3((unsigned)heads), dim3(kEvictThreads), smem, s, p) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  if (!p.split) return BOLT3_OK;
  const int64_t per = kThreads / 32 * 4 * (HD == 128 ? 1 : 2), want = (p.most + per - 1) / per, fit = (148 * 4 + heads - 1) / heads;
  const unsigned slices = (unsigned)(want < fit ? want : fit);
  return launch_overlapped(paged_move_kernel<HD>, dim3((unsigned)heads, slices), dim3(kThreads), 0, s, p) == cudaSuccess
             ? BOLT3_OK : BOLT3_ERR_CUDA;
}

}  // namespace

extern "C" int bolt3_paged_append(const bolt3_paged_append_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_paged_append");
  if (!a || !a->q || !a->k || !a->v || !a->q_out || !a->pages || !a->table) return BOLT3_ERR_ARG;
  if (a->lens != nullptr && a->pos_dev != nullptr) return BOLT3_ERR_ARG;
  if (a->pos != nullptr && a->lens == nullptr) return BOLT3_ERR_ARG;
  if ((a->weight == nullptr) != (a->order == nullptr)) return BOLT3_ERR_ARG;
  if (a->pos_dev != nullptr && a->pos_span < 1) return BOLT3_ERR_ARG;
  if (a->B <= 0 || a->T <= 0 || a->T > (1 << 20) || a->H <= 0 || a->HKV <= 0 || a->H > 4096 || a->HKV > 2048 ||
      a->H + 2 * a->HKV > 4096)
    return BOLT3_ERR_SHAPE;
  if ((int64_t)a->B * a->T > 0x7fffffff || (int64_t)a->B * a->HKV > 0x7fffffff) return BOLT3_ERR_SHAPE;
  Pages pages;
  if (!pages_ok(a->n_pages, a->page, a->width, a->table_stride, a->HKV, a->HD, &pages, a->table)) return BOLT3_ERR_SHAPE;
  const int64_t cap = a->width * a->page, dmax = a->pos_dev != nullptr ? a->pos_span - 1 : 0;
  if (a->n < 0 || cap < a->T || (a->lens == nullptr && a->n > cap - a->T - dmax)) return BOLT3_ERR_CAPACITY;
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->pages |
                       (uintptr_t)a->q_norm_w | (uintptr_t)a->k_norm_w;
  const int64_t st = a->q_sb | a->q_st | a->k_sb | a->k_st | a->v_sb | a->v_st;
  if ((al & 15) || (st & 7)) return BOLT3_ERR_ALIGN;
  // with lens, n bounds the lengths and the table the rows
  const Length len{a->lens, a->pos_dev, a->n, a->pos_ref, a->pos_span,
                   a->lens != nullptr && a->n < cap - a->T ? a->n + a->T : cap, a->T};
  const int rows = a->H + 2 * a->HKV, rpi = kThreads / (a->HD / 8);
  // few tokens: a block per iteration's rows, so that a one-token step still fills the machine; from two blocks of four
  // tokens for every SM on, blocks of four
  const int64_t tokens = (int64_t)a->B * a->T;
  const bool few = tokens < 148 * 8;
  const dim3 grid((unsigned)(few ? tokens : (tokens + 3) / 4), (unsigned)(few ? (rows + rpi - 1) / rpi : 1));
  cudaStream_t s = (cudaStream_t)stream;
  auto kern = a->HD == 128 ? (few ? paged_append_kernel<128, 1> : paged_append_kernel<128, 4>)
                           : (few ? paged_append_kernel<64, 1> : paged_append_kernel<64, 4>);
  return launch_overlapped(kern, grid, dim3(kThreads), 0, s, *a, len, pages, rpi) == cudaSuccess ? BOLT3_OK : BOLT3_ERR_CUDA;
}

extern "C" size_t bolt3_paged_evict_workspace(int B, int HKV, int64_t n, int64_t keep) {
  if (B <= 0 || HKV <= 0 || n < 0 || keep < 1 || n > 0x7fffffff) return 0;
  return (size_t)B * (size_t)HKV * ((size_t)most_moves(n, keep) * 8 + 4);
}

extern "C" int bolt3_paged_evict(const bolt3_paged_evict_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_paged_evict");
  if (!a || !a->pages || !a->table || !a->weight || !a->order || !a->workspace) return BOLT3_ERR_ARG;
  if (a->keep < 1 || a->recent < 0 || a->recent > a->keep) return BOLT3_ERR_ARG;
  if (a->B <= 0 || (int64_t)a->B * a->HKV > 0x7fffffff) return BOLT3_ERR_SHAPE;
  Evict p;
  if (!pages_ok(a->n_pages, a->page, a->width, a->table_stride, a->HKV, a->HD, &p.pages, a->table)) return BOLT3_ERR_SHAPE;
  if (a->n < 0 || a->n > a->width * a->page) return BOLT3_ERR_CAPACITY;
  if (a->workspace_bytes < bolt3_paged_evict_workspace(a->B, a->HKV, a->n, a->keep)) return BOLT3_ERR_CAPACITY;
  if (((uintptr_t)a->pages | (uintptr_t)a->workspace) & 15) return BOLT3_ERR_ALIGN;
  p.a = *a;
  p.most = most_moves(a->n, a->keep);
  p.moves = reinterpret_cast<int2*>(a->workspace);
  p.count = reinterpret_cast<int32_t*>(p.moves + (int64_t)a->B * a->HKV * p.most);
  p.split = p.most > kInline && (int64_t)a->B * a->HKV < 148;
  cudaStream_t s = (cudaStream_t)stream;
  return a->HD == 128 ? launch_evict<128>(p, s) : launch_evict<64>(p, s);
}
