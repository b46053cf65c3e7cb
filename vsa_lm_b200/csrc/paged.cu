// The paged bf16 cache of a softmax anchor: new tokens into the pages (per-head RMSNorm, rotation, one rounding), and
// the eviction of rows by recorded attention weight.
//
// append, per head row x of HD values: x <- x * rsqrt(mean(x^2) + eps) * w, then the rotation of the pairs (i, i + HD/2)
// by pos * inv_freq[i], in fp32, one rounding to bf16; values are copied. The angle's product is taken in fp64 and reduced
// to one turn before the fp32 sine: at position 100000 an fp32 product is off by 0.004 of a radian, more than a bf16 step.
// Bound by HBM: (2 H + 4 HKV) HD bf16 per token. A warp takes a token's rows (few tokens: a share of them), HD / 16 lanes to a
// row, a lane holding eight neighbouring values of each half, so that a rotation's pair is in one lane; its lanes share the
// token's sines and cosines out among themselves and keep them for all rows. 64 x 128 tokens of 32 + 2 x 8 heads of 128: 38.5 us,
// 5.2 TB/s.
//
// evict: a CTA per (sequence, KV head). The threshold weight comes from a radix selection over the weights as ordered 32-bit
// keys (digits of 11, 11 and 10 bits, counted in shared memory); then every warp walks a stretch of rows, so that one sum over
// the warps gives the ranks of equal weights, and one those of dropped rows below `keep` and of kept rows behind it,
// which are paired by rank. Only those rows move. Bound by HBM: 8 bytes per row, and 8 HD + 16 per moved row. 512 heads of 2176
// rows, 128 of them moved: 20 us.
#include <cudaTypedefs.h>

#include <mutex>

#include "paged.cuh"
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

// Where a token's rows go
struct Token {
  int64_t token, s, row, pos;                        // its number, the rows its sequence held (-1: idle), its row, its position
  int b, page;                                       // -1: none
};

B3_DEV Token token_at(const bolt3_paged_append_args& a, const Length& len, const Pages& pages, int64_t token, int lane) {
  Token tk;
  bool bad = false;
  tk.token = token;
  tk.b = (int)(token / a.T);
  const int t = (int)(token - (int64_t)tk.b * a.T);
  tk.s = len.rows(tk.b, bad);                        // the same for the whole warp
  tk.row = tk.s + t;
  tk.page = -1;
  if (tk.s >= 0) {
    tk.page = pages.page_of(tk.b, tk.row);
    bad |= tk.page < 0;
  }
  if (bad && lane == 0 && a.status) atomicOr(a.status, 8);
  tk.pos = tk.s < 0 ? 0 : a.pos != nullptr ? (int64_t)a.pos[tk.b] + t : a.pos0 + (tk.row - a.n);
  return tk;
}

// The norms' weights, of queries and of keys, into shared memory, the first four of every lane's eight (append_rows) before the
// other four: a load's lanes read neighbouring 16 bytes. A __syncthreads() comes after
template <int HD>
B3_DEV bool load_norms(const bolt3_paged_append_args& a, float4* s_norm) {
  if (threadIdx.x < HD / 2) {
    const float* w = threadIdx.x < HD / 4 ? a.q_norm_w : a.k_norm_w;
    const int i = threadIdx.x % (HD / 8), at = threadIdx.x - i + i % 2 * (HD / 16) + i / 2;
    if (w != nullptr) s_norm[at] = __ldg(reinterpret_cast<const float4*>(w) + threadIdx.x % (HD / 4));
  }
  return a.q_norm_w != nullptr || a.k_norm_w != nullptr;
}

// The cosines of two neighbouring pairs of dimensions of a token, then their sines, for all pairs, by the lanes of a warp; the
// i-th 16 bytes of every lane's four (append_rows) stand together (a lane's own together: 4 banks for 8 lanes, and 50 us
// rather than 41 for 64 x 128 tokens of 32 + 2 x 8 heads of 128)
template <int HD>
B3_DEV void turns_of(const bolt3_paged_append_args& a, const Token& tk, float* turns, int lane) {
#pragma unroll
  for (int i = lane; i < HD / 2; i += 32) {
    float sn = 0.f, cs = 1.f;
    if (a.inv_freq != nullptr) {
      const double turn = (double)tk.pos * (double)a.inv_freq[i] * 0.15915494309189533577;   // 1 / (2 pi)
      __sincosf((float)((turn - rint(turn)) * 6.28318530717958647693), &sn, &cs);   // within 2^-21 of either, in [-pi, pi]
    }
    float* at = turns + (i / 2 % 4 * (HD / 16) + i / 8) * 4 + i % 2;
    at[0] = cs;
    at[2] = sn;
  }
}

// Rows r0 .. of a token, one for each HD / 16 lanes: this lane's values 8 part .. of row r in o0, HD / 2 + 8 part .. in o1. Rows
// from `end` on store nothing, but their lanes take part: the shuffles name the warp
template <int HD>
B3_DEV void append_rows(const bolt3_paged_append_args& a, const Token& tk, uint4 o0, uint4 o1, int r0, int r, int end, uint32_t at_turn,
                        uint32_t at_norm, bool norms) {
  constexpr int LPR = HD / 16;
  const int part = (threadIdx.x & 31) % LPR;
  const bool is_q = r < a.H, is_k = !is_q && r < a.H + a.HKV;
  auto lds = [](uint32_t at, uint64_t& lo, uint64_t& hi) {   // where it stands: kept in registers over the rows they cost the loads in flight
    asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];\n" : "=l"(lo), "=l"(hi) : "r"(at));
  };
  if (r0 < a.H + a.HKV) {                            // the same for the whole warp: some of its rows are queries or keys
    uint64_t x[4], y[4];                             // the values, two neighbours at a time
    {
      const uint32_t w0[4] = {o0.x, o0.y, o0.z, o0.w}, w1[4] = {o1.x, o1.y, o1.z, o1.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = pair(__uint_as_float(w0[i] << 16), __uint_as_float(w0[i] & 0xffff0000u));
        y[i] = pair(__uint_as_float(w1[i] << 16), __uint_as_float(w1[i] & 0xffff0000u));
      }
    }
    if (norms) {
      uint64_t s0 = mul2(x[0], x[0]), s1 = mul2(y[0], y[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        s0 = fma2(x[i], x[i], s0);
        s1 = fma2(y[i], y[i], s1);
      }
      const float2 s2 = unpair(add2(s0, s1));
      float ss = s2.x + s2.y;
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (is_q ? a.q_norm_w != nullptr : is_k && a.k_norm_w != nullptr) {
        const float inv = rsqrtf(ss * (1.f / HD) + a.eps);
        const uint64_t inv2 = pair(inv, inv);
        const uint32_t w = at_norm + (is_q ? 0 : HD * 4);
        uint64_t wx[4], wy[4];
        lds(w, wx[0], wx[1]);
        lds(w + HD, wx[2], wx[3]);
        lds(w + HD * 2, wy[0], wy[1]);
        lds(w + HD * 3, wy[2], wy[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = mul2(x[i], mul2(inv2, wx[i]));
          y[i] = mul2(y[i], mul2(inv2, wy[i]));
        }
      }
    }
    if (is_q || is_k) {
      uint32_t w0[4], w1[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint64_t c, d;                               // cosines and sines of a pair of pairs
        lds(at_turn + HD * i, c, d);
        const float2 u = unpair(fma2(x[i], c, mul2(y[i], d ^ 0x8000000080000000ull))), v = unpair(fma2(y[i], c, mul2(x[i], d)));
        w0[i] = pack_bf16(u.x, u.y);
        w1[i] = pack_bf16(v.x, v.y);
      }
      o0 = make_uint4(w0[0], w0[1], w0[2], w0[3]);
      o1 = make_uint4(w1[0], w1[1], w1[2], w1[3]);
    }
  }
  if (r >= end) return;
  bf16* out;
  if (is_q) {
    if (tk.s < 0) o0 = o1 = make_uint4(0, 0, 0, 0);
    out = reinterpret_cast<bf16*>(a.q_out) + (tk.token * a.H + r) * HD + 8 * part;
  } else {
    if (tk.page < 0) return;
    const int h = is_k ? r - a.H : r - a.H - a.HKV;
    const int64_t row = ((is_k ? 0 : a.n_pages) + tk.page) * a.HKV + h;
    out = reinterpret_cast<bf16*>(a.pages) + (row * a.page + (tk.row & (a.page - 1))) * HD + 8 * part;
    if (is_k && part == 0 && a.weight != nullptr) {
      const int64_t at = ((int64_t)tk.b * a.HKV + h) * a.width * a.page + tk.row;
      a.weight[at] = 0.f;
      a.order[at] = (int32_t)min(tk.pos, (int64_t)0x7fffffff);
    }
  }
  reinterpret_cast<uint4*>(out)[0] = o0;
  reinterpret_cast<uint4*>(out + HD / 2)[0] = o1;
}

// A warp takes rows [c rows_per, ..) of the H + 2 HKV rows of a token, of `chunks` such stretches. The row after the one at work
// is in flight, and 32 warps of an SM hide the rest: 64 x 128 tokens of 32 + 2 x 8 heads of 128 in 39 us, where a copy of as many
// bytes takes 35 (two rows in flight and 24 warps 41 us, four and 16 48 us, 40 warps spill: 48 us; rows by bulk copies through
// a ring of shared memory are not faster)
template <int HD>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(const __grid_constant__ bolt3_paged_append_args a,
                                                                const __grid_constant__ Length len,
                                                                const __grid_constant__ Pages pages, int chunks, int rows_per) {
  constexpr int LPR = HD / 16, RPI = 32 / LPR;       // lanes of a row, rows of an iteration
  __shared__ float4 s_turn[kThreads / 32][HD / 4];   // of a warp's token (turns_of)
  __shared__ float4 s_norm[2][HD / 4];               // of queries, of keys
  const int lane = threadIdx.x & 31, part = lane % LPR, sub = lane / LPR;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), token = item / chunks;
  grid_dep_launch();
  grid_dep_wait();
  const bool norms = load_norms<HD>(a, s_norm[0]);
  __syncthreads();
  if (token >= (int64_t)a.B * a.T) return;
  const int c = (int)(item - token * chunks), b = (int)(token / a.T), t = (int)(token - (int64_t)b * a.T);
  const int n_rows = a.H + 2 * a.HKV, first = c * rows_per, end = min(n_rows, first + rows_per);
  const bf16* q = reinterpret_cast<const bf16*>(a.q) + b * a.q_sb + t * a.q_st + 8 * part;
  const bf16* k = reinterpret_cast<const bf16*>(a.k) + b * a.k_sb + t * a.k_st + 8 * part;
  const bf16* v = reinterpret_cast<const bf16*>(a.v) + b * a.v_sb + t * a.v_st + 8 * part;
  uint4 raw[2];                                      // values 8 part .., HD / 2 + 8 part ..
  auto fetch = [&](int r) {
    if (r >= end) return;
    const bf16* src = r < a.H ? q + r * HD : r < a.H + a.HKV ? k + (r - a.H) * HD : v + (r - a.H - a.HKV) * HD;
    raw[0] = __ldg(reinterpret_cast<const uint4*>(src));
    raw[1] = __ldg(reinterpret_cast<const uint4*>(src + HD / 2));
  };
  fetch(first + sub);
  const Token tk = token_at(a, len, pages, token, lane);
  if (first < a.H + a.HKV) turns_of<HD>(a, tk, reinterpret_cast<float*>(s_turn[threadIdx.x >> 5]), lane);
  __syncwarp();
  const uint32_t at_turn = (uint32_t)__cvta_generic_to_shared(s_turn[threadIdx.x >> 5] + part);
  const uint32_t at_norm = (uint32_t)__cvta_generic_to_shared(s_norm[0] + part);
  for (int r0 = first; r0 < end; r0 += RPI) {
    const uint4 o0 = raw[0], o1 = raw[1];
    fetch(r0 + sub + RPI);                           // rows past the end compute on what stands in the registers
    append_rows<HD>(a, tk, o0, o1, r0, r0 + sub, end, at_turn, at_norm, norms);
  }
}

// -------------------------------------------------------------------------------------------- evict

constexpr int kBins = 2048;
constexpr int kCached = 12288;                       // rows whose keys and positions are kept in shared memory
constexpr int kListed = 1024;                        // moves of a head whose list is kept in shared memory

struct Evict {
  bolt3_paged_evict_args a;
  Pages pages;
  int64_t most;                                      // moves that a head can have
  int2* moves;                                       // [head][most] (to, from), where they are not listed in shared memory
  int32_t* count;                                    // [head], where `split`
  int split;                                         // a second kernel moves the rows
};

// v summed over the earlier warps of the block, and over all; v the same for all lanes of a warp
template <int W>
B3_DEV uint64_t warps_before(uint64_t v, uint64_t* s_warp, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) s_warp[warp] = v;
  __syncthreads();
  uint64_t up = lane < W ? s_warp[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += x;
  }
  total = __shfl_sync(0xffffffffu, up, 31);
  return __shfl_sync(0xffffffffu, up, warp) - v;
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

template <int HD, int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 4 : 1) paged_evict_kernel(const __grid_constant__ Evict p) {
  constexpr int W = NT / 32;
  extern __shared__ __align__(16) uint32_t s_dyn[];                // keys of the first rows, positions of the first rows, the list of moves
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint64_t s_warp[32];
  __shared__ uint32_t s_digit;
  __shared__ int s_left, s_whole, s_bad;
  const bolt3_paged_evict_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.x, b = head / a.HKV, h = head % a.HKV;
  const int64_t cap = a.width * a.page;
  grid_dep_launch();
  grid_dep_wait();
  const int64_t held = a.lens != nullptr ? (int64_t)a.lens[b] : a.n;
  const bool bad = held < -1 || held > a.n;          // (n <= cap is the host's check)
  if (tid == 0) {
    if (bad && h == 0 && a.status) atomicOr(a.status, 8);
    if (h == 0 && a.lens_out != nullptr) a.lens_out[b] = bad ? -1 : (int32_t)min(held, a.keep);
    if (p.split) p.count[head] = 0;
    s_bad = 0;
  }
  if (bad || held <= a.keep) return;                 // the same for all threads
  const int n = (int)held, keep = (int)a.keep;
  const float* weight = a.weight + ((int64_t)b * a.HKV + h) * cap;
  const int32_t* order = a.order + ((int64_t)b * a.HKV + h) * cap;
  const int cached = min(n, kCached);
  uint32_t* s_key = s_dyn;
  int32_t* s_order = reinterpret_cast<int32_t*>(s_dyn + cached);
  // NaN as +infinity, -0 as 0 (the sum is +0); no key is 0
  auto key_of = [&](float w) { return w != w ? 0xff800000u : fkey(w + 0.f); };
  __syncthreads();

  // positions and weights into shared memory, the newest position; every page that a row may leave or reach is in the pool
  int newest = (int)0x80000000;
  for (int i0 = tid; i0 < n; i0 += 4 * NT) {
    int32_t o[4];
    float w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * NT;
      if (i < n) o[u] = order[i];
      if (i < cached) w[u] = weight[i];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * NT;
      if (i < n) newest = max(newest, o[u]);
      if (i < cached) {
        s_key[i] = key_of(w[u]);
        s_order[i] = o[u];
      }
    }
  }
  for (int i = tid; i <= (n - 1) >> p.pages.log; i += NT)
    if (p.pages.page_of(b, (int64_t)i << p.pages.log) < 0) s_bad = 1;
  for (int i = tid; i < kBins; i += NT) s_hist[i] = 0;
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) s_warp[warp] = (uint64_t)(uint32_t)newest;
  __syncthreads();
  if (s_bad) {
    if (tid == 0 && a.status) atomicOr(a.status, 8);
    return;
  }
  newest = __reduce_max_sync(0xffffffffu, lane < W ? (int)(uint32_t)s_warp[lane] : (int)0x80000000);
  const int64_t above = (int64_t)newest - a.recent;
  // New rows rank before all others. Where they all stay, they need no order among themselves; where they do not, the
  // other rows are out
  uint64_t total;
  int fresh = 0;
  for (int i = tid; i < n; i += NT) fresh += (i < cached ? s_order[i] : order[i]) > above;
  warps_before<W>((uint64_t)__reduce_add_sync(0xffffffffu, fresh), s_warp, total);
  const bool all_fresh_stay = (int64_t)total <= keep;
  auto rank_key = [&](int32_t o, uint32_t k) {
    const bool f = o > above;
    return all_fresh_stay ? (f ? 0xffffffffu : k) : (f ? k : 0u);
  };
  auto get = [&](int i) { return i < cached ? s_key[i] : rank_key(order[i], key_of(weight[i])); };

  // the keep-th largest key, digit by digit: rows of the digits so far are candidates, `left` of them stay. Done early where a
  // digit's rows all stay
  uint32_t prefix = 0;
  int left = keep;
  bool whole = false;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    if (whole) break;                                // the same for all threads
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const uint32_t mask = (1u << bits) - 1;
    if (pass > 0) {
      for (int i = tid; i < kBins; i += NT) s_hist[i] = 0;
      __syncthreads();
    }
    for (int i = tid; i < n; i += NT) {
      uint32_t k;
      if (pass == 0 && i < cached) s_key[i] = k = rank_key(s_order[i], s_key[i]);
      else k = get(i);
      if (pass == 0 || k >> (shift + bits) == prefix >> (shift + bits)) atomicAdd(&s_hist[(k >> shift) & mask], 1u);
    }
    __syncthreads();
    // bins from the largest digit on, a few to a thread
    constexpr int PER = kBins / NT;
    uint32_t c[PER], sum = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) sum += c[u] = s_hist[kBins - 1 - (tid * PER + u)];
    uint32_t up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    uint32_t before = (uint32_t)warps_before<W>((uint64_t)__shfl_sync(0xffffffffu, up, 31), s_warp, total) + up - sum;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if ((int)before < left && (int)(before + c[u]) >= left) {
        s_digit = kBins - 1 - (tid * PER + u);
        s_left = left - (int)before;
        s_whole = (int)(before + c[u]) == left;
      }
      before += c[u];
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
    whole = s_whole;
  }
  // rows above `prefix` stay, and the first `left` of those equal to it; a whole digit: those from it on (no key is 0, and not
  // all rows stay, so it is not 0)
  if (whole) {
    prefix -= 1;
    left = 0;
  }
  // a warp takes a stretch of rows, 32 at a time, so that ranks in the order of rows are sums over warps and bits before a lane's
  const int per = (n + NT - 1) / NT * 32, i0 = min(n, warp * per), i1 = min(n, i0 + per);
  const uint32_t lower = (1u << lane) - 1;
  int rank0 = 0;
  if (left > 0) {
    int equal = 0;
    for (int i = i0 + lane; i - lane < i1; i += 32) equal += __popc(__ballot_sync(0xffffffffu, i < i1 && get(i) == prefix));
    rank0 = (int)warps_before<W>((uint64_t)equal, s_warp, total);
  }
  auto stays = [&](int i, int& rank) {
    const uint32_t k = i < i1 ? get(i) : 0u;
    bool st = k > prefix;
    if (left > 0) {
      const uint32_t eq = __ballot_sync(0xffffffffu, i < i1 && k == prefix);
      st |= (eq >> lane & 1) && rank + __popc(eq & lower) < left;
      rank += __popc(eq);
    }
    return st;
  };
  uint64_t mine = 0;                                 // dropped rows below keep, kept rows from it on
  int rank = rank0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const bool st = stays(i, rank);
    mine += __popc(__ballot_sync(0xffffffffu, i < i1 && i < keep && !st)) +
            ((uint64_t)__popc(__ballot_sync(0xffffffffu, i < i1 && i >= keep && st)) << 32);
  }
  const uint64_t before = warps_before<W>(mine, s_warp, total);
  int hole = (int)(uint32_t)before, mover = (int)(before >> 32);
  const int n_moves = (int)(uint32_t)total;
  int2* moves = p.most <= kListed ? reinterpret_cast<int2*>(s_dyn + 2 * cached) : p.moves + (int64_t)head * p.most;
  rank = rank0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const bool st = stays(i, rank), drops = i < i1 && i < keep && !st, moves_in = i < i1 && i >= keep && st;
    const uint32_t d = __ballot_sync(0xffffffffu, drops), m = __ballot_sync(0xffffffffu, moves_in);
    if (drops) moves[hole + __popc(d & lower)].x = i;
    if (moves_in) moves[mover + __popc(m & lower)].y = i;
    hole += __popc(d);
    mover += __popc(m);
  }
  if (p.split) {
    if (tid == 0) p.count[head] = n_moves;
    return;
  }
  __syncthreads();
  move_rows<HD>(p, b, h, moves, warp, n_moves, W, lane);
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
// Whether a kernel of its own moves the rows, several blocks to a head: 8 heads of 6107 rows with 2011 moves each 18.5 us, moved by
// each head's CTA 27; with 1024 moves, whose list is in shared memory, the CTA is as fast (4 heads 17.1 us, apart 17.4)
bool split_moves(int64_t heads, int64_t most) { return most > kListed && heads < 148; }

template <int HD, int NT>
int launch_select(const Evict& p, cudaStream_t s) {
  const size_t cached = p.a.n < kCached ? (size_t)p.a.n : (size_t)kCached;
  const size_t smem = cached * 8 + (p.most <= kListed ? (size_t)p.most * 8 : 0);
  if (cudaFuncSetAttribute(paged_evict_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCached * 8 + kListed * 8) != cudaSuccess)
    return BOLT3_ERR_CUDA;
  return launch_overlapped(paged_evict_kernel<HD, NT>, dim3((unsigned)(p.a.B * p.a.HKV)), dim3(NT), smem, s, p) == cudaSuccess
             ? BOLT3_OK : BOLT3_ERR_CUDA;
}

template <int HD>
int launch_evict(const Evict& p, cudaStream_t s) {
  const int64_t heads = (int64_t)p.a.B * p.a.HKV;
  // Times with cold caches. A thread per few rows where an SM has a head at most (4 heads of 4224 rows: 1024 threads 16.4 us, 512 20.5, 256 28.7; 148 heads
  // 18.4, 22.5, 30.7), and where shared memory holds two heads' rows on an SM at most (400 heads of 12000 rows, 3808 moves: 334, 446, 717).
  // Else smaller blocks, of which an SM holds two of 512 threads by registers (400 heads of 4224 rows: 45.1, 39.4, 38.9; of 8320 53.2,
  // 49.2, 49.2; 512 heads 69.6, 57.3, 79.8), or four of 256: where there are more heads than that holds of 512, up to 4096 rows (512 heads
  // of 2176 rows: 49.1, 38.9, 34.8; 296 heads 28.7, 24.6, 28.7)
  const bool many = heads > 148, full = p.a.n > 10240;
  const int rc = p.a.n > 4096 && (!many || full) ? launch_select<HD, 1024>(p, s)
               : p.a.n <= 4096 && heads > 148 * 2 ? launch_select<HD, 256>(p, s) : launch_select<HD, 512>(p, s);
  if (rc != BOLT3_OK) return rc;
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
  // positions are recorded in 32 bits
  if (a->order != nullptr && a->pos == nullptr && (a->pos0 < -(1ll << 31) + a->n || a->pos0 > 0x7fffffffll - a->T - dmax)) return BOLT3_ERR_CAPACITY;
  if (a->n < 0 || cap < a->T || (a->lens == nullptr && a->n > cap - a->T - dmax)) return BOLT3_ERR_CAPACITY;
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->pages |
                       (uintptr_t)a->q_norm_w | (uintptr_t)a->k_norm_w;
  const int64_t st = a->q_sb | a->q_st | a->k_sb | a->k_st | a->v_sb | a->v_st;
  if ((al & 15) || (st & 7)) return BOLT3_ERR_ALIGN;
  // with lens, n bounds the lengths and the table the rows
  const Length len{a->lens, a->pos_dev, a->n, a->pos_ref, a->pos_span,
                   a->lens != nullptr && a->n < cap - a->T ? a->n + a->T : cap, a->T};
  // A warp per token, or per share of its rows: as many as make the fewest steps of the longest warp, where 32 warps of an SM work
  // at once and each begins with what takes one step and a half (its token's sines). 24 sequences of 128 tokens of 32 + 2 x 8
  // heads of 128: 3 shares 15.6 us, 1 18.0; 40 sequences: 3 shares 26.7 us, 1 30.2
  const int rows = a->H + 2 * a->HKV, rpi = 32 / (a->HD / 16), groups = (rows + rpi - 1) / rpi;
  const int64_t tokens = (int64_t)a->B * a->T;
  cudaStream_t s = (cudaStream_t)stream;
  int chunks = 1, rows_per = groups * rpi;
  double least = 0;
  for (int per = groups; per >= 1; per = per > 16 ? per / 2 : per - 1) {
    const int c = (groups + per - 1) / per;
    const double cost = (double)((tokens * c + 148 * 32 - 1) / (148 * 32)) * (per + 1.5);
    if (per == groups || cost < least) {
      least = cost;
      chunks = c;
      rows_per = per * rpi;
    }
  }
  const int64_t blocks = (tokens * chunks + kThreads / 32 - 1) / (kThreads / 32);
  return launch_overlapped(a->HD == 128 ? paged_append_kernel<128> : paged_append_kernel<64>, dim3((unsigned)blocks), dim3(kThreads), 0, s,
                           *a, len, pages, chunks, rows_per) == cudaSuccess ? BOLT3_OK : BOLT3_ERR_CUDA;
}

extern "C" size_t bolt3_paged_evict_workspace(int B, int HKV, int64_t n, int64_t keep) {
  if (B <= 0 || HKV <= 0 || n < 0 || keep < 1 || n > 0x7fffffff) return 0;
  const int64_t heads = (int64_t)B * HKV, most = most_moves(n, keep);
  return most > kListed ? (size_t)heads * ((size_t)most * 8 + (split_moves(heads, most) ? 4 : 0)) : 0;
}

extern "C" int bolt3_paged_evict(const bolt3_paged_evict_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_paged_evict");
  if (!a || !a->pages || !a->table || !a->weight || !a->order) return BOLT3_ERR_ARG;
  if (a->keep < 1 || a->recent < 0 || a->recent > a->keep) return BOLT3_ERR_ARG;
  if (a->B <= 0 || (int64_t)a->B * a->HKV > 0x7fffffff) return BOLT3_ERR_SHAPE;
  Evict p;
  if (!pages_ok(a->n_pages, a->page, a->width, a->table_stride, a->HKV, a->HD, &p.pages, a->table)) return BOLT3_ERR_SHAPE;
  if (a->n < 0 || a->n > a->width * a->page) return BOLT3_ERR_CAPACITY;
  const size_t need = bolt3_paged_evict_workspace(a->B, a->HKV, a->n, a->keep);
  if (need > 0 && !a->workspace) return BOLT3_ERR_ARG;
  if (a->workspace_bytes < need) return BOLT3_ERR_CAPACITY;
  if (((uintptr_t)a->pages | (uintptr_t)a->workspace) & 15) return BOLT3_ERR_ALIGN;
  // the first head of a sequence writes its new length where the others may not have read the old one yet
  if (a->lens != nullptr && a->lens_out != nullptr && a->lens < a->lens_out + a->B && a->lens_out < a->lens + a->B) return BOLT3_ERR_ARG;
  p.a = *a;
  p.most = most_moves(a->n, a->keep);
  p.moves = reinterpret_cast<int2*>(a->workspace);
  p.count = reinterpret_cast<int32_t*>(p.moves + (int64_t)a->B * a->HKV * p.most);
  p.split = split_moves((int64_t)a->B * a->HKV, p.most);
  cudaStream_t s = (cudaStream_t)stream;
  return a->HD == 128 ? launch_evict<128>(p, s) : launch_evict<64>(p, s);
}
