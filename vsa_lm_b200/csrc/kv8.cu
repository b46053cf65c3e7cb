// The 8-bit KV cache of a softmax anchor: new tokens in (per-head RMSNorm, rotation, quantisation in one
// pass) and rows back out as bf16.
//
// append, per head row x of HD values: x <- x * rsqrt(mean(x^2) + eps) * w, then the rotation of the pairs
// (i, i + HD/2) by the angle fp32(position) * inv_freq[i], all in fp32. A query row is rounded to bf16 once;
// a key or value row goes to int8 with scale = max(max |x| / 127, 2^-40).
// Bound by HBM: per token (H + 2 HKV) HD bf16 in, H HD bf16 and 2 HKV (HD + 4) bytes out.
// A row is HD / 8 lanes of 16 bytes: the norm's sum and the row's maximum are shuffles within these lanes,
// and the rotation's partner is HD / 16 lanes away. A block takes four tokens (few tokens: a share of one token's
// rows), so that a sine and a cosine are taken once per (token, frequency), by all threads at once, while the
// first four rows of every thread are on their way.
#include "../../include/bolt3.h"
#include "kv8.cuh"
#include "trace.h"

namespace {

using namespace b3;
using namespace kv8;

constexpr int kThreads = 256;

template <int LPR>
B3_DEV float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LPR>
B3_DEV float row_max_nan(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

constexpr int kAhead = 4;                            // rows that a thread has in flight

// blockIdx.x = TPB tokens, blockIdx.y = share of their rows
template <int HD, int TPB>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const __grid_constant__ bolt3_kv8_append_args a,
                                                              const __grid_constant__ Length len, int rows_per_block) {
  constexpr int LPR = HD / 8;                        // lanes of a row
  constexpr int RPI = kThreads / LPR;                // rows of one iteration
  __shared__ float2 trig[TPB][HD / 2];
  __shared__ int64_t s_row[TPB];                     // the token's cache row, or -1
  const int tid = threadIdx.x, part = tid % LPR;
  const int64_t tok0 = (int64_t)blockIdx.x * TPB, tokens = (int64_t)a.B * a.T;
  const int n_rows = a.H + 2 * a.HKV;
  const int first = TPB == 1 ? blockIdx.y * rows_per_block : 0;
  const int end = TPB == 1 ? min(n_rows, first + rows_per_block) : (int)min((int64_t)TPB, tokens - tok0) * n_rows;
  grid_dep_launch();
  grid_dep_wait();
  if (tid < TPB && tok0 + tid < tokens) {
    bool bad = false;
    const int b = (int)((tok0 + tid) / a.T), t = (int)((tok0 + tid) % a.T);
    const int64_t s = len.rows(b, bad);
    if (bad && a.status) atomicOr(a.status, 8);
    s_row[tid] = s < 0 ? -1 : s + t;
  }
  __syncthreads();
  for (int i = tid; a.inv_freq != nullptr && i < TPB * (HD / 2); i += kThreads) {
    const int k = i / (HD / 2), f = i % (HD / 2);
    if (tok0 + k < tokens && s_row[k] >= 0) {
      float sn, cs;
      sincosf(__fmul_rn((float)(a.pos0 + (s_row[k] - a.n)), a.inv_freq[f]), &sn, &cs);
      trig[k][f] = make_float2(cs, sn);
    }
  }
  // whole groups of LPR lanes share a row, but the shuffles name the warp: rows past the end compute on zeros
  // and store nothing
  for (int r0 = first; r0 < end; r0 += kAhead * RPI) {
    uint4 raw[kAhead];
    int row[kAhead], tk[kAhead];                     // row of its token, token of the block
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int item = r0 + u * RPI + tid / LPR;
      const bool live = item < end;
      tk[u] = TPB == 1 || !live ? 0 : item / n_rows;
      const int r = live ? item - tk[u] * n_rows : 0;
      row[u] = live ? r : -1;
      const bool is_q = r < a.H, is_k = !is_q && r < a.H + a.HKV;
      const int h = is_q ? r : is_k ? r - a.H : r - a.H - a.HKV;
      const int64_t tok = tok0 + tk[u], b = tok / a.T, t = tok - b * a.T;
      const bf16* src = reinterpret_cast<const bf16*>(is_q ? a.q : is_k ? a.k : a.v);
      src += b * (is_q ? a.q_sb : is_k ? a.k_sb : a.v_sb) + t * (is_q ? a.q_st : is_k ? a.k_st : a.v_st) + (int64_t)h * HD;
      raw[u] = make_uint4(0, 0, 0, 0);
      if (live && s_row[tk[u]] >= 0) raw[u] = __ldg(reinterpret_cast<const uint4*>(src) + part);
    }
    if (r0 == first) __syncthreads();                // the sines and cosines
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (r0 + u * RPI >= end) break;                // the same for all threads
      const int r = row[u];
      const bool is_q = r < a.H, is_k = !is_q && r < a.H + a.HKV;
      const int64_t at = s_row[tk[u]];
      float x[8];
      {
        const float2 p0 = unpack_bf16(raw[u].x), p1 = unpack_bf16(raw[u].y), p2 = unpack_bf16(raw[u].z), p3 = unpack_bf16(raw[u].w);
        x[0] = p0.x; x[1] = p0.y; x[2] = p1.x; x[3] = p1.y; x[4] = p2.x; x[5] = p2.y; x[6] = p3.x; x[7] = p3.y;
      }
      const float* w = is_q ? a.q_norm_w : is_k ? a.k_norm_w : nullptr;
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
      ss = row_sum<LPR>(ss);
      if (w != nullptr) {
        const float inv = rsqrtf(ss * (1.f / HD) + a.eps);
        const float4 w0 = reinterpret_cast<const float4*>(w)[2 * part], w1 = reinterpret_cast<const float4*>(w)[2 * part + 1];
        const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * ww[i];
      }
      if (a.inv_freq != nullptr) {
        const bool second = part >= LPR / 2;         // this lane's values are the pairs' second halves
        const float4* cs = reinterpret_cast<const float4*>(trig[tk[u]] + (second ? part - LPR / 2 : part) * 8);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float4 z = cs[i / 2];                // cos, sin of this value, cos, sin of the next
          const float o0 = __shfl_xor_sync(0xffffffffu, x[i], LPR / 2), o1 = __shfl_xor_sync(0xffffffffu, x[i + 1], LPR / 2);
          if (is_q || is_k) {
            x[i] = second ? fmaf(x[i], z.x, o0 * z.y) : fmaf(x[i], z.x, -o0 * z.y);
            x[i + 1] = second ? fmaf(x[i + 1], z.z, o1 * z.w) : fmaf(x[i + 1], z.z, -o1 * z.w);
          }
        }
      }
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(x[i]));
      m = row_max_nan<LPR>(m);
      if (r < 0) continue;
      const int64_t tok = tok0 + tk[u];
      const int h = is_q ? r : is_k ? r - a.H : r - a.H - a.HKV;
      if (is_q) {
        uint4 o;
        o.x = pack_bf16(x[0], x[1]); o.y = pack_bf16(x[2], x[3]); o.z = pack_bf16(x[4], x[5]); o.w = pack_bf16(x[6], x[7]);
        if (at < 0) o = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.q_out) + (tok * a.H + h) * HD)[part] = o;
      } else if (at >= 0) {
        const float sc = max_nan(__fdiv_rn(m, 127.f), kScaleFloor);
        const int64_t out = (((int64_t)(is_k ? 0 : a.B) + tok / a.T) * a.HKV + h) * a.cap + at;
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo |= ((uint32_t)__float2int_rn(__fdiv_rn(x[i], sc)) & 255u) << (8 * i);
          hi |= ((uint32_t)__float2int_rn(__fdiv_rn(x[4 + i], sc)) & 255u) << (8 * i);
        }
        reinterpret_cast<uint2*>(a.data + out * HD)[part] = make_uint2(lo, hi);
        if (part == 0) a.scale[out] = sc;
      }
    }
  }
}

// a thread is 16 values of a row: blockIdx.x runs over a (keys / values, sequence, head)'s T * HD / 16 pieces
template <int HD>
__global__ void __launch_bounds__(kThreads) kv8_read_kernel(const __grid_constant__ bolt3_kv8_read_args a,
                                                            const __grid_constant__ Length len) {
  constexpr int PPR = HD / 16;
  grid_dep_launch();
  grid_dep_wait();
  const int b = (int)((blockIdx.y / a.HKV) % a.B);
  bool bad = false;
  const int64_t s = len.rows(b, bad);
  if (bad && blockIdx.x == 0 && threadIdx.x == 0 && a.status) atomicOr(a.status, 8);
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.T * PPR) return;
  const int64_t t = i / PPR;
  const int p = (int)(i % PPR);
  uint4 o0 = make_uint4(0, 0, 0, 0), o1 = o0;
  if (s >= 0) {
    const int64_t row = (int64_t)blockIdx.y * a.cap + s + t;
    const uint4 raw = reinterpret_cast<const uint4*>(a.data + row * HD)[p];
    const float sc = a.scale[row];
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int v = (int)w[j];
      o[2 * j] = pack_bf16((float)(v << 24 >> 24) * sc, (float)(v << 16 >> 24) * sc);
      o[2 * j + 1] = pack_bf16((float)(v << 8 >> 24) * sc, (float)(v >> 24) * sc);
    }
    o0 = make_uint4(o[0], o[1], o[2], o[3]);
    o1 = make_uint4(o[4], o[5], o[6], o[7]);
  }
  uint4* dst = reinterpret_cast<uint4*>(a.out) + ((int64_t)blockIdx.y * a.T * PPR + i) * 2;
  dst[0] = o0;
  dst[1] = o1;
}

}  // namespace

extern "C" int bolt3_kv8_append(const bolt3_kv8_append_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_kv8_append");
  if (!a || !a->q || !a->k || !a->v || !a->q_out || !a->data || !a->scale) return BOLT3_ERR_ARG;
  if (a->lens != nullptr && a->pos_dev != nullptr) return BOLT3_ERR_ARG;
  if (a->pos_dev != nullptr && a->pos_span < 1) return BOLT3_ERR_ARG;
  if (a->B <= 0 || a->T <= 0 || a->T > (1 << 20) || a->H <= 0 || a->HKV <= 0 || a->H > 4096 || a->HKV > 2048 ||
      a->H + 2 * a->HKV > 4096 || (a->HD != 64 && a->HD != 128))
    return BOLT3_ERR_SHAPE;
  if ((int64_t)a->B * a->T > 0x7fffffff || (int64_t)a->B * a->HKV > 0x7fffffff) return BOLT3_ERR_SHAPE;
  const int64_t dmax = a->pos_dev != nullptr ? a->pos_span - 1 : 0;
  if (a->n < 0 || a->cap < a->T || (a->lens == nullptr && a->n > a->cap - a->T - dmax)) return BOLT3_ERR_CAPACITY;
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->data |
                       (uintptr_t)a->scale | (uintptr_t)a->q_norm_w | (uintptr_t)a->k_norm_w;
  const int64_t st = a->q_sb | a->q_st | a->k_sb | a->k_st | a->v_sb | a->v_st;
  if ((al & 15) || (st & 7)) return BOLT3_ERR_ALIGN;
  const Length len{a->lens, a->pos_dev, a->n, a->pos_ref, a->pos_span, a->cap, a->T};
  const int rows = a->H + 2 * a->HKV, rpi = kThreads / (a->HD / 8);
  // few tokens: a block per iteration's rows, so that a one-token step still fills the machine; from two blocks of four
  // tokens for every SM on, blocks of four
  const int64_t tokens = (int64_t)a->B * a->T;
  const bool few = tokens < 148 * 8;
  const dim3 grid((unsigned)(few ? tokens : (tokens + 3) / 4), (unsigned)(few ? (rows + rpi - 1) / rpi : 1));
  cudaStream_t s = (cudaStream_t)stream;
  auto kern = a->HD == 128 ? (few ? kv8_append_kernel<128, 1> : kv8_append_kernel<128, 4>)
                           : (few ? kv8_append_kernel<64, 1> : kv8_append_kernel<64, 4>);
  return launch_overlapped(kern, grid, dim3(kThreads), 0, s, *a, len, rpi) == cudaSuccess ? BOLT3_OK : BOLT3_ERR_CUDA;
}

extern "C" int bolt3_kv8_read(const bolt3_kv8_read_args* a, void* stream) {
  const b3::TraceRange trace_range("bolt3_kv8_read");
  if (!a || !a->data || !a->scale || !a->out) return BOLT3_ERR_ARG;
  if (a->B <= 0 || a->HKV <= 0 || a->T <= 0 || (a->HD != 64 && a->HD != 128)) return BOLT3_ERR_SHAPE;
  if ((int64_t)a->B * a->HKV > 32767) return BOLT3_ERR_SHAPE;   // 2 B HKV blocks in grid.y
  if (a->t0 < 0 || a->T > a->cap || (a->lens == nullptr && a->t0 > a->cap - a->T)) return BOLT3_ERR_CAPACITY;
  if (((uintptr_t)a->data | (uintptr_t)a->out | (uintptr_t)a->scale) & 15) return BOLT3_ERR_ALIGN;
  const int64_t blocks = (a->T * (a->HD / 16) + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return BOLT3_ERR_SHAPE;
  const Length len{a->lens, nullptr, a->t0, 0, 0, a->cap, a->T};
  const dim3 grid((unsigned)blocks, (unsigned)(2 * a->B * a->HKV));
  cudaStream_t s = (cudaStream_t)stream;
  return launch_overlapped(a->HD == 128 ? kv8_read_kernel<128> : kv8_read_kernel<64>, grid, dim3(kThreads), 0, s, *a, len) ==
                 cudaSuccess ? BOLT3_OK : BOLT3_ERR_CUDA;
}
