// The 8-bit KV cache of a softmax anchor: new tokens in (per-head RMSNorm, rotation, quantisation in one
// pass) and rows back out as bf16.
//
// append, per head row x of HD values: x <- x * rsqrt(mean(x^2) + eps) * w, then the rotation of the pairs
// (i, i + HD/2) by the angle fp32(position) * inv_freq[i], all in fp32. A query row is rounded to bf16 once;
// a key or value row goes to int8 with scale = max(max |x| / 127, 2^-40).
// Bound by HBM: per token (H + 2 HKV) HD bf16 in, H HD bf16 and 2 HKV (HD + 4) bytes out.
// A row is HD / 8 lanes, a lane holding four neighbouring values of each half: a rotation's pair is in one lane,
// the norm's sum and the row's maximum are shuffles within the row's lanes. A block takes four tokens (few tokens: a share
// of one token's rows), so that a sine and a cosine are taken once per (token, frequency), by all threads at once, while
// the first four rows of every thread are on their way. With a row's neighbouring pairs in different lanes, 64-bit index
// divisions and a true division per value the same work took a quarter longer.
//
// read: a thread takes 16 values; bound by HBM, HD + 4 bytes in and 2 HD out per row.
//
// Measured on a B200: append and read of 37 x 101 tokens, 15 + 2 x 5 heads of 64, 14.5 us (their bytes take 4.4; bound by
// instructions, about 200 per 8 values); of 64 x 1 token, 32 + 2 x 8 heads of 128, 5.1 us (two launches of 2.5); read of
// 16 x 8 x 2047 rows of 128, 36 us (5.6 TB/s).
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
  __shared__ float4 trig[TPB][HD / 4];               // cos, sin of a pair of dimensions, cos, sin of the next
  // of each token: its cache row (-1: idle), its first q, k and v element, and the cache row of its first head's keys
  __shared__ int64_t s_row[TPB], s_src[TPB][3], s_out[TPB];
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
    s_src[tid][0] = b * a.q_sb + t * a.q_st;
    s_src[tid][1] = b * a.k_sb + t * a.k_st;
    s_src[tid][2] = b * a.v_sb + t * a.v_st;
    s_out[tid] = (int64_t)b * a.HKV * a.cap + s + t;
  }
  __syncthreads();
  for (int i = tid; a.inv_freq != nullptr && i < TPB * (HD / 2); i += kThreads) {
    const int k = i / (HD / 2), f = i % (HD / 2);
    if (tok0 + k < tokens && s_row[k] >= 0) {
      float sn, cs;
      sincosf(__fmul_rn((float)(a.pos0 + (s_row[k] - a.n)), a.inv_freq[f]), &sn, &cs);
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
      const int64_t at = s_row[tk[u]];
      float x[8];                                    // values 4 part .., HD / 2 + 4 part ..
      {
        const float2 p0 = unpack_bf16(raw[u][0].x), p1 = unpack_bf16(raw[u][0].y), p2 = unpack_bf16(raw[u][1].x), p3 = unpack_bf16(raw[u][1].y);
        x[0] = p0.x; x[1] = p0.y; x[2] = p1.x; x[3] = p1.y; x[4] = p2.x; x[5] = p2.y; x[6] = p3.x; x[7] = p3.y;
      }
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
      if (a.inv_freq != nullptr && (is_q || is_k)) {
        const float4* cs = trig[tk[u]] + 2 * part;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float4 z = cs[i / 2];                // of pairs i and i + 1
          const float a0 = x[i], b0 = x[4 + i], a1 = x[i + 1], b1 = x[5 + i];
          x[i] = fmaf(a0, z.x, -b0 * z.y);
          x[4 + i] = fmaf(b0, z.x, a0 * z.y);
          x[i + 1] = fmaf(a1, z.z, -b1 * z.w);
          x[5 + i] = fmaf(b1, z.z, a1 * z.w);
        }
      }
      const int h = is_q ? r : is_k ? r - a.H : r - a.H - a.HKV;
      if (is_q && r >= 0) {
        uint2 o0 = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        uint2 o1 = make_uint2(pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
        if (at < 0) o0 = o1 = make_uint2(0, 0);
        bf16* out = reinterpret_cast<bf16*>(a.q_out) + ((tok0 + tk[u]) * a.H + h) * HD;
        reinterpret_cast<uint2*>(out)[part] = o0;
        reinterpret_cast<uint2*>(out + HD / 2)[part] = o1;
      }
      const bool stores = r >= 0 && !is_q && at >= 0;
      if (!__any_sync(0xffffffffu, stores)) continue;
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(x[i]));
      m = row_max_nan<LPR>(m);
      const float sc = max_nan(__fdiv_rn(m, 127.f), kScaleFloor);
      // x / sc to the nearest integer: by the reciprocal, whose product is within 127 * 2^-22 of the quotient; only where
      // that leaves the rounding open (and for rows that are not finite) by division
      const float inv = __frcp_rn(sc);
      uint32_t word[2] = {0, 0};
      bool open = !(m < 3e38f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = x[i] * inv, z = y + 12582912.f;   // 1.5 * 2^23: the integer stands in the low bits
        open |= fabsf(fabsf(y - (z - 12582912.f)) - 0.5f) < 1e-4f;
        word[i / 4] |= (__float_as_uint(z) & 255u) << (8 * (i & 3));
      }
      if (open) {
        word[0] = word[1] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) word[i / 4] |= ((uint32_t)__float2int_rn(__fdiv_rn(x[i], sc)) & 255u) << (8 * (i & 3));
      }
      if (stores) {
        const int64_t out = s_out[tk[u]] + ((int64_t)(is_k ? 0 : a.B) * a.HKV + h) * a.cap;
        reinterpret_cast<uint32_t*>(a.data + out * HD)[part] = word[0];
        reinterpret_cast<uint32_t*>(a.data + out * HD + HD / 2)[part] = word[1];
        if (part == 0) a.scale[out] = sc;
      }
    }
  }
}

// a thread is 16 values of a row; `per` blocks for the T * HD / 16 pieces of a (keys / values, sequence, head)
template <int HD>
__global__ void __launch_bounds__(kThreads) kv8_read_kernel(const __grid_constant__ bolt3_kv8_read_args a,
                                                            const __grid_constant__ Length len, unsigned per) {
  constexpr int PPR = HD / 16;
  const int64_t slice = blockIdx.x / per;
  const unsigned blk = blockIdx.x - (unsigned)slice * per;
  grid_dep_launch();
  grid_dep_wait();
  const int b = (int)((slice / a.HKV) % a.B);
  bool bad = false;
  const int64_t s = len.rows(b, bad);
  if (bad && blk == 0 && threadIdx.x == 0 && a.status) atomicOr(a.status, 8);
  const int64_t i = (int64_t)blk * kThreads + threadIdx.x;
  if (i >= a.T * PPR) return;
  const int64_t t = i / PPR;
  const int p = (int)(i % PPR);
  uint4 o0 = make_uint4(0, 0, 0, 0), o1 = o0;
  if (s >= 0) {
    const int64_t row = slice * a.cap + s + t;
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
  uint4* dst = reinterpret_cast<uint4*>(a.out) + (slice * a.T * PPR + i) * 2;
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
  if (a->t0 < 0 || a->T > a->cap || (a->lens == nullptr && a->t0 > a->cap - a->T)) return BOLT3_ERR_CAPACITY;
  if (((uintptr_t)a->data | (uintptr_t)a->out | (uintptr_t)a->scale) & 15) return BOLT3_ERR_ALIGN;
  const int64_t slices = 2 * (int64_t)a->B * a->HKV, per = (a->T * (a->HD / 16) + kThreads - 1) / kThreads;
  if (per > 0x7fffffff / slices) return BOLT3_ERR_SHAPE;
  const Length len{a->lens, nullptr, a->t0, 0, 0, a->cap, a->T};
  const dim3 grid((unsigned)(slices * per));
  cudaStream_t s = (cudaStream_t)stream;
  return launch_overlapped(a->HD == 128 ? kv8_read_kernel<128> : kv8_read_kernel<64>, grid, dim3(kThreads), 0, s, *a, len,
                           (unsigned)per) ==
                 cudaSuccess ? BOLT3_OK : BOLT3_ERR_CUDA;
}
