// k_qknorm.cu -- RMS norm of every query and key head and the position
// rotation, in one pass over rows of Q|K|V, and its backward pass.
//
//   xn = x r, r = 1 / sqrt(mean x^2 + eps),  y = R(pos) (xn o g)
// per head vector x of head_dim values, with one gain g for the query heads
// and one for the key heads.  R turns the pairs (a, b) of the first rot_dim
// values by the angle whose cosine and sine the tables hold for the row's
// position: (a c - b s, a s + b c); pairs are (m, m + rot_dim / 2), as in
// rope-half (lisp/nelisp-gpu-kernels.el:857-882), or (2m, 2m + 1), as in
// rope-apply.  Backward, with u = R^T dy and w = u o g:
//   dg = sum over rows and heads of u o xn,  dx = r (w - xn mean(w o xn)).
//
// Bound by memory: every value is read once (x; x and dy) and written once.
// A group of G lanes holds a head vector, each lane two 16-byte chunks that
// are partners of the rotation, so a head needs one reduction over the group
// and no exchange of values.  A warp takes one row and walks its heads with
// the row's cosines and sines, and the gain, in registers; U vectors are
// requested before the first is used.  All arithmetic is in 32 bits; the one
// rounding to the output type is at the store.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "nl_internal.h"

namespace nl {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct QkArgs {
  const void *x;                 // rows of Q|K|V
  uint64_t x_stride;
  const float *g[2];             // gains of the query and the key heads
  const float *co, *si;          // [rope_rows][rot / 2]
  const int32_t *pos;
  const void *dy[2];             // backward: gradients of q and k
  uint64_t dy_stride[2];
  void *out[2];                  // q and k; backward: dx of the two parts
  uint64_t out_stride[2];
  float *partial;                // backward: [blocks][2][head_dim]
  uint32_t n, heads, kv_heads, head_dim, rot, rope_rows;
  uint32_t per_job, jobs_per_row;  // heads a warp takes, and jobs a row has
  float eps;
};

template <typename T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4 &w, float *v) {
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y);
    v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 put(const float *v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
  }
};
template <> struct Chunk<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4 &w, float *v) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 put(const float *v) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t *>(&p);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// Where this lane of a group stands: its two chunks of a head vector and
// whether they are rotated.  Pairs of a rotated lane are (v[e], v[N + e]) in
// the half form and (v[2e], v[2e + 1]) in the adjacent form; either way their
// angles are lane * N + e.
struct Place {
  uint32_t c0, c1;
  bool live, turned;
};
template <typename T, bool HALF>
__device__ __forceinline__ Place place_of(uint32_t j, uint32_t head_dim, uint32_t rot) {
  constexpr uint32_t N = Chunk<T>::N;
  const uint32_t half = rot / 2 / N;
  Place p;
  p.live = j < head_dim / (2 * N);
  p.turned = j < half;
  p.c0 = HALF && p.turned ? j : 2 * j;
  p.c1 = HALF && p.turned ? j + half : 2 * j + 1;
  return p;
}

template <int N, bool HALF>
__device__ __forceinline__ void turn(float *v, const float *c, const float *s) {
#pragma unroll
  for (int e = 0; e < N; e++) {
    float &a = v[HALF ? e : 2 * e], &b = v[HALF ? N + e : 2 * e + 1];
    const float a0 = a, b0 = b;
    a = a0 * c[e] - b0 * s[e];
    b = a0 * s[e] + b0 * c[e];
  }
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp, one row, the heads [h0, h1) of one part (queries or keys), a
// group of G lanes per head.
template <typename T, int G, bool HALF, bool BWD, int U>
__device__ __forceinline__ void walk(const QkArgs &a, int part, uint32_t row, uint32_t h0,
                                     uint32_t h1, const Place &p, bool real, const float *c,
                                     const float *s, float *dg) {
  constexpr int N = Chunk<T>::N, H = 32 / G;
  if (h0 >= h1) return;
  const uint32_t lane = threadIdx.x & 31, mine = lane / G;
  const T *x = (const T *)a.x + (uint64_t)row * a.x_stride +
               (part ? (uint64_t)a.heads * a.head_dim : 0);
  const T *dy = BWD ? (const T *)a.dy[part] + (uint64_t)row * a.dy_stride[part] : nullptr;
  T *out = (T *)a.out[part] + (uint64_t)row * a.out_stride[part];
  float g[2 * N];
#pragma unroll
  for (int e = 0; e < 2 * N; e++) g[e] = 0.0f;
  if (p.live) {
#pragma unroll
    for (int e = 0; e < N; e++) {
      g[e] = __ldg(a.g[part] + p.c0 * N + e);
      g[N + e] = __ldg(a.g[part] + p.c1 * N + e);
    }
  }
  const float inv_d = 1.0f / (float)a.head_dim;
  for (uint32_t h = h0; h < h1; h += H * U) {
    uint4 w[U][2], d[BWD ? U : 1][2];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t hh = h + u * H + mine;
      const bool on = p.live && hh < h1 && real;
      const uint64_t at = (uint64_t)hh * a.head_dim;
      w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
      if (BWD) d[u][0] = d[u][1] = make_uint4(0, 0, 0, 0);
      if (on) {
        w[u][0] = *reinterpret_cast<const uint4 *>(x + at + p.c0 * N);
        w[u][1] = *reinterpret_cast<const uint4 *>(x + at + p.c1 * N);
        if (BWD) {
          d[u][0] = *reinterpret_cast<const uint4 *>(dy + at + p.c0 * N);
          d[u][1] = *reinterpret_cast<const uint4 *>(dy + at + p.c1 * N);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t hh = h + u * H + mine;
      float v[2 * N];
      Chunk<T>::get(w[u][0], v);
      Chunk<T>::get(w[u][1], v + N);
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 2 * N; e++) ss = fmaf(v[e], v[e], ss);
      const float r = rsqrtf(fmaf(group_sum<G>(ss), inv_d, a.eps));
      if (!BWD) {
#pragma unroll
        for (int e = 0; e < 2 * N; e++) v[e] = v[e] * r * g[e];
        if (p.turned) turn<N, HALF>(v, c, s);
      } else {
        float q[2 * N];
        Chunk<T>::get(d[u][0], q);
        Chunk<T>::get(d[u][1], q + N);
        if (p.turned) turn<N, HALF>(q, c, s);      // s is negated by the caller
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 2 * N; e++) {
          v[e] *= r;
          dg[e] = fmaf(q[e], v[e], dg[e]);
          q[e] *= g[e];
          dot = fmaf(q[e], v[e], dot);
        }
        dot = group_sum<G>(dot) * inv_d;
#pragma unroll
        for (int e = 0; e < 2 * N; e++) v[e] = r * fmaf(-v[e], dot, q[e]);
      }
      if (p.live && hh < h1) {
        const uint64_t at = (uint64_t)hh * a.head_dim;
        if (!real) {
#pragma unroll
          for (int e = 0; e < 2 * N; e++) v[e] = 0.0f;
        }
        *reinterpret_cast<uint4 *>(out + at + p.c0 * N) = Chunk<T>::put(v);
        *reinterpret_cast<uint4 *>(out + at + p.c1 * N) = Chunk<T>::put(v + N);
      }
    }
  }
}

template <typename T, int G, bool HALF, bool BWD, int U>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ QkArgs a) {
  constexpr int N = Chunk<T>::N;
  pdl_trigger();
  pdl_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Place p = place_of<T, HALF>(lane % G, a.head_dim, a.rot);
  float dg[2][2 * N];
  if (BWD) {
#pragma unroll
    for (int e = 0; e < 2 * N; e++) dg[0][e] = dg[1][e] = 0.0f;
  }
  const uint64_t jobs = (uint64_t)a.n * a.jobs_per_row;
  for (uint64_t job = (uint64_t)blockIdx.x * kWarps + warp; job < jobs;
       job += (uint64_t)gridDim.x * kWarps) {
    const uint32_t row = (uint32_t)(job / a.jobs_per_row);
    const uint32_t h0 = (uint32_t)(job % a.jobs_per_row) * a.per_job;
    const uint32_t h1 = min(h0 + a.per_job, a.heads + a.kv_heads);
    const int32_t pos = __ldg(a.pos + row);
    const bool real = (uint32_t)pos < a.rope_rows;
    float c[N], s[N];
    if (p.turned && real) {
      const uint64_t at = (uint64_t)pos * (a.rot / 2) + (lane % G) * N;
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const float4 cc = __ldg(reinterpret_cast<const float4 *>(a.co + at + e));
        const float4 sc = __ldg(reinterpret_cast<const float4 *>(a.si + at + e));
        c[e] = cc.x; c[e + 1] = cc.y; c[e + 2] = cc.z; c[e + 3] = cc.w;
        s[e] = sc.x; s[e + 1] = sc.y; s[e + 2] = sc.z; s[e + 3] = sc.w;
      }
      if (BWD) {
#pragma unroll
        for (int e = 0; e < N; e++) s[e] = -s[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) c[e] = s[e] = 0.0f;
    }
    walk<T, G, HALF, BWD, U>(a, 0, row, min(h0, a.heads), min(h1, a.heads), p, real, c, s, dg[0]);
    walk<T, G, HALF, BWD, U>(a, 1, row, max(h0, a.heads) - a.heads, max(h1, a.heads) - a.heads, p,
                             real, c, s, dg[1]);
  }
  if (BWD) {
    // this block's share of the gain gradients, summed in a fixed order
    __shared__ float red[kWarps][2 * N * G];
#pragma unroll
    for (int part = 0; part < 2; part++) {
#pragma unroll
      for (int e = 0; e < 2 * N; e++) {
        float v = dg[part][e];
#pragma unroll
        for (int o = G; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane < G) red[warp][lane * 2 * N + e] = v;
      }
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < 2 * N * G; i += kThreads) {
        const Place q = place_of<T, HALF>(i / (2 * N), a.head_dim, a.rot);
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) v += red[w][i];
        const uint32_t e = i % (2 * N);
        if (q.live)
          a.partial[((uint64_t)blockIdx.x * 2 + part) * a.head_dim +
                    (e < N ? q.c0 * N + e : q.c1 * N + e - N)] = v;
      }
      __syncthreads();
    }
  }
}

// dG[part][i] = the sum of the blocks' shares, in a fixed order: a block takes
// eight columns, 32 threads a column.
__global__ void __launch_bounds__(256)
qk_gain_sum_kernel(const float *partial, uint32_t blocks, uint32_t head_dim, float *dgq,
                   float *dgk) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red[32][9];
  const uint32_t col = threadIdx.x & 7, k = threadIdx.x >> 3, at = blockIdx.x * 8 + col;
  float v = 0.0f;
  for (uint32_t b = k; b < blocks; b += 32) v += partial[(uint64_t)b * 2 * head_dim + at];
  red[k][col] = v;
  __syncthreads();
  if (k == 0) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i++) t += red[i][col];
    if (at < head_dim) dgq[at] = t;
    else dgk[at - head_dim] = t;
  }
}

template <typename T, int G, bool HALF, bool BWD, int U>
cudaError_t start(QkArgs &a, uint32_t blocks, cudaStream_t st) {
  return launch_pdl(qk_norm_rope_kernel<T, G, HALF, BWD, U>, dim3(blocks), dim3(kThreads), 0, st,
                    a);
}
template <typename T, bool BWD>
cudaError_t start_t(QkArgs &a, bool half, uint32_t group, uint32_t blocks, cudaStream_t st) {
  constexpr int U = BWD ? 2 : 4;
  switch (group * 2 + (half ? 1 : 0)) {
    case 8: return start<T, 4, false, BWD, U>(a, blocks, st);
    case 9: return start<T, 4, true, BWD, U>(a, blocks, st);
    case 16: return start<T, 8, false, BWD, U>(a, blocks, st);
    case 17: return start<T, 8, true, BWD, U>(a, blocks, st);
    case 32: return start<T, 16, false, BWD, U>(a, blocks, st);
    case 33: return start<T, 16, true, BWD, U>(a, blocks, st);
  }
  if constexpr (sizeof(T) == 4) {   // 256 values of 16 bits take 16 lanes
    return half ? start<T, 32, true, BWD, U>(a, blocks, st)
                : start<T, 32, false, BWD, U>(a, blocks, st);
  }
  return cudaErrorInvalidValue;
}

// Lanes that hold a head vector, two 16-byte chunks each.
uint32_t group_of(int dtype, uint32_t head_dim) {
  const uint32_t lanes = head_dim / (dtype == NL_BF16 ? 16 : 8);
  uint32_t g = 4;
  while (g < lanes) g *= 2;
  return g;
}

constexpr uint32_t kMaxBlocks = 148 * 4;

// How a launch divides n rows of HEADS heads: a warp takes whole rows once
// there are enough of them to fill the GPU's warps, and otherwise as few heads
// as a warp holds at a time.
uint32_t divide(QkArgs &a, uint32_t at_once) {
  const uint32_t all = a.heads + a.kv_heads;
  a.per_job = all;
  while (a.per_job > at_once &&
         (uint64_t)a.n * ((all + a.per_job - 1) / a.per_job) < (uint64_t)kMaxBlocks * kWarps)
    a.per_job = (a.per_job + 1) / 2;
  a.per_job = (a.per_job + at_once - 1) / at_once * at_once;
  a.jobs_per_row = (all + a.per_job - 1) / a.per_job;
  const uint64_t blocks = ceil_div64((uint64_t)a.n * a.jobs_per_row, kWarps);
  return (uint32_t)(blocks < kMaxBlocks ? blocks : kMaxBlocks);
}

int check_common(const char *what, int dtype, const QkArgs &a, int pairs) {
  if (dtype != NL_F32 && dtype != NL_BF16)
    return set_error(NL_ERROR, "%s: type %d is neither NL_F32 nor NL_BF16", what, dtype);
  if (pairs != NL_PAIRS_HALF && pairs != NL_PAIRS_ADJACENT)
    return set_error(NL_ERROR, "%s: pairs %d", what, pairs);
  const uint32_t unit = dtype == NL_BF16 ? 16 : 8;
  if (!a.heads || !a.kv_heads || a.heads > 65536 || a.kv_heads > 65536)
    return set_error(NL_ERROR, "%s: heads %u, kv heads %u", what, a.heads, a.kv_heads);
  if (!a.head_dim || a.head_dim > 256 || a.head_dim % unit || !a.rot || a.rot > a.head_dim ||
      a.rot % unit)
    return set_error(NL_ERROR,
                     "%s: head size %u (at most 256) and rotated part %u must be multiples of %u",
                     what, a.head_dim, a.rot, unit);
  return NL_OK;
}

int check_rows(const char *what, const char *name, int dtype, const void *p, uint64_t stride,
               uint64_t width) {
  const uint32_t per = dtype == NL_BF16 ? 8 : 4;
  if (!p || !aligned16(p) || stride < width || stride % per)
    return set_error(NL_ERROR,
                     "%s: %s rows must be 16-byte aligned, with a stride (%llu) that is a multiple "
                     "of %u and at least %llu",
                     what, name, (unsigned long long)stride, per, (unsigned long long)width);
  return NL_OK;
}

int check_tables(const char *what, const QkArgs &a) {
  if (!a.g[0] || !a.g[1] || !a.pos || !a.co || !a.si || !aligned16(a.co) || !aligned16(a.si))
    return set_error(NL_ERROR, "%s: a null gain, position or table, or an unaligned table", what);
  return NL_OK;
}

}  // namespace
}  // namespace nl

using namespace nl;

extern "C" int nl_qk_norm_rope_dev(int dtype, const void *QKV, uint64_t x_stride, const float *GQ,
                                   const float *GK, const float *CO, const float *SI,
                                   const int32_t *POS, void *Q, uint64_t q_stride, void *K,
                                   uint64_t k_stride, uint32_t n, uint32_t heads,
                                   uint32_t kv_heads, uint32_t head_dim, uint32_t rot_dim,
                                   uint32_t rope_rows, int pairs, float eps, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  const char *what = "qk-norm-rope";
  QkArgs a = {};
  a.x = QKV; a.x_stride = x_stride; a.g[0] = GQ; a.g[1] = GK; a.co = CO; a.si = SI; a.pos = POS;
  a.out[0] = Q; a.out[1] = K; a.out_stride[0] = q_stride; a.out_stride[1] = k_stride;
  a.n = n; a.heads = heads; a.kv_heads = kv_heads; a.head_dim = head_dim; a.rot = rot_dim;
  a.rope_rows = rope_rows; a.eps = eps;
  if ((rc = check_common(what, dtype, a, pairs))) return rc;
  if (n == 0) return NL_OK;
  const uint64_t qw = (uint64_t)heads * head_dim, kw = (uint64_t)kv_heads * head_dim;
  if ((rc = check_rows(what, "QKV", dtype, QKV, x_stride, qw + kw)) ||
      (rc = check_rows(what, "Q", dtype, Q, q_stride, qw)) ||
      (rc = check_rows(what, "K", dtype, K, k_stride, kw)) || (rc = check_tables(what, a)))
    return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t group = group_of(dtype, head_dim), blocks = divide(a, 32 / group);
  const bool half = pairs == NL_PAIRS_HALF;
  const cudaError_t e = dtype == NL_BF16 ? start_t<__nv_bfloat16, false>(a, half, group, blocks, st)
                                         : start_t<float, false>(a, half, group, blocks, st);
  count_launches(1);
  return cuda_status(e, what);
}

extern "C" size_t nl_qk_norm_rope_bwd_workspace_bytes(uint32_t head_dim) {
  return (size_t)kMaxBlocks * 2 * head_dim * sizeof(float);
}

extern "C" int nl_qk_norm_rope_bwd_dev(int dtype, const void *QKV, uint64_t x_stride,
                                       const float *GQ, const float *GK, const float *CO,
                                       const float *SI, const int32_t *POS, const void *DQ,
                                       uint64_t dq_stride, const void *DK, uint64_t dk_stride,
                                       void *DQKV, uint64_t dx_stride, float *DGQ, float *DGK,
                                       uint32_t n, uint32_t heads, uint32_t kv_heads,
                                       uint32_t head_dim, uint32_t rot_dim, uint32_t rope_rows,
                                       int pairs, float eps, void *workspace, size_t ws_bytes,
                                       void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  const char *what = "qk-norm-rope-bwd";
  QkArgs a = {};
  a.x = QKV; a.x_stride = x_stride; a.g[0] = GQ; a.g[1] = GK; a.co = CO; a.si = SI; a.pos = POS;
  a.dy[0] = DQ; a.dy[1] = DK; a.dy_stride[0] = dq_stride; a.dy_stride[1] = dk_stride;
  a.out_stride[0] = a.out_stride[1] = dx_stride;
  a.n = n; a.heads = heads; a.kv_heads = kv_heads; a.head_dim = head_dim; a.rot = rot_dim;
  a.rope_rows = rope_rows; a.eps = eps;
  if ((rc = check_common(what, dtype, a, pairs))) return rc;
  if (!DGQ || !DGK) return set_error(NL_ERROR, "%s: a null gain gradient", what);
  cudaStream_t st = (cudaStream_t)stream;
  uint32_t blocks = 0;
  if (n) {
    const uint64_t qw = (uint64_t)heads * head_dim, kw = (uint64_t)kv_heads * head_dim;
    if ((rc = check_rows(what, "QKV", dtype, QKV, x_stride, qw + kw)) ||
        (rc = check_rows(what, "DQ", dtype, DQ, dq_stride, qw)) ||
        (rc = check_rows(what, "DK", dtype, DK, dk_stride, kw)) ||
        (rc = check_rows(what, "DQKV", dtype, DQKV, dx_stride, qw + kw)) ||
        (rc = check_tables(what, a)))
      return rc;
    const size_t need = nl_qk_norm_rope_bwd_workspace_bytes(head_dim);
    if (workspace && ws_bytes < need)
      return set_error(NL_ERROR, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
    if (!workspace) workspace = library_workspace(need, st);
    if (!workspace || !aligned16(workspace))
      return set_error(NL_ERROR, "%s: no aligned workspace of %zu bytes", what, need);
    a.partial = (float *)workspace;
    a.out[0] = DQKV;
    a.out[1] = (char *)DQKV + qw * (dtype == NL_BF16 ? 2 : 4);
    const uint32_t group = group_of(dtype, head_dim);
    blocks = divide(a, 32 / group);
    const bool half = pairs == NL_PAIRS_HALF;
    const cudaError_t e = dtype == NL_BF16
                              ? start_t<__nv_bfloat16, true>(a, half, group, blocks, st)
                              : start_t<float, true>(a, half, group, blocks, st);
    count_launches(1);
    if (e != cudaSuccess) return cuda_status(e, what);
  }
  const cudaError_t e = launch_pdl(qk_gain_sum_kernel, dim3(2 * head_dim / 8), dim3(256), 0, st,
                                   (const float *)workspace, blocks, head_dim, DGQ, DGK);
  count_launches(1);
  return cuda_status(e, what);
}
