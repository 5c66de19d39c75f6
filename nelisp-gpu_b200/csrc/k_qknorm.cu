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
// and no exchange of values.  A warp takes one row and walks its query or its
// key heads with the row's products of gain, cosine and sine in registers;
// blocks belong to one of the two parts, so a thread holds one gain (and one
// set of gain gradients).  The next vectors are on their way to shared memory
// meanwhile, in runs of whole vectors whatever the pairs.  Arithmetic is two
// floats an instruction, all in 32 bits; the one rounding to the output type is
// at the store.  8,192 rows of 40 heads of 128, bfloat16, one row in twenty
// padding: 30.9 us, 5.6 TB/s, 0.85 of a copy; backward, 8,191 rows of 40 heads of
// 64: 28.4 us, 4.5 TB/s, bound by the latency of a step that few warps hide.  A part
// with fewer heads than a warp holds at a time leaves the other lanes idle: 8,192
// rows of 8 heads and 1 of 64, bfloat16, take 11.6 us where 32 and 8 take 15.9.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "f32x2.cuh"
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
  float *partial;                // backward: [blocks][head_dim]
  uint32_t n, heads[2], head_dim, rot, rope_rows;
  uint32_t per_job[2], jobs_per_row[2], blocks[2];  // heads a warp takes; how a part is divided
  float eps;
};

// Where this lane of a group stands: its two chunks of a head vector.  Pair e
// of a rotated lane turns by angle lane * N + e; in the half form its values
// are the chunks' values e, in the adjacent form values 2e and 2e + 1 of the
// two chunks in a row.  Lanes past the rotated part turn by no angle.
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

// The first and second values of a lane's N pairs, from its chunks and back.
template <typename T, bool HALF>
__device__ __forceinline__ void split(const uint4 &w0, const uint4 &w1, Pair *a, Pair *b) {
  constexpr int N = Chunk<T>::N;
  if (HALF) {
    Chunk<T>::get(w0, a);
    Chunk<T>::get(w1, b);
  } else {
    Pair v[N];
    Chunk<T>::get(w0, v);
    Chunk<T>::get(w1, v + N / 2);
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      const float2 x = unpair(v[2 * i]), y = unpair(v[2 * i + 1]);
      a[i] = pair(x.x, y.x);
      b[i] = pair(x.y, y.y);
    }
  }
}
template <typename T, bool HALF>
__device__ __forceinline__ void merge(const Pair *a, const Pair *b, uint4 &w0, uint4 &w1) {
  constexpr int N = Chunk<T>::N;
  if (HALF) {
    w0 = Chunk<T>::put(a);
    w1 = Chunk<T>::put(b);
  } else {
    Pair v[N];
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      const float2 x = unpair(a[i]), y = unpair(b[i]);
      v[2 * i] = pair(x.x, y.x);
      v[2 * i + 1] = pair(x.y, y.y);
    }
    w0 = Chunk<T>::put(v);
    w1 = Chunk<T>::put(v + N / 2);
  }
}

template <int G>
__device__ __forceinline__ float group_sum(Pair p) {
  const float2 f = unpair(p);
  float v = f.x + f.y;
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 16 bytes to shared memory on their way while others are worked on, or zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from),
               "r"(some ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;\n" ::: "memory");
}
template <int AHEAD> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(AHEAD) : "memory");
}

// DEPTH steps of U vectors a group are on their way to shared memory.
template <typename T, int G, bool HALF, bool BWD, int U, int DEPTH, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM)
qk_norm_rope_kernel(const __grid_constant__ QkArgs a) {
  constexpr int N = Chunk<T>::N, P = N / 2, H = 32 / G, CH = BWD ? 4 : 2;
  extern __shared__ uint4 ring[];
  pdl_trigger();
  pdl_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = lane / G;
  const int part = blockIdx.x >= a.blocks[0];
  const uint32_t block = blockIdx.x - (part ? a.blocks[0] : 0), heads = a.heads[part];
  const uint32_t per_row = a.jobs_per_row[part];
  const Place p = place_of<T, HALF>(lane % G, a.head_dim, a.rot);
  const uint32_t at0 = p.c0 * N, at1 = p.c1 * N;
  Pair ga[P], gb[P];
  {
    float v[2 * N];
#pragma unroll
    for (int e = 0; e < N; e++) {
      v[e] = p.live ? __ldg(a.g[part] + (HALF ? at0 + e : (e < P ? at0 : at1 - N) + 2 * e)) : 0.0f;
      v[N + e] =
          p.live ? __ldg(a.g[part] + (HALF ? at1 + e : (e < P ? at0 : at1 - N) + 2 * e + 1)) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < P; i++) {
      ga[i] = pair(v[2 * i], v[2 * i + 1]);
      gb[i] = pair(v[N + 2 * i], v[N + 2 * i + 1]);
    }
  }
  Pair da[P], db[P];             // backward: the gain's gradient so far
#pragma unroll
  for (int i = 0; i < P; i++) da[i] = db[i] = 0;
  const float inv_d = 1.0f / (float)a.head_dim;
  const uint64_t jobs = (uint64_t)a.n * per_row;
  // the position and the angles of a job's row, asked for a job ahead
  const uint64_t step = (uint64_t)a.blocks[part] * kWarps;
  auto position = [&](uint64_t job) {
    return job < jobs ? __ldg(a.pos + (per_row == 1 ? job : job / per_row)) : -1;
  };
  float c[N], s[N];
  auto angles = [&](int32_t pos) {
#pragma unroll
    for (int e = 0; e < N; e++) c[e] = 1.0f, s[e] = 0.0f;
    if (p.turned && (uint32_t)pos < a.rope_rows) {
      const uint64_t at = (uint64_t)pos * (a.rot / 2) + (lane % G) * N;
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const float4 cc = __ldg(reinterpret_cast<const float4 *>(a.co + at + e));
        const float4 sc = __ldg(reinterpret_cast<const float4 *>(a.si + at + e));
        c[e] = cc.x; c[e + 1] = cc.y; c[e + 2] = cc.z; c[e + 3] = cc.w;
        s[e] = sc.x; s[e + 1] = sc.y; s[e + 2] = sc.z; s[e + 3] = sc.w;
      }
    }
  };
  const uint64_t first = (uint64_t)block * kWarps + warp;
  int32_t pos = position(first), pos_next = position(first + step);
  angles(pos);
  // The vectors to come, over the ends of jobs: a group copies one in two runs,
  // whatever chunks its lanes then take.
  uint4 *slots = ring + warp * (DEPTH * U * CH * 32) + mine * (2 * G);
  const uint32_t j = lane % G, chunks = a.head_dim / N;
  const uint32_t slots_at = (uint32_t)__cvta_generic_to_shared(slots + j);
  uint64_t next_job = first;
  uint32_t next_h = 0, next_end = 0, into = 0, from = 0;
  const T *next_x = nullptr, *next_dy = nullptr;
  auto aim = [&]() {
    const uint32_t row = per_row == 1 ? (uint32_t)next_job : (uint32_t)(next_job / per_row);
    next_h = per_row == 1 ? 0 : (uint32_t)(next_job % per_row) * a.per_job[part];
    next_end = min(next_h + a.per_job[part], heads);
    next_x = (const T *)a.x + (uint64_t)row * a.x_stride +
             (uint64_t)((part ? a.heads[0] : 0) + next_h + mine) * a.head_dim + j * N;
    if (BWD)
      next_dy = (const T *)a.dy[part] + (uint64_t)row * a.dy_stride[part] +
                (uint64_t)(next_h + mine) * a.head_dim + j * N;
  };
  auto fetch = [&]() {
    if (next_job < jobs) {
      const uint32_t to = slots_at + into * (U * CH * 512);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool some = next_h + mine + u * H < next_end;
        const bool in0 = some && j < chunks, in1 = some && j + G < chunks;
        const T *v = next_x + u * H * a.head_dim;
        copy16(to + u * CH * 512, in0 ? v : (const T *)a.x, in0);
        copy16(to + u * CH * 512 + G * 16, in1 ? v + G * N : (const T *)a.x, in1);
        if (BWD) {
          const T *g = next_dy + u * H * a.head_dim;
          copy16(to + u * CH * 512 + 1024, in0 ? g : (const T *)a.x, in0);
          copy16(to + u * CH * 512 + 1024 + G * 16, in1 ? g + G * N : (const T *)a.x, in1);
        }
      }
      into = into + 1 == DEPTH ? 0 : into + 1;
      next_h += H * U;
      next_x += H * U * a.head_dim;
      if (BWD) next_dy += H * U * a.head_dim;
      if (next_h >= next_end) {
        next_job += step;
        if (next_job < jobs) aim();
      }
    }
    copy_commit();
  };
  if (next_job < jobs) aim();
#pragma unroll
  for (int i = 0; i < DEPTH; i++) fetch();
  for (uint64_t job = first; job < jobs; job += step) {
    const uint32_t row = per_row == 1 ? (uint32_t)job : (uint32_t)(job / per_row);
    const uint32_t h0 = per_row == 1 ? 0 : (uint32_t)(job % per_row) * a.per_job[part];
    const uint32_t h1 = min(h0 + a.per_job[part], heads);
    const bool real = (uint32_t)pos < a.rope_rows;
    T *out = (T *)a.out[part] + (uint64_t)row * a.out_stride[part];
    // Forward: ca = ga c, sa = ga s, cb = gb c, sb = -gb s, for
    // y_a = r (a ca + b sb), y_b = r (a sa + b cb).  Backward: ca = c, sa = s,
    // sb = -s, for u_a = dy_a c + dy_b s, u_b = dy_b c - dy_a s.
    Pair ca[P], sa[P], cb[BWD ? 1 : P], sb[P];
#pragma unroll
    for (int i = 0; i < P; i++) {
      const Pair c2 = pair(c[2 * i], c[2 * i + 1]), s2 = pair(s[2 * i], s[2 * i + 1]);
      const Pair m2 = pair(-s[2 * i], -s[2 * i + 1]);
      ca[i] = BWD ? c2 : mul2(ga[i], c2);
      sa[i] = BWD ? s2 : mul2(ga[i], s2);
      sb[i] = BWD ? m2 : mul2(gb[i], m2);
      if (!BWD) cb[i % (BWD ? 1 : P)] = mul2(gb[i], c2);
    }
    pos = pos_next;
    pos_next = position(job + 2 * step);
    angles(pos);
    for (uint32_t h = h0; h < h1; h += H * U) {
      uint4 w[U][CH];
      copy_wait<DEPTH - 1>();
      __syncwarp();
      const uint4 *here = slots + from * (U * CH * 32);
      from = from + 1 == DEPTH ? 0 : from + 1;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < CH; i++)
          w[u][i] = p.live ? here[(u * CH + i / 2 * 2) * 32 + (i % 2 ? p.c1 : p.c0)]
                           : make_uint4(0, 0, 0, 0);
      if (!real) {                 // a row of padding: nothing it holds counts
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int i = 0; i < CH; i++) w[u][i] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t hh = h + u * H + mine;
        Pair va[P], vb[P], ss = 0;
        split<T, HALF>(w[u][0], w[u][1], va, vb);
#pragma unroll
        for (int i = 0; i < P; i++) ss = fma2(vb[i], vb[i], fma2(va[i], va[i], ss));
        // 0 where there is nothing: with no eps a vector of zeros would make NaN
        const float sum = group_sum<G>(ss);
        const float r = real && hh < h1 ? rsqrtf(fmaf(sum, inv_d, a.eps)) : 0.0f;
        const Pair r2 = pair(r, r);
        if (!BWD) {
#pragma unroll
          for (int i = 0; i < P; i++) {
            const Pair x0 = mul2(va[i], r2), x1 = mul2(vb[i], r2);
            va[i] = fma2(x0, ca[i], mul2(x1, sb[i]));
            vb[i] = fma2(x0, sa[i], mul2(x1, cb[i % (BWD ? 1 : P)]));
          }
        } else {
          // t = u x: dg += r t, and dx = r (g u - x r^2 mean(g t)), in an order in which
          // nothing leaves float32's range that the gradient does not leave: r^3, or
          // the mean times it, did for rows of a size of 1e14
          Pair ua[P], ub[P], dot = 0;
          split<T, HALF>(w[u][CH - 2], w[u][CH - 1], ua, ub);
#pragma unroll
          for (int i = 0; i < P; i++) {
            const Pair y0 = ua[i], y1 = ub[i];
            ua[i] = fma2(y0, ca[i], mul2(y1, sa[i]));
            ub[i] = fma2(y1, ca[i], mul2(y0, sb[i]));
            const Pair t0 = mul2(ua[i], va[i]), t1 = mul2(ub[i], vb[i]);
            da[i] = fma2(t0, r2, da[i]);
            db[i] = fma2(t1, r2, db[i]);
            dot = fma2(t1, gb[i], fma2(t0, ga[i], dot));
          }
          const float k = -r * (r * (group_sum<G>(dot) * inv_d));
          const Pair k2 = pair(k, k);
#pragma unroll
          for (int i = 0; i < P; i++) {
            va[i] = mul2(fma2(va[i], k2, mul2(ua[i], ga[i])), r2);
            vb[i] = mul2(fma2(vb[i], k2, mul2(ub[i], gb[i])), r2);
          }
        }
        if (p.live && hh < h1) {
          uint4 y0, y1;
          merge<T, HALF>(va, vb, y0, y1);
          T *to = out + (uint64_t)hh * a.head_dim;
          *reinterpret_cast<uint4 *>(to + at0) = y0;
          *reinterpret_cast<uint4 *>(to + at1) = y1;
        }
      }
      __syncwarp();
      fetch();                     // into the slots just read
    }
  }
  if (BWD) {
    // this block's share of the gain's gradient, summed in a fixed order
    __shared__ float red[kWarps][2 * N * G];
#pragma unroll
    for (int i = 0; i < 2 * P; i++) {
      const float2 f = unpair(i < P ? da[i % P] : db[i % P]);
      float v[2] = {f.x, f.y};
#pragma unroll
      for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int o = G; o < 32; o <<= 1) v[e] += __shfl_xor_sync(0xffffffffu, v[e], o);
        if (lane < G) red[warp][lane * 2 * N + 2 * i + e] = v[e];
      }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * N * G; i += kThreads) {
      const Place q = place_of<T, HALF>(i / (2 * N), a.head_dim, a.rot);
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) v += red[w][i];
      // slot e < N is the first value of pair e, N + e the second
      const uint32_t e = i % (2 * N), k = e % N, second = e / N;
      const uint32_t at = HALF ? (second ? q.c1 : q.c0) * N + k : q.c0 * N + 2 * k + second;
      if (q.live) a.partial[(uint64_t)blockIdx.x * a.head_dim + at] = v;
    }
  }
}

// dG[part][i] = the sum of the blocks' shares, in a fixed order: a block takes
// eight columns, 32 threads a column.
__global__ void __launch_bounds__(256)
qk_gain_sum_kernel(const float *partial, uint32_t blocks_q, uint32_t blocks_k, uint32_t head_dim,
                   float *dgq, float *dgk) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red[32][9];
  const uint32_t col = threadIdx.x & 7, k = threadIdx.x >> 3, part = blockIdx.y;
  const uint32_t at = blockIdx.x * 8 + col, blocks = part ? blocks_k : blocks_q;
  if (part) partial += (uint64_t)blocks_q * head_dim;
  float v = 0.0f;
#pragma unroll 4
  for (uint32_t b = k; b < blocks; b += 32) v += partial[(uint64_t)b * head_dim + at];
  red[k][col] = v;
  __syncthreads();
  if (k == 0) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i++) t += red[i][col];
    (part ? dgk : dgq)[at] = t;
  }
}

template <typename T, bool BWD> constexpr int per_sm = BWD && sizeof(T) == 2 ? 1 : 2;

template <typename T, int G, bool HALF, bool BWD>
cudaError_t start(QkArgs &a, cudaStream_t st) {
  // Vectors a group takes at a time, steps on their way, blocks an SM.  Forward,
  // 8192 rows of 40 heads of 128, bf16: 30.6 us with 1, 3 and 2; 33.1 with 1, 2,
  // 2; 31.6 with 2, 2, 2.  With loads to registers instead 35.1, and with a lane
  // copying its own chunks 31.5, but 20.0 and not 14.3 where these are two
  // neighbours (3000 rows of 20 heads of 256, adjacent pairs).  4096 rows of 40
  // heads, f32: 30.4 us with 2, 2 and 2; 31.3 with 2, 3, 2.
  // Backward, 8192 rows of 40 heads, bf16, of 128 / of 64 (adjacent pairs): 45.8 /
  // 28.4 with 1, 4 and 1 block; 50.9 / 32.3 with 1, 3 and 2 (whose 128 registers
  // spill), 46.3 / 36.5 with 2, 2 and 1, 62.0 / 33.4 with 1, loads to registers
  // and 2.  4096 rows of 40 heads of 128, f32: 45.4 with 2, 2 and 2; 45.6 with 2, 4
  // and 1; 4096 rows of 40 heads of 64: 25.7 and 26.5.
  constexpr int U = sizeof(T) == 4 ? 2 : 1, DEPTH = sizeof(T) == 4 ? 2 : BWD ? 4 : 3,
                PER_SM = per_sm<T, BWD>;
  constexpr auto kernel = qk_norm_rope_kernel<T, G, HALF, BWD, U, DEPTH, PER_SM>;
  constexpr int bytes = kWarps * DEPTH * U * (BWD ? 2048 : 1024);
  static bool configured = false;
  if (!configured) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  return launch_pdl(kernel, dim3(a.blocks[0] + a.blocks[1]), dim3(kThreads), (size_t)bytes, st, a);
}
template <typename T, bool BWD>
cudaError_t start_t(QkArgs &a, bool half, uint32_t group, cudaStream_t st) {
  switch (group * 2 + (half ? 1 : 0)) {
    case 8: return start<T, 4, false, BWD>(a, st);
    case 9: return start<T, 4, true, BWD>(a, st);
    case 16: return start<T, 8, false, BWD>(a, st);
    case 17: return start<T, 8, true, BWD>(a, st);
    case 32: return start<T, 16, false, BWD>(a, st);
    case 33: return start<T, 16, true, BWD>(a, st);
  }
  if constexpr (sizeof(T) == 4) {   // 256 values of 16 bits take 16 lanes
    return half ? start<T, 32, true, BWD>(a, st) : start<T, 32, false, BWD>(a, st);
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

constexpr uint32_t kMaxBlocks = 148 * 2;

// What a row costs a warp besides its heads, in heads.
constexpr uint32_t kRowCost = 4;

// How a launch divides n rows of the two parts' heads: the blocks (at most
// MAX_BLOCKS) in proportion to the heads; a warp takes whole rows once there
// are enough of them to fill the blocks' warps, and otherwise as few heads as a
// warp holds at a time.
void divide(QkArgs &a, uint32_t at_once, uint32_t max_blocks) {
  const uint32_t all = a.heads[0] + a.heads[1];
  for (int p = 0; p < 2; p++) {
    uint64_t most = (uint64_t)max_blocks * (a.heads[p] + kRowCost) / (all + 2 * kRowCost);
    if (most < 1) most = 1;
    if (p == 1 && most + a.blocks[0] > max_blocks) most = max_blocks - a.blocks[0];
    uint32_t per = a.heads[p];
    while (per > at_once && (uint64_t)a.n * ((a.heads[p] + per - 1) / per) < most * kWarps)
      per = (per + 1) / 2;
    per = (per + at_once - 1) / at_once * at_once;
    a.per_job[p] = per;
    a.jobs_per_row[p] = (a.heads[p] + per - 1) / per;
    const uint64_t blocks = ceil_div64((uint64_t)a.n * a.jobs_per_row[p], kWarps);
    a.blocks[p] = (uint32_t)(blocks < most ? blocks : most);
  }
}

int check_common(const char *what, int dtype, const QkArgs &a, int pairs) {
  if (dtype != NL_F32 && dtype != NL_BF16)
    return set_error(NL_ERROR, "%s: type %d is neither NL_F32 nor NL_BF16", what, dtype);
  if (pairs != NL_PAIRS_HALF && pairs != NL_PAIRS_ADJACENT)
    return set_error(NL_ERROR, "%s: pairs %d", what, pairs);
  const uint32_t unit = dtype == NL_BF16 ? 16 : 8;
  if (!a.heads[0] || !a.heads[1] || a.heads[0] > 65536 || a.heads[1] > 65536)
    return set_error(NL_ERROR, "%s: heads %u, kv heads %u", what, a.heads[0], a.heads[1]);
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

// The fields that the two directions share.
template <typename A> static QkArgs common_of(const A &x) {
  QkArgs a = {};
  a.x = x.qkv; a.x_stride = x.x_stride;
  a.g[0] = x.gq; a.g[1] = x.gk; a.co = x.co; a.si = x.si; a.pos = x.pos;
  a.n = x.n; a.heads[0] = x.heads; a.heads[1] = x.kv_heads; a.head_dim = x.head_dim;
  a.rot = x.rot_dim; a.rope_rows = x.rope_rows; a.eps = x.eps;
  return a;
}

extern "C" int nl_qk_norm_rope_dev(const nl_qk_norm_rope_args *args, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  const char *what = "qk-norm-rope";
  if (!args) return set_error(NL_ERROR, "%s: null arguments", what);
  const nl_qk_norm_rope_args &x = *args;
  const int dtype = x.dtype, pairs = x.pairs;
  QkArgs a = common_of(x);
  a.out[0] = x.q; a.out[1] = x.k; a.out_stride[0] = x.q_stride; a.out_stride[1] = x.k_stride;
  if ((rc = check_common(what, dtype, a, pairs))) return rc;
  if (x.n == 0) return NL_OK;
  const uint64_t qw = (uint64_t)x.heads * x.head_dim, kw = (uint64_t)x.kv_heads * x.head_dim;
  if ((rc = check_rows(what, "QKV", dtype, x.qkv, x.x_stride, qw + kw)) ||
      (rc = check_rows(what, "Q", dtype, x.q, x.q_stride, qw)) ||
      (rc = check_rows(what, "K", dtype, x.k, x.k_stride, kw)) || (rc = check_tables(what, a)))
    return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t group = group_of(dtype, x.head_dim);
  divide(a, 32 / group, kMaxBlocks);
  const bool half = pairs == NL_PAIRS_HALF;
  const cudaError_t e = dtype == NL_BF16 ? start_t<__nv_bfloat16, false>(a, half, group, st)
                                         : start_t<float, false>(a, half, group, st);
  count_launches(1);
  return cuda_status(e, what);
}

extern "C" size_t nl_qk_norm_rope_bwd_workspace_bytes(uint32_t head_dim) {
  return (size_t)kMaxBlocks * head_dim * sizeof(float);
}

extern "C" int nl_qk_norm_rope_bwd_dev(const nl_qk_norm_rope_bwd_args *args, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  const char *what = "qk-norm-rope-bwd";
  if (!args) return set_error(NL_ERROR, "%s: null arguments", what);
  const nl_qk_norm_rope_bwd_args &x = *args;
  const int dtype = x.dtype, pairs = x.pairs;
  QkArgs a = common_of(x);
  a.dy[0] = x.dq; a.dy[1] = x.dk; a.dy_stride[0] = x.dq_stride; a.dy_stride[1] = x.dk_stride;
  a.out_stride[0] = a.out_stride[1] = x.dx_stride;
  if ((rc = check_common(what, dtype, a, pairs))) return rc;
  if (!x.dgq || !x.dgk) return set_error(NL_ERROR, "%s: a null gain gradient", what);
  cudaStream_t st = (cudaStream_t)stream;
  if (x.n) {
    const uint64_t qw = (uint64_t)x.heads * x.head_dim, kw = (uint64_t)x.kv_heads * x.head_dim;
    if ((rc = check_rows(what, "QKV", dtype, x.qkv, x.x_stride, qw + kw)) ||
        (rc = check_rows(what, "DQ", dtype, x.dq, x.dq_stride, qw)) ||
        (rc = check_rows(what, "DK", dtype, x.dk, x.dk_stride, kw)) ||
        (rc = check_rows(what, "DQKV", dtype, x.dqkv, x.dx_stride, qw + kw)) ||
        (rc = check_tables(what, a)))
      return rc;
    const size_t need = nl_qk_norm_rope_bwd_workspace_bytes(x.head_dim);
    if (x.workspace && x.ws_bytes < need)
      return set_error(NL_ERROR, "%s: workspace of %zu bytes, %zu needed", what, x.ws_bytes, need);
    void *workspace = x.workspace ? x.workspace : library_workspace(need, st);
    if (!workspace || !aligned16(workspace))
      return set_error(NL_ERROR, "%s: no aligned workspace of %zu bytes", what, need);
    a.partial = (float *)workspace;
    a.out[0] = x.dqkv;
    a.out[1] = (char *)x.dqkv + qw * (dtype == NL_BF16 ? 2 : 4);
    const uint32_t group = group_of(dtype, x.head_dim);
    divide(a, 32 / group,
           148 * (dtype == NL_BF16 ? per_sm<__nv_bfloat16, true> : per_sm<float, true>));
    const bool half = pairs == NL_PAIRS_HALF;
    const cudaError_t e = dtype == NL_BF16 ? start_t<__nv_bfloat16, true>(a, half, group, st)
                                           : start_t<float, true>(a, half, group, st);
    count_launches(1);
    if (e != cudaSuccess) return cuda_status(e, what);
  }
  const cudaError_t e = launch_pdl(qk_gain_sum_kernel, dim3(x.head_dim / 8, 2), dim3(256), 0, st,
                                   (const float *)a.partial, a.blocks[0], a.blocks[1], x.head_dim,
                                   x.dgq, x.dgk);
  count_launches(1);
  return cuda_status(e, what);
}
