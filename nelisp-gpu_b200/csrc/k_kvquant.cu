// k_kvquant.cu -- keys and values quantised as they are written to a paged
// cache, read back, and moved inside it (kv_quant.cuh has the layout).
//
//   8 bits  s = fl(max|x| / 127), c = rint(fl(x fl(127 / max|x|)))
//   4 bits  lo = min x rounded down to bfloat16, s = fl(fl(max x - lo) / 15)
//           rounded up to bfloat16, c = min(15, rint(fl(fl(x - lo) fl(1 / s))))
// fl: one rounding to float32, and no product is contracted into a following
// sum, so the codes are the same bits on any IEEE machine.  Rounding lo down
// and s up keeps every value inside [lo, lo + 15 s]: nothing is clipped by
// more than the last rounding.  A scale below 2^-112 becomes zero.  A vector
// with a NaN or an infinity (or, in 4 bits, a range beyond float32) has no
// such form: its scale is NaN, so it reads back, and attends, as NaN.
//
// Bound by memory.  As in k_qknorm.cu a group of lanes holds a head vector,
// two 16-byte chunks a lane half a vector apart, so each request of a group is
// one contiguous run.  A warp takes a token's key and value heads (some of
// them, while there are few tokens), so the slot is looked up once and a head
// is a step on both sides; U vectors are requested before the first is used.
// Their extremes are joined together, each lane ends with one vector's, divides
// for that one alone, and the group shares the quotients: a division costs as
// much as two values.  Codes and floats are turned into one another by adding
// 2^23 and its like, two at a time: the conversion instructions run at a
// sixteenth of the rate and bound the first form of these kernels.  Append and
// read of 4,095 tokens of 20 heads of 128, float32, 8 bits: 33.9 us together, 6.2
// TB/s, 0.95 of a copy; of 16,384 tokens of 8 heads, bfloat16, 4 bits: 29.5 us,
// 5.8 TB/s, where issue is the bound.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "f32x2.cuh"
#include "kv_quant.cuh"

namespace nl {

int kv_check_pool(const char *what, int fmt, const KvPool &p) {
  if (fmt != NL_KV_I8 && fmt != NL_KV_I4)
    return set_error(NL_ERROR, "%s: format %d is neither NL_KV_I8 nor NL_KV_I4", what, fmt);
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return set_error(NL_ERROR, "%s: head size %u (64, 128 or 256)", what, p.head_dim);
  if (!p.kv_heads || !p.block_size)
    return set_error(NL_ERROR, "%s: kv heads %u, block size %u", what, p.kv_heads, p.block_size);
  const uint64_t slots = (uint64_t)p.num_blocks * p.block_size;
  if (slots > INT32_MAX || slots * p.kv_heads > UINT32_MAX)
    return set_error(NL_ERROR,
                     "%s: %llu token slots x %u kv heads: at most 2^31 - 1 slots and 2^32 - 1 rows",
                     what, (unsigned long long)slots, p.kv_heads);
  for (int i = 0; i < 2; i++)
    if (p.num_blocks && (!p.code[i] || !p.param[i] || !aligned16(p.code[i]) ||
                         ((uintptr_t)p.param[i] & 3u)))
      return set_error(NL_ERROR, "%s: a null or unaligned cache pointer (codes: 16 bytes)", what);
  return NL_OK;
}

namespace {

constexpr int kThreads = 256;

struct KvRows {
  const void *in[2];             // append: keys and values, rows of kv_heads * head_dim
  void *out[2];                  // read
  uint64_t stride[2];
  const int32_t *slot;
  uint32_t n, per_job, jobs;     // tokens; heads a warp takes, and how many warps a token
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The unsigned integer that holds the codes of a chunk of N values.
template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };

// Codes of N values as 32-bit words (one word, its low half for four 4-bit
// codes).  Adding 1.5 * 2^23 (and 128) rounds to an integer, ties to even, in
// the low bits of the sum.
template <int BITS, int N>
__device__ __forceinline__ void encode(const Pair *v, float lo, float inv, uint32_t *w) {
  const float magic = 12582912.0f + (BITS == 8 ? 128.0f : 0.0f);
  uint32_t c[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    // one at a time: the packed product and sum were contracted, and the code
    // is that of the rounded product
    const float2 f = unpair(v[i / 2]);
    float x = i & 1 ? f.y : f.x;
    if (BITS == 4) x = __fsub_rn(x, lo);
    x = __fmul_rn(x, inv);         // (4 bits: it rounds to at most 15, by lo and s)
    c[i] = __float_as_uint(__fadd_rn(x, magic));
  }
  if (BITS == 8) {
#pragma unroll
    for (int i = 0; i < N; i += 4) w[i / 4] = low_bytes(c[i], c[i + 1], c[i + 2], c[i + 3]);
  } else {
    // bytes of the even and the odd codes, the odd ones four bits up
    uint32_t x = 0;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint32_t even = __byte_perm(c[i], c[i + 2], 0x0040) & 0x0f0fu;
      const uint32_t odd = __byte_perm(c[i + 1], c[i + 3], 0x0040) & 0x0f0fu;
      x |= (even | odd << 4) << (4 * i);
    }
    w[0] = x;
  }
}

// The values of N codes: 2^23 + code is exact, and so is the difference.
template <int BITS, int N>
__device__ __forceinline__ void decode(const uint32_t *w, float s, float lo, Pair *v) {
  const float back = -(8388608.0f + (BITS == 8 ? 128.0f : 0.0f));
  const Pair back2 = pair(back, back), s2 = pair(s, s), lo2 = pair(lo, lo);
#pragma unroll
  for (int i = 0; i < N / 2; i++) {
    uint32_t c[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int k = 2 * i + e;
      c[e] = BITS == 8 ? __byte_perm(w[k / 4], 0x4b000000u, 0x7440 + k % 4)
                       : (w[0] >> (4 * k) & 15u) | 0x4b000000u;
    }
    Pair x = mul2(add2(pair(__uint_as_float(c[0]), __uint_as_float(c[1])), back2), s2);
    if (BITS == 4) x = add2(x, lo2);   // s c has 12 bits: exact, so rounded once
    v[i] = x;
  }
}

__device__ __forceinline__ float bf16_up(float x) {   // of a positive finite x
  return __uint_as_float((__float_as_uint(x) + 0xffffu) & 0xffff0000u);
}

// A warp's job: some of a token's heads, the values' after the keys'.  Nothing orders
// the jobs, nor a vector's codes and its word: two tokens of one append with one slot
// leave a mixture there, which the caller is told.  (One owner a slot would take
// either a word per slot of the pool or every token's slot compared with all others.)
struct Job {
  uint32_t token, h0, h1;
  uint32_t row;                  // of head 0 in the pool, or ~0
};
__device__ __forceinline__ Job job_of(const KvRows &r, const KvPool &p, uint64_t i) {
  Job j;
  j.token = r.jobs == 1 ? (uint32_t)i : (uint32_t)(i / r.jobs);
  j.h0 = (uint32_t)(i - (uint64_t)j.token * r.jobs) * r.per_job;
  j.h1 = min(j.h0 + r.per_job, 2 * p.kv_heads);
  const uint32_t slot = (uint32_t)__ldg(r.slot + j.token), block = slot / p.block_size;
  j.row = block < p.num_blocks ? kv_row(p, block, slot - block * p.block_size, 0) : ~0u;
  return j;
}
// Head HH of a token: keys or values, which of them, and its row in the pool.
struct Head {
  uint32_t kv, head, at;
};
__device__ __forceinline__ Head head_of(const KvPool &p, const Job &job, uint32_t hh) {
  Head h;
  h.kv = hh >= p.kv_heads;
  h.head = h.kv ? hh - p.kv_heads : hh;
  h.at = job.row + h.head * p.block_size;
  return h;
}

// The largest and the smallest of a lane's part of a vector (8 bits: the largest
// magnitude, and nothing), NaN if any is.
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T, int BITS>
__device__ __forceinline__ void extremes(const uint4 (&w)[2], float *hi, float *lo) {
  const uint32_t v[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
  if constexpr (sizeof(T) == 4) {
    auto of = [&](int i) {
      const float f = __uint_as_float(v[i]);
      return BITS == 8 ? fabsf(f) : f;
    };
    float h = of(0), l = of(0);
#pragma unroll
    for (int i = 1; i < 8; i++) {
      h = max_nan(h, of(i));
      if (BITS == 4) l = min_nan(l, of(i));
    }
    *hi = h;
    *lo = l;
  } else {                         // two at a time; exact
    auto of = [&](int i) { return BITS == 8 ? v[i] & 0x7fff7fffu : v[i]; };
    uint32_t h = of(0), l = of(0);
#pragma unroll
    for (int i = 1; i < 8; i++) {
      h = max2_nan(h, of(i));
      if (BITS == 4) l = min2_nan(l, of(i));
    }
    *hi = max_nan(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
    *lo = min_nan(__uint_as_float(l << 16), __uint_as_float(l & 0xffff0000u));
  }
}
// Of U values a lane, the join over the lanes of a group of G: lane j of it gets
// that of value j / (G / U), in log2(G) + U - 1 - log2(U) exchanges.
template <int G, int U, typename F>
__device__ __forceinline__ float across(float (&v)[U], uint32_t j, F join) {
  int o = G / 2;
#pragma unroll
  for (int n = U / 2; n > 0; n /= 2, o /= 2) {
    const bool high = j & o;
#pragma unroll
    for (int i = 0; i < n; i++) {
      const float give = high ? v[i] : v[i + n], have = high ? v[i + n] : v[i];
      v[i] = join(have, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
#pragma unroll
  for (; o > 0; o /= 2) v[0] = join(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
  return v[0];
}

template <typename T, int HD, int BITS, int U>
__global__ void __launch_bounds__(kThreads)
kv_append_kernel(const __grid_constant__ KvRows r, const __grid_constant__ KvPool p) {
  constexpr int N = Chunk<T>::N, G = HD / (2 * N), H = 32 / G, CB = N * BITS / 8;
  using W = typename Word<CB>::type;
  pdl_trigger();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31, j = lane % G, mine = lane / G;
  const uint64_t jobs = (uint64_t)r.n * r.jobs;
  for (uint64_t i = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < jobs;
       i += (uint64_t)gridDim.x * (kThreads / 32)) {
    const Job job = job_of(r, p, i);
    const T *x[2] = {(const T *)r.in[0] + (uint64_t)job.token * r.stride[0],
                     (const T *)r.in[1] + (uint64_t)job.token * r.stride[1]};
    for (uint32_t h = job.h0; h < job.h1; h += H * U) {
      uint4 w[U][2];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t hh = h + u * H + mine;
        w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
        if (hh < job.h1) {
          const Head at = head_of(p, job, hh);
          const uint4 *v = reinterpret_cast<const uint4 *>((at.kv ? x[1] : x[0]) +
                                                           (uint64_t)at.head * HD);
          w[u][0] = __ldcs(v + j);
          w[u][1] = __ldcs(v + j + G);
        }
      }
      // a lane makes the parameters of one of the U vectors, and the group shares
      // them: the divisions are most of what a vector costs besides its values
      float hi[U], lo[U];
#pragma unroll
      for (int u = 0; u < U; u++) extremes<T, BITS>(w[u], &hi[u], &lo[u]);
      const float top = across<G, U>(hi, j, max_nan);
      float s, low = 0.0f, inv = 0.0f;
      uint32_t word;
      bool bad;
      if (BITS == 8) {
        const bool some = top >= 127.0f * kKvTiny;
        s = some ? __fdiv_rn(top, 127.0f) : 0.0f;
        if (some) inv = __fdiv_rn(127.0f, top);
        bad = !(top < INFINITY);
        word = bad ? 0x7fc00000u : __float_as_uint(s);
      } else {
        low = __bfloat162float(__float2bfloat16_rd(across<G, U>(lo, j, min_nan)));
        const float range = __fsub_rn(top, low);
        s = bf16_up(__fdiv_rn(range, 15.0f));
        const bool some = s >= kKvTiny;
        if (some) inv = __fdiv_rn(1.0f, s);
        else s = 0.0f;
        bad = !(range < INFINITY);
        word = bad ? 0x7fc0u
                   : __float_as_uint(s) >> 16 | (__float_as_uint(low) & 0xffff0000u);
      }
      if (bad) inv = -1.0f;        // the scale says so: the codes are those of zero
      if (j % (G / U) == 0) {
        const uint32_t hh = h + j / (G / U) * H + mine;
        if (hh < job.h1 && job.row != ~0u) {
          const Head at = head_of(p, job, hh);
          (at.kv ? p.param[1] : p.param[0])[at.at] = word;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t hh = h + u * H + mine, from = mine * G + u * (G / U);
        float by = __shfl_sync(0xffffffffu, inv, from);
        float off = BITS == 4 ? __shfl_sync(0xffffffffu, low, from) : 0.0f;
        Pair v[N];
        Chunk<T>::get(w[u][0], v);
        Chunk<T>::get(w[u][1], v + N / 2);
        if (by < 0.0f) {
#pragma unroll
          for (int e = 0; e < N; e++) v[e] = 0;
          by = off = 0.0f;
        }
        if (hh < job.h1 && job.row != ~0u) {
          const Head at = head_of(p, job, hh);
          uint8_t *to = (at.kv ? p.code[1] : p.code[0]) +
                        (uint64_t)at.at * (HD * BITS / 8) + j * CB;
#pragma unroll
          for (int k = 0; k < 2; k++) {
            uint32_t c[2];
            encode<BITS, N>(v + k * (N / 2), off, by, c);
            W t;
            if constexpr (CB == 8) t = make_uint2(c[0], c[1]);
            else t = (W)c[0];
            *reinterpret_cast<W *>(to + k * G * CB) = t;
          }
        }
      }
    }
  }
}

template <typename T, int HD, int BITS, int U>
__global__ void __launch_bounds__(kThreads)
kv_read_kernel(const __grid_constant__ KvRows r, const __grid_constant__ KvPool p) {
  constexpr int N = Chunk<T>::N, G = HD / (2 * N), H = 32 / G, CB = N * BITS / 8;
  using W = typename Word<CB>::type;
  pdl_trigger();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31, j = lane % G, mine = lane / G;
  const uint64_t jobs = (uint64_t)r.n * r.jobs;
  for (uint64_t i = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < jobs;
       i += (uint64_t)gridDim.x * (kThreads / 32)) {
    const Job job = job_of(r, p, i);
    T *y[2] = {(T *)r.out[0] + (uint64_t)job.token * r.stride[0],
               (T *)r.out[1] + (uint64_t)job.token * r.stride[1]};
    for (uint32_t h = job.h0; h < job.h1; h += H * U) {
      W w[U][2];
      uint32_t word[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t hh = h + u * H + mine;
        word[u] = 0;
        w[u][0] = w[u][1] = W{};
        if (hh < job.h1 && job.row != ~0u) {
          const Head at = head_of(p, job, hh);
          const uint8_t *from = (at.kv ? p.code[1] : p.code[0]) +
                                (uint64_t)at.at * (HD * BITS / 8) + j * CB;
          word[u] = (at.kv ? p.param[1] : p.param[0])[at.at];
          w[u][0] = *reinterpret_cast<const W *>(from);
          w[u][1] = *reinterpret_cast<const W *>(from + G * CB);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t hh = h + u * H + mine;
        if (hh >= job.h1) continue;
        const float s = __uint_as_float(BITS == 8 ? word[u] : word[u] << 16);
        const float lo = BITS == 8 ? 0.0f : __uint_as_float(word[u] & 0xffff0000u);
        const Head at = head_of(p, job, hh);
        uint4 *to = reinterpret_cast<uint4 *>((at.kv ? y[1] : y[0]) + (uint64_t)at.head * HD) + j;
#pragma unroll
        for (int k = 0; k < 2; k++) {
          uint32_t c[2];
          if constexpr (CB == 8) c[0] = w[u][k].x, c[1] = w[u][k].y;
          else c[0] = w[u][k], c[1] = 0;
          Pair v[N / 2];
          decode<BITS, N>(c, s, lo, v);
          __stcs(to + k * G, Chunk<T>::put(v));
        }
      }
    }
  }
}

// Rows moved inside the pool, one block per (sequence, head): every source is
// in shared memory before the first destination is written, and of pairs with one
// destination the last alone is written, as one after the other would leave it.
__global__ void __launch_bounds__(kThreads)
kv_move_kernel(const __grid_constant__ KvPool p, const int32_t *src, const int32_t *dst,
               uint32_t count) {
  extern __shared__ uint4 held[];
  pdl_trigger();
  pdl_wait();
  const uint32_t head = blockIdx.x, kv = blockIdx.z;
  src += (uint64_t)blockIdx.y * count;
  dst += (uint64_t)blockIdx.y * count;
  const uint32_t chunks = p.head_dim * p.bits / 128, per = chunks + 1;   // and the parameter
  const uint64_t bytes = (uint64_t)chunks * 16;
  __shared__ uint32_t target[64], kept[64];      // the pairs' destinations, or ~0
  if (threadIdx.x < count) {
    const uint32_t from = (uint32_t)src[threadIdx.x], to = (uint32_t)dst[threadIdx.x];
    const bool both = from / p.block_size < p.num_blocks && to / p.block_size < p.num_blocks;
    target[threadIdx.x] = both ? to : ~0u;
  }
  for (uint32_t i = threadIdx.x; i < count * per; i += kThreads) {
    const uint32_t slot = (uint32_t)src[i / per], block = slot / p.block_size, k = i % per;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (block < p.num_blocks) {
      const uint32_t at = kv_row(p, block, slot % p.block_size, head);
      if (k < chunks) v = reinterpret_cast<const uint4 *>(p.code[kv] + at * bytes)[k];
      else v.x = p.param[kv][at];
    }
    held[i] = v;
  }
  __syncthreads();
  if (threadIdx.x < count) {
    const uint32_t to = target[threadIdx.x];
    bool later = false;
    for (uint32_t k = threadIdx.x + 1; k < count; k++) later |= target[k] == to;
    kept[threadIdx.x] = later ? ~0u : to;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < count * per; i += kThreads) {
    const uint32_t to = kept[i / per], k = i % per;
    if (to == ~0u) continue;
    const uint32_t at = kv_row(p, to / p.block_size, to % p.block_size, head);
    if (k < chunks) reinterpret_cast<uint4 *>(p.code[kv] + at * bytes)[k] = held[i];
    else p.param[kv][at] = held[i].x;
  }
}

// U vectors a group at a time (append + read of 4095 tokens of 20 heads of 128,
// f32, 8 bits: 40.9 us with 2, 37.6 with 4; 16384 of 8 heads, bf16, 4 bits: 34.1
// with 2, 31.3 with 4).  Up to 16 blocks an SM, and a token's heads divided so
// that there are as many jobs as warps (f32: 47.5 us with 4 blocks, 37.6 with 8,
// 35.8 with 16 or 32), whole steps of U vectors each; with too few tokens for
// that a vector a group, for the shortest call.
template <typename T, int HD, int BITS>
cudaError_t start(bool append, KvRows &r, const KvPool &p, cudaStream_t st) {
  constexpr int U = 4;
  constexpr uint32_t H = 32 / (HD / (2 * Chunk<T>::N)), warps = kThreads / 32;
  constexpr uint64_t most = 148 * 16;
  const uint32_t heads = 2 * p.kv_heads, steps = (heads + H * U - 1) / (H * U);
  if ((uint64_t)r.n * steps >= 148 * warps) {
    const uint64_t split = ceil_div64(most * warps, r.n);
    const uint32_t jobs = split < steps ? (uint32_t)split : steps;
    r.per_job = (steps + jobs - 1) / jobs * (H * U);
  } else {
    r.per_job = H;
  }
  r.jobs = (heads + r.per_job - 1) / r.per_job;
  const uint64_t want = ceil_div64((uint64_t)r.n * r.jobs, warps);
  const dim3 grid((unsigned)(want < most ? want : most));
  return append ? launch_pdl(kv_append_kernel<T, HD, BITS, U>, grid, dim3(kThreads), 0, st, r, p)
                : launch_pdl(kv_read_kernel<T, HD, BITS, U>, grid, dim3(kThreads), 0, st, r, p);
}
template <typename T>
cudaError_t start_t(bool append, KvRows &r, const KvPool &p, cudaStream_t st) {
  switch (p.head_dim + p.bits) {
    case 64 + 8: return start<T, 64, 8>(append, r, p, st);
    case 128 + 8: return start<T, 128, 8>(append, r, p, st);
    case 256 + 8: return start<T, 256, 8>(append, r, p, st);
    case 64 + 4: return start<T, 64, 4>(append, r, p, st);
    case 128 + 4: return start<T, 128, 4>(append, r, p, st);
    default: return start<T, 256, 4>(append, r, p, st);
  }
}

int rows_call(const char *what, bool append, const nl_kv_rows_args *args, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  if (!args) return set_error(NL_ERROR, "%s: null arguments", what);
  const int dtype = args->dtype, fmt = args->cache.fmt;
  const uint32_t n = args->n;
  KvPool p = kv_pool_of(args->cache);
  KvRows r = {{args->k, args->v}, {args->k, args->v}, {args->k_stride, args->v_stride},
              args->slot, 0, 0, 0};
  if (dtype != NL_F32 && dtype != NL_BF16)
    return set_error(NL_ERROR, "%s: type %d is neither NL_F32 nor NL_BF16", what, dtype);
  if ((rc = kv_check_pool(what, fmt, p))) return rc;
  if (n == 0) return NL_OK;
  if (!r.slot) return set_error(NL_ERROR, "%s: null slots", what);
  if (p.kv_heads > 1u << 30)       // twice as many, and a step more, are counted in 32 bits
    return set_error(NL_ERROR, "%s: %u kv heads", what, p.kv_heads);
  const uint32_t unit = dtype == NL_BF16 ? 8 : 4;
  for (int i = 0; i < 2; i++) {
    const void *x = append ? r.in[i] : r.out[i];
    if (!x || !aligned16(x) || r.stride[i] % unit ||
        r.stride[i] < (uint64_t)p.kv_heads * p.head_dim)
      return set_error(NL_ERROR,
                       "%s: %s rows must be 16-byte aligned, with a stride (%llu) that is a "
                       "multiple of %u and at least kv heads x head size",
                       what, i ? "V" : "K", (unsigned long long)r.stride[i], unit);
  }
  r.n = n;
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == NL_BF16 ? start_t<__nv_bfloat16>(append, r, p, st)
                                         : start_t<float>(append, r, p, st);
  count_launches(1);
  return cuda_status(e, what);
}

}  // namespace
}  // namespace nl

using namespace nl;

extern "C" int nl_kv_append_dev(const nl_kv_rows_args *args, void *stream) {
  return rows_call("kv-append", true, args, stream);
}

extern "C" int nl_kv_read_dev(const nl_kv_rows_args *args, void *stream) {
  return rows_call("kv-read", false, args, stream);
}

extern "C" int nl_kv_move_dev(const nl_kv_move_args *args, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  if (!args) return set_error(NL_ERROR, "kv-move: null arguments");
  const KvPool p = kv_pool_of(args->cache);
  if ((rc = kv_check_pool("kv-move", args->cache.fmt, p))) return rc;
  const uint32_t batch = args->batch, count = args->count;
  if (batch == 0 || count == 0) return NL_OK;
  if (!args->src || !args->dst) return set_error(NL_ERROR, "kv-move: null slots");
  if (count > 64 || batch > 65535)
    return set_error(NL_ERROR, "kv-move: count %u (at most 64), batch %u (at most 65535)", count,
                     batch);
  const size_t smem = (size_t)count * (p.head_dim * p.bits / 128 + 1) * 16;   // at most 17 KB
  const cudaError_t e = launch_pdl(kv_move_kernel, dim3(p.kv_heads, batch, 2), dim3(kThreads), smem,
                                   (cudaStream_t)stream, p, args->src, args->dst, count);
  count_launches(1);
  return cuda_status(e, "kv-move");
}
