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
// one contiguous run; U vectors are requested before the first is used.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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
  uint32_t vectors;              // 2 * n * kv_heads: a token's key heads, then its value heads
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

// x is at most 2^21 in magnitude and BIAS an integer: the low bits of the
// result are those of the integer BIAS + rint(x) (ties to even: 1.5 * 2^23 is
// even, and so is every BIAS used).
template <int BIAS>
__device__ __forceinline__ uint32_t round_bits(float x) {
  return __float_as_uint(__fadd_rn(x, 12582912.0f + (float)BIAS));
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// N values (a 16-byte chunk) and back, as floats.
template <typename T> struct Values;
template <> struct Values<float> {
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
template <> struct Values<__nv_bfloat16> {
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

// The unsigned integer that holds the codes of a chunk of N values.
template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };

// Codes of N values as 32-bit words (one word, its low half for four 4-bit
// codes).
template <int BITS, int N>
__device__ __forceinline__ void encode(const float *v, float lo, float inv, uint32_t *w) {
  if (BITS == 8) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      w[i / 4] = low_bytes(round_bits<128>(__fmul_rn(v[i], inv)),
                           round_bits<128>(__fmul_rn(v[i + 1], inv)),
                           round_bits<128>(__fmul_rn(v[i + 2], inv)),
                           round_bits<128>(__fmul_rn(v[i + 3], inv)));
  } else {
    uint32_t c[N];
#pragma unroll
    for (int i = 0; i < N; i++)
      c[i] = round_bits<0>(fminf(__fmul_rn(__fsub_rn(v[i], lo), inv), 15.0f)) & 15u;
    uint32_t x = 0;
#pragma unroll
    for (int i = 0; i < N; i++) x |= c[i] << (4 * i);
    w[0] = x;
  }
}

__device__ __forceinline__ float bf16_up(float x) {   // of a positive finite x
  return __uint_as_float((__float_as_uint(x) + 0xffffu) & 0xffff0000u);
}

template <typename T, int HD, int BITS, int U>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ KvRows r, const __grid_constant__ KvPool p) {
  constexpr int N = Values<T>::N, G = HD / (2 * N), H = 32 / G, CB = N * BITS / 8;
  using W = typename Word<CB>::type;
  pdl_trigger();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31, j = lane % G;
  const uint64_t step = (uint64_t)gridDim.x * (kThreads / 32) * (H * U);
  uint64_t base = ((uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * (H * U);
  for (; base < r.vectors; base += step) {
    uint4 w[U][2];
    uint32_t at[U];               // row in the pool, or ~0
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint64_t i = base + u * H + lane / G;
      at[u] = ~0u;
      w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
      if (i < r.vectors) {
        const uint32_t token = (uint32_t)i / (2 * p.kv_heads);
        const uint32_t rest = (uint32_t)i % (2 * p.kv_heads);
        const uint32_t kv = rest / p.kv_heads, head = rest % p.kv_heads;
        const uint32_t slot = (uint32_t)__ldg(r.slot + token);
        const T *x = (const T *)r.in[kv] + (uint64_t)token * r.stride[kv] + (uint64_t)head * HD;
        w[u][0] = __ldcs(reinterpret_cast<const uint4 *>(x) + j);
        w[u][1] = __ldcs(reinterpret_cast<const uint4 *>(x) + j + G);
        const uint32_t block = slot / p.block_size;
        if (block < p.num_blocks) at[u] = kv_row(p, block, slot % p.block_size, head);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint64_t i = base + u * H + lane / G;
      const uint32_t kv = (uint32_t)i % (2 * p.kv_heads) / p.kv_heads;
      float v[2 * N];
      Values<T>::get(w[u][0], v);
      Values<T>::get(w[u][1], v + N);
      float hi = BITS == 8 ? fabsf(v[0]) : v[0], lo = v[0];
#pragma unroll
      for (int e = 1; e < 2 * N; e++) {
        hi = max_nan(hi, BITS == 8 ? fabsf(v[e]) : v[e]);
        if (BITS == 4) lo = min_nan(lo, v[e]);
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) {
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        if (BITS == 4) lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      }
      float s, inv = 0.0f;
      uint32_t word;
      if (BITS == 8) {
        const bool some = hi >= 127.0f * kKvTiny;
        s = some ? __fdiv_rn(hi, 127.0f) : 0.0f;
        if (some) inv = __fdiv_rn(127.0f, hi);
        if (!(hi < INFINITY)) s = __uint_as_float(0x7fc00000u), inv = 0.0f;
        word = __float_as_uint(s);
      } else {
        lo = __bfloat162float(__float2bfloat16_rd(lo));
        const float range = __fsub_rn(hi, lo);
        s = bf16_up(__fdiv_rn(range, 15.0f));
        const bool some = s >= kKvTiny;
        if (some) inv = __fdiv_rn(1.0f, s);
        else s = 0.0f;
        word = __float_as_uint(s) >> 16 | (__float_as_uint(lo) & 0xffff0000u);
        if (!(range < INFINITY)) word = 0x7fc0u, inv = 0.0f;
      }
      if (at[u] != ~0u) {
        const bool bad = BITS == 8 ? !(hi < INFINITY) : word == 0x7fc0u;
        uint32_t c[2][N * BITS / 8 < 4 ? 1 : N * BITS / 32];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          if (bad) {
#pragma unroll
            for (int e = 0; e < N; e++) v[k * N + e] = 0.0f;
          }
          encode<BITS, N>(v + k * N, bad ? 0.0f : lo, inv, c[k]);
        }
        uint8_t *row = p.code[kv] + (uint64_t)at[u] * (HD * BITS / 8);
#pragma unroll
        for (int k = 0; k < 2; k++) {
          W t;
          if constexpr (CB == 8) t = make_uint2(c[k][0], c[k][1]);
          else t = (W)c[k][0];
          *reinterpret_cast<W *>(row + (j + k * G) * CB) = t;
        }
        if (j == 0) p.param[kv][at[u]] = word;
      }
    }
  }
}

template <typename T, int HD, int BITS, int U>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ KvRows r, const __grid_constant__ KvPool p) {
  constexpr int N = Values<T>::N, G = HD / (2 * N), H = 32 / G, CB = N * BITS / 8;
  using W = typename Word<CB>::type;
  pdl_trigger();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31, j = lane % G;
  const uint64_t step = (uint64_t)gridDim.x * (kThreads / 32) * (H * U);
  uint64_t base = ((uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * (H * U);
  for (; base < r.vectors; base += step) {
    W w[U][2];
    uint32_t word[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint64_t i = base + u * H + lane / G;
      word[u] = 0;
      w[u][0] = w[u][1] = W{};
      if (i < r.vectors) {
        const uint32_t token = (uint32_t)i / (2 * p.kv_heads);
        const uint32_t rest = (uint32_t)i % (2 * p.kv_heads);
        const uint32_t kv = rest / p.kv_heads, head = rest % p.kv_heads;
        const uint32_t slot = (uint32_t)__ldg(r.slot + token), block = slot / p.block_size;
        if (block < p.num_blocks) {
          const uint32_t at = kv_row(p, block, slot % p.block_size, head);
          const uint8_t *row = p.code[kv] + (uint64_t)at * (HD * BITS / 8);
          word[u] = p.param[kv][at];
          w[u][0] = *reinterpret_cast<const W *>(row + j * CB);
          w[u][1] = *reinterpret_cast<const W *>(row + (j + G) * CB);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint64_t i = base + u * H + lane / G;
      if (i >= r.vectors) continue;
      const uint32_t token = (uint32_t)i / (2 * p.kv_heads);
      const uint32_t rest = (uint32_t)i % (2 * p.kv_heads);
      const uint32_t kv = rest / p.kv_heads, head = rest % p.kv_heads;
      const float s = __uint_as_float(BITS == 8 ? word[u] : word[u] << 16);
      const float lo = BITS == 8 ? 0.0f : __uint_as_float(word[u] & 0xffff0000u);
      uint4 *y = reinterpret_cast<uint4 *>((T *)r.out[kv] + (uint64_t)token * r.stride[kv] +
                                           (uint64_t)head * HD);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        uint32_t c[2];
        if constexpr (CB == 8) c[0] = w[u][k].x, c[1] = w[u][k].y;
        else c[0] = w[u][k];
        float v[N];
#pragma unroll
        for (int e = 0; e < N; e++) {
          if (BITS == 8) {
            v[e] = s * (float)((int)(c[e / 4] >> (8 * (e % 4)) & 255u) - 128);
          } else {   // s c has 12 bits: exact, so one rounding either way
            v[e] = __fadd_rn(__fmul_rn(s, (float)(c[0] >> (4 * e) & 15u)), lo);
          }
        }
        y[j + k * G] = Values<T>::put(v);
      }
    }
  }
}

// Rows moved inside the pool, one block per (sequence, head): every source is
// in shared memory before the first destination is written.
__global__ void __launch_bounds__(kThreads)
kv_move_kernel(const __grid_constant__ KvPool p, const int32_t *src, const int32_t *dst, uint32_t count) {
  extern __shared__ uint4 held[];
  pdl_trigger();
  pdl_wait();
  const uint32_t head = blockIdx.x, kv = blockIdx.z;
  src += (uint64_t)blockIdx.y * count;
  dst += (uint64_t)blockIdx.y * count;
  const uint32_t chunks = p.head_dim * p.bits / 128, per = chunks + 1;   // and the parameter
  const uint64_t bytes = (uint64_t)chunks * 16;
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
  for (uint32_t i = threadIdx.x; i < count * per; i += kThreads) {
    const uint32_t from = (uint32_t)src[i / per], to = (uint32_t)dst[i / per], k = i % per;
    const uint32_t block = to / p.block_size;
    if (from / p.block_size >= p.num_blocks || block >= p.num_blocks) continue;
    const uint32_t at = kv_row(p, block, to % p.block_size, head);
    if (k < chunks) reinterpret_cast<uint4 *>(p.code[kv] + at * bytes)[k] = held[i];
    else p.param[kv][at] = held[i].x;
  }
}

// Both directions take U vectors a group at a time: 4 for rows of 16 bits or
// 32 bits alike, so a warp has 4 KB requested.
constexpr int kU = 4;

template <typename T, int HD, int BITS>
cudaError_t start(bool append, const KvRows &r, const KvPool &p, cudaStream_t st) {
  constexpr uint64_t per_block = (kThreads / 32) * (32 / (HD / (2 * Values<T>::N))) * kU;
  const uint64_t want = ceil_div64(r.vectors, per_block);
  const dim3 grid((unsigned)(want < 148 * 8 ? want : 148 * 8));
  return append ? launch_pdl(kv_append_kernel<T, HD, BITS, kU>, grid, dim3(kThreads), 0, st, r, p)
                : launch_pdl(kv_read_kernel<T, HD, BITS, kU>, grid, dim3(kThreads), 0, st, r, p);
}
template <typename T>
cudaError_t start_t(bool append, const KvRows &r, const KvPool &p, cudaStream_t st) {
  switch (p.head_dim + p.bits) {
    case 64 + 8: return start<T, 64, 8>(append, r, p, st);
    case 128 + 8: return start<T, 128, 8>(append, r, p, st);
    case 256 + 8: return start<T, 256, 8>(append, r, p, st);
    case 64 + 4: return start<T, 64, 4>(append, r, p, st);
    case 128 + 4: return start<T, 128, 4>(append, r, p, st);
    default: return start<T, 256, 4>(append, r, p, st);
  }
}

int rows_call(const char *what, bool append, int fmt, int dtype, KvRows &r, KvPool &p, uint32_t n,
              void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  if (dtype != NL_F32 && dtype != NL_BF16)
    return set_error(NL_ERROR, "%s: type %d is neither NL_F32 nor NL_BF16", what, dtype);
  if ((rc = kv_check_pool(what, fmt, p))) return rc;
  p.bits = (uint32_t)fmt;
  if (n == 0) return NL_OK;
  if (!r.slot) return set_error(NL_ERROR, "%s: null slots", what);
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
  if (2 * (uint64_t)n * p.kv_heads > UINT32_MAX)
    return set_error(NL_ERROR, "%s: %u tokens x %u kv heads: at most 2^31 - 1 head vectors", what,
                     n, p.kv_heads);
  r.vectors = 2 * n * p.kv_heads;
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == NL_BF16 ? start_t<__nv_bfloat16>(append, r, p, st)
                                         : start_t<float>(append, r, p, st);
  count_launches(1);
  return cuda_status(e, what);
}

}  // namespace
}  // namespace nl

using namespace nl;

extern "C" int nl_kv_append_dev(int fmt, int dtype, const void *K, uint64_t k_stride,
                                const void *V, uint64_t v_stride, const int32_t *SLOT, void *KC,
                                uint32_t *KP, void *VC, uint32_t *VP, uint32_t n,
                                uint32_t kv_heads, uint32_t head_dim, uint32_t block_size,
                                uint32_t num_blocks, void *stream) {
  KvRows r = {{K, V}, {nullptr, nullptr}, {k_stride, v_stride}, SLOT, 0};
  KvPool p = {{(uint8_t *)KC, (uint8_t *)VC}, {KP, VP}, num_blocks, block_size, kv_heads,
              head_dim, 0};
  return rows_call("kv-append", true, fmt, dtype, r, p, n, stream);
}

extern "C" int nl_kv_read_dev(int fmt, int dtype, const int32_t *SLOT, const void *KC,
                              const uint32_t *KP, const void *VC, const uint32_t *VP, void *K,
                              uint64_t k_stride, void *V, uint64_t v_stride, uint32_t n,
                              uint32_t kv_heads, uint32_t head_dim, uint32_t block_size,
                              uint32_t num_blocks, void *stream) {
  KvRows r = {{nullptr, nullptr}, {K, V}, {k_stride, v_stride}, SLOT, 0};
  KvPool p = {{(uint8_t *)const_cast<void *>(KC), (uint8_t *)const_cast<void *>(VC)},
              {const_cast<uint32_t *>(KP), const_cast<uint32_t *>(VP)}, num_blocks, block_size,
              kv_heads, head_dim, 0};
  return rows_call("kv-read", false, fmt, dtype, r, p, n, stream);
}

extern "C" int nl_kv_move_dev(int fmt, const int32_t *SRC, const int32_t *DST, void *KC,
                              uint32_t *KP, void *VC, uint32_t *VP, uint32_t batch,
                              uint32_t count, uint32_t kv_heads, uint32_t head_dim,
                              uint32_t block_size, uint32_t num_blocks, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  KvPool p = {{(uint8_t *)KC, (uint8_t *)VC}, {KP, VP}, num_blocks, block_size, kv_heads,
              head_dim, 0};
  if ((rc = kv_check_pool("kv-move", fmt, p))) return rc;
  p.bits = (uint32_t)fmt;
  if (batch == 0 || count == 0) return NL_OK;
  if (!SRC || !DST) return set_error(NL_ERROR, "kv-move: null slots");
  if (count > 64 || batch > 65535 || kv_heads > 65535)
    return set_error(NL_ERROR, "kv-move: count %u (at most 64), batch %u, kv heads %u", count,
                     batch, kv_heads);
  const size_t smem = (size_t)count * (head_dim * p.bits / 128 + 1) * 16;   // at most 17 KB
  const cudaError_t e = launch_pdl(kv_move_kernel, dim3(kv_heads, batch, 2), dim3(kThreads), smem,
                                   (cudaStream_t)stream, p, SRC, DST, count);
  count_launches(1);
  return cuda_status(e, "kv-move");
}
