// k_treeattn.cu -- attention of a tree of drafted tokens over the quantised
// paged cache (kv_quant.cuh); one node is an ordinary decode step.
//
// For a query row q (a node and a head), over the keys t it sees,
//   score_t = scale q.k_t,  o = sum_t softmax_t(score) v_t,
// with k_t = s c (8 bits) or s c + lo (4 bits; c is then taken less 8, and lo
// with 8 s more), so that
//   q.k_t = s (q.c) + lo sum(q),   sum_t p_t v_t = sum_t (p_t s_t) c_t + sum_t p_t lo_t:
// the matrix products run on the codes themselves, small integers that are
// exact in float16, and the scales meet the scores and the weights in 32 bits.
// The other operand is normalised to a power of two (a query row by its
// largest value, the weights p_t s_t by the largest scale met so far) and
// rounded to float16: one term (11 bits) where the output is bfloat16, whose
// 8 bits hide it; a second term, the remainder (22 bits), where it is float32.
//
// Rows of one key head -- nodes x the query heads that share it -- are taken
// 16 at a time (mma.sync m16n8k16).  The work is the list of (sequence, key
// head, 16 rows) items, each a run of 128-key tiles; every CTA takes an equal
// run of that list whatever the sequences' lengths, keeps the softmax state of
// one item at a time, and writes the output itself where it has the whole
// item, or a partial state that a second kernel joins.  A warp has its own 32
// keys of each tile and its own cp.async ring, so nothing synchronises the
// CTA until an item ends.
//
// Key order.  Within 16 keys the two 8-key score tiles hold keys 4t, 4t+1 and
// 4t+2, 4t+3 in the columns of lane t, so a lane's weights are four successive
// keys and V is read four rows a lane.  The K index of the score product is
// permuted so a lane's part of a key is whole 16-byte chunks; the columns of
// the second product so a lane's part of a value row is contiguous.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_quant.cuh"

namespace nl {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kKeys = 32;                  // keys of a warp's tile
constexpr int kTile = kKeys * kWarps;      // keys of a CTA's tile
constexpr int kRows = 16;                  // query rows of an item
constexpr uint32_t kMaxCtas = 148 * 4;
constexpr uint32_t kNone = ~0u;

struct TreeArgs {
  const void *q;
  void *o;
  float *lse;
  const int32_t *table, *len;
  const uint64_t *mask;
  float *part_o, *part_ml;       // partial states: [2 * ctas][kRows][HD], [..][kRows][2]
  uint64_t q_stride, o_stride;
  KvPool pool;
  uint32_t batch, nodes, heads, group, rows, row_tiles, max_blocks, ctas;
  float scale;                   // scale * log2(e)
};

// ---- the list of work -----------------------------------------------------

__device__ __forceinline__ uint32_t prefix_of(const TreeArgs &a, uint32_t b) {
  return (uint32_t)max(__ldg(a.len + b), 0);
}
// Tokens of sequence b that the table can hold.
__device__ __forceinline__ uint32_t keys_of(const TreeArgs &a, uint32_t b) {
  const uint64_t n = (uint64_t)prefix_of(a, b) + a.nodes;
  const uint64_t most = (uint64_t)a.max_blocks * a.pool.block_size;
  return (uint32_t)(n < most ? n : most);
}
// Tiles of one of its items: at least one, so that every row is written.
__device__ __forceinline__ uint32_t tiles_of(const TreeArgs &a, uint32_t b) {
  const uint32_t n = keys_of(a, b);
  return n ? (n + kTile - 1) / kTile : 1u;
}

struct Share {
  uint64_t total, before;        // all tiles; those of the sequences before b
  uint32_t b;                    // the sequence that tile AT falls into
};
__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t all_tiles(const TreeArgs &a) {
  const uint32_t lane = threadIdx.x & 31;
  uint64_t v = 0;
  for (uint32_t b = lane; b < a.batch; b += 32) v += tiles_of(a, b);
  return warp_sum(v) * (a.pool.kv_heads * a.row_tiles);
}
// The sequence that tile AT of the list falls into, and the tiles before it.
__device__ __forceinline__ void locate(const TreeArgs &a, uint64_t at, uint32_t *b_out,
                                       uint64_t *before_out) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t items = (uint64_t)a.pool.kv_heads * a.row_tiles;
  uint64_t before = 0;
  for (uint32_t base = 0; base < a.batch; base += 32) {
    uint64_t mine = base + lane < a.batch ? tiles_of(a, base + lane) * items : 0, end = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= (uint32_t)o) end += up;
    }
    end += before;
    const uint32_t past = __ballot_sync(0xffffffffu, base + lane < a.batch && at < end);
    if (past) {
      const int first = __ffs(past) - 1;
      *b_out = base + first;
      *before_out = __shfl_sync(0xffffffffu, end - mine, first);
      return;
    }
    before = __shfl_sync(0xffffffffu, end, 31);
  }
  *b_out = a.batch;
  *before_out = before;
}
// CTA c of w takes the tiles [share(c), share(c + 1)).
__device__ __forceinline__ uint64_t share(uint64_t total, uint32_t w, uint32_t c) {
  return total / w * c + total % w * c / w;
}
__device__ __forceinline__ uint32_t owner(uint64_t total, uint32_t w, uint64_t at) {
  uint32_t c = (uint32_t)((double)at * w / (double)total);
  if (c >= w) c = w - 1;
  while (c + 1 < w && share(total, w, c + 1) <= at) c++;
  while (c > 0 && share(total, w, c) > at) c--;
  return c;
}

// ---- small device helpers ---------------------------------------------------

__device__ __forceinline__ uint32_t su32(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src),
               "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;\n" ::: "memory");
}
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t *>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2 *>(&v); }

// o += the two-term product.  The tensor core cuts, not rounds, what it adds to
// an accumulator, and over a long context that drifts; where the output is
// float32 each 16 keys are summed apart and added in float32.
template <int Terms>
__device__ __forceinline__ void weigh(float (&o)[4], const uint4 (&p)[Terms], uint32_t b0,
                                      uint32_t b1) {
  if (Terms == 1) {
    mma16(o, p[0], b0, b1);
  } else {
    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = Terms - 1; e >= 0; e--) mma16(d, p[e], b0, b1);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] += d[i];
  }
}

// Two bytes u, v (0 .. 255) of W, placed as float16 1024 + u, 1024 + v by the
// selector, less 1152: the signed codes u - 128, v - 128, exactly.
__device__ __forceinline__ uint32_t codes8(uint32_t w, uint32_t sel) {
  return h2(__hsub2(as_h2(__byte_perm(w, 0x64646464u, sel)), as_h2(0x64806480u)));
}
// The nibbles at bits 0 and 16 (4 and 20) of W, less 8, as float16.
__device__ __forceinline__ uint32_t codes4_low(uint32_t w) {
  return h2(__hsub2(as_h2((w & 0x000f000fu) | 0x64006400u), as_h2(0x64086408u)));
}
__device__ __forceinline__ uint32_t codes4_high(uint32_t w) {
  return h2(__hfma2(as_h2((w & 0x00f000f0u) | 0x64006400u), as_h2(0x2c002c00u),
                    as_h2(0xd480d480u)));   // (1024 + 16 c) / 16 - 64 - 8
}
// Scale and offset of a parameter word.  Four-bit codes are used less 8, so
// the offset is that of the middle of the range: with it at the low end the
// two sums q.c and lo sum(q) would be large and of opposite signs.
template <int BITS> __device__ __forceinline__ float scale_of(uint32_t w) {
  return __uint_as_float(BITS == 8 ? w : w << 16);
}
__device__ __forceinline__ float middle_of(uint32_t w) {
  return fmaf(8.0f, __uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// ---- geometry -----------------------------------------------------------------

template <int HD, int BITS> struct Geo {
  static constexpr int RB = HD * BITS / 8;            // bytes of a row
  static constexpr int Chunks = RB / 16;
  static constexpr int Steps = HD / 16;               // k16 steps of the score product
  static constexpr int Words = HD * BITS / 128;       // words of a key a lane holds
  static constexpr int NT = HD / 8;                   // column tiles of the second product
  static constexpr int Stage = 2 * kKeys * RB + 2 * kKeys * 4 + 16;   // codes, words, valid keys
  static constexpr int Stages = RB <= 64 ? 4 : RB <= 128 ? 3 : 2;
  static constexpr int Ring = kWarps * Stages * Stage;
  // Byte of chunk c of key k: keys two rows apart (read together by the lanes
  // of a score tile) and value rows four apart (by those of the second
  // product) are kept off each other's banks.
  static __device__ __forceinline__ uint32_t k_at(uint32_t key, uint32_t c) {
    return key * RB + (RB >= 128 ? c ^ ((key & 1) << 2) : c) * 16;
  }
  static __device__ __forceinline__ uint32_t v_at(uint32_t key, uint32_t c) {
    return (((key * Chunks + c) ^ (((key >> 2) & 3) << 1))) * 16;
  }
  // Column d of the output that column n of column tile nt holds.
  static __device__ __forceinline__ uint32_t column(uint32_t n, uint32_t nt) {
    if (HD == 256 && BITS == 8) return nt / 16 * 128 + 16 * n + nt % 16;
    return HD / 8 * n + nt;
  }
  // Where element d of a query row goes among the operand fragments: step,
  // lane of the quad, which of the two registers, which half.
  static __device__ __forceinline__ void spot(uint32_t d, uint32_t *step, uint32_t *t, uint32_t *p,
                                              uint32_t *i) {
    if (BITS == 8) {
      const uint32_t c = d / 16;
      *t = c & 3;
      *step = c / 4 * 4 + d % 16 / 4;
      *p = d % 4 / 2;
      *i = d % 2;
    } else {
      constexpr uint32_t per = HD == 64 ? 16 : 32;    // elements of a lane's contiguous part
      const uint32_t c = d / per, e = d % 8;
      *t = c & 3;
      *step = 2 * (c / 4 * 4 + d % per / 8) + ((e >> 1) & 1);
      *p = e & 1;
      *i = e >> 2;
    }
  }
};

template <int HD> constexpr int kPitch = HD + 4;       // floats of a row when states are joined

template <typename T, int HD, int BITS> struct Smem {
  static constexpr int Terms = sizeof(T) == 4 ? 2 : 1;
  static constexpr int Q = Terms * Geo<HD, BITS>::Steps * 512;
  static constexpr int Join = kWarps * kRows * kPitch<HD> * 4;
  static constexpr int Ring = Geo<HD, BITS>::Ring > Join ? Geo<HD, BITS>::Ring : Join;
  // query fragments, row factors and sums, masks, per-warp (max, sum), ring
  static constexpr int Bytes = Q + kRows * 8 + kRows * 8 + kWarps * kRows * 8 + Ring;
};

template <typename T> __device__ __forceinline__ float load1(const T *p);
template <> __device__ __forceinline__ float load1<float>(const float *p) { return __ldg(p); }
template <> __device__ __forceinline__ float load1<__nv_bfloat16>(const __nv_bfloat16 *p) {
  return __bfloat162float(__ldg(p));
}
__device__ __forceinline__ void store1(float *p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, int HD, int BITS>
__global__ void __launch_bounds__(kThreads)
tree_attn_kernel(const __grid_constant__ TreeArgs a) {
  using G = Geo<HD, BITS>;
  using S = Smem<T, HD, BITS>;
  constexpr int Terms = S::Terms;
  extern __shared__ __align__(16) uint8_t smem[];
  uint4 *qf = reinterpret_cast<uint4 *>(smem);                       // [Terms][Steps][32]
  float2 *row_q = reinterpret_cast<float2 *>(smem + S::Q);           // factor, sum of a row
  uint64_t *row_mask = reinterpret_cast<uint64_t *>(row_q + kRows);
  float2 *ml = reinterpret_cast<float2 *>(row_mask + kRows);         // [kWarps][kRows]
  uint8_t *ring = reinterpret_cast<uint8_t *>(ml + kWarps * kRows);

  pdl_trigger();
  pdl_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint64_t total = all_tiles(a);
  const uint32_t workers = total < a.ctas ? (uint32_t)total : a.ctas;
  if (blockIdx.x >= workers) return;
  uint64_t at = share(total, workers, blockIdx.x);
  const uint64_t end = share(total, workers, blockIdx.x + 1);
  uint32_t b;
  uint64_t before;
  locate(a, at, &b, &before);
  const uint32_t items = a.pool.kv_heads * a.row_tiles;
  uint8_t *mine = ring + warp * (G::Stages * G::Stage);
  const uint64_t used = a.nodes < 64 ? (1ull << a.nodes) - 1 : ~0ull;

  while (at < end) {
    // ---- the next item, or part of one ----
    const uint32_t tiles = tiles_of(a, b);
    if (at >= before + (uint64_t)tiles * items) {
      before += (uint64_t)tiles * items;
      b++;
      continue;
    }
    const uint32_t item = (uint32_t)((at - before) / tiles), t0 = (uint32_t)((at - before) % tiles);
    const uint32_t t1 = end - at < tiles - t0 ? t0 + (uint32_t)(end - at) : tiles;
    const uint32_t head = item / a.row_tiles, row0 = item % a.row_tiles * kRows;
    const uint32_t prefix = prefix_of(a, b), keys = keys_of(a, b);

    // ---- its query rows, as operand fragments ----
    __syncthreads();               // the last item's states are joined
    {
      constexpr int Per = HD / 8;  // values of a row a thread takes, 8 threads a row
      const uint32_t r = threadIdx.x / 8, part = threadIdx.x % 8, row = row0 + r;
      const bool live = row < a.rows;
      const uint32_t node = live ? row / a.group : 0;
      const T *q = (const T *)a.q + ((uint64_t)b * a.nodes + node) * a.q_stride +
                   (uint64_t)(head * a.group + (live ? row % a.group : 0)) * HD + part * Per;
      float v[Per], top = 0.0f, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < Per; i++) {
        v[i] = live ? load1(q + i) : 0.0f;
        top = fmaxf(top, fabsf(v[i]));
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // the power of two that brings the largest value to [2^13, 2^14)
      int up = 140 - (int)(__float_as_uint(top) >> 23);
      if (top == 0.0f || !(top < INFINITY)) up = 0;
      up = min(up, 126);
      const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
      for (int i = 0; i < Per; i++) {
        v[i] *= mul;
        sum += v[i];
        uint32_t step, quad, p, half;
        G::spot(part * Per + i, &step, &quad, &p, &half);
        const uint32_t byte = (step * 32 + (r & 7) * 4 + quad) * 16 + (2 * p + (r >> 3)) * 4 +
                              half * 2;
        const __half hi = __float2half_rn(v[i]);
        *reinterpret_cast<__half *>(smem + byte) = hi;
        if (Terms == 2)
          *reinterpret_cast<__half *>(smem + G::Steps * 512 + byte) =
              __float2half_rn(v[i] - __half2float(hi));
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (part == 0) {
        // never zero: a factor of zero would make NaN of a masked score
        row_q[r] = make_float2(fmaxf(a.scale * __uint_as_float((uint32_t)(127 - up) << 23),
                                     1.17549435e-38f), sum);
        row_mask[r] = live ? a.mask[(uint64_t)b * a.nodes + node] & used : 0;
      }
    }
    __syncthreads();

    float o[G::NT][4];
#pragma unroll
    for (int i = 0; i < G::NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, base[2] = {0.0f, 0.0f};
    float vs = 1.0f;               // the weights are p s vs
    uint32_t vlimit = 0;           // scales below these bits fit vs
    const float f[2] = {row_q[g].x, row_q[g + 8].x};
    const float qsum[2] = {row_q[g].y, row_q[g + 8].y};

    // ---- this warp's tiles of the run, through its ring ----
    auto request = [&](uint32_t tile, uint32_t slot) {
      const uint32_t k0 = tile * kTile + warp * kKeys, key = k0 + lane;
      uint32_t row = kNone;
      if (key < keys) {
        const uint32_t block =
            (uint32_t)__ldg(a.table + (uint64_t)b * a.max_blocks + key / a.pool.block_size);
        if (block < a.pool.num_blocks)
          row = kv_row(a.pool, block, key % a.pool.block_size, head);
      }
      const uint32_t valid = __ballot_sync(0xffffffffu, row != kNone);
      uint8_t *st = mine + slot * G::Stage;
      const uint32_t s0 = su32(st), words = s0 + 2 * kKeys * G::RB;
      const bool on = row != kNone;
      copy4(words + lane * 4, a.pool.param[0] + (on ? row : 0), on);
      copy4(words + 128 + lane * 4, a.pool.param[1] + (on ? row : 0), on);
      if (lane == 0) *reinterpret_cast<uint32_t *>(st + 2 * kKeys * G::RB + 256) = valid;
#pragma unroll
      for (int i = 0; i < G::Chunks; i++) {
        const uint32_t k = (i * 32 + lane) / G::Chunks, c = (i * 32 + lane) % G::Chunks;
        const uint32_t from = __shfl_sync(0xffffffffu, row, k);
        const bool have = from != kNone;
        const uint64_t byte = (uint64_t)(have ? from : 0) * G::RB + c * 16;
        copy16(s0 + G::k_at(k, c), a.pool.code[0] + byte, have);
        copy16(s0 + kKeys * G::RB + G::v_at(k, c), a.pool.code[1] + byte, have);
      }
    };
    uint32_t asked = t0;
#pragma unroll
    for (int i = 0; i < G::Stages - 1; i++) {
      if (asked < t1) request(asked, (asked - t0) % G::Stages);
      asked++;
      copy_commit();
    }
    for (uint32_t tile = t0; tile < t1; tile++) {
      if (asked < t1) request(asked, (asked - t0) % G::Stages);
      asked++;
      copy_commit();
      copy_wait<G::Stages - 1>();
      __syncwarp();
      const uint8_t *st = mine + (tile - t0) % G::Stages * G::Stage;
      const uint8_t *kc = st, *vc = st + kKeys * G::RB;
      const uint32_t *kw = reinterpret_cast<const uint32_t *>(st + 2 * kKeys * G::RB);
      const uint32_t *vw = kw + 32;
      const uint32_t valid = vw[32];
      const uint32_t k0 = tile * kTile + warp * kKeys;

      // scores of 16 rows x 32 keys, in units of the normalised query
      float s[4][4];
#pragma unroll
      for (int n = 0; n < 4; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
      const uint32_t krow = 4 * (g >> 1) + (g & 1);
#pragma unroll
      for (int h = 0; h < (G::Words + 3) / 4; h++) {
        uint32_t w[4][4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
          const uint32_t key = 16 * (n >> 1) + 2 * (n & 1) + krow;
          if (G::Words == 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(kc + key * G::RB + t * 8);
            w[n][0] = x.x; w[n][1] = x.y;
          } else {
            const uint4 x = *reinterpret_cast<const uint4 *>(kc + G::k_at(key, t + 4 * h));
            w[n][0] = x.x; w[n][1] = x.y; w[n][2] = x.z; w[n][3] = x.w;
          }
        }
#pragma unroll
        for (int i = 0; i < (G::Words < 4 ? G::Words : 4); i++) {
#pragma unroll
          for (int half = 0; half < (BITS == 8 ? 1 : 2); half++) {
            const int step = BITS == 8 ? 4 * h + i : 2 * (4 * h + i) + half;
            uint4 q[Terms];
#pragma unroll
            for (int e = 0; e < Terms; e++) q[e] = qf[(e * G::Steps + step) * 32 + lane];
#pragma unroll
            for (int n = 0; n < 4; n++) {
              uint32_t b0, b1;
              if (BITS == 8) {
                b0 = codes8(w[n][i], 0x4140);
                b1 = codes8(w[n][i], 0x4342);
              } else {
                const uint32_t x = half ? w[n][i] >> 8 : w[n][i];
                b0 = codes4_low(x);
                b1 = codes4_high(x);
              }
#pragma unroll
              for (int e = Terms - 1; e >= 0; e--) mma16(s[n], q[e], b0, b1);
            }
          }
        }
      }

      // scales, offsets and masks
      const bool whole = k0 + kKeys <= prefix && valid == 0xffffffffu;
      uint32_t see[2] = {0xffffffffu, 0xffffffffu};
      if (!whole) {
        const uint32_t pre = k0 >= prefix ? 0u
                             : prefix - k0 >= 32 ? 0xffffffffu : (1u << (prefix - k0)) - 1u;
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const uint64_t w = row_mask[g + 8 * r];
          uint32_t nodes = 0;
          if (k0 >= prefix) nodes = k0 - prefix < 64 ? (uint32_t)(w >> (k0 - prefix)) : 0u;
          else if (prefix - k0 < 32) nodes = (uint32_t)(w << (prefix - k0));
          see[r] = (pre | nodes) & valid;
        }
      }
      float x[2][8];               // [row][key 4 kk + i of this lane]
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const uint4 wd = *reinterpret_cast<const uint4 *>(kw + 16 * kk + 4 * t);
        const uint32_t wv[4] = {wd.x, wd.y, wd.z, wd.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float sc = scale_of<BITS>(wv[i]), mid = middle_of(wv[i]);
#pragma unroll
          for (int r = 0; r < 2; r++) {
            float v = s[2 * kk + (i >> 1)][2 * r + (i & 1)] * sc;
            if (BITS == 4) v = fmaf(mid, qsum[r], v);
            if (!whole && !(see[r] >> (16 * kk + 4 * t + i) & 1)) v = -INFINITY;
            x[r][4 * kk + i] = v;
            top[r] = fmaxf(top[r], v);
          }
        }
      }
      float keep[2];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        top[r] = fmaxf(top[r], m[r]);
        keep[r] = top[r] == m[r] ? 1.0f : ex2((m[r] - top[r]) * f[r]);
      }
      // the largest finite scale of the values decides the weights' power of two
      uint32_t big = BITS == 8 ? vw[lane] : vw[lane] << 16;
      big = __reduce_max_sync(0xffffffffu, big < 0x7f800000u ? big : 0u);
      float ratio = 1.0f;
      if (big >= vlimit && big != 0) {
        const uint32_t e = (big >> 23) + 1;             // scales below 2^(e - 127)
        vlimit = e << 23;
        const float next = __uint_as_float((269u - e) << 23);   // to below 2^15
        ratio = next / vs;
        vs = next;
      }
      if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f) || ratio != 1.0f) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
          l[r] *= keep[r];
          base[r] *= keep[r];
          const float c = keep[r] * ratio;
#pragma unroll
          for (int i = 0; i < G::NT; i++) {
            o[i][2 * r] *= c;
            o[i][2 * r + 1] *= c;
          }
        }
      }
      float off[2];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        m[r] = top[r];
        off[r] = top[r] == -INFINITY ? 0.0f : -top[r] * f[r];
      }

      // weights, and the second product
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const uint4 wd = *reinterpret_cast<const uint4 *>(vw + 16 * kk + 4 * t);
        const uint32_t wv[4] = {wd.x, wd.y, wd.z, wd.w};
        float p[2][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float sc = scale_of<BITS>(wv[i]) * vs, mid = middle_of(wv[i]);
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const float e = ex2(fmaf(x[r][4 * kk + i], f[r], off[r]));
            l[r] += e;
            const bool seen = whole || (see[r] >> (16 * kk + 4 * t + i) & 1);
            if (BITS == 4 && seen) base[r] = fmaf(e, mid, base[r]);
            p[r][i] = seen ? e * sc : 0.0f;
          }
        }
        uint4 pa[Terms];
#pragma unroll
        for (int e = 0; e < Terms; e++) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float *v = &p[j & 1][2 * (j >> 1)];
            const __half2 hi = __floats2half2_rn(v[0], v[1]);
            w[j] = h2(hi);
            if (e + 1 < Terms) {
              v[0] -= __low2float(hi);
              v[1] -= __high2float(hi);
            }
          }
          pa[e] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        // a lane's part of the four value rows, in groups of 4 (8 bits) or 8
        // (4 bits) columns a word
        constexpr int VW = G::RB / 32;                   // words of a row a lane holds
        uint32_t w[4][VW];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t key = 16 * kk + 4 * t + i;
          if (VW == 1) {
            w[i][0] = *reinterpret_cast<const uint32_t *>(vc + G::v_at(key, g / 4) + g % 4 * 4);
          } else if (VW == 2) {
            const uint2 y = *reinterpret_cast<const uint2 *>(vc + G::v_at(key, g / 2) + g % 2 * 8);
            w[i][0] = y.x; w[i][VW - 1] = y.y;
          } else {
#pragma unroll
            for (int h = 0; h < VW / 4; h++) {
              const uint4 y = *reinterpret_cast<const uint4 *>(vc + G::v_at(key, g + 8 * h));
              w[i][4 * h] = y.x; w[i][4 * h + 1] = y.y; w[i][4 * h + 2] = y.z;
              w[i][4 * h + 3] = y.w;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < VW; j++) {
          if (BITS == 8) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
              const uint32_t sel = u ? 0x7362 : 0x5140;
              const uint32_t ab = __byte_perm(w[0][j], w[1][j], sel);
              const uint32_t cd = __byte_perm(w[2][j], w[3][j], sel);
#pragma unroll
              for (int c = 0; c < 2; c++) {
                const uint32_t b0 = codes8(ab, c ? 0x4342 : 0x4140);
                const uint32_t b1 = codes8(cd, c ? 0x4342 : 0x4140);
                weigh<Terms>(o[4 * j + 2 * u + c], pa, b0, b1);
              }
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; u++) {                // byte u: columns 2u, 2u + 1
              const uint32_t sel = u < 2 ? 0x5410 : 0x7632;
              uint32_t ab = __byte_perm(w[0][j], w[1][j], sel);
              uint32_t cd = __byte_perm(w[2][j], w[3][j], sel);
              if (u & 1) ab >>= 8, cd >>= 8;
              weigh<Terms>(o[8 * j + 2 * u], pa, codes4_low(ab), codes4_low(cd));
              weigh<Terms>(o[8 * j + 2 * u + 1], pa, codes4_high(ab), codes4_high(cd));
            }
          }
        }
      }
      __syncwarp();                // the stage may be requested again
    }
    copy_wait<0>();

    // ---- join the warps' states ----
#pragma unroll
    for (int r = 0; r < 2; r++) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      base[r] += __shfl_xor_sync(0xffffffffu, base[r], 1);
      base[r] += __shfl_xor_sync(0xffffffffu, base[r], 2);
      m[r] = m[r] == -INFINITY ? m[r] : m[r] * f[r];
      if (t == 0) ml[warp * kRows + g + 8 * r] = make_float2(m[r], l[r]);
    }
    __syncthreads();               // and every warp is done with its ring
    float *join = reinterpret_cast<float *>(ring);
    {
      const float back = 1.0f / vs;
#pragma unroll
      for (int r = 0; r < 2; r++) {
        float *to = join + (warp * kRows + g + 8 * r) * kPitch<HD>;
#pragma unroll
        for (int i = 0; i < G::NT; i++) {
          to[G::column(2 * t, i)] = fmaf(o[i][2 * r], back, base[r]);
          to[G::column(2 * t + 1, i)] = fmaf(o[i][2 * r + 1], back, base[r]);
        }
      }
    }
    __syncthreads();
    {
      constexpr int Per = HD / 8;
      const uint32_t r = threadIdx.x / 8, part = threadIdx.x % 8, row = row0 + r;
      float top = -INFINITY, sum = 0.0f, c[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; w++) top = fmaxf(top, ml[w * kRows + r].x);
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        const float2 v = ml[w * kRows + r];
        c[w] = v.x == -INFINITY ? 0.0f : ex2(v.x - top);
        // a row of NaN scores has the maximum -inf and a sum that is NaN
        if (v.x == -INFINITY && v.y != v.y) c[w] = 1.0f;
        sum = fmaf(c[w], v.y, sum);
      }
      const bool first = t0 == 0, last = t1 == tiles;
      const uint32_t slot = 2 * blockIdx.x + (first ? 1 : 0);
      const bool empty = row_mask[r] == 0 || sum == 0.0f;
      const float inv = 1.0f / sum;
      const uint32_t node = row / a.group, h = head * a.group + row % a.group;
      const uint64_t out_row = (uint64_t)b * a.nodes + node;
#pragma unroll
      for (int i = 0; i < Per; i++) {
        const uint32_t d = i * 8 + part;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++)
          v = c[w] == 0.0f ? v : fmaf(c[w], join[(w * kRows + r) * kPitch<HD> + d], v);
        if (!(first && last)) {
          a.part_o[((uint64_t)slot * kRows + r) * HD + d] = v;
        } else if (row < a.rows) {
          store1((T *)a.o + out_row * a.o_stride + (uint64_t)h * HD + d, empty ? 0.0f : v * inv);
        }
      }
      if (part == 0) {
        if (!(first && last)) {
          a.part_ml[((uint64_t)slot * kRows + r) * 2] = top;
          a.part_ml[((uint64_t)slot * kRows + r) * 2 + 1] = sum;
        } else if (row < a.rows && a.lse) {
          a.lse[out_row * a.heads + h] =
              empty ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        }
      }
    }
    at += t1 - t0;
  }
}

// Joins the partial states of the items that several CTAs share: a block per
// output row.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads)
tree_join_kernel(const __grid_constant__ TreeArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red[kWarps][HD + 2];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t h = blockIdx.x % a.heads, bn = blockIdx.x / a.heads;
  const uint32_t b = bn / a.nodes, row = bn % a.nodes * a.group + h % a.group;
  const uint64_t total = all_tiles(a);
  const uint32_t workers = total < a.ctas ? (uint32_t)total : a.ctas;
  uint64_t before = 0;
  {
    for (uint32_t i = lane; i < b; i += 32) before += tiles_of(a, i);
    before = warp_sum(before) * ((uint64_t)a.pool.kv_heads * a.row_tiles);
  }
  const uint32_t tiles = tiles_of(a, b);
  const uint64_t s0 = before + (uint64_t)(h / a.group * a.row_tiles + row / kRows) * tiles;
  const uint32_t c0 = owner(total, workers, s0), c1 = owner(total, workers, s0 + tiles - 1);
  if (c0 == c1) return;
  constexpr int Per = HD / 32;
  float v[Per], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < Per; i++) v[i] = 0.0f;
  for (uint32_t c = c0 + warp; c <= c1; c += kWarps) {
    const uint64_t at = (uint64_t)(2 * c + (c == c0 ? 1 : 0)) * kRows + row % kRows;
    const float pm = a.part_ml[2 * at], pl = a.part_ml[2 * at + 1];
    if (pm == -INFINITY && pl == 0.0f) continue;
    const float top = fmaxf(m, pm);
    const float old = m == top ? 1.0f : ex2(m - top), add = pm == top ? 1.0f : ex2(pm - top);
    m = top;
    l = fmaf(l, old, pl * add);
#pragma unroll
    for (int i = 0; i < Per; i++) v[i] = fmaf(v[i], old, a.part_o[at * HD + i * 32 + lane] * add);
  }
#pragma unroll
  for (int i = 0; i < Per; i++) red[warp][i * 32 + lane] = v[i];
  if (lane == 0) red[warp][HD] = m, red[warp][HD + 1] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.0f, c[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; w++) top = fmaxf(top, red[w][HD]);
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    c[w] = red[w][HD] == top ? 1.0f : ex2(red[w][HD] - top);
    sum = fmaf(c[w], red[w][HD + 1], sum);
  }
  const uint64_t words = a.mask[bn] & (a.nodes < 64 ? (1ull << a.nodes) - 1 : ~0ull);
  const bool empty = words == 0 || sum == 0.0f;
  const float inv = 1.0f / sum;
  for (uint32_t d = threadIdx.x; d < HD; d += kThreads) {
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; w++) y = fmaf(c[w], red[w][d], y);
    store1((T *)a.o + (uint64_t)bn * a.o_stride + (uint64_t)h * HD + d, empty ? 0.0f : y * inv);
  }
  if (threadIdx.x == 0 && a.lse)
    a.lse[(uint64_t)bn * a.heads + h] =
        empty ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

template <typename T, int HD, int BITS>
cudaError_t start(TreeArgs &a, cudaStream_t st) {
  constexpr int smem = Smem<T, HD, BITS>::Bytes;
  static int per_sm = 0;
  if (!per_sm) {
    cudaError_t e = cudaFuncSetAttribute(tree_attn_kernel<T, HD, BITS>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    int n = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, tree_attn_kernel<T, HD, BITS>, kThreads,
                                                      smem);
    if (e != cudaSuccess) return e;
    per_sm = n < 1 ? 1 : n > 4 ? 4 : n;
  }
  a.ctas = 148u * per_sm;
  cudaError_t e = launch_pdl(tree_attn_kernel<T, HD, BITS>, dim3(a.ctas), dim3(kThreads), smem, st,
                             a);
  if (e != cudaSuccess) return e;
  count_launches(2);
  return launch_pdl(tree_join_kernel<T, HD>, dim3(a.batch * a.nodes * a.heads), dim3(kThreads), 0,
                    st, a);
}
template <typename T>
cudaError_t start_t(TreeArgs &a, cudaStream_t st) {
  switch (a.pool.head_dim + a.pool.bits) {
    case 64 + 8: return start<T, 64, 8>(a, st);
    case 128 + 8: return start<T, 128, 8>(a, st);
    case 256 + 8: return start<T, 256, 8>(a, st);
    case 64 + 4: return start<T, 64, 4>(a, st);
    case 128 + 4: return start<T, 128, 4>(a, st);
    default: return start<T, 256, 4>(a, st);
  }
}

}  // namespace
}  // namespace nl

using namespace nl;

extern "C" size_t nl_tree_attn_workspace_bytes(uint32_t nodes, uint32_t heads, uint32_t kv_heads,
                                               uint32_t head_dim) {
  (void)nodes; (void)heads; (void)kv_heads;
  return (size_t)2 * kMaxCtas * kRows * (head_dim + 2) * sizeof(float);
}

extern "C" int nl_tree_attn_dev(int fmt, int dtype, const void *Q, uint64_t q_stride,
                                const void *KC, const uint32_t *KP, const void *VC,
                                const uint32_t *VP, const int32_t *TABLE, const int32_t *LEN,
                                const uint64_t *MASK, void *O, uint64_t o_stride, float *LSE,
                                uint32_t batch, uint32_t nodes, uint32_t heads, uint32_t kv_heads,
                                uint32_t head_dim, uint32_t block_size, uint32_t num_blocks,
                                uint32_t max_blocks, float scale, void *workspace,
                                size_t ws_bytes, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  const char *what = "tree-attn";
  if (dtype != NL_F32 && dtype != NL_BF16)
    return set_error(NL_ERROR, "%s: type %d is neither NL_F32 nor NL_BF16", what, dtype);
  TreeArgs a = {};
  a.pool = {{(uint8_t *)const_cast<void *>(KC), (uint8_t *)const_cast<void *>(VC)},
            {const_cast<uint32_t *>(KP), const_cast<uint32_t *>(VP)}, num_blocks, block_size,
            kv_heads, head_dim, (uint32_t)fmt};
  if ((rc = kv_check_pool(what, fmt, a.pool))) return rc;
  if (!heads || heads % kv_heads || heads > 65536)
    return set_error(NL_ERROR, "%s: heads %u, kv heads %u", what, heads, kv_heads);
  if (nodes > 64) return set_error(NL_ERROR, "%s: %u nodes (at most 64)", what, nodes);
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return set_error(NL_ERROR, "%s: scale %g is not positive and finite", what, scale);
  if (batch == 0 || nodes == 0) return NL_OK;
  if ((uint64_t)batch * nodes * heads > INT32_MAX)
    return set_error(NL_ERROR, "%s: %u sequences x %u nodes x %u heads", what, batch, nodes, heads);
  if (!LEN || !MASK || ((uintptr_t)MASK & 7u) || (!TABLE && max_blocks))
    return set_error(NL_ERROR, "%s: null lengths, masks or table, or unaligned masks", what);
  const uint32_t unit = dtype == NL_BF16 ? 8 : 4;
  const uint64_t width = (uint64_t)heads * head_dim;
  if (!Q || !O || !aligned16(Q) || !aligned16(O) || q_stride % unit || o_stride % unit ||
      q_stride < width || o_stride < width)
    return set_error(NL_ERROR,
                     "%s: Q and O rows must be 16-byte aligned, with strides (%llu, %llu) that are "
                     "multiples of %u and at least heads x head size",
                     what, (unsigned long long)q_stride, (unsigned long long)o_stride, unit);
  cudaStream_t st = (cudaStream_t)stream;
  const size_t need = nl_tree_attn_workspace_bytes(nodes, heads, kv_heads, head_dim);
  if (workspace && ws_bytes < need)
    return set_error(NL_ERROR, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
  if (!workspace) workspace = library_workspace(need, st);
  if (!workspace || !aligned16(workspace))
    return set_error(NL_ERROR, "%s: no aligned workspace of %zu bytes", what, need);
  a.q = Q; a.o = O; a.lse = LSE; a.table = TABLE; a.len = LEN; a.mask = MASK;
  a.q_stride = q_stride; a.o_stride = o_stride;
  a.batch = batch; a.nodes = nodes; a.heads = heads; a.group = heads / kv_heads;
  a.rows = a.group * nodes; a.row_tiles = (a.rows + kRows - 1) / kRows;
  a.max_blocks = max_blocks;
  a.scale = scale * 1.4426950408889634f;
  if (!num_blocks)                 // nothing is read of an empty pool, but its addresses are formed
    for (int i = 0; i < 2; i++)
      a.pool.code[i] = (uint8_t *)workspace, a.pool.param[i] = (uint32_t *)workspace;
  a.part_o = (float *)workspace;
  a.part_ml = a.part_o + (size_t)2 * kMaxCtas * kRows * head_dim;
  return cuda_status(dtype == NL_BF16 ? start_t<__nv_bfloat16>(a, st) : start_t<float>(a, st),
                     what);
}
