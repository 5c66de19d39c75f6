// tree_attn.cuh -- attention of a tree of drafted tokens over the quantised
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
// The codes are the first operand of mma.sync m16n8k16 in both products --
// 16 keys x 8 rows of scores, 16 columns x 8 rows of output -- so a decode
// step with few rows wastes nothing: rows are padded to 8, not 16, and the
// state of 8 rows is 32 registers at 128 columns.  The scores come out with a
// key per lane group and leave as the second operand with a row per lane
// group: one movmatrix per 8 x 8 weights.
//
// Rows of one key head -- nodes x the query heads that share it -- are taken
// 8 NR WR at a time, an item: NR tiles of 8 rows a warp, WR warps for
// different rows of the same keys.  The work is the list of the items' runs of
// key tiles; every CTA takes an equal run of that list whatever the sequences'
// lengths, keeps the softmax state of one item at a time, and writes the
// output itself where it has the whole item, or a partial state that a second
// kernel joins.  The WR warps of 32 keys share a cp.async ring, and nothing
// else synchronises the CTA until an item ends.
//
// What bounds it: with few rows the loads.  8 sequences of 4,096 keys, 32 heads
// of 128, float32, 8 bits: 61.5 us for 277 MB, 0.69 of a copy's rate; the same
// without the products 50, the join 3.  With many rows the issue of products and
// weights: the table at start_rows; in bfloat16 the tcgen05 form
// (k_treeattn_umma.cu) takes over there.
//
// Key order.  Row r of a 16-key tile is key 4 (r % 8 / 2) + r % 2 + 2 (r / 8):
// the second product then takes four successive value rows a lane.  The K
// index of the score product is permuted so a lane's part of a key is whole
// 16-byte chunks, and the columns of the second product so a lane's part of a
// value row is contiguous.
#pragma once

#define NL_TREE_KERNELS
#include "tree_work.cuh"

namespace nl {
namespace {

constexpr int kTreeWarps = 4, kTreeThreads = 32 * kTreeWarps;
constexpr int kTreeKeys = 32;              // keys of a warp's tile

// ---- geometry -----------------------------------------------------------------

template <int HD, int BITS> struct Geo {
  static constexpr int RB = HD * BITS / 8;            // bytes of a row
  static constexpr int Chunks = RB / 16;
  static constexpr int Steps = HD / 16;               // k16 steps of the score product
  static constexpr int Words = HD * BITS / 128;       // words of a key a lane holds
  static constexpr int MT = HD / 16;                  // 16-column tiles of the second product
  static constexpr int Stage = 2 * kTreeKeys * RB + 2 * kTreeKeys * 4 + 16;   // codes, words, valid
  // Byte of chunk c of key k: key rows read together by the lanes of a score
  // tile (two apart) and value rows read together by those of the second
  // product (four apart) are kept off each other's banks.
  static __device__ __forceinline__ uint32_t k_at(uint32_t key, uint32_t c) {
    return key * RB + (RB >= 128 ? c ^ ((key & 1) << 2) : c) * 16;
  }
  static __device__ __forceinline__ uint32_t v_at(uint32_t key, uint32_t c) {
    return (((key * Chunks + c) ^ (((key >> 2) & 3) << 1))) * 16;
  }
  // Column d of the output that lane group g holds as its column nt.
  static __device__ __forceinline__ uint32_t column(uint32_t g, uint32_t nt) {
    if (HD == 256 && BITS == 8) return nt / 16 * 128 + 16 * g + nt % 16;
    return HD / 8 * g + nt;
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

template <typename T, int HD, int BITS, int NR, int WR, bool PACK> struct Plan {
  using G = Geo<HD, BITS>;
  // PACK: at most four rows, whose two terms are columns r and r + 4 of one
  // tile instead of two products.
  static constexpr int Terms = sizeof(T) == 4 && !PACK ? 2 : 1;
  static constexpr int WK = kTreeWarps / WR;                // warps with keys of their own
  static constexpr int Rows = 8 * NR * WR, Tile = kTreeKeys * WK;
  static constexpr int Q = Terms * Rows * HD * 2;           // query fragments
  static constexpr int Stages = WR > 1 ? 4 : G::RB <= 64 ? 4 : G::RB <= 128 ? 3 : 2;
  static constexpr int Ring = WK * Stages * G::Stage;
  static constexpr int Pitch = HD + 4;                     // floats of a row when states are joined
  static constexpr int Join = WK * Rows * Pitch * 4;        // over the fragments and the ring
  // row factors, row sums, masks, per-warp (max, sum), per-warp limits
  static constexpr int Small = Rows * 4 + Rows * 4 + Rows * 8 + WK * Rows * 8 + WK * Rows * 4;
  static constexpr int Bytes = Small + (Q + Ring > Join ? Q + Ring : Join);
};

// N values from a place aligned to all of them, or to 16 bytes.
template <int N> __device__ __forceinline__ void load_row(const float *p, float *v) {
  if constexpr (N == 2) {
    const float2 x = __ldg(reinterpret_cast<const float2 *>(p));
    v[0] = x.x; v[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4 *>(p + i));
      v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
    }
  }
}
template <int N> __device__ __forceinline__ void load_row(const __nv_bfloat16 *p, float *v) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p + i));
    v[i] = __uint_as_float(x.x << 16); v[i + 1] = __uint_as_float(x.x & 0xffff0000u);
    v[i + 2] = __uint_as_float(x.y << 16); v[i + 3] = __uint_as_float(x.y & 0xffff0000u);
  }
}
__device__ __forceinline__ void store1(float *p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, int HD, int BITS, int NR, int WR, bool PACK>
__global__ void __launch_bounds__(kTreeThreads)
tree_attn_kernel(const __grid_constant__ TreeArgs a) {
  using G = Geo<HD, BITS>;
  using P = Plan<T, HD, BITS, NR, WR, PACK>;
  constexpr int Terms = P::Terms, WK = P::WK, Stages = P::Stages;
  constexpr bool Flush = sizeof(T) == 4;         // each 16 keys summed apart
  constexpr uint32_t Live = PACK ? 4 : P::Rows;  // rows of an item
  // threads of a row where it is read and where its state is joined
  constexpr uint32_t PerRow = Live <= 4 ? 32 : Live <= 8 ? 16 : 8;
  extern __shared__ __align__(16) uint8_t smem[];
  float *row_f = reinterpret_cast<float *>(smem);                    // factor of a row's scores
  float *row_sum = row_f + P::Rows;                                  // sum of its query
  uint64_t *row_mask = reinterpret_cast<uint64_t *>(row_sum + P::Rows);
  float2 *ml = reinterpret_cast<float2 *>(row_mask + P::Rows);       // [WK][Rows]
  uint32_t *row_lim = reinterpret_cast<uint32_t *>(ml + WK * P::Rows);  // [WK][Rows], if apart
  uint8_t *qf = reinterpret_cast<uint8_t *>(row_lim + WK * P::Rows);
  uint8_t *ring = qf + P::Q;
  float *join = reinterpret_cast<float *>(qf);

  pdl_wait();
  pdl_trigger();                 // after the wait: the join reads the lengths before its own
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t wr = warp % WR, wk = warp / WR;
  const List list = list_of(a);
  const uint32_t total = list.total, workers = list.workers;
  if (blockIdx.x >= workers) return;
  uint32_t at = share(total, workers, blockIdx.x);
  const uint32_t begin = at;
  uint32_t part0 = 0;            // the first tile of this CTA's part of an item, over its runs
  const uint32_t end = share(total, workers, blockIdx.x + 1);
  uint32_t b;
  uint32_t before;
  locate(a, at, &b, &before);
  const uint32_t items = a.pool.kv_heads * a.row_tiles;
  uint8_t *mine = ring + wk * (Stages * G::Stage);
  const uint64_t used = a.nodes < 64 ? (1ull << a.nodes) - 1 : ~0ull;
  // Byte of lane (row % 8, quad)'s fragment of a step: one tile of 8 rows
  // (8 bytes) or two side by side (16).
  auto fragment = [](uint32_t row, uint32_t step, uint32_t quad) {
    const uint32_t l = (row & 7) * 4 + quad;
    if (NR == 1) return ((row / 8 * G::Steps + step) * 32 + l) * 8;
    return ((row / 16 * G::Steps + step) * 32 + l) * 16 + (row / 8 & 1) * 8;
  };

  while (at < end) {
    // ---- the next item, or part of one ----
    const uint32_t tiles = tiles_of(a, b), cost = tiles + a.item_cost;
    if (at >= before + cost * items) {
      before += cost * items;
      b++;
      continue;
    }
    const uint32_t item = (at - before) / cost, c0 = (at - before) % cost;
    uint32_t c1 = end - at < cost - c0 ? c0 + (end - at) : cost;
    // Where the sums stay in the tensor core's accumulator a part is taken in
    // runs, each joined with the state that the one before left in the workspace.
    bool resumed = false, more = false;
    if constexpr (!Flush) {
      const uint32_t most = max(c0, a.item_cost) + kTreeRun;
      resumed = c0 != 0 && at != begin;
      more = c1 > most;
      c1 = min(c1, most);
    }
    at += c1 - c0;
    if (c1 <= a.item_cost) continue;             // its share ends before the first tile
    const uint32_t t0 = c0 > a.item_cost ? c0 - a.item_cost : 0, t1 = c1 - a.item_cost;
    if (Flush || !resumed) part0 = t0;
    const uint32_t head = item / a.row_tiles, row0 = item % a.row_tiles * Live;
    const uint32_t prefix = prefix_of(a, b), keys = keys_of(a, b);

    // ---- keys on their way ----
    // The pool row of this lane's key of a tile, kNone where there is none.
    auto find = [&](uint32_t tile) {
      const uint32_t key = tile * P::Tile + wk * kTreeKeys + lane;
      if (tile >= t1 || key >= keys) return kNone;
      const uint32_t page = a.block_shift < 32 ? key >> a.block_shift : key / a.pool.block_size;
      const uint32_t off = key - page * a.pool.block_size;
      const uint32_t block = (uint32_t)__ldg(a.table + (uint64_t)b * a.max_blocks + page);
      return block < a.pool.num_blocks ? kv_row(a.pool, block, off, head) : kNone;
    };
    auto request = [&](uint32_t row, uint32_t slot) {
      const uint32_t valid = __ballot_sync(0xffffffffu, row != kNone);
      uint8_t *st = mine + slot * G::Stage;
      const uint32_t s0 = su32(st), words = s0 + 2 * kTreeKeys * G::RB;
      const bool on = row != kNone;
      if (WR == 1 || wr == 0) {
        copy4(words + lane * 4, a.pool.param[0] + (on ? row : 0), on);
        copy4(words + 128 + lane * 4, a.pool.param[1] + (on ? row : 0), on);
        if (lane == 0) *reinterpret_cast<uint32_t *>(st + 2 * kTreeKeys * G::RB + 256) = valid;
      }
#pragma unroll
      for (int i = 0; i < (G::Chunks + WR - 1) / WR; i++) {
        const uint32_t n = (i * WR + wr) * 32 + lane;
        if (G::Chunks % WR != 0 && n >= kTreeKeys * G::Chunks) break;   // the whole warp
        const uint32_t k = n / G::Chunks, c = n % G::Chunks;
        const uint32_t from = __shfl_sync(0xffffffffu, row, k);
        const bool have = from != kNone;
        const uint64_t byte = (uint64_t)(have ? from : 0) * G::RB + c * 16;
        copy16(s0 + G::k_at(k, c), a.pool.code[0] + byte, have);
        copy16(s0 + kTreeKeys * G::RB + G::v_at(k, c), a.pool.code[1] + byte, have);
      }
    };
    __syncthreads();               // the last item's states are joined
    uint32_t next = find(t0);
#pragma unroll
    for (int i = 0; i < Stages - 1; i++) {
      if (t0 + i < t1) request(next, i);
      copy_commit();
      next = find(t0 + i + 1);
    }

    // ---- the query rows, as operand fragments ----
    for (uint32_t r = threadIdx.x / PerRow; r < Live; r += kTreeThreads / PerRow) {
      constexpr int Per = HD / PerRow;
      const uint32_t part = threadIdx.x % PerRow, row = row0 + r;
      const bool live = row < a.rows;
      const uint32_t node = live ? row / a.group : 0;
      const T *q = (const T *)a.q + ((uint64_t)b * a.nodes + node) * a.q_stride +
                   (uint64_t)(head * a.group + (live ? row % a.group : 0)) * HD + part * Per;
      const uint64_t mask = live ? a.mask[(uint64_t)b * a.nodes + node] & used : 0;
      float v[Per], top = 0.0f, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < Per; i++) v[i] = 0.0f;
      if (live) load_row<Per>(q, v);
#pragma unroll
      for (int i = 0; i < Per; i++) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
      for (int o = PerRow / 2; o > 0; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // the power of two that brings the largest value to [2^13, 2^14)
      int up = 140 - (int)(__float_as_uint(top) >> 23);
      if (top == 0.0f || !(top < INFINITY)) up = 0;
      up = min(up, kTreeUp);
      const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
      for (int i = 0; i < Per; i++) {
        v[i] *= mul;
        sum += v[i];
        uint32_t step, quad, p, half;
        G::spot(part * Per + i, &step, &quad, &p, &half);
        const uint32_t byte = fragment(r, step, quad) + p * 4 + half * 2;
        const __half hi = __float2half_rn(v[i]);
        const __half low = __float2half_rn(v[i] - __half2float(hi));
        *reinterpret_cast<__half *>(qf + byte) = hi;
        if (Terms == 2) *reinterpret_cast<__half *>(qf + P::Rows * HD * 2 + byte) = low;
        if (PACK)
          *reinterpret_cast<__half *>(qf + fragment(r + 4, step, quad) + p * 4 + half * 2) = low;
      }
#pragma unroll
      for (int o = PerRow / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (part == 0) {
#pragma unroll
        for (uint32_t c = r; c < P::Rows; c += PACK ? 4 : P::Rows) {
          row_f[c] = fmaxf(a.scale * __uint_as_float((uint32_t)(127 - up) << 23), kTreeFactor);
          row_sum[c] = sum;
          row_mask[c] = mask;
        }
      }
    }
    __syncthreads();

    const uint32_t r0 = wr * (8 * NR) + 2 * t;      // rows r0 + 8 n and the next are this lane's
    float o[G::MT][NR][4];
#pragma unroll
    for (int i = 0; i < G::MT; i++)
#pragma unroll
      for (int n = 0; n < NR; n++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
    float m[NR][2], l[NR][2], base[NR][2];
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
      for (int r = 0; r < 2; r++) m[n][r] = -INFINITY, l[n][r] = base[n][r] = 0.0f;
    float vs = 1.0f;               // the weights are p s vs
    uint32_t vlimit = kTreeNone;   // scales below these bits fit vs
    // Rows see different nodes, so there a row has a limit of its own, and where
    // the limits differ (VLIMIT is kTreeOwn) its reference M is not the maximum so
    // far but off it by as many powers of two: a node that a row does not see costs
    // it no bits.
    uint32_t *lim = row_lim + wk * P::Rows + r0;

    for (uint32_t tile = t0; tile < t1; tile++) {
      copy_wait<Stages - 2>();
      if (WR == 1) __syncwarp();
      else asm volatile("bar.sync %0, %1;\n" ::"r"(1 + wk), "n"(32 * WR) : "memory");
      // the slot of the tile before this one: every warp of the ring is past it
      if (tile + Stages - 1 < t1) request(next, (tile - t0 + Stages - 1) % Stages);
      copy_commit();
      next = find(tile + Stages);

      const uint8_t *st = mine + (tile - t0) % Stages * G::Stage;
      const uint8_t *kc = st, *vc = st + kTreeKeys * G::RB;
      const uint32_t *kw = reinterpret_cast<const uint32_t *>(st + 2 * kTreeKeys * G::RB);
      const uint32_t *vw = kw + 32;
      const uint32_t valid = vw[32];
      const uint32_t k0 = tile * P::Tile + wk * kTreeKeys;
      const uint32_t krow = 4 * (g >> 1) + (g & 1);  // and two keys on

      // scores of 32 keys x 8 NR rows, in units of the normalised queries
      float s[2][NR][4];
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int n = 0; n < NR; n++) s[k][n][0] = s[k][n][1] = s[k][n][2] = s[k][n][3] = 0.0f;
#pragma unroll
      for (int h = 0; h < (G::Words + 3) / 4; h++) {
        uint32_t w[2][2][4];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const uint32_t key = 16 * k + 2 * u + krow;
            if (G::Words == 2) {
              const uint2 x = *reinterpret_cast<const uint2 *>(kc + key * G::RB + t * 8);
              w[k][u][0] = x.x; w[k][u][1] = x.y;
            } else {
              const uint4 x = *reinterpret_cast<const uint4 *>(kc + G::k_at(key, t + 4 * h));
              w[k][u][0] = x.x; w[k][u][1] = x.y; w[k][u][2] = x.z; w[k][u][3] = x.w;
            }
          }
#pragma unroll
        for (int i = 0; i < (G::Words < 4 ? G::Words : 4); i++) {
#pragma unroll
          for (int half = 0; half < (BITS == 8 ? 1 : 2); half++) {
            const int step = BITS == 8 ? 4 * h + i : 2 * (4 * h + i) + half;
            uint32_t q[Terms][NR][2];
#pragma unroll
            for (int e = 0; e < Terms; e++) {
              const uint8_t *from = qf + e * (P::Rows * HD * 2);
              if (NR == 1) {
                const uint2 x =
                    *reinterpret_cast<const uint2 *>(from + fragment(8 * wr + g, step, t));
                q[e][0][0] = x.x; q[e][0][1] = x.y;
              } else {
#pragma unroll
                for (int n = 0; n < NR; n += 2) {
                  const uint4 x = *reinterpret_cast<const uint4 *>(
                      from + fragment(8 * NR * wr + 8 * n + g, step, t));
                  q[e][n][0] = x.x; q[e][n][1] = x.y;
                  q[e][n + 1 < NR ? n + 1 : 0][0] = x.z; q[e][n + 1 < NR ? n + 1 : 0][1] = x.w;
                }
              }
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
              uint4 c;
              if (BITS == 8) {
                c = make_uint4(codes8(w[k][0][i], 0x4140), codes8(w[k][1][i], 0x4140),
                               codes8(w[k][0][i], 0x4342), codes8(w[k][1][i], 0x4342));
              } else {
                const uint32_t x = half ? w[k][0][i] >> 8 : w[k][0][i];
                const uint32_t y = half ? w[k][1][i] >> 8 : w[k][1][i];
                c = make_uint4(codes4_low(x), codes4_low(y), codes4_high(x), codes4_high(y));
              }
#pragma unroll
              for (int e = Terms - 1; e >= 0; e--)
#pragma unroll
                for (int n = 0; n < NR; n++) mma16(s[k][n], c, q[e][n][0], q[e][n][1]);
            }
          }
        }
      }

      if (PACK) {                  // the other term's column is two lanes on
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[k][0][i] += __shfl_xor_sync(0xffffffffu, s[k][0][i], 2);
      }

      // scales, offsets and masks: s becomes the score over the row's factor
      const bool whole = k0 + kTreeKeys <= prefix && valid == 0xffffffffu;
      float f[NR][2], top[NR][2];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint32_t wa = kw[16 * k + krow], wb = kw[16 * k + krow + 2];
        const float sa = scale_of<BITS>(wa), sb = scale_of<BITS>(wb);
        const float ma = middle_of(wa), mb = middle_of(wb);
#pragma unroll
        for (int n = 0; n < NR; n++) {
          float2 sum = make_float2(0.0f, 0.0f);
          if (BITS == 4) sum = *reinterpret_cast<const float2 *>(row_sum + r0 + 8 * n);
          float (&x)[4] = s[k][n];
          x[0] *= sa; x[1] *= sa; x[2] *= sb; x[3] *= sb;
          if (BITS == 4) {
            x[0] = fmaf(ma, sum.x, x[0]); x[1] = fmaf(ma, sum.y, x[1]);
            x[2] = fmaf(mb, sum.x, x[2]); x[3] = fmaf(mb, sum.y, x[3]);
          }
        }
      }
      uint32_t see[NR][2];
      if (!whole) {
        const uint32_t pre = k0 >= prefix ? 0u
                             : prefix - k0 >= 32 ? 0xffffffffu : (1u << (prefix - k0)) - 1u;
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const uint64_t w = row_mask[r0 + 8 * n + r];
            uint32_t nodes = 0;
            if (k0 >= prefix) nodes = k0 - prefix < 64 ? (uint32_t)(w >> (k0 - prefix)) : 0u;
            else if (prefix - k0 < 32) nodes = (uint32_t)(w << (prefix - k0));
            see[n][r] = ((pre | nodes) & valid) >> krow;     // this lane's keys: 0, 2, 16, 18
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
              for (int u = 0; u < 2; u++)
                if (!(see[n][r] >> (16 * k + 2 * u) & 1)) s[k][n][2 * u + r] = -INFINITY;
          }
      }
      bool moved = false;
#pragma unroll
      for (int n = 0; n < NR; n++) {
        const float2 ff = *reinterpret_cast<const float2 *>(row_f + r0 + 8 * n);
        f[n][0] = ff.x; f[n][1] = ff.y;
#pragma unroll
        for (int r = 0; r < 2; r++) {
          float v = fmaxf(fmaxf(s[0][n][r], s[0][n][2 + r]), fmaxf(s[1][n][r], s[1][n][2 + r]));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          top[n][r] = fmaxf(v, m[n][r]);
          moved |= top[n][r] != m[n][r];
        }
      }
      // the largest finite scale of the values decides the weights' power of two
      uint32_t one = BITS == 8 ? vw[lane] : vw[lane] << 16;
      one = one < 0x7f800000u ? one : 0u;
      const uint32_t big = __reduce_max_sync(0xffffffffu, one);
      float ratio = 1.0f;
      if (big >= vlimit) {
        const bool apart = vlimit == kTreeOwn;
        const uint32_t before = vlimit == kTreeNone ? 0 : 269u - (__float_as_uint(vs) >> 23);
        uint32_t e = limit_of(big);
        bool rows = false;                              // looked at one by one
        if (k0 + kTreeKeys > prefix) {                  // some keys are nodes
          const uint32_t low = __reduce_min_sync(0xffffffffu, one ? limit_of(one) : ~0u);
          const bool met = __any_sync(0xffffffffu, one != 0 && k0 + lane < prefix);
          rows = apart || rows_apart(before, low, e, met || tile + 1 == t1);
        }
        if (rows) {
          uint32_t own[NR][2], most = 0, least = ~0u;
#pragma unroll
          for (int n = 0; n < NR; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
              uint32_t v = 0;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const uint32_t at = 16 * (i >> 1) + 2 * (i & 1);
                const uint32_t w = __float_as_uint(scale_of<BITS>(vw[at + krow]));
                if ((see[n][r] >> at & 1) && w < 0x7f800000u) v = max(v, w);
              }
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, x));
              own[n][r] = max(apart ? lim[8 * n + r] : before, v ? limit_of(v) : 0u);
              most = max(most, own[n][r]);
              if (own[n][r]) least = min(least, own[n][r]);
            }
          most = __reduce_max_sync(0xffffffffu, most);
          least = __reduce_min_sync(0xffffffffu, least);
          e = common_limit(before, least, most);
          bool differ = false;
#pragma unroll
          for (int n = 0; n < NR; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
              // the maximum so far, and the reference that many powers of two off it
              float v = fmaxf(fmaxf(s[0][n][r], s[0][n][2 + r]), fmaxf(s[1][n][r], s[1][n][2 + r]));
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
              const int was = apart ? apart_by(before, lim[8 * n + r]) : 0;
              const float unit = 1.0f / f[n][r];
              if (m[n][r] != -INFINITY) v = fmaxf(v, fmaf((float)was, unit, m[n][r]));
              top[n][r] = v == -INFINITY ? v : fmaf((float)-apart_by(e, own[n][r]), unit, v);
              differ |= own[n][r] != e;
            }
          __syncwarp();                                 // every lane has read the limits
#pragma unroll
          for (int n = 0; n < NR; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) lim[8 * n + r] = own[n][r];   // of all lanes the same
          __syncwarp();
          vlimit = __any_sync(0xffffffffu, differ) ? kTreeOwn : e ? e << 23 : kTreeNone;
        } else {
          vlimit = e << 23;
        }
        if (e) {
          const float next_vs = __uint_as_float((269u - e) << 23);   // to below 2^15
          ratio = next_vs / vs;
          vs = next_vs;
        }
        moved = true;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < NR; n++) {
          float c[2];
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const float keep = top[n][r] == m[n][r] ? 1.0f : ex2((m[n][r] - top[n][r]) * f[n][r]);
            l[n][r] *= keep;
            base[n][r] *= keep;
            c[r] = keep * ratio;
            m[n][r] = top[n][r];
          }
#pragma unroll
          for (int i = 0; i < G::MT; i++) {
            o[i][n][0] *= c[0]; o[i][n][1] *= c[1];
            o[i][n][2] *= c[0]; o[i][n][3] *= c[1];
          }
        }
      }

      // weights, and the second product
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint32_t wa = vw[16 * k + krow], wb = vw[16 * k + krow + 2];
        const float sc[2] = {scale_of<BITS>(wa) * vs, scale_of<BITS>(wb) * vs};
        const float mid[2] = {middle_of(wa), middle_of(wb)};
        uint32_t p[Terms][NR][2];
#pragma unroll
        for (int n = 0; n < NR; n++) {
          float off[2];
#pragma unroll
          for (int r = 0; r < 2; r++) off[r] = m[n][r] == -INFINITY ? 0.0f : -m[n][r] * f[n][r];
#pragma unroll
          for (int u = 0; u < 2; u++) {
            float e[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
              e[r] = ex2(fmaf(s[k][n][2 * u + r], f[n][r], off[r]));
              l[n][r] += e[r];
              const bool seen = whole || (see[n][r] >> (16 * k + 2 * u) & 1);
              if (BITS == 4 && seen) base[n][r] = fmaf(e[r], mid[u], base[n][r]);
              e[r] = seen ? e[r] * sc[u] : 0.0f;
            }
            __half2 hi = __floats2half2_rn(e[0], e[1]);
            if (PACK) {
              const __half2 low =
                  __floats2half2_rn(e[0] - __low2float(hi), e[1] - __high2float(hi));
              if (t & 2) hi = low;
            }
            p[0][n][u] = transpose8(h2(hi));
            if (Terms == 2)
              p[Terms - 1][n][u] = transpose8(
                  h2(__floats2half2_rn(e[0] - __low2float(hi), e[1] - __high2float(hi))));
          }
        }
        // a lane's part of the four value rows, in groups of 4 (8 bits) or 8
        // (4 bits) columns a word
        constexpr int VW = G::RB / 32;                   // words of a row a lane holds
        constexpr int VL = VW < 4 ? VW : 4;              // at a time
#pragma unroll
        for (int h = 0; h < VW / VL; h++) {
          uint32_t w[4][VL];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t key = 16 * k + 4 * t + i;
            if (VW == 1) {
              w[i][0] = *reinterpret_cast<const uint32_t *>(vc + G::v_at(key, g / 4) + g % 4 * 4);
            } else if (VW == 2) {
              const uint2 y =
                  *reinterpret_cast<const uint2 *>(vc + G::v_at(key, g / 2) + g % 2 * 8);
              w[i][0] = y.x; w[i][VL - 1] = y.y;
            } else {
              const uint4 y = *reinterpret_cast<const uint4 *>(vc + G::v_at(key, g + 8 * h));
              w[i][0] = y.x; w[i][1 % VL] = y.y; w[i][2 % VL] = y.z; w[i][3 % VL] = y.w;
            }
          }
#pragma unroll
          for (int j = 0; j < VL; j++) {
            if (BITS == 8) {
#pragma unroll
              for (int u = 0; u < 2; u++) {              // bytes 2u, 2u + 1
                const uint32_t sel = u ? 0x7362 : 0x5140;
                const uint32_t ab = __byte_perm(w[0][j], w[1][j], sel);
                const uint32_t cd = __byte_perm(w[2][j], w[3][j], sel);
                const uint4 c = make_uint4(codes8(ab, 0x4140), codes8(ab, 0x4342),
                                           codes8(cd, 0x4140), codes8(cd, 0x4342));
#pragma unroll
                for (int n = 0; n < NR; n++)
                  weigh<Terms, NR, Flush>(o[2 * (VL * h + j) + u][n], c, p, n);
              }
            } else {
#pragma unroll
              for (int u = 0; u < 4; u++) {              // byte u: columns 2u, 2u + 1
                const uint32_t sel = u < 2 ? 0x5410 : 0x7632;
                uint32_t ab = __byte_perm(w[0][j], w[1][j], sel);
                uint32_t cd = __byte_perm(w[2][j], w[3][j], sel);
                if (u & 1) ab >>= 8, cd >>= 8;
                const uint4 c = make_uint4(codes4_low(ab), codes4_high(ab), codes4_low(cd),
                                           codes4_high(cd));
#pragma unroll
                for (int n = 0; n < NR; n++)
                  weigh<Terms, NR, Flush>(o[4 * (VL * h + j) + u][n], c, p, n);
              }
            }
          }
        }
      }
    }
    copy_wait<0>();

    // ---- join the warps' states ----
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], x);
          if (BITS == 4) base[n][r] += __shfl_xor_sync(0xffffffffu, base[n][r], x);
        }
        const uint32_t row = r0 + 8 * n + r;
        const float mm = m[n][r] == -INFINITY ? m[n][r] : m[n][r] * row_f[row];
        if (g == 0) ml[wk * P::Rows + row] = make_float2(mm, l[n][r]);
      }
    __syncthreads();               // every warp is done with the fragments and its ring
    {
      const float back = 1.0f / vs;
#pragma unroll
      for (int n = 0; n < NR; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          float *to = join + (wk * P::Rows + r0 + 8 * n + r) * P::Pitch;
          const float add = PACK && (t & 2) ? 0.0f : base[n][r];
#pragma unroll
          for (int i = 0; i < G::MT; i++)
            *reinterpret_cast<float2 *>(to + G::column(g, 2 * i)) =
                make_float2(fmaf(o[i][n][r], back, add), fmaf(o[i][n][2 + r], back, add));
        }
    }
    __syncthreads();
    for (uint32_t r = threadIdx.x / PerRow; r < Live; r += kTreeThreads / PerRow) {
      constexpr int Per = HD / PerRow;
      const uint32_t part = threadIdx.x % PerRow, row = row0 + r;
      float top = -INFINITY, sum = 0.0f, c[WK];
#pragma unroll
      for (int w = 0; w < WK; w++) top = fmaxf(top, ml[w * P::Rows + r].x);
      const bool part_of = more || !(part0 == 0 && t1 == tiles);
      const uint32_t slot = 2 * blockIdx.x + (part0 == 0 ? 1 : 0);
      float run = 0.0f;              // what the runs before weigh
      if constexpr (!Flush) {
        if (resumed) {
          const float2 before =
              *reinterpret_cast<const float2 *>(a.part_ml + ((uint64_t)slot * P::Rows + r) * 2);
          top = fmaxf(top, before.x);
          run = before.x == -INFINITY ? (before.y != before.y ? 1.0f : 0.0f) : ex2(before.x - top);
          sum = run * before.y;
        }
        __syncwarp();                // the row's threads have read it
      }
#pragma unroll
      for (int w = 0; w < WK; w++) {
        const float2 v = ml[w * P::Rows + r];
        c[w] = v.x == -INFINITY ? 0.0f : ex2(v.x - top);
        // a row of NaN scores has the maximum -inf and a sum that is NaN
        if (v.x == -INFINITY && v.y != v.y) c[w] = 1.0f;
        sum = fmaf(c[w], v.y, sum);
      }
      if constexpr (!Flush) {
        if (resumed) {               // the runs before join the first warp's state
#pragma unroll 1
          for (int i = 0; i < Per; i++) {
            float *x = join + r * P::Pitch + i * PerRow + part;
            const float before = a.part_o[((uint64_t)slot * P::Rows + r) * HD + i * PerRow + part];
            *x = (c[0] != 0.0f ? c[0] * *x : 0.0f) + (run != 0.0f ? run * before : 0.0f);
          }
          c[0] = 1.0f;
        }
      }
      const bool empty = row_mask[r] == 0 || sum == 0.0f;
      const float inv = 1.0f / sum;
      const uint32_t node = row / a.group, h = head * a.group + row % a.group;
      const uint64_t out_row = (uint64_t)b * a.nodes + node;
#pragma unroll
      for (int i = 0; i < Per; i++) {
        const uint32_t d = i * PerRow + part;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WK; w++)
          if (c[w] != 0.0f) {
            const float *x = join + (w * P::Rows + r) * P::Pitch + d;
            v = fmaf(c[w], PACK ? x[0] + x[4 * P::Pitch] : x[0], v);
          }
        if (part_of) {
          a.part_o[((uint64_t)slot * P::Rows + r) * HD + d] = v;
        } else if (row < a.rows) {
          store1((T *)a.o + out_row * a.o_stride + (uint64_t)h * HD + d, empty ? 0.0f : v * inv);
        }
      }
      if (part == 0) {
        if (part_of) {
          a.part_ml[((uint64_t)slot * P::Rows + r) * 2] = top;
          a.part_ml[((uint64_t)slot * P::Rows + r) * 2 + 1] = sum;
        } else if (row < a.rows && a.lse) {
          a.lse[out_row * a.heads + h] =
              empty ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        }
      }
    }
  }
}

// Joins the partial states of the items that several CTAs share.  The shares'
// boundaries are the only places where an item can be cut: block (c, y) joins
// four rows of the item that boundary c + 1 cuts, if it is the first to cut it.
// A warp takes a row while the parts are few, the block a row at a time else.
template <typename T, int HD>
__global__ void __launch_bounds__(kTreeThreads)
tree_join_kernel(const __grid_constant__ TreeArgs a) {
  pdl_trigger();
  __shared__ float red[kTreeWarps][HD + 2];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Whatever wrote the lengths is done: the attention kernel lets this one start
  // once it has waited for that itself.
  const List list = list_of(a);
  const uint32_t total = list.total, workers = list.workers, cut = blockIdx.x + 1;
  // (Every block waits, also where it has nothing to join: once this grid is
  // done, whatever follows it takes the attention kernel to be done.)
  if (cut >= workers) {
    pdl_wait();
    return;
  }
  const uint32_t at = share(total, workers, cut);
  uint32_t b;
  uint32_t before;
  locate(a, at, &b, &before);
  const uint32_t tiles = tiles_of(a, b), cost = tiles + a.item_cost;
  const uint32_t off = (at - before) % cost, item = (at - before) / cost;
  const uint32_t s0 = at - off + a.item_cost;     // the item's first tile
  const bool cuts = off > a.item_cost && share(total, workers, cut - 1) <= s0;
  const uint32_t c0 = cut - 1, c1 = owner(total, workers, s0 + tiles - 1);
  const uint32_t head = item / a.row_tiles, row0 = item % a.row_tiles * a.rows_at_once;
  constexpr int Per = HD / 32;
  pdl_wait();
  if (!cuts) return;
  const bool alone = c1 - c0 < 32;                // a warp per row
  for (uint32_t r = alone ? warp : 0; r < 4; r += alone ? 4 : 1) {
    const uint32_t here = blockIdx.y * 4 + r, row = row0 + here;
    if (row >= a.rows) break;                      // of the warp, or of the block
    float v[Per], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < Per; i++) v[i] = 0.0f;
    // 32 parts at a time: a lane finds the weight of one
    const uint32_t step = alone ? 1 : kTreeWarps;
    for (uint32_t c = c0 + (alone ? 0 : warp); c <= c1; c += 32 * step) {
      const uint32_t mine = c + lane * step;
      float pm = -INFINITY, pl = 0.0f;
      if (mine <= c1) {
        const uint64_t from = (uint64_t)(2 * mine + (mine == c0 ? 1 : 0)) * a.rows_at_once + here;
        const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + 2 * from);
        pm = ml.x;
        pl = ml.y;
      }
      float top = fmaxf(m, pm);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // a part without keys weighs nothing; one of NaN may have left no maximum
      const float by = pm == -INFINITY && pl == 0.0f ? 0.0f : pm == top ? 1.0f : ex2(pm - top);
      const float old = m == top ? 1.0f : ex2(m - top);
      float sum = by == 0.0f && pl == pl ? 0.0f : pl * by;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l = fmaf(l, old, sum);
      m = top;
#pragma unroll
      for (int i = 0; i < Per; i++) v[i] *= old;
      const uint32_t n = min(32u, (c1 - c) / step + 1);
#pragma unroll 4
      for (uint32_t p = 0; p < n; p++) {
        const uint32_t part = c + p * step;
        const float w = __shfl_sync(0xffffffffu, by, p);
        const float *from = a.part_o + ((uint64_t)(2 * part + (part == c0 ? 1 : 0)) *
                                            a.rows_at_once + here) * HD + lane;
#pragma unroll
        for (int i = 0; i < Per; i++) {
          const float x = from[i * 32];
          v[i] = w == 0.0f ? v[i] : fmaf(x, w, v[i]);
        }
      }
    }
    if (!alone) {
      __syncthreads();                             // the last row's states are read
#pragma unroll
      for (int i = 0; i < Per; i++) red[warp][i * 32 + lane] = v[i];
      if (lane == 0) red[warp][HD] = m, red[warp][HD + 1] = l;
      __syncthreads();
      float c[kTreeWarps];
      m = -INFINITY;
      l = 0.0f;
#pragma unroll
      for (int w = 0; w < kTreeWarps; w++) m = fmaxf(m, red[w][HD]);
#pragma unroll
      for (int w = 0; w < kTreeWarps; w++) {
        c[w] = red[w][HD] == m ? 1.0f : ex2(red[w][HD] - m);
        l = fmaf(c[w], red[w][HD + 1], l);
      }
#pragma unroll
      for (int i = 0; i < Per; i++) {
        v[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < kTreeWarps; w++) v[i] = fmaf(c[w], red[w][i * 32 + lane], v[i]);
      }
    }
    const uint64_t bn = (uint64_t)b * a.nodes + row / a.group;
    const uint32_t h = head * a.group + row % a.group;
    const uint64_t words = a.mask[bn] & (a.nodes < 64 ? (1ull << a.nodes) - 1 : ~0ull);
    const bool empty = words == 0 || l == 0.0f;
    const float inv = 1.0f / l;
    if (alone || warp == 0) {
#pragma unroll
      for (int i = 0; i < Per; i++)
        store1((T *)a.o + bn * a.o_stride + (uint64_t)h * HD + i * 32 + lane,
               empty ? 0.0f : v[i] * inv);
      if (lane == 0 && a.lse)
        a.lse[bn * a.heads + h] = empty ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
  }
}

template <typename T, int HD, int BITS, int NR, int WR, bool PACK = false>
cudaError_t start(TreeArgs &a, cudaStream_t st) {
  using P = Plan<T, HD, BITS, NR, WR, PACK>;
  static int per_sm = 0;
  if (!per_sm) {
    cudaError_t e = cudaFuncSetAttribute(tree_attn_kernel<T, HD, BITS, NR, WR, PACK>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, P::Bytes);
    if (e != cudaSuccess) return e;
    int n = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(
        &n, tree_attn_kernel<T, HD, BITS, NR, WR, PACK>, kTreeThreads, P::Bytes);
    if (e != cudaSuccess) return e;
    per_sm = n < 1 ? 1 : n > 4 ? 4 : n;
  }
  a.ctas = 148u * per_sm;
  a.tile = P::Tile;
  // About 512 keys.  (With WR, 2 WR, 4 WR, 8 WR, us: 16 sequences of 1,000 keys, 8 key
  // heads, 4 rows, f32 17.4, 17.4, 19.0, 20.4; 3 of 4,096, 32 heads 29.9, 30.4, 31.4,
  // 33.3; but 30 of 700, 8 heads, 4 rows, bf16, 4 bits 24.5, 23.6, 23.2, 20.2; one of
  // 4,000, 64 rows, f32 42.1, 42.2, 42.4, 39.8; long or many items within 2%.)
  a.item_cost = 4 * WR;
  cudaError_t e = launch_pdl(tree_attn_kernel<T, HD, BITS, NR, WR, PACK>, dim3(a.ctas),
                             dim3(kTreeThreads), (size_t)P::Bytes, st, a);
  count_launches(1);
  return e;
}
template <typename T, int HD, int BITS>
cudaError_t start_rows(TreeArgs &a, cudaStream_t st) {
  // Row tiles of a warp: as many as it has registers for, since every warp that
  // shares keys converts their codes again (us, 4 sequences of 32,768 keys, 8 key
  // heads of 128, 8 bits / 4 bits):
  //   rows               16         32         64         128
  //   bf16  4 a warp   69/ 73    100/106    176/193    330/367
  //         half       85/ 98    114/129    209/235    383/424
  //   f32   4 a warp   88/ 87    193/149    275/287    510/552
  //         half      108/112    159/156    293/304    544/565
  // (half: 1 of 16 rows, 2 of more, 128 as two items of 64.)  32 rows of float32 in 8
  // bits are the exception: one warp with four tiles holds both terms of both
  // products and shares its keys with no other.  (Four tiles take all 255 registers
  // and spill up to 100 bytes, as do two of 256 values, up to 190.)
  constexpr int Most = HD == 256 ? 2 : 4;
  constexpr int Part = sizeof(T) == 4 && HD == 128 && BITS == 8 ? 2 : Most;
  // Up to four rows of float32: both terms in one 8-row tile (8 sequences of 4,096
  // keys, 32 heads, 8 bits: 61.6 us where as two tiles it took 69.0).
  if constexpr (sizeof(T) == 4) {
    if (a.rows <= 4) return start<T, HD, BITS, 1, 1, true>(a, st);
  }
  if (a.rows_at_once == 8) return start<T, HD, BITS, 1, 1>(a, st);
  if (a.rows_at_once == 16) return start<T, HD, BITS, 2, 1>(a, st);
  if (a.rows_at_once == 32) return start<T, HD, BITS, Part, 4 / Part>(a, st);
  if (a.rows_at_once == 64) return start<T, HD, BITS, Most, 8 / Most>(a, st);
  if constexpr (Most == 4) return start<T, HD, BITS, Most, 4>(a, st);
  return cudaErrorInvalidValue;
}

}  // namespace

template <int HD>
cudaError_t tree_attn_start(TreeArgs &a, bool bf16, cudaStream_t st) {
  if (a.pool.bits == 8)
    return bf16 ? start_rows<__nv_bfloat16, HD, 8>(a, st) : start_rows<float, HD, 8>(a, st);
  return bf16 ? start_rows<__nv_bfloat16, HD, 4>(a, st) : start_rows<float, HD, 4>(a, st);
}

template <int HD>
cudaError_t tree_join_start(TreeArgs &a, bool bf16, cudaStream_t st) {
  const dim3 grid(a.ctas, (a.rows_at_once + 3) / 4), block(kTreeThreads);
  count_launches(1);
  return bf16 ? launch_pdl(tree_join_kernel<__nv_bfloat16, HD>, grid, block, 0, st, a)
              : launch_pdl(tree_join_kernel<float, HD>, grid, block, 0, st, a);
}

}  // namespace nl
