// tree_work.cuh -- what the kernels of the tree attention share: their
// arguments, the list of work and how CTAs divide it, and the codes as float16.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_quant.cuh"

namespace nl {

constexpr uint32_t kTreeMaxCtas = 148 * 4;
constexpr uint32_t kTreeMaxItemCost = 16;

struct TreeArgs {
  const void *q;
  void *o;
  float *lse;
  const int32_t *table, *len;
  const uint64_t *mask;
  float *part_o, *part_ml;       // partial states: [2 * ctas][rows_at_once][HD], [..][2]
  uint64_t q_stride, o_stride;
  KvPool pool;
  uint32_t batch, nodes, heads, group, rows, row_tiles, max_blocks, ctas;
  uint32_t rows_at_once, tile;   // rows of an item; keys of a CTA's tile
  // What an item costs besides its tiles (its queries, the first fill, the
  // join), in tiles: the shares count it, or a CTA whose share is many short
  // items would end long after the others.
  uint32_t item_cost;
  uint32_t block_shift;          // log2(block_size), or 32 if it is not a power of two
  float scale;                   // scale * log2(e)
};

// The launches for one head size (k_treeattn_h*.cu): NR and WR follow from
// the rows.
template <int HD> cudaError_t tree_attn_start(TreeArgs &a, bool bf16, cudaStream_t st);
// The joining kernel alone.
template <int HD> cudaError_t tree_join_start(TreeArgs &a, bool bf16, cudaStream_t st);
// The tcgen05 form (k_treeattn_umma.cu): the rows of an item it would take, or
// 0 where it does not apply, and its launch.
uint32_t tree_umma_rows(const TreeArgs &a, bool bf16);
cudaError_t tree_umma_start(TreeArgs &a, cudaStream_t st);

#ifdef NL_TREE_KERNELS
namespace {

constexpr uint32_t kNone = ~0u;

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
  return n ? (n + a.tile - 1) / a.tile : 1u;
}

// (The entry point refuses lists of 2^32 places and more: in 64 bits the
// divisions here took a microsecond of a call with a few keys, and registers of
// the others.)
// The list's length -- an item counts its tiles and its own cost -- and the CTAs
// it is divided among.  Where all sequences are equally long, a number of CTAs
// that the items divide evenly gives every CTA a part of one item only, which saves
// it an item's own cost, and leaves some CTAs without work: it is taken where a
// CTA's part grows by no more than that.  (Even / by places, us: 32 items of 8 rows
// of 64 values, bf16, 32,768 keys, on 576 or 592 CTAs, 39.8 / 52.9; 128 items of 32
// rows, bf16, 4 bits, on 128 or 148, 500 keys 19.8 / 25.7, 2,000: 34.9 / 39.0, 64 rows,
// 8 bits, 1,000 keys 28.4 / 35.3; but 128 of 32 rows, 8,192 keys 101 / 96, 32,768: 374 /
// 322; 256 of a row, f32, 4,096 keys, on 256 or 296 61.7 / 61.4.)
struct List {
  uint32_t total, workers;
};
__device__ __forceinline__ List list_of(const TreeArgs &a) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t sum = 0;
  uint32_t least = ~0u, most = 0;
  for (uint32_t b = lane; b < a.batch; b += 32) {
    const uint32_t t = tiles_of(a, b);
    sum += t + a.item_cost;
    least = min(least, t);
    most = max(most, t);
  }
  List l;
  const uint32_t items = a.pool.kv_heads * a.row_tiles;
  l.total = __reduce_add_sync(0xffffffffu, sum) * items;
  l.workers = min(l.total, a.ctas);
  const uint32_t all = items * a.batch;
  const uint32_t tiles = __reduce_max_sync(0xffffffffu, most);
  if (__reduce_min_sync(0xffffffffu, least) == tiles && all <= l.workers) {
    const uint32_t even = l.workers / all * all;
    // all (tiles + cost) (1 / even - 1 / workers) <= cost
    const float grows = (float)all * (float)(tiles + a.item_cost) * (float)(l.workers - even);
    if (grows <= (float)even * (float)l.workers * (float)a.item_cost) l.workers = even;
  }
  return l;
}
// The sequence that place AT of the list falls into, and the places before it.
__device__ __forceinline__ void locate(const TreeArgs &a, uint32_t at, uint32_t *b_out,
                                       uint32_t *before_out) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t items = a.pool.kv_heads * a.row_tiles;
  uint32_t before = 0;
  for (uint32_t base = 0; base < a.batch; base += 32) {
    const uint32_t mine =
        base + lane < a.batch ? (tiles_of(a, base + lane) + a.item_cost) * items : 0;
    uint32_t end = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, end, o);
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
// CTA c of w takes the places [share(c), share(c + 1)).
__device__ __forceinline__ uint32_t share(uint32_t total, uint32_t w, uint32_t c) {
  return total / w * c + total % w * c / w;      // w is at most kTreeMaxCtas
}
__device__ __forceinline__ uint32_t owner(uint32_t total, uint32_t w, uint32_t at) {
  uint32_t c = (uint32_t)((float)at * ((float)w / (float)total));      // or a neighbour of it
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

// The 8 x 8 matrix of 16-bit values whose row g, columns 2t and 2t + 1, lane
// (g, t) holds, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// The tensor core cuts, not rounds, what it adds to an accumulator: with values of
// one sign the sum falls behind by 0.5e-7 of itself an addition here, 1e-7 by
// tcgen05 (measured; 8 bits, 100,000 keys in one part: mean error -3.0e-4 and
// -6.5e-4).  Where the output is float32 each 16 keys are summed apart and added in
// float32.  Where it is bfloat16, whose rounding is 2^-9, a part longer than
// kTreeRun tiles of 32 keys (two additions each) or kTreeRunUmma of 128 (eight each)
// is taken in runs of that many, joined in float32: at most 2,048 additions and
// 2^-12.  (Sums taken out of the accumulator within the loop over the tiles made
// every call of the tcgen05 form 8 to 12% slower, however rare and small the code; a
// run costs about seven tiles, 3% of a long part.)
constexpr uint32_t kTreeRun = 512, kTreeRunUmma = 256;

// o += codes x weights.
template <int Terms, int NR, bool Flush>
__device__ __forceinline__ void weigh(float (&o)[4], const uint4 &c,
                                      const uint32_t (&p)[Terms][NR][2], int n) {
  if (!Flush) {
    mma16(o, c, p[0][n][0], p[0][n][1]);
  } else {
    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = Terms - 1; e >= 0; e--) mma16(d, c, p[e][n][0], p[e][n][1]);
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
// The limits of value scales, as exponents: scales below 2^(e - 127), 0 before
// any was met.  Where the rows' own limits differ, E is the one the common power of
// two of the weights goes by -- that of the keys before, or the least, unless the
// largest is more than kTreeApart above it -- and a row's weights are raised over
// it by the powers of two that apart_by says.  (Largest cases: 2^60 up or down
// leaves sums of weights their whole range, and what is cut at 2^60 comes out of the
// 15 bits that float16 has to spare.)
constexpr int kTreeApart = 60;
// What stands for a limit before any scale was met, and where rows have their own:
// less than any scale's bits but zero's, so that a scale met is looked at.
constexpr uint32_t kTreeNone = 1, kTreeOwn = 2;
__device__ __forceinline__ uint32_t limit_of(uint32_t scale) {
  return max((scale >> 23) + 1, 16u);            // the least scale is 2^-112
}
// Whether that has to be looked at row by row, for a tile of nodes whose scales lie
// in [LOW, E]: 2^kTreeSpare of difference fits the bits that float16 has to spare, and
// then one limit serves all rows, unless a row may meet its first scale later (not
// ALL: a prefix key that all rows see has one, or the tile is the last).  (Most calls
// run the code for that nowhere: with it in every first tile of nodes 16 ragged
// sequences of 32 rows took 5 us more.)
constexpr uint32_t kTreeSpare = 10;
__device__ __forceinline__ bool rows_apart(uint32_t before, uint32_t low, uint32_t e, bool all) {
  return before ? e > before + kTreeSpare : !all || e > low + kTreeSpare;
}
__device__ __forceinline__ uint32_t common_limit(uint32_t before, uint32_t least, uint32_t most) {
  const int from = before ? (int)before : most ? (int)least : 0;
  return (uint32_t)max(from, (int)most - kTreeApart);
}
__device__ __forceinline__ int apart_by(uint32_t e, uint32_t own) {
  return own ? max(-kTreeApart, min((int)e - (int)own, kTreeApart)) : 0;
}
// A query row is raised by at most 2^kTreeUp to float16's range (below, what it
// loses is less than 2^-100 of a score), and its factor is at least kTreeFactor:
// a factor of zero would make NaN of a masked score, and 2^kTreeApart over it has to
// be finite.
constexpr int kTreeUp = 100;
constexpr float kTreeFactor = 7.70371978e-34f;   // 2^-110
// Scale and offset of a parameter word.  Four-bit codes are used less 8, so
// the offset is that of the middle of the range: with it at the low end the
// two sums q.c and lo sum(q) would be large and of opposite signs.
template <int BITS> __device__ __forceinline__ float scale_of(uint32_t w) {
  return __uint_as_float(BITS == 8 ? w : w << 16);
}
__device__ __forceinline__ float middle_of(uint32_t w) {
  return fmaf(8.0f, __uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

}  // namespace
#endif  // NL_TREE_KERNELS

}  // namespace nl
