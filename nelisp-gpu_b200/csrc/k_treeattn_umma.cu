// k_treeattn_umma.cu -- tree attention with many rows a key head on the
// 5th-generation tensor cores (bfloat16 activations, heads of 64 or 128).
//
// The mathematics is tree_attn.cuh's.  Both products have the codes as their
// first operand, so M = 128 is always full whatever the number of rows N:
//   scores  S^T [128 keys x N rows]  = K codes (TMEM) x Q^T (shared memory)
//   output  O^T [128 values x N rows] += V^T codes (shared memory) x P^T (shared memory)
// with float32 accumulators in TMEM.  A score arrives with its key's thread:
// the key's scale is a register, and no row maximum is taken at all in the
// usual tile -- weights are formed against each row's reference, the maximum
// of the keys up to the last time one exceeded it by 2^8 (a vote over the CTA
// per tile), and float16 has the room: scales are brought below 2^7.
//
// 16 warps, one CTA per SM, tiles of 128 keys:
//   warps 0-7   two groups, half the rows each, a thread per key: scores from
//               TMEM, weights to shared memory (the N x 128 operand with N
//               contiguous), sums of the weights in registers; at the end of
//               an item the output from TMEM, a thread per value;
//   warps 8-11  codes to float16, a thread per key: keys to a TMEM stage,
//               values to a shared-memory stage ([key][value], read as V^T);
//   warp 12     TMA of the code tiles, one box per run of a page;
//   warp 13     allocates TMEM and issues the MMAs of both products;
//               warps 14 and 15 have nothing to do.
// The 128 registers a thread of the launch are shared out anew: 168 for the
// score warps, which hold the sums of their rows, 104 for warps 8-11, 72 for
// warps 12-15 (2 x 168 + 104 + 72 = 4 x 128).
// The stages run on over the end of an item: the next item's codes are on
// their way and converted while the last one's output is written.
//
// Per tile of 128 keys and heads of 128, shared memory moves about 1400 (N =
// 64, 8 bits) cycles' worth at 128 bytes each, DRAM 1445 at the SM's share of
// the copy rate, so the two are in balance there; with 4 bits or 128 rows the
// shared memory and the score arithmetic bound it.
//
// Every wait is bounded.  One that gives up sets the library's wait flag, and
// its thread then waits no more but runs on to the end: no barrier of the CTA
// is left short, the copies are waited for and TMEM is freed.

#include <cuda.h>

#define NL_TREE_KERNELS
#include "tree_work.cuh"

namespace nl {
namespace {

constexpr int kThreads = 512;
constexpr int kSoft = 256;                 // threads of the score warps
constexpr int kTileKeys = 128;
constexpr uint32_t kWaitRounds = 4096, kSuspendNs = 1000000;
constexpr float kFar = 1.0e30f;            // a row that has met no key: -reference

template <int HD, int BITS, int N> struct Plan {
  static constexpr int RB = HD * BITS / 8;
  static constexpr int Chunks = RB / 16;
  static constexpr int Codes = kTileKeys * RB;               // one side's codes of a tile
  static constexpr int Stages = 2 * Codes * 3 <= 48 * 1024 ? 3 : N == 64 ? 3 : 2;
  static constexpr int VTile = HD * kTileKeys * 2;            // values as float16
  static constexpr int PBufs = N == 64 ? 2 : 1;
  static constexpr int PTile = N * kTileKeys * 2;
  static constexpr int QTile = N * HD * 2;
  // offsets from a 1024-byte boundary
  static constexpr int V = Stages * 2 * Codes, P = V + 2 * VTile, Q = P + PBufs * PTile;
  static constexpr int Ref = Q + QTile;                       // float2 per row
  static constexpr int Sum = Ref + N * 8;                     // floats
  static constexpr int Keep = Sum + N * 4;
  static constexpr int Masks = Keep + N * 4;
  static constexpr int Offs = Masks + N * 8;                  // output offsets
  static constexpr int Warp = Offs + N * 8;                   // [4][N] floats
  static constexpr int Bars = Warp + 4 * N * 4;
  static constexpr int Used = Bars + 256 + 1024;
  static constexpr int Bytes = Used > 120 * 1024 ? Used : 120 * 1024;   // one CTA per SM (TMEM)
  // TMEM columns
  static constexpr uint32_t KCols = HD / 2;
  static constexpr uint32_t TK = 0, TS = 2 * KCols, TO = TS + 2 * N;
  static_assert(TO + N <= 512 && Used <= 227 * 1024, "tile");
};

__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(b), "r"(n));
}
__device__ __forceinline__ void bar_expect(uint32_t b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(b), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(b) : "memory");
}
// A bounded wait; ALIVE goes false when one gives up, and no later one waits.
__device__ __forceinline__ void bar_wait(uint32_t b, uint32_t parity, bool &alive, int *err) {
  if (!alive) return;
  for (uint32_t i = 0; i < kWaitRounds; i++) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(b), "r"(parity), "r"(kSuspendNs) : "memory");
    if (done) return;
  }
  report_wait_timeout(err);
  alive = false;
}
__device__ __forceinline__ void tma2d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                      uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
}
__device__ __forceinline__ void soft_sync() {
  asm volatile("bar.sync 1, %0;\n" ::"n"(kSoft) : "memory");
}
// Whether any of the score warps' threads says so.
__device__ __forceinline__ bool soft_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, %2, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r) : "r"((uint32_t)v), "n"(kSoft) : "memory");
  return r != 0;
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
        "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(
          at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
// Shared-memory operands in the 128-byte swizzle, rows of 128 bytes in groups
// of eight 1024 bytes apart: rows of the M or N index with 64 K values
// (K-major), or rows of the K index with 64 M or N values, 64-value blocks
// BLOCK bytes apart (M/N-major).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t block) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// float16 x float16 -> float32, M = 128; MN: both operands M/N-major.
template <int N, bool MN> constexpr uint32_t instr_desc() {
  return (1u << 4) | (MN ? (1u << 15) | (1u << 16) : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(
                   bar) : "memory");
}

// The order in which a word's codes leave the conversion: natural for 8 bits;
// nibbles 0, 4, 1, 5, 2, 6, 3, 7 for 4.
template <int BITS> __device__ __forceinline__ uint32_t natural(uint32_t p) {
  return BITS == 8 ? p : (p & ~7u) | ((p & 1) << 2) | ((p >> 1) & 3);
}
// One word of codes as float16 pairs: two registers (8 bits) or four (4 bits).
template <int BITS>
__device__ __forceinline__ void expand(uint32_t w, uint32_t *to) {
  if (BITS == 8) {
    to[0] = codes8(w, 0x4140);
    to[1] = codes8(w, 0x4342);
  } else {
    const uint32_t x = w >> 8;
    to[0] = codes4_low(w);
    to[1] = codes4_high(w);
    to[2] = codes4_low(x);
    to[3] = codes4_high(x);
  }
}

// The sum over a warp's lanes of each of 32 values: lane i gets that of v[i].
__device__ __forceinline__ float sums32(float (&v)[32]) {
  const uint32_t lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool high = lane & o;
#pragma unroll
    for (int i = 0; i < o; i++) {
      const float give = high ? v[i] : v[i + o], keep = high ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

// The walk over the parts of items that a CTA has, the same in every role.
struct Walk {
  uint64_t at, end, before;
  uint32_t b, items;
  uint32_t head, row0, t0, t1, tiles;
  __device__ __forceinline__ bool begin(const TreeArgs &a) {
    const uint64_t total = all_cost(a);
    const uint32_t workers = total < a.ctas ? (uint32_t)total : a.ctas;
    if (blockIdx.x >= workers) return false;
    at = share(total, workers, blockIdx.x);
    end = share(total, workers, blockIdx.x + 1);
    items = a.pool.kv_heads * a.row_tiles;
    locate(a, at, &b, &before);
    return true;
  }
  __device__ __forceinline__ bool next(const TreeArgs &a) {
    while (at < end) {
      tiles = tiles_of(a, b);
      const uint32_t cost = tiles + a.item_cost;
      if (at >= before + (uint64_t)cost * items) {
        before += (uint64_t)cost * items;
        b++;
        continue;
      }
      const uint32_t item = (uint32_t)((at - before) / cost), c0 = (uint32_t)((at - before) % cost);
      const uint32_t c1 = end - at < cost - c0 ? c0 + (uint32_t)(end - at) : cost;
      at += c1 - c0;
      if (c1 <= a.item_cost) continue;
      t0 = c0 > a.item_cost ? c0 - a.item_cost : 0;
      t1 = c1 - a.item_cost;
      head = item / a.row_tiles;
      row0 = item % a.row_tiles * a.rows_at_once;
      return true;
    }
    return false;
  }
};

template <int HD, int BITS, int N>
__global__ void __launch_bounds__(kThreads, 1)
tree_umma_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, uint32_t box, int *err) {
  using L = Plan<HD, BITS, N>;
  constexpr int Half = N / 2;                // rows of a group of score warps
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                            ~(uintptr_t)1023);
  const uint32_t s0 = su32(sm);
  float2 *ref = reinterpret_cast<float2 *>(sm + L::Ref);      // a row's factor, -reference
  float *qsum = reinterpret_cast<float *>(sm + L::Sum);       // the sum of its query
  float *keep = reinterpret_cast<float *>(sm + L::Keep);      // what a new reference leaves of sums
  uint64_t *masks = reinterpret_cast<uint64_t *>(sm + L::Masks);
  uint64_t *offs = reinterpret_cast<uint64_t *>(sm + L::Offs);
  float *warp_part = reinterpret_cast<float *>(sm + L::Warp);
  const uint32_t bars = s0 + L::Bars;
  const uint32_t full = bars, empty = bars + 24, kready = bars + 48, qkdone = bars + 64,
                 sfree = bars + 80, vready = bars + 96, pready = bars + 112, pvdone = bars + 128,
                 qready = bars + 144;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + L::Bars + 160);
  uint32_t *vote = tmem_slot + 1;            // the largest scale of a tile
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::Stages; i++) {
      bar_init(full + 8 * i, 1);
      bar_init(empty + 8 * i, 4);
    }
    for (int i = 0; i < 2; i++) {
      bar_init(kready + 8 * i, 4);
      bar_init(qkdone + 8 * i, 1);
      bar_init(sfree + 8 * i, 8);
      bar_init(vready + 8 * i, 4);
      bar_init(pready + 8 * i, 8);
      bar_init(pvdone + 8 * i, 1);
    }
    bar_init(qready, 8);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 13) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     su32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  bool alive = true;
  Walk w;
  if (w.begin(a)) {
    uint32_t it = 0;                         // tiles so far, over all items
    if (warp >= 12) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
      if (warp == 12) {
        // ---- TMA of the codes: a run of BOX keys of a page at a time, one lane each ----
        const uint32_t runs = kTileKeys / box;
        while (w.next(a)) {
          const uint32_t keys = keys_of(a, w.b);
          for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
            const uint32_t st = it % L::Stages;
            const uint32_t key = tile * kTileKeys + lane * box;
            uint32_t row = kNone;
            if (lane < runs && key < keys) {
              const uint32_t page = key / a.pool.block_size;
              const uint32_t block = (uint32_t)__ldg(a.table + (uint64_t)w.b * a.max_blocks + page);
              if (block < a.pool.num_blocks)
                row = kv_row(a.pool, block, key - page * a.pool.block_size, w.head);
            }
            bar_wait(empty + 8 * st, (it / L::Stages & 1) ^ 1, alive, err);
            const uint32_t count = __popc(__ballot_sync(0xffffffffu, row != kNone));
            // what is not copied keeps older codes: finite, and weighed by zero
            if (lane == 0) bar_expect(full + 8 * st, count * 2 * box * L::RB);
            __syncwarp();
            if (row != kNone) {
              const uint32_t to = s0 + st * (2 * L::Codes) + lane * box * L::RB;
              tma2d(to, &tm_k, 0, (int)row, full + 8 * st);
              tma2d(to + L::Codes, &tm_v, 0, (int)row, full + 8 * st);
            }
          }
        }
        // the last copies, before the CTA may end
        alive = true;
        for (uint32_t i = it > (uint32_t)L::Stages ? it - L::Stages : 0; i < it; i++)
          bar_wait(full + 8 * (i % L::Stages), i / L::Stages & 1, alive, err);
      } else if (warp == 13) {
        // ---- the MMAs: scores of tile i, then the output of tile i - 1 ----
        uint32_t item = 0;
        bool owed = false, first = true;       // a second product not issued yet; its item's first
        auto second = [&](uint32_t i, bool fresh) {
          const uint32_t st = i & 1;
          bar_wait(vready + 8 * st, i >> 1 & 1, alive, err);
          bar_wait(pready + 8 * st, i >> 1 & 1, alive, err);
          fence_after();
          const uint32_t v0 = s0 + L::V + st * L::VTile;
          const uint32_t p0 = s0 + L::P + (L::PBufs == 2 ? st * L::PTile : 0);
  #pragma unroll
          for (int k = 0; k < kTileKeys / 16; k++)
            mma_ss(tmem + L::TO, smem_desc(v0 + 2048 * k, HD == 128 ? kTileKeys * 128 : 0),
                   smem_desc(p0 + 2048 * k, kTileKeys * 128), instr_desc<N, true>(),
                   fresh && k == 0 ? 0u : 1u);
          mma_commit(pvdone + 8 * st);
        };
        while (w.next(a)) {
          if (owed && lane == 0) second(it - 1, first);
          owed = false;
          first = true;
          if (lane == 0) bar_wait(qready, item & 1, alive, err);
          item++;
          for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
            if (lane == 0) {
              const uint32_t st = it & 1;
              bar_wait(kready + 8 * st, it >> 1 & 1, alive, err);
              bar_wait(sfree + 8 * st, (it >> 1 & 1) ^ 1, alive, err);
              fence_after();
  #pragma unroll
              for (int k = 0; k < HD / 16; k++)
                mma_ts(tmem + L::TS + st * N, tmem + L::TK + st * L::KCols + 8 * k,
                       smem_desc(s0 + L::Q + k / 4 * (N * 128) + k % 4 * 32, 16),
                       instr_desc<N, false>(), k ? 1u : 0u);
              mma_commit(qkdone + 8 * st);
              if (owed) {
                second(it - 1, first);
                first = false;
              }
            }
            owed = true;
          }
          __syncwarp();
        }
        if (owed && lane == 0) second(it - 1, first);
        __syncwarp();
      }
    } else if (warp >= 8) {
      // ---- codes to float16, a thread per key ----
      asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n");
      const uint32_t tid = threadIdx.x - kSoft;
      const uint32_t quad = (warp & 3) * 32, key = quad + lane;    // its TMEM lane
      while (w.next(a)) {
        for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
          const uint32_t st = it % L::Stages, h = it & 1;
          const uint8_t *kc = sm + st * (2 * L::Codes), *vc = kc + L::Codes;
          bar_wait(full + 8 * st, it / L::Stages & 1, alive, err);
          bar_wait(qkdone + 8 * h, (it >> 1 & 1) ^ 1, alive, err);
          fence_after();
          // byte of chunk c of a key's row, swizzled by the copy over the row's bytes
          auto chunk = [](uint32_t k, uint32_t c) {
            const uint32_t x = L::RB == 128 ? k & 7 : L::RB == 64 ? k >> 1 & 3 : k >> 2 & 1;
            return k * L::RB + ((c ^ x) << 4);
          };
          constexpr int Each = BITS == 8 ? 4 : 2;       // chunks that make 32 TMEM columns
#pragma unroll
          for (int c0 = 0; c0 < L::Chunks; c0 += Each) {
            uint32_t v[32];
#pragma unroll
            for (int c = 0; c < Each; c++) {
              const uint4 x = *reinterpret_cast<const uint4 *>(kc + chunk(key, c0 + c));
              constexpr int W = BITS == 8 ? 2 : 4;
              uint32_t *to = v + c * 4 * W;
              expand<BITS>(x.x, to); expand<BITS>(x.y, to + W);
              expand<BITS>(x.z, to + 2 * W); expand<BITS>(x.w, to + 3 * W);
            }
            tmem_st32(tmem + (quad << 16) + L::TK + h * L::KCols + c0 / Each * 32, v);
          }
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(kready + 8 * h);
          // values: 16-byte chunks in turn, so that neither the reads nor the
          // writes of eight lanes share a bank
          bar_wait(pvdone + 8 * h, (it >> 1 & 1) ^ 1, alive, err);
          uint8_t *vt = sm + L::V + h * L::VTile;
#pragma unroll
          for (int i = 0; i < L::Chunks; i++) {
            const uint32_t n = i * 128 + tid, k = n / L::Chunks, c = n % L::Chunks;
            const uint4 x = *reinterpret_cast<const uint4 *>(vc + chunk(k, c));
            constexpr int Out = BITS == 8 ? 2 : 4;      // chunks of float16 it makes
            uint32_t v[4 * Out];
            if (BITS == 8) {
              expand<8>(x.x, v); expand<8>(x.y, v + 2); expand<8>(x.z, v + 4); expand<8>(x.w, v + 6);
            } else {
              expand<4>(x.x, v); expand<4>(x.y, v + 4);
              expand<4>(x.z, v + 8 % (4 * Out)); expand<4>(x.w, v + 12 % (4 * Out));
            }
            const uint32_t block = c * Out / 8, oc = c * Out % 8;
            uint8_t *row = vt + block * (kTileKeys * 128) + k * 128;
            const uint32_t turn = BITS == 8 ? block : block ^ ((k & 1) << 1);
#pragma unroll
            for (int s = 0; s < Out; s++) {
              uint4 y = make_uint4(v[4 * s], v[4 * s + 1], v[4 * s + 2], v[4 * s + 3]);
#pragma unroll
              for (int u = 0; u < Out; u++)
                if ((s ^ turn) == (uint32_t)u)
                  y = make_uint4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
              *reinterpret_cast<uint4 *>(row + (((oc + (s ^ turn)) ^ (k & 7)) << 4)) = y;
            }
          }
          fence_async();
          __syncwarp();
          if (lane == 0) {
            bar_arrive(vready + 8 * h);
            bar_arrive(empty + 8 * st);
          }
        }
      }
    } else {
      // ---- scores to weights, a thread per key; half the rows a group ----
      asm volatile("setmaxnreg.inc.sync.aligned.u32 168;\n");
      const uint32_t group = warp >> 2, quad = (warp & 3) * 32, mykey = quad + lane;
      const uint32_t tid = threadIdx.x, n0 = group * Half;
      const uint64_t used = a.nodes < 64 ? (1ull << a.nodes) - 1 : ~0ull;
      while (w.next(a)) {
        const uint32_t prefix = prefix_of(a, w.b), keys = keys_of(a, w.b);
        // the parameter words of this thread's key of a tile, found a tile ahead
        auto block_of = [&](uint32_t tile) {
          const uint32_t key = tile * kTileKeys + mykey;
          if (tile >= w.t1 || key >= keys) return kNone;
          return (uint32_t)__ldg(a.table + (uint64_t)w.b * a.max_blocks + key / a.pool.block_size);
        };
        auto words_of = [&](uint32_t tile, uint32_t block, uint32_t *kw, uint32_t *vw) {
          *kw = *vw = 0;
          if (block >= a.pool.num_blocks) return false;
          const uint32_t row =
              kv_row(a.pool, block, (tile * kTileKeys + mykey) % a.pool.block_size, w.head);
          *kw = __ldg(a.pool.param[0] + row);
          *vw = __ldg(a.pool.param[1] + row);
          return true;
        };
        uint32_t block1 = block_of(w.t0), kw1, vw1;

        // the queries of the item, float16, K-major
        {
          constexpr int Per = N * HD / kSoft, Lanes = HD / Per;      // values a thread takes
          const uint32_t n = tid / Lanes, part = tid % Lanes, row = w.row0 + n;
          const bool live = row < a.rows;
          const uint32_t node = live ? row / a.group : 0;
          const uint64_t out_row = (uint64_t)w.b * a.nodes + node;
          const uint32_t col = (w.head * a.group + (live ? row % a.group : 0));
          const uint4 *q = reinterpret_cast<const uint4 *>(
              (const __nv_bfloat16 *)a.q + out_row * a.q_stride + (uint64_t)col * HD + part * Per);
          uint4 raw[Per / 8];
          float top = 0.0f, sum = 0.0f;
#pragma unroll
          for (int i = 0; i < Per / 8; i++) raw[i] = live ? __ldg(q + i) : make_uint4(0, 0, 0, 0);
          auto value = [&](int i) {
            const uint4 &x = raw[i / 8];
            const uint32_t u = i % 8 / 2 == 0 ? x.x : i % 8 / 2 == 1 ? x.y : i % 8 / 2 == 2 ? x.z : x.w;
            return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
          };
#pragma unroll
          for (int i = 0; i < Per; i++) top = fmaxf(top, fabsf(value(i)));
#pragma unroll
          for (int o = Lanes / 2; o > 0; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          int up = 140 - (int)(__float_as_uint(top) >> 23);
          if (top == 0.0f || !(top < INFINITY)) up = 0;
          up = min(up, 126);
          const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
          for (int i = 0; i < Per; i += 8) {
            uint32_t u[4];
#pragma unroll
            for (int p = 0; p < 8; p += 2) {
              const float x = value(i + natural<BITS>(p)) * mul;
              const float y = value(i + natural<BITS>(p + 1)) * mul;
              sum += x + y;
              u[p / 2] = h2(__floats2half2_rn(x, y));
            }
            const uint32_t k = part * Per + i, c = k % 64 / 8;
            *reinterpret_cast<uint4 *>(sm + L::Q + k / 64 * (N * 128) + n * 128 +
                                       ((c ^ (n & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
#pragma unroll
          for (int o = Lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          if (part == 0) {
            // a factor is never zero: it would make NaN of a masked score
            ref[n] = make_float2(fmaxf(a.scale * __uint_as_float((uint32_t)(127 - up) << 23),
                                       1.17549435e-38f), kFar);
            qsum[n] = sum;
            masks[n] = live ? a.mask[out_row] & used : 0;
            offs[n] = live ? out_row * a.o_stride + (uint64_t)col * HD : ~0ull;
          }
        }
        fence_async();
        soft_sync();
        if (lane == 0) bar_arrive(qready);

        float l[Half], base[BITS == 4 ? Half : 1];
#pragma unroll
        for (int i = 0; i < Half; i++) l[i] = 0.0f;
        if (BITS == 4) {
#pragma unroll
          for (int i = 0; i < Half; i++) base[i] = 0.0f;
        }
        float vs = 1.0f;
        uint32_t vlimit = 0;
        bool have1 = words_of(w.t0, block1, &kw1, &vw1);
        block1 = block_of(w.t0 + 1);

        for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
          const uint32_t st = it & 1;
          const bool have = have1;
          const uint32_t kw = kw1, vw = vw1;
          have1 = words_of(tile + 1, block1, &kw1, &vw1);
          block1 = block_of(tile + 2);
          const float sk = scale_of<BITS>(kw), mk = middle_of(kw);
          const float sv = scale_of<BITS>(vw), mv = middle_of(vw);
          const uint32_t vbits = __float_as_uint(sv) < 0x7f800000u ? __float_as_uint(sv) : 0u;
          const uint32_t key = tile * kTileKeys + mykey;
          // tiles of prefix keys that all exist need no masks
          const bool whole = __all_sync(0xffffffffu, have && key < prefix);
          // whether row n sees this key
          auto seen = [&](uint32_t n) {
            return have && (key < prefix ? masks[n] != 0
                                         : key - prefix < 64 && (masks[n] >> (key - prefix) & 1));
          };
          // the scores of 32 rows from n: over the rows' references, in powers of two
          auto score = [&](uint32_t (&s)[32], uint32_t n) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              if (BITS == 4) {
                const float4 x = *reinterpret_cast<const float4 *>(qsum + n + i);
                q[0] = x.x; q[1] = x.y; q[2] = x.z; q[3] = x.w;
              }
#pragma unroll
              for (int j = 0; j < 4; j += 2) {
                const float4 r = *reinterpret_cast<const float4 *>(ref + n + i + j);
                float x = __uint_as_float(s[i + j]) * sk, y = __uint_as_float(s[i + j + 1]) * sk;
                if (BITS == 4) x = fmaf(mk, q[j], x), y = fmaf(mk, q[j + 1], y);
                s[i + j] = __float_as_uint(fmaf(x, r.x, r.y));
                s[i + j + 1] = __float_as_uint(fmaf(y, r.z, r.w));
              }
            }
            if (!whole) {
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (!seen(n + i)) s[i] = 0xff800000u;        // -inf
            }
          };
          bar_wait(qkdone + 8 * st, it >> 1 & 1, alive, err);
          fence_after();
          const uint32_t ts = tmem + (quad << 16) + L::TS + st * N + n0;
          uint32_t s[32];
          bool over = vbits >= vlimit && vbits != 0;
#pragma unroll
          for (int c = 0; c < Half / 32; c++) {
            tmem_ld32(ts + 32 * c, s);
            score(s, n0 + 32 * c);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; i++) top = fmaxf(top, __uint_as_float(s[i]));
            over |= top > 8.0f;
          }
          if (soft_any(over)) {
            // ---- new references: the maxima of the keys so far ----
#pragma unroll
            for (int c = 0; c < Half / 32; c++) {
              tmem_ld32(ts + 32 * c, s);
#pragma unroll
              for (int i = 0; i < 32; i++) {
                const uint32_t n = n0 + 32 * c + i;
                float x = __uint_as_float(s[i]) * sk;
                if (BITS == 4) x = fmaf(mk, qsum[n], x);
                x *= ref[n].x;
                if (!whole && !seen(n)) x = -INFINITY;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                if (lane == 0) warp_part[(warp & 3) * N + n] = x;
              }
            }
            if (tid == 0) *vote = 0;
            soft_sync();
            const uint32_t top_bits = __reduce_max_sync(0xffffffffu, vbits);
            if (group == 0 && lane == 0) atomicMax(vote, top_bits);
            soft_sync();
            float ratio = 1.0f;
            const uint32_t big = *vote;
            if (big >= vlimit && big != 0) {
              const uint32_t e = (big >> 23) + 1;           // scales below 2^(e - 127)
              vlimit = e << 23;
              const float next_vs = __uint_as_float((261u - e) << 23);   // to below 2^7
              ratio = next_vs / vs;
              vs = next_vs;
            }
            if (tid < N) {
              const float top = fmaxf(fmaxf(warp_part[tid], warp_part[N + tid]),
                                      fmaxf(warp_part[2 * N + tid], warp_part[3 * N + tid]));
              const float old = -ref[tid].y;                 // -kFar: no key met yet
              keep[tid] = top > old ? ex2(old - top) : 1.0f;
              if (top > old) ref[tid].y = -top;
            }
            soft_sync();
            // the sums, and the output so far once its last product is done
#pragma unroll
            for (int i = 0; i < Half; i++) {
              const float k = keep[n0 + i];
              l[i] *= k;
              if (BITS == 4) base[i % (BITS == 4 ? Half : 1)] *= k;
            }
            if (tile > w.t0) {
              bar_wait(pvdone + 8 * ((it - 1) & 1), (it - 1) >> 1 & 1, alive, err);
              fence_after();
              const uint32_t to = tmem + (quad << 16) + L::TO + n0;
#pragma unroll
              for (int c = 0; c < Half / 32; c++) {
                uint32_t o[32];
                tmem_ld32(to + 32 * c, o);
#pragma unroll
                for (int i = 0; i < 32; i++)
                  o[i] = __float_as_uint(__uint_as_float(o[i]) * (keep[n0 + 32 * c + i] * ratio));
                tmem_st32(to + 32 * c, o);
              }
              tmem_wait_st();
            }
            if (Half == 32) {
              tmem_ld32(ts, s);
              score(s, n0);
            }
          }
          // ---- the weights ----
          const float wv = sv * vs;
          if (L::PBufs == 2) bar_wait(pvdone + 8 * st, (it >> 1 & 1) ^ 1, alive, err);
          else if (it) bar_wait(pvdone + 8 * ((it - 1) & 1), (it - 1) >> 1 & 1, alive, err);
          uint8_t *pt = sm + L::P + (L::PBufs == 2 ? st * L::PTile : 0) + mykey * 128;
#pragma unroll
          for (int c = 0; c < Half / 32; c++) {
            if (Half > 32) {
              tmem_ld32(ts + 32 * c, s);
              score(s, n0 + 32 * c);
            }
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float e[2];
#pragma unroll
              for (int j = 0; j < 2; j++) {
                const int n = 32 * c + i + j;
                const float x = __uint_as_float(s[i + j]);
                e[j] = ex2(x);
                l[n] += e[j];
                // an unseen key's value may be NaN
                const bool in = whole || x != -INFINITY;
                if (BITS == 4 && in) base[n % (BITS == 4 ? Half : 1)] =
                    fmaf(e[j], mv, base[n % (BITS == 4 ? Half : 1)]);
                e[j] = in ? e[j] * wv : 0.0f;
              }
              p[i / 2] = h2(__floats2half2_rn(e[0], e[1]));
            }
            const uint32_t n = n0 + 32 * c;
            uint8_t *to = pt + n / 64 * (kTileKeys * 128);
#pragma unroll
            for (int j = 0; j < 4; j++)
              *reinterpret_cast<uint4 *>(to + (((n % 64 / 8 + j) ^ (mykey & 7)) << 4)) =
                  make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
          }
          fence_before();
          fence_async();
          __syncwarp();
          if (lane == 0) {
            bar_arrive(sfree + 8 * st);
            bar_arrive(pready + 8 * st);
          }
        }

        // ---- the end of the item: sums over the keys, and the output ----
        const bool part_of = !(w.t0 == 0 && w.t1 == w.tiles);
        const uint32_t slot = 2 * blockIdx.x + (w.t0 == 0 ? 1 : 0);
#pragma unroll
        for (int c = 0; c < Half / 32; c++) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; i++) v[i] = l[32 * c + i];
          warp_part[(warp & 3) * N + n0 + 32 * c + lane] = sums32(v);
        }
        soft_sync();
        if (tid < N) {
          const float sum = (warp_part[tid] + warp_part[N + tid]) +
                            (warp_part[2 * N + tid] + warp_part[3 * N + tid]);
          const bool empty = masks[tid] == 0 || sum == 0.0f;
          const float top = ref[tid].y == kFar ? -INFINITY : -ref[tid].y;
          const uint32_t row = w.row0 + tid;
          if (part_of) {
            a.part_ml[((uint64_t)slot * N + tid) * 2] = top;
            a.part_ml[((uint64_t)slot * N + tid) * 2 + 1] = sum;
          } else if (row < a.rows && a.lse) {
            a.lse[((uint64_t)w.b * a.nodes + row / a.group) * a.heads + w.head * a.group +
                  row % a.group] = empty ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
          }
          // what the output is multiplied by: 0 stands for a row without keys
          keep[tid] = part_of ? 1.0f : empty ? 0.0f : 1.0f / sum;
          qsum[tid] = 0.0f;
        }
        if (BITS == 4) {
          soft_sync();                       // the sums of the weights are read
#pragma unroll
          for (int c = 0; c < Half / 32; c++) {
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; i++) v[i] = base[(32 * c + i) % (BITS == 4 ? Half : 1)];
            warp_part[(warp & 3) * N + n0 + 32 * c + lane] = sums32(v);
          }
          soft_sync();
          if (tid < N)
            qsum[tid] = (warp_part[tid] + warp_part[N + tid]) +
                        (warp_part[2 * N + tid] + warp_part[3 * N + tid]);
        }
        soft_sync();
        bar_wait(pvdone + 8 * ((it - 1) & 1), (it - 1) >> 1 & 1, alive, err);
        fence_after();
        const float back = 1.0f / vs;
        const uint32_t d = natural<BITS>(mykey);       // the value this TMEM lane holds
#pragma unroll
        for (int c = 0; c < Half / 32; c++) {
          uint32_t o[32];
          tmem_ld32(tmem + (quad << 16) + L::TO + n0 + 32 * c, o);
          if (HD == 128 || quad < 64) {
#pragma unroll
            for (int i = 0; i < 32; i++) {
              const uint32_t n = n0 + 32 * c + i;
              const float v = fmaf(__uint_as_float(o[i]), back, qsum[n]), by = keep[n];
              if (part_of) {
                a.part_o[((uint64_t)slot * N + n) * HD + d] = v;
              } else if (offs[n] != ~0ull) {
                ((__nv_bfloat16 *)a.o)[offs[n] + d] =
                    __float2bfloat16_rn(by == 0.0f ? 0.0f : v * by);
              }
            }
          }
        }
        fence_before();
        soft_sync();                         // the rows are read: the next item may write them
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 13) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                             const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static bool tried = false;
  if (!tried) {
    tried = true;
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
    cudaGetLastError();
  }
  return fn;
}

// Keys of a copy: the longest run that every page is made of and a tile too.
uint32_t box_of(uint32_t block_size) {
  uint32_t n = 16;
  while (n < (uint32_t)kTileKeys && block_size % (2 * n) == 0) n *= 2;
  return n;
}

template <int HD, int BITS, int N>
cudaError_t start(TreeArgs &a, cudaStream_t st) {
  using L = Plan<HD, BITS, N>;
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(
        tree_umma_kernel<HD, BITS, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::Bytes);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  const uint32_t box = box_of(a.pool.block_size);
  const uint64_t rows = (uint64_t)a.pool.num_blocks * a.pool.kv_heads * a.pool.block_size;
  CUtensorMap map[2];
  for (int i = 0; i < 2; i++) {
    const cuuint64_t dims[2] = {L::RB, rows}, strides[1] = {L::RB};
    const cuuint32_t boxes[2] = {L::RB, box}, es[2] = {1, 1};
    const CUtensorMapSwizzle swizzle = L::RB == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                       : L::RB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                     : CU_TENSOR_MAP_SWIZZLE_32B;
    if (encode_fn()(&map[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a.pool.code[i], dims, strides, boxes,
                    es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  a.ctas = 148;
  a.tile = kTileKeys;
  a.item_cost = 4;
  int *err = wait_flag_device();
  if (!err) return cudaErrorMemoryAllocation;
  count_launches(1);
  return launch_pdl(tree_umma_kernel<HD, BITS, N>, dim3(a.ctas), dim3(kThreads), (size_t)L::Bytes,
                    st, a, map[0], map[1], box, err);
}

}  // namespace

uint32_t tree_umma_rows(const TreeArgs &a, bool bf16) {
  if (!bf16 || a.pool.head_dim > 128 || a.pool.block_size % 16 || a.rows <= 16 ||
      (uint64_t)a.pool.num_blocks * a.pool.kv_heads * a.pool.block_size > INT32_MAX ||
      !a.pool.num_blocks || (uint64_t)a.batch * a.nodes * a.heads >= kNone || !encode_fn())
    return 0;
  return a.pool.bits == 8 && a.rows > 64 ? 128 : 64;
}

cudaError_t tree_umma_start(TreeArgs &a, cudaStream_t st) {
  const bool h128 = a.pool.head_dim == 128;
  if (a.pool.bits == 4) return h128 ? start<128, 4, 64>(a, st) : start<64, 4, 64>(a, st);
  if (a.rows_at_once == 64) return h128 ? start<128, 8, 64>(a, st) : start<64, 8, 64>(a, st);
  return h128 ? start<128, 8, 128>(a, st) : start<64, 8, 128>(a, st);
}

}  // namespace nl
