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
// of the keys up to the last time one exceeded it by 2^8 (a vote of the 128
// threads per tile), and float16 has the room: scales are brought below 2^7.
//
// One CTA per SM, tiles of 128 keys, a warp group (four warps) per role:
//   N / 16 groups of score warps, 16 rows each, a thread per key: scores from
//               TMEM, weights to shared memory (the N x 128 operand with N
//               contiguous), sums of the weights in registers; at the end of
//               an item the output, a thread per value.  A group has its own
//               references and votes, so they do not wait for each other;
//   keys        codes to float16 in a TMEM stage, a thread per key, and the
//               keys' parameter words to shared memory;
//   values      codes to float16 in a shared-memory stage ([key][value], read
//               as V^T), a thread per key;
//   control     one warp for the TMA of the code tiles, one box per run of a
//               page; one that allocates TMEM and issues the MMAs of the scores;
//               one that issues those of the output (and one idle).  The two
//               run as whole warps of which one thread issues, so that the
//               descriptors are formed in uniform registers: from a single
//               thread's branch the issue of a tile took longer than its work.
// The registers of the launch are shared out anew among the roles.
//
// What bounds it: a tile takes about 3,000 cycles (131,071 keys, 16 nodes of 4
// heads, 8 bits: 102 us, 2.7 TB/s, 336 TF/s) with the tensor cores 18% busy,
// issue 67%, and shared memory -- codes in and out, values out and in again,
// weights, the rows' factors and references -- about 80%.  No role is the one:
// each is 2,000 to 2,300 cycles busy a tile at 5 to 8 cycles an instruction, and
// waits the rest of it for another.  Registers matter: the list of work in 64
// bits, which spilled, took 5% longer (now 32 rows in 8 bits spill some 100 bytes a
// thread, 64 of 128 values in 8 bits 4, the others none).  So does code: instructions that every CTA runs
// once are fetched as it does.  Measured and not taken: two streams
// of score warps on alternate tiles (32 rows, 4 bits: 64.3 us, not 63.2), the vote
// by a barrier that is waited for after the exponentials (15% slower), the scores'
// columns released before the weights (5%), deeper batches of loads in the
// conversions (1 to 5%).
//
// Every wait is bounded.  One that gives up sets the library's wait flag, and
// its thread then waits no more but runs on to the end: no barrier of the CTA
// is left short, the copies are waited for and TMEM is freed.

#include <cuda.h>

#define NL_TREE_KERNELS
#include "f32x2.cuh"
#include "tree_work.cuh"

namespace nl {
namespace {

constexpr int H = 16;                      // rows of a group of score warps
constexpr int kTileKeys = 128;
constexpr uint32_t kWaitTries = 1u << 22;
constexpr float kFar = 1.0e30f;            // a row that has met no key: -reference

template <int HD, int BITS, int N> struct Plan {
  static constexpr int Groups = N / H;
  static constexpr int Soft = 128 * Groups;                   // threads of the score warps
  static constexpr int Threads = Soft + 3 * 128;
  static constexpr int Regs = 65536 / Threads / 8 * 8;        // a thread, at launch
  static constexpr int RegsCtl = N == 32 ? 64 : 40;           // with 7 groups there are no more
  static constexpr int RegsSoft = (Regs * (Groups + 3) - 56 - 56 - RegsCtl) / Groups / 8 * 8;
  static constexpr int RB = HD * BITS / 8;
  static constexpr int Chunks = RB / 16;
  static constexpr int Codes = kTileKeys * RB;               // one side's codes of a tile
  static constexpr int Stages = 3;
  static constexpr int VTile = HD * kTileKeys * 2;            // values as float16
  static constexpr int PTile = 128 * kTileKeys;               // weights, rows of 128 bytes
  static constexpr int QTile = N * HD * 2;
  // offsets from a 1024-byte boundary
  static constexpr int V = Stages * 2 * Codes, P = V + 2 * VTile, Q = P + 2 * PTile;
  static constexpr int Factor = Q + QTile;                    // floats
  static constexpr int Sum = Factor + N * 4;
  static constexpr int Ref = Sum + N * 4;
  static constexpr int Keep = Ref + N * 4;
  static constexpr int Masks = Keep + N * 4;
  static constexpr int Offs = Masks + N * 8;                  // output offsets
  static constexpr int Warp = Offs + N * 8;                   // [4][N]
  static constexpr int Base = Warp + 4 * N * 4;               // [4][N] (4 bits)
  static constexpr int Words = Base + (BITS == 4 ? 4 * N * 4 : 0);   // [4][128] uint4
  static constexpr int Scale = Words + 4 * kTileKeys * 16;    // [4][N]
  static constexpr int Lim = Scale + 4 * N * 4;
  static constexpr int Bars = Lim + N * 4;
  static constexpr int Used = Bars + 256 + 1024;
  static constexpr int Bytes = Used > 120 * 1024 ? Used : 120 * 1024;   // one CTA per SM (TMEM)
  // TMEM columns: two stages of keys and of scores, the output
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
// Without a suspend-time hint: with one a waiter may sleep on, and a tile
// passes through ten waits.
__device__ __forceinline__ void bar_wait(uint32_t b, uint32_t parity, bool &alive, int *err) {
  if (!alive) return;
#pragma unroll 1
  for (uint32_t i = 0; i < kWaitTries; i++) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(b), "r"(parity) : "memory");
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
template <int THREADS> __device__ __forceinline__ void soft_sync() {
  asm volatile("bar.sync 1, %0;\n" ::"n"(THREADS) : "memory");
}
// The same for the 128 threads of one group, and whether any of them says so.
__device__ __forceinline__ void group_sync(uint32_t group) {
  asm volatile("bar.sync %0, 128;\n" ::"r"(2 + group) : "memory");
}
__device__ __forceinline__ bool group_any(uint32_t group, bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 128, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r) : "r"((uint32_t)v), "r"(2 + group) : "memory");
  return r != 0;
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ float tmem_ld1(uint32_t at) {
  uint32_t v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n"
               "tcgen05.wait::ld.sync.aligned;\n" : "=r"(v) : "r"(at) : "memory");
  return __uint_as_float(v);
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};\n" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15])
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
// Issued by the thread whose ME is set; every lane comes here with the same
// operands.
__device__ __forceinline__ uint32_t elect() {
  uint32_t me;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(me));
  return me;
}
__device__ __forceinline__ void mma_ts(uint32_t me, uint32_t d, uint32_t a, uint64_t b,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(me));
}
__device__ __forceinline__ void mma_ss(uint32_t me, uint32_t d, uint64_t a, uint64_t b,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(me));
}
__device__ __forceinline__ void mma_commit(uint32_t me, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
          bar), "r"(me) : "memory");
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

// The largest, or the sum, over a warp's lanes of each of 16 values: lanes i and
// i + 16 get that of v[i].
template <bool SUM> __device__ __forceinline__ float across(uint32_t (&v)[H]) {
  const uint32_t lane = threadIdx.x & 31;
  auto join = [](float x, float y) { return SUM ? x + y : fmaxf(x, y); };
#pragma unroll
  for (int o = H / 2; o > 0; o >>= 1) {
    const bool high = lane & o;
#pragma unroll
    for (int i = 0; i < o; i++) {
      const uint32_t give = high ? v[i] : v[i + o], have = high ? v[i + o] : v[i];
      v[i] = __float_as_uint(join(__uint_as_float(have),
                                  __uint_as_float(__shfl_xor_sync(0xffffffffu, give, o))));
    }
  }
  const float r = __uint_as_float(v[0]);
  return join(r, __shfl_xor_sync(0xffffffffu, r, 16));
}

// The walk over the parts of items that a CTA has, the same in every role.  A part
// is taken in runs of at most kTreeRunUmma tiles, each joined with the state that the
// one before (RESUMED) left in the workspace.
struct Walk {
  uint32_t at, end, before;
  uint32_t b, items;
  uint32_t head, row0, t0, t1, tiles;
  bool any, resumed, more;
  bool from0;                    // the part begins the item
  __device__ __forceinline__ bool begin(const TreeArgs &a) {
    const List list = list_of(a);
    if (blockIdx.x >= list.workers) return false;
    at = share(list.total, list.workers, blockIdx.x);
    end = share(list.total, list.workers, blockIdx.x + 1);
    items = a.pool.kv_heads * a.row_tiles;
    locate(a, at, &b, &before);
    any = false;
    return true;
  }
  __device__ __forceinline__ bool next(const TreeArgs &a) {
    while (at < end) {
      tiles = tiles_of(a, b);
      const uint32_t cost = tiles + a.item_cost;
      if (at >= before + cost * items) {
        before += cost * items;
        b++;
        continue;
      }
      const uint32_t item = (at - before) / cost, c0 = (at - before) % cost;
      const uint32_t all = end - at < cost - c0 ? c0 + (end - at) : cost;
      const uint32_t c1 = min(all, max(c0, a.item_cost) + kTreeRunUmma);
      resumed = any && c0 != 0;
      more = c1 < all;
      at += c1 - c0;
      any = true;
      if (c1 <= a.item_cost) continue;
      t0 = c0 > a.item_cost ? c0 - a.item_cost : 0;
      t1 = c1 - a.item_cost;
      if (!resumed) from0 = t0 == 0;
      head = item / a.row_tiles;
      row0 = item % a.row_tiles * a.rows_at_once;
      return true;
    }
    return false;
  }
};

template <int HD, int BITS, int N>
__global__ void __launch_bounds__(Plan<HD, BITS, N>::Threads, 1)
tree_umma_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, uint32_t box, int *err) {
  using L = Plan<HD, BITS, N>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                            ~(uintptr_t)1023);
  const uint32_t s0 = su32(sm);
  float *factor = reinterpret_cast<float *>(sm + L::Factor);  // of a row's scores
  float *qsum = reinterpret_cast<float *>(sm + L::Sum);       // the sum of its query
  float *ref = reinterpret_cast<float *>(sm + L::Ref);        // less its reference
  float *keep = reinterpret_cast<float *>(sm + L::Keep);      // what a new one leaves of the sums
  uint64_t *masks = reinterpret_cast<uint64_t *>(sm + L::Masks);
  uint64_t *offs = reinterpret_cast<uint64_t *>(sm + L::Offs);
  float *warp_part = reinterpret_cast<float *>(sm + L::Warp);
  float *warp_base = reinterpret_cast<float *>(sm + L::Base);
  float *warp_scale = reinterpret_cast<float *>(sm + L::Scale);   // largest scale a row sees
  uint32_t *lim = reinterpret_cast<uint32_t *>(sm + L::Lim);      // of a row so far, if apart
  const uint32_t bars = s0 + L::Bars;
  const uint32_t full = bars, empty = bars + 24, kready = bars + 48, qkdone = bars + 80,
                 sfree = bars + 96, vready = bars + 112, pready = bars + 128, pvdone = bars + 144,
                 qready = bars + 160;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + L::Bars + 176);
  uint32_t *votes = tmem_slot + 1;           // the largest scale of a group's tile
  uint4 *words = reinterpret_cast<uint4 *>(sm + L::Words);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // 0: the score groups; then keys, values, control
  const uint32_t role = warp < 4 * L::Groups ? 0 : warp / 4 - L::Groups + 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::Stages; i++) {
      bar_init(full + 8 * i, 1);
      bar_init(empty + 8 * i, 8);
    }
    for (int i = 0; i < 2; i++) {
      bar_init(kready + 8 * i, 4);
      bar_init(qkdone + 8 * i, 1);
      bar_init(sfree + 8 * i, 4 * L::Groups);
      bar_init(vready + 8 * i, 4);
      bar_init(pready + 8 * i, 4 * L::Groups);
      bar_init(pvdone + 8 * i, 1);
    }
    bar_init(qready, 4 * L::Groups);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (role == 3 && warp % 4 == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     su32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();                 // after the wait: the join reads the lengths before its own

  bool alive = true;
  Walk w;
  if (w.begin(a)) {
    uint32_t it = 0;                         // tiles so far, over all items
    if (role == 3) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(L::RegsCtl));
      if (warp % 4 == 0) {
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
      } else if (warp % 4 == 1) {
        // ---- the score products ----
        const uint32_t me = elect();
        uint32_t item = 0;
        while (w.next(a)) {
          bar_wait(qready, item & 1, alive, err);
          item++;
          for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
            const uint32_t st = it & 1, ph = it >> 1 & 1;
            bar_wait(kready + 8 * st, ph, alive, err);
            bar_wait(sfree + 8 * st, ph ^ 1, alive, err);
            fence_after();
            const uint64_t q = smem_desc(s0 + L::Q, 16);
#pragma unroll
            for (int k = 0; k < HD / 16; k++)
              mma_ts(me, tmem + L::TS + st * N, tmem + L::TK + st * L::KCols + 8 * k,
                     q + (k / 4 * (N * 128) + k % 4 * 32) / 16, instr_desc<N, false>(),
                     k ? 1u : 0u);
            mma_commit(me, qkdone + 8 * st);
          }
        }
      } else if (warp % 4 == 2) {
        // ---- the output products ----
        const uint32_t me = elect();
        while (w.next(a)) {
          for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
            const uint32_t st = it & 1, ph = it >> 1 & 1;
            bar_wait(vready + 8 * st, ph, alive, err);
            bar_wait(pready + 8 * st, ph, alive, err);
            fence_after();
            // 16 keys on is 2048 bytes on: 128 in a descriptor's address field
            const uint64_t v = smem_desc(s0 + L::V + st * L::VTile,
                                         HD == 128 ? kTileKeys * 128 : 0);
            const uint64_t p = smem_desc(s0 + L::P + st * L::PTile, 16);
#pragma unroll
            for (int k = 0; k < kTileKeys / 16; k++)
              mma_ss(me, tmem + L::TO, v + 128 * k, p + 128 * k, instr_desc<N, true>(),
                     k == 0 && tile == w.t0 ? 0u : 1u);
            mma_commit(me, pvdone + 8 * st);
          }
        }
      }
    } else if (role) {
      // byte of chunk c of a key's row, swizzled by the copy over the row's bytes
      const uint32_t quad = (warp & 3) * 32, key = quad + lane;
      const uint32_t x = L::RB == 128 ? key & 7 : L::RB == 64 ? key >> 1 & 3 : key >> 2 & 1;
      const uint32_t from = key * L::RB + (x << 4);
      if (role == 1) {
        // ---- keys, to TMEM.  (Codes left 1024 too large, with that much of the
        // query's sum taken off the scores, would halve the work here, but the
        // cut sums of the tensor core then cost the scores 5 bits.) ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        while (w.next(a)) {
          const uint32_t keys = keys_of(a, w.b);
          // the parameter words of this thread's key, and whether there is one:
          // the block is looked up two tiles ahead, the words one
          auto page_of = [&](uint32_t token) {
            return a.block_shift < 32 ? token >> a.block_shift : token / a.pool.block_size;
          };
          auto block_of = [&](uint32_t tile) {
            const uint32_t token = tile * kTileKeys + key;
            if (tile >= w.t1 || token >= keys) return kNone;
            return (uint32_t)__ldg(a.table + (uint64_t)w.b * a.max_blocks + page_of(token));
          };
          auto words_of = [&](uint32_t tile, uint32_t block) {
            uint4 word = make_uint4(0, 0, 0, 0);
            if (block < a.pool.num_blocks) {
              const uint32_t token = tile * kTileKeys + key;
              const uint32_t row =
                  kv_row(a.pool, block, token - page_of(token) * a.pool.block_size, w.head);
              word.x = __ldg(a.pool.param[0] + row);
              word.y = __ldg(a.pool.param[1] + row);
              word.z = 1;
            }
            return word;
          };
          uint4 next = words_of(w.t0, block_of(w.t0));
          uint32_t block = block_of(w.t0 + 1);
          for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
            const uint32_t st = it % L::Stages, h = it & 1;
            const uint4 word = next;
            next = words_of(tile + 1, block);
            block = block_of(tile + 2);
            const uint8_t *kc = sm + st * (2 * L::Codes);
            bar_wait(full + 8 * st, it / L::Stages & 1, alive, err);
            bar_wait(qkdone + 8 * h, (it >> 1 & 1) ^ 1, alive, err);
            fence_after();
            constexpr int Each = BITS == 8 ? 2 : 1;       // chunks that make 16 TMEM columns
            constexpr int W = BITS == 8 ? 2 : 4;          // columns a word makes
#pragma unroll
            for (int c0 = 0; c0 < L::Chunks; c0 += Each) {
              uint32_t v[16];
#pragma unroll
              for (int c = 0; c < Each; c++) {
                const uint4 y = *reinterpret_cast<const uint4 *>(kc + (from ^ ((c0 + c) << 4)));
                uint32_t *to = v + c * 4 * W;
                expand<BITS>(y.x, to); expand<BITS>(y.y, to + W);
                expand<BITS>(y.z, to + 2 * W); expand<BITS>(y.w, to + 3 * W);
              }
              tmem_st16(tmem + (quad << 16) + L::TK + h * L::KCols + c0 / Each * 16, v);
            }
            // four tiles of them: the product just waited for was issued after every
            // score warp was past the tile before its stage's last
            words[(it & 3) * kTileKeys + key] = word;
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) {
              bar_arrive(kready + 8 * h);
              bar_arrive(empty + 8 * st);
            }
          }
        }
      } else {
        // ---- values: the signed codes, to shared memory; eight lanes' rows are
        // swizzled apart, so neither reads nor writes share a bank ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        const uint32_t row = key * 128 + ((key & 7) << 4);
        while (w.next(a)) {
          for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
            const uint32_t st = it % L::Stages, h = it & 1;
            const uint8_t *vc = sm + st * (2 * L::Codes) + L::Codes;
            uint8_t *vt = sm + L::V + h * L::VTile;
            bar_wait(full + 8 * st, it / L::Stages & 1, alive, err);
            bar_wait(pvdone + 8 * h, (it >> 1 & 1) ^ 1, alive, err);
#pragma unroll 2
            for (int c = 0; c < L::Chunks; c++) {
              const uint4 y = *reinterpret_cast<const uint4 *>(vc + (from ^ (c << 4)));
              constexpr int Out = BITS == 8 ? 2 : 4;      // chunks of float16 it makes
              const uint32_t in[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
              for (int s = 0; s < Out; s++) {
                uint32_t v[4];
                if (BITS == 8) {
                  expand<8>(in[2 * s % 4], v);
                  expand<8>(in[(2 * s + 1) % 4], v + 2);
                } else {
                  expand<4>(in[s], v);
                }
                const int oc = c * Out + s;
                *reinterpret_cast<uint4 *>(vt + oc / 8 * (kTileKeys * 128) +
                                           (row ^ ((oc & 7) << 4))) =
                    make_uint4(v[0], v[1], v[2], v[3]);
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
      }
    } else {
      // ---- scores to weights, a thread per key; 16 rows a group ----
      if constexpr (L::RegsSoft >= L::Regs)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(L::RegsSoft));
      const uint32_t group = warp >> 2, quad = (warp & 3) * 32, mykey = quad + lane;
      const uint32_t tid = threadIdx.x;
      const uint32_t n0 = group * H;         // its first row
      uint32_t *vote = votes + group;
      const uint64_t used = a.nodes < 64 ? (1ull << a.nodes) - 1 : ~0ull;
      while (w.next(a)) {
        const uint32_t prefix = prefix_of(a, w.b);
        // the queries of the item, float16, K-major
        {
          constexpr int Per = N * HD / L::Soft, Lanes = HD / Per;      // values a thread takes
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
            const uint32_t w2 = i % 8 / 2;
            const uint32_t u = w2 == 0 ? x.x : w2 == 1 ? x.y : w2 == 2 ? x.z : x.w;
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
            factor[n] = fmaxf(a.scale * __uint_as_float((uint32_t)(127 - up) << 23),
                              1.17549435e-38f);
            ref[n] = kFar;
            qsum[n] = sum;
            masks[n] = live ? a.mask[out_row] & used : 0;
            offs[n] = live ? out_row * a.o_stride + (uint64_t)col * HD : ~0ull;
          }
        }
        fence_async();
        soft_sync<L::Soft>();
        if (lane == 0) bar_arrive(qready);

        constexpr int NB = BITS == 4 ? H / 2 : 1;
        Pair l[H / 2], base[NB];
#pragma unroll
        for (int i = 0; i < H / 2; i++) l[i] = base[i % NB] = 0;
        float vs = 1.0f;
        uint32_t vlimit = kTreeNone;
        // Rows see different nodes, so there a row has a limit of its own, and where
        // the limits differ (VLIMIT is kTreeOwn) its reference is moved by as many
        // powers of two: a node that a row does not see costs its weights no bits.

        for (uint32_t tile = w.t0; tile < w.t1; tile++, it++) {
          const uint32_t st = it & 1, ph = it >> 1 & 1;
          // (the key warps' words came before the barrier that the product waited for)
          bar_wait(qkdone + 8 * st, ph, alive, err);
          fence_after();
          const uint4 word = words[(it & 3) * kTileKeys + mykey];
          const uint32_t kw = word.x, vw = word.y;
          const bool have = word.z != 0;
          const float sk = scale_of<BITS>(kw);
          const float mk = middle_of(kw);
          const Pair sk2 = pair(sk, sk), mk2 = pair(mk, mk);
          const float sv = scale_of<BITS>(vw);
          // (a value that is not finite reaches the output by its weight alone)
          const float mid = BITS == 4 ? middle_of(vw) : 0.0f;
          const bool finite = fabsf(mid) < INFINITY;
          const float mv = finite ? mid : 0.0f;
          const uint32_t vbits = __float_as_uint(sv) < 0x7f800000u ? __float_as_uint(sv) : 0u;
          const uint32_t key = tile * kTileKeys + mykey;
          // tiles of prefix keys that all exist need no masks
          const bool whole = __all_sync(0xffffffffu, have && key < prefix);
          const bool nodes_here = (tile + 1) * kTileKeys > prefix;
          auto sees = [&](int i) {
            const uint64_t m = masks[n0 + i];
            const uint32_t node = key - prefix;
            return have && (key < prefix ? m != 0 : node < 64 && (m >> node & 1));
          };
          // the scores of the group's rows on this key, in powers of two: over the
          // rows' references, or as they are
          auto score = [&](uint32_t (&s)[H], bool over_ref) {
            const uint32_t n = n0;
#pragma unroll
            for (int i = 0; i < H; i += 4) {
              float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (BITS == 4) q = *reinterpret_cast<const float4 *>(qsum + n + i);
              const float4 f = *reinterpret_cast<const float4 *>(factor + n + i);
              float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (over_ref) r = *reinterpret_cast<const float4 *>(ref + n + i);
#pragma unroll
              for (int j = 0; j < 4; j += 2) {
                Pair x = pair(__uint_as_float(s[i + j]), __uint_as_float(s[i + j + 1]));
                x = mul2(x, sk2);
                if (BITS == 4) x = fma2(mk2, j ? pair(q.z, q.w) : pair(q.x, q.y), x);
                x = fma2(x, j ? pair(f.z, f.w) : pair(f.x, f.y),
                         j ? pair(r.z, r.w) : pair(r.x, r.y));
                const float2 y = unpair(x);
                s[i + j] = __float_as_uint(y.x);
                s[i + j + 1] = __float_as_uint(y.y);
              }
            }
            if (!whole) {
#pragma unroll
              for (int i = 0; i < H; i++)
                if (!sees(i)) s[i] = 0xff800000u;          // -inf
            }
          };
          const uint32_t ts = tmem + (quad << 16) + L::TS + st * N + n0;
          uint32_t s[H];
          for (bool again = false;; again = true) {
            tmem_ld16(ts, s);
            score(s, true);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < H; i++) top = fmaxf(top, __uint_as_float(s[i]));
            const bool over = top > 8.0f || vbits >= vlimit;
            if (again || !group_any(group, over)) break;
            // ---- new references: the maxima of the keys so far ----
            const bool apart = vlimit == kTreeOwn;
            const uint32_t before = vlimit == kTreeNone ? 0 : 261u - (__float_as_uint(vs) >> 23);
            tmem_ld16(ts, s);
            score(s, false);
            const float mine = across<false>(s);
            if (lane < H) warp_part[(warp & 3) * N + n0 + lane] = mine;
            uint32_t *low_vote = votes + 4 + group, *met = votes + 8 + group;
            if (quad == 0 && lane == 0) *vote = before << 23, *low_vote = ~0u, *met = 0;
            group_sync(group);
            const uint32_t high = __reduce_max_sync(0xffffffffu, vbits);
            if (lane == 0 && high != 0) atomicMax(vote, limit_of(high) << 23);
            bool rows = false;                 // limits looked at row by row
            if (nodes_here) {
              const uint32_t low = __reduce_min_sync(0xffffffffu, vbits ? limit_of(vbits) : ~0u);
              if (lane == 0) atomicMin(low_vote, low);
              if (vbits != 0 && key < prefix) *met = 1;
              group_sync(group);
              rows = apart ||
                     rows_apart(before, *low_vote, *vote >> 23, *met || tile + 1 == w.t1);
              if (rows) {
                // (not unrolled: the code of all sixteen rows here, run or not, made
                // every call 2 to 7% slower)
#pragma unroll 1
                for (int i = 0; i < H; i++) {
                  const uint32_t most = __reduce_max_sync(0xffffffffu, sees(i) ? vbits : 0u);
                  if (lane == 0) warp_scale[(warp & 3) * N + n0 + i] = __uint_as_float(most);
                }
                group_sync(group);
              }
            }
            if (mykey < H) {
              const uint32_t n = n0 + mykey;
              const float *p = warp_part + n;
              const float most = fmaxf(fmaxf(p[0], p[N]), fmaxf(p[2 * N], p[3 * N]));
              int was = 0, now = 0;                          // powers of two of the reference
              if (rows) {
                const float *z = warp_scale + n;
                const float scale = fmaxf(fmaxf(z[0], z[N]), fmaxf(z[2 * N], z[3 * N]));
                const uint32_t had = apart ? lim[n] : before;
                const uint32_t own =
                    max(had, scale > 0.0f ? limit_of(__float_as_uint(scale)) : 0u);
                const uint32_t e = common_limit(before, __reduce_min_sync(0xffffu, own ? own : ~0u),
                                                __reduce_max_sync(0xffffu, own));
                const bool differ = __any_sync(0xffffu, own != e);
                was = apart_by(before, had);
                now = apart_by(e, own);
                lim[n] = own;
                if (mykey == 0) *vote = e << 23 | (differ ? 1u : 0u);
              }
              // (kFar: no key met yet)
              const float old = ref[n] == kFar ? -kFar : (float)was - ref[n];
              keep[n] = (most > old ? ex2(old - most) : 1.0f) *
                        __uint_as_float((uint32_t)(127 + now - was) << 23);
              if (most > old) ref[n] = (float)now - most;
              else if (ref[n] != kFar) ref[n] = (float)now - old;
            }
            group_sync(group);
            float ratio = 1.0f;
            const uint32_t e = *vote >> 23;                  // scales below 2^(e - 127)
            vlimit = *vote & 1u ? kTreeOwn : e ? e << 23 : kTreeNone;
            if (e != before) {
              const float next_vs = __uint_as_float((261u - e) << 23);   // to below 2^7
              ratio = next_vs / vs;
              vs = next_vs;
            }
            // the sums, and the output so far once its last product is done
#pragma unroll
            for (int i = 0; i < H / 2; i++) {
              const float2 k = *reinterpret_cast<const float2 *>(keep + n0 + 2 * i);
              l[i] = mul2(l[i], pair(k.x, k.y));
              if (BITS == 4) base[i % NB] = mul2(base[i % NB], pair(k.x, k.y));
            }
            if (tile > w.t0) {
              bar_wait(pvdone + 8 * (st ^ 1), (it - 1) >> 1 & 1, alive, err);
              fence_after();
              const uint32_t to = tmem + (quad << 16) + L::TO + n0;
              tmem_ld16(to, s);
#pragma unroll
              for (int i = 0; i < H; i++)
                s[i] = __float_as_uint(__uint_as_float(s[i]) * (keep[n0 + i] * ratio));
              tmem_st16(to, s);
              tmem_wait_st();
            }
          }
          // ---- the weights ----
          const float wv = sv * vs;
          // an unseen key's value may be NaN
          const bool odd = !(fabsf(wv) < INFINITY && finite);
          const Pair wv2 = pair(wv, wv), mv2 = pair(mv, mv);
          bar_wait(pvdone + 8 * st, ph ^ 1, alive, err);       // the buffer's last reader
          uint8_t *pt = sm + L::P + st * L::PTile + mykey * 128;
          uint32_t p[H / 2];
#pragma unroll
          for (int i = 0; i < H / 2; i++) {
            const Pair e = pair(ex2(__uint_as_float(s[2 * i])), ex2(__uint_as_float(s[2 * i + 1])));
            l[i] = add2(l[i], e);
            const float2 y = unpair(mul2(e, wv2));
            if (BITS == 4) base[i % NB] = fma2(e, mv2, base[i % NB]);
            p[i] = h2(__floats2half2_rn(y.x, y.y));
          }
          if (odd) {
            // this key's value is NaN: to the rows that see it, and to no other
#pragma unroll
            for (int i = 0; i < H / 2; i++) {
              const bool in0 = s[2 * i] != 0xff800000u, in1 = s[2 * i + 1] != 0xff800000u;
              p[i] = (in0 ? 0x7e00u : 0u) | (in1 ? 0x7e000000u : 0u);
            }
          }
#pragma unroll
          for (int j = 0; j < H / 8; j++)
            *reinterpret_cast<uint4 *>(pt + (((n0 / 8 + j) ^ (mykey & 7)) << 4)) =
                make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
          fence_before();
          fence_async();
          __syncwarp();
          if (lane == 0) {
            bar_arrive(sfree + 8 * st);
            bar_arrive(pready + 8 * st);
          }
        }

        // ---- the end of the item: sums over the keys, and the output ----
        const bool part_of = w.more || !(w.from0 && w.t1 == w.tiles);
        const uint32_t slot = 2 * blockIdx.x + (w.from0 ? 1 : 0);
        {
          uint32_t v[H];
#pragma unroll
          for (int i = 0; i < H / 2; i++) {
            const float2 y = unpair(l[i]);
            v[2 * i] = __float_as_uint(y.x);
            v[2 * i + 1] = __float_as_uint(y.y);
          }
          const float sum = across<true>(v);
          if (lane < H) warp_part[(warp & 3) * N + n0 + lane] = sum;
          if (BITS == 4) {
#pragma unroll
            for (int i = 0; i < H / 2; i++) {
              const float2 y = unpair(base[i % NB]);
              v[2 * i] = __float_as_uint(y.x);
              v[2 * i + 1] = __float_as_uint(y.y);
            }
            const float mid = across<true>(v);
            if (lane < H) warp_base[(warp & 3) * N + n0 + lane] = mid;
          }
        }
        group_sync(group);
        if (mykey < H) {
          const uint32_t n = n0 + mykey, row = w.row0 + n;
          const float *p = warp_part + n, *q = warp_base + n;
          float sum = (p[0] + p[N]) + (p[2 * N] + p[3 * N]);
          float top = ref[n] == kFar ? -INFINITY : -ref[n];
          float *ml = a.part_ml + ((uint64_t)slot * N + n) * 2;
          // what this run and those before it weigh (one of NaN may have no maximum)
          float now = 1.0f, old = 0.0f;
          if (w.resumed) {
            const float x = ml[0], y = ml[1], both = fmaxf(top, x);
            now = top == both ? 1.0f : ex2(top - both);
            old = x == both ? 1.0f : ex2(x - both);
            sum = now * sum + old * y;
            top = both;
          }
          const bool empty = masks[n] == 0 || sum == 0.0f;
          if (part_of) {
            ml[0] = top;
            ml[1] = sum;
          } else if (row < a.rows && a.lse) {
            a.lse[((uint64_t)w.b * a.nodes + row / a.group) * a.heads + w.head * a.group +
                  row % a.group] = empty ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
          }
          // what the output is multiplied by, 0 for a row without keys, and what
          // the offsets add to it
          float by = part_of ? 1.0f : empty ? 0.0f : 1.0f / sum;
          factor[n] = by * old;
          by *= now;
          keep[n] = by / vs;
          qsum[n] = BITS == 4 && by != 0.0f ? by * ((q[0] + q[N]) + (q[2 * N] + q[3 * N])) : 0.0f;
        }
        group_sync(group);
        bar_wait(pvdone + 8 * (it - 1 & 1), (it - 1) >> 1 & 1, alive, err);
        fence_after();
        const uint32_t d = natural<BITS>(mykey);       // the value this TMEM lane holds
        if (w.resumed) {
          float *part = a.part_o + ((uint64_t)slot * N + n0) * HD + d;
#pragma unroll 1
          for (int i = 0; i < H; i++) {
            const uint32_t n = n0 + i;
            const float x = tmem_ld1(tmem + (quad << 16) + L::TO + n), k = keep[n], f = factor[n];
            if (HD == 128 || quad < 64) {
              float v = k == 0.0f ? 0.0f : fmaf(x, k, qsum[n]);
              if (f != 0.0f) v = fmaf(part[i * HD], f, v);
              const uint64_t at = offs[n];
              if (part_of) part[i * HD] = v;
              else if (at != ~0ull) ((__nv_bfloat16 *)a.o)[at + d] = __float2bfloat16_rn(v);
            }
          }
        } else {
          uint32_t o[H];
          tmem_ld16(tmem + (quad << 16) + L::TO + n0, o);
          if (HD == 128 || quad < 64) {
            float *part = a.part_o + ((uint64_t)slot * N + n0) * HD + d;
#pragma unroll
            for (int i = 0; i < H; i++) {
              const uint32_t n = n0 + i;
              const float k = keep[n];
              const float v = k == 0.0f ? 0.0f : fmaf(__uint_as_float(o[i]), k, qsum[n]);
              const uint64_t at = offs[n];
              if (part_of) part[i * HD] = v;
              else if (at != ~0ull) ((__nv_bfloat16 *)a.o)[at + d] = __float2bfloat16_rn(v);
            }
          }
        }
        fence_before();
        soft_sync<L::Soft>();              // the rows are read: the next item may write them
      }
    }
  }
  fence_before();
  __syncthreads();
  if (role == 3 && warp % 4 == 1) {
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
  // (With 5, 7, 10, us: 16 ragged sequences to 8,192 keys, 32 rows, 4 bits 64.7, 62.7,
  // 61.9, with 3 88; 4 ragged to 16,384, 256 rows 123, 100, 103, with 3 169; 8 of 2,000,
  // 64 rows 33.6, 35.1, 36.4; 32 of 500 44.4, 42.7, 42.3.)
  a.item_cost = 7;
  int *err = wait_flag_device();
  if (!err) return cudaErrorMemoryAllocation;
  count_launches(1);
  return launch_pdl(tree_umma_kernel<HD, BITS, N>, dim3(a.ctas), dim3(L::Threads), (size_t)L::Bytes,
                    st, a, map[0], map[1], box, err);
}

}  // namespace

// The rows of an item of this form, 0 where the other one serves.  It takes
// about 3,000 cycles a tile whatever the rows, the other one a time that grows
// with them and with the head size, so this one is for many (us, 4 sequences of
// 32,768 keys, 8 key heads, 8 bits / 4 bits):
//   rows            8        16       20        32         48        64
//   128 values
//     this form   82/85    81/86    82/ 85    82/ 85     97/111    99/112
//     the other   57/59    69/73    97/103   100/106    174/190   177/194
//   64 values
//     this form   91/102   91/102   91/102    91/103     92/102    93/105
//     the other   40/40    47/50    63/ 71    65/ 73    115/128   118/131
// More than 16 rows of 128 values, then, or 32 of 64.  Few and short sequences
// would have it otherwise (8 bits, 128 values, 8 key heads; this form / the other):
//   keys                     500          1,000        2,000        4,000
//   1 sequence, 24 rows   16.3/14.4    17.9/15.9    17.0/18.5    18.8/24.6
//   64 rows               21.8/21.8    23.3/25.4    21.4/31.7    23.0/39.3
//   8 sequences, 24 rows  19.9/22.6    24.1/24.0    27.8/30.3    37.1/40.8
//   64 rows               22.6/32.3    32.0/38.3    35.6/49.4    46.2/71.3
// but the lengths are on the device, and the rule goes by what the host knows: a
// single sequence of up to 1,000 keys and 17 to 32 rows pays 13 to 25% for it.  (256 values have no room
// in TMEM and shared memory; a run of a page that is no multiple of 16 keys has
// no copy of whole boxes; float32 needs its sums out of the tensor core often.)
uint32_t tree_umma_rows(const TreeArgs &a, bool bf16) {
  if (!bf16 || a.pool.head_dim > 128 || a.pool.block_size % 16 ||
      (uint64_t)a.rows * a.pool.head_dim <= 2048 ||
      (uint64_t)a.pool.num_blocks * a.pool.kv_heads * a.pool.block_size > INT32_MAX ||
      !a.pool.num_blocks || (uint64_t)a.batch * a.nodes * a.heads >= kNone || !encode_fn())
    return 0;
  return a.rows > 32 ? 64 : 32;
}

cudaError_t tree_umma_start(TreeArgs &a, cudaStream_t st) {
  const bool h128 = a.pool.head_dim == 128;
  const bool few = a.rows_at_once == 32;
  if (a.pool.bits == 4) {
    if (few) return start<128, 4, 32>(a, st);          // 64 values have more rows than 32
    return h128 ? start<128, 4, 64>(a, st) : start<64, 4, 64>(a, st);
  }
  if (few) return start<128, 8, 32>(a, st);
  return h128 ? start<128, 8, 64>(a, st) : start<64, 8, 64>(a, st);
}

}  // namespace nl
