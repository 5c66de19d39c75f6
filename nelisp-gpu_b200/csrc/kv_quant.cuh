// kv_quant.cuh -- the quantised paged key / value cache: its layout, shared by
// the kernels that write, read and attend to it.
//
//   codes  [num_blocks][kv_heads][block_size][head_dim * bits / 8] bytes
//   params [num_blocks][kv_heads][block_size] words
// for keys and values each.  A row is one head vector of one token; token
// slot s of the pool is offset s % block_size of block s / block_size.
// 8 bits: code 128 + c, the word is the float32 scale, value = s c.
// 4 bits: element 2i in the low and 2i + 1 in the high half of byte i; the
// word holds two bfloat16, the scale below the offset, value = s c + lo.
// Both words are zero-cost to load with the row: 4 bytes beside 32 .. 256.
#pragma once

#include <stdint.h>

#include "nl_internal.h"

namespace nl {

struct KvPool {
  uint8_t *code[2];       // keys, values
  uint32_t *param[2];
  uint32_t num_blocks, block_size, kv_heads, head_dim, bits;
};

// A scale below this stands for zero: its reciprocal would leave the range of
// float32 (127 / max at 2^-121), and the words below it are denormal.
constexpr float kKvTiny = 1.92592994e-34f;   // 2^-112

// The index of a head vector's row, for row counts below 2^32.
__device__ __forceinline__ uint32_t kv_row(const KvPool &p, uint32_t block, uint32_t off,
                                           uint32_t head) {
  return (block * p.kv_heads + head) * p.block_size + off;
}

static inline KvPool kv_pool_of(const nl_kv_cache &c) {
  return {{(uint8_t *)c.kc, (uint8_t *)c.vc}, {c.kp, c.vp}, c.num_blocks, c.block_size,
          c.kv_heads, c.head_dim, (uint32_t)c.fmt};
}
// NL_OK if the pool's description can be served (k_kvquant.cu).
int kv_check_pool(const char *what, int fmt, const KvPool &p);

}  // namespace nl
