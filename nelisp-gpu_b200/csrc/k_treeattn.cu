// k_treeattn.cu -- the entry point of the attention of drafted-token trees over
// the quantised paged cache.  The kernels are in tree_attn.cuh, compiled per
// head size in k_treeattn_h*.cu.

#include <algorithm>

#include "tree_work.cuh"

namespace nl {

// Rows are padded to 8, 16, 32, 64 or 128: a warp holds the state of 32 rows
// of 128 values (16 of 256), and up to four warps share the keys they read.
uint32_t tree_rows_at_once(uint32_t rows, uint32_t head_dim) {
  const uint32_t most = head_dim == 256 ? 64 : 128;
  uint32_t n = 8;
  while (n < rows && n < most) n *= 2;
  return n;
}

}  // namespace nl

using namespace nl;

extern "C" size_t nl_tree_attn_workspace_bytes(uint32_t nodes, uint32_t heads, uint32_t kv_heads,
                                               uint32_t head_dim) {
  if (!kv_heads || !nodes) return 16;
  const uint32_t rows = tree_rows_at_once(heads / kv_heads * nodes, head_dim);
  return (size_t)2 * kTreeMaxCtas * rows * (head_dim + 2) * sizeof(float);
}

extern "C" int nl_tree_attn_dev(const nl_tree_attn_args *args, void *stream) {
  int rc = api_ready();
  if (rc) return rc;
  const char *what = "tree-attn";
  if (!args) return set_error(NL_ERROR, "%s: null arguments", what);
  const nl_tree_attn_args &x = *args;
  const uint32_t batch = x.batch, nodes = x.nodes, heads = x.heads, kv_heads = x.cache.kv_heads,
                 head_dim = x.cache.head_dim, block_size = x.cache.block_size;
  const float scale = x.scale;
  if (x.dtype != NL_F32 && x.dtype != NL_BF16)
    return set_error(NL_ERROR, "%s: type %d is neither NL_F32 nor NL_BF16", what, x.dtype);
  TreeArgs a = {};
  a.pool = kv_pool_of(x.cache);
  if ((rc = kv_check_pool(what, x.cache.fmt, a.pool))) return rc;
  if (!heads || heads % kv_heads || heads > 65536)
    return set_error(NL_ERROR, "%s: heads %u, kv heads %u", what, heads, kv_heads);
  if (nodes > 64) return set_error(NL_ERROR, "%s: %u nodes (at most 64)", what, nodes);
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return set_error(NL_ERROR, "%s: scale %g is not positive and finite", what, scale);
  if (batch == 0 || nodes == 0) return NL_OK;
  if ((uint64_t)batch * nodes * heads > INT32_MAX)
    return set_error(NL_ERROR, "%s: %u sequences x %u nodes x %u heads", what, batch, nodes, heads);
  if (!x.len || !x.mask || ((uintptr_t)x.mask & 7u) || (!x.table && x.max_blocks))
    return set_error(NL_ERROR, "%s: null lengths, masks or table, or unaligned masks", what);
  const uint32_t unit = x.dtype == NL_BF16 ? 8 : 4;
  const uint64_t width = (uint64_t)heads * head_dim;
  if (!x.q || !x.o || !aligned16(x.q) || !aligned16(x.o) || x.q_stride % unit ||
      x.o_stride % unit || x.q_stride < width || x.o_stride < width)
    return set_error(NL_ERROR,
                     "%s: Q and O rows must be 16-byte aligned, with strides (%llu, %llu) that are "
                     "multiples of %u and at least heads x head size",
                     what, (unsigned long long)x.q_stride, (unsigned long long)x.o_stride, unit);
  cudaStream_t st = (cudaStream_t)stream;
  const size_t need = nl_tree_attn_workspace_bytes(nodes, heads, kv_heads, head_dim);
  if (x.workspace && x.ws_bytes < need)
    return set_error(NL_ERROR, "%s: workspace of %zu bytes, %zu needed", what, x.ws_bytes, need);
  void *workspace = x.workspace ? x.workspace : library_workspace(need, st);
  if (!workspace || !aligned16(workspace))
    return set_error(NL_ERROR, "%s: no aligned workspace of %zu bytes", what, need);
  a.q = x.q; a.o = x.o; a.lse = x.lse; a.table = x.table; a.len = x.len; a.mask = x.mask;
  a.q_stride = x.q_stride; a.o_stride = x.o_stride;
  a.batch = batch; a.nodes = nodes; a.heads = heads; a.group = heads / kv_heads;
  a.rows = a.group * nodes;
  const bool bf16 = x.dtype == NL_BF16;
  const uint32_t umma_rows = tree_umma_rows(a, bf16);
  a.rows_at_once = umma_rows ? umma_rows : tree_rows_at_once(a.rows, head_dim);
  a.row_tiles = (a.rows + a.rows_at_once - 1) / a.rows_at_once;
  // The list of the work, in tiles of at least 32 keys, is counted in 32 bits.
  const uint64_t most = std::min((uint64_t)x.max_blocks * block_size, (uint64_t)INT32_MAX + nodes);
  const unsigned __int128 places =
      (unsigned __int128)(most / 32 + 1 + kTreeMaxItemCost) * kv_heads * a.row_tiles * batch;
  if (places > UINT32_MAX)
    return set_error(NL_ERROR, "%s: %u sequences of up to %llu tokens: too much for one call", what,
                     batch, (unsigned long long)most);
  a.block_shift = 32;
  for (uint32_t s = 0; s < 32; s++)
    if (block_size == 1u << s) a.block_shift = s;
  a.max_blocks = x.max_blocks;
  a.scale = scale * 1.4426950408889634f;
  if (!x.cache.num_blocks)         // nothing is read of an empty pool, but its addresses are formed
    for (int i = 0; i < 2; i++)
      a.pool.code[i] = (uint8_t *)workspace, a.pool.param[i] = (uint32_t *)workspace;
  a.part_o = (float *)workspace;
  // Sized for 2 x 592 parts of tree_rows_at_once rows; the tcgen05 form has 2 x 148 of
  // 32 rows (of 17 to 32, which that rounds to 32) or of 64 (of more: 64 or 128).
  a.part_ml = a.part_o +
              (size_t)2 * kTreeMaxCtas * tree_rows_at_once(a.rows, head_dim) * head_dim;
  cudaError_t e = umma_rows         ? tree_umma_start(a, st)
                  : head_dim == 64  ? tree_attn_start<64>(a, bf16, st)
                  : head_dim == 128 ? tree_attn_start<128>(a, bf16, st)
                                    : tree_attn_start<256>(a, bf16, st);
  if (e == cudaSuccess)
    e = head_dim == 64    ? tree_join_start<64>(a, bf16, st)
        : head_dim == 128 ? tree_join_start<128>(a, bf16, st)
                          : tree_join_start<256>(a, bf16, st);
  return cuda_status(e, what);
}
