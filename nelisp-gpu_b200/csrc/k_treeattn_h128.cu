// k_treeattn_h128.cu -- tree attention for heads of 128 values.
#include "tree_attn.cuh"

namespace nl {
template cudaError_t tree_attn_start<128>(TreeArgs &a, bool bf16, cudaStream_t st);
template cudaError_t tree_join_start<128>(TreeArgs &a, bool bf16, cudaStream_t st);
}
