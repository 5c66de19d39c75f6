// k_treeattn_h256.cu -- tree attention for heads of 256 values.
#include "tree_attn.cuh"

namespace nl {
template cudaError_t tree_attn_start<256>(TreeArgs &a, bool bf16, cudaStream_t st);
template cudaError_t tree_join_start<256>(TreeArgs &a, bool bf16, cudaStream_t st);
}
