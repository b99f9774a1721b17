// paged_tc.h -- the tensor-core form of paged attention (paged_attention_tc.cu).
#pragma once

#include "paged.h"

namespace hesa_cuda {

constexpr int kTcRows = 128;   // rows of a tile

// Keys of a block (a.blocks_per_split counts these) and dims of V that a CTA works
// on: what fits into 512 columns of TMEM beside q.
__host__ __device__ constexpr int tc_keys(int head_dim) { return head_dim == 256 ? 64 : 128; }
__host__ __device__ constexpr int tc_dims(int head_dim) { return head_dim == 256 ? 128 : head_dim; }

// Whether the pages can be read with tiled copies; head_dim 256 has no other way.
bool paged_attention_tiled(const PagedLayer& c);

cudaError_t paged_attention_tc(const AttnArgs& a, int tiles, cudaStream_t s);

}  // namespace hesa_cuda
