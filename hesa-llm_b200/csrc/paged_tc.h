// paged_tc.h -- the tensor-core form of paged attention (paged_attention_tc.cu).
#pragma once

#include "paged.h"

namespace hesa_cuda {

constexpr int kTcRows = 128;   // rows of a tile
constexpr int kTcKeys = 128;   // keys of a block; a.blocks_per_split counts these

// head_dim 64 or 128
cudaError_t paged_attention_tc(const AttnArgs& a, int tiles, cudaStream_t s);

}  // namespace hesa_cuda
