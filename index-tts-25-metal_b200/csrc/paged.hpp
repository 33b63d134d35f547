// Paged K/V cache operators: launchers of the kernels (paged_tables.cu,
// paged_append.cu, paged_attn*.cu) behind include/itts_paged.h
// (itts_paged.cpp checks the arguments before any of these runs).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "itts_paged.h"

namespace itts {
namespace paged {

cudaError_t launch_tables(const itts_paged_tables_args& a, cudaStream_t s);
cudaError_t launch_append(const itts_paged_append_args& a, cudaStream_t s);
cudaError_t launch_attention(const itts_paged_attention_args& a, cudaStream_t s);
size_t attention_workspace(int head_dim);

}  // namespace paged
}  // namespace itts
