// The paged-attention kernel for many query rows (paged_attention_chunk.cu), for the entry point in paged_attention.cu.
#pragma once
#include <cuda_runtime.h>

#include "pyc_b200.h"

namespace b200 {

struct PagedParams;

int paged_chunk_ctas();
size_t paged_chunk_partial_bytes(int head_dim);
// p.rows_above / rows_upto say which requests it takes; p.cost and p.unsplit are set here.
int launch_paged_chunk(pyc_dtype dtype, int head_dim, PagedParams p, const void* k_cache, const void* v_cache, cudaStream_t s);

}  // namespace b200
