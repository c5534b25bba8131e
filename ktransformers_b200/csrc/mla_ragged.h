// The latent decode kernel (mla.cu) for a ragged batch of tokens, inside the library: token t, at position pos[t] (< 0: no keys) of the sequence in page-table row row[t] (a ring), sees
// positions 0 .. pos[t].  q_abs [T][H][512], q_rot [T][H][64], out [T][H][512], bf16; page_size a multiple of 32.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>

namespace ktb {

size_t mla_ragged_workspace(int n_tokens, int num_heads, int max_kv);
int mla_ragged(const void* q_abs, const void* q_rot, int num_heads, float scale, const int* pos, const int* row, const int* page_table, int max_pages, int page_size, const void* cache, long cache_rows,
               void* out, int n_tokens, int max_kv, void* workspace, size_t workspace_bytes, cudaStream_t stream);

}  // namespace ktb
