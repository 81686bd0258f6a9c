// qw_chunk_attn.h -- host interface of the ragged chunk attention (qw_chunk_attn.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace qw {

constexpr int kChunkMaxBatch = 1024;  // sequences of one call (their schedule lies in shared memory)
constexpr int kChunkCounterBytes = 3 * 256 * 4;  // the workspace begins with counters, zero between calls
                                                 // (but for one whose bounded wait gave up)

struct ChunkArgs {
    const void *q, *k, *v;  // q (rows, ld_q): heads side by side; k, v: one layer's pages
    const int *page_table, *slots, *row_start, *kv_len;
    void *out;
    float *lse;
    int *err;
    void *workspace;
    long long ld_q, ld_out;
    int batch, rows, H, Hkv, G, d, ps, log2_ps, num_pages, max_pages, window;
    float sl2;  // scale * log2(e)
};

cudaError_t chunk_attn_tc_launch(const ChunkArgs &a, cudaStream_t st);    // bf16 (qw_chunk_attn_tc.cu)
cudaError_t chunk_attn_simt_launch(const ChunkArgs &a, cudaStream_t st);  // fp32 (qw_chunk_attn.cu)
size_t chunk_attn_tc_workspace(int head_dim);
// more units than the line of any lengths of these arguments has (the kernel numbers them in 32 bits)
uint64_t chunk_attn_tc_most_units(const ChunkArgs &a);

}  // namespace qw
