// Attention over selected key blocks with its gradient: what its translation units share.
#pragma once
#include <cuda.h>

#include "wa_internal.cuh"

namespace wa {

// Device pieces of a call's workspace.
struct SelectedPlan {
    int Nq, Nkv, group, words, row_words;      // query / key blocks, query heads of a key head, words of a bit per key block / per query block
    size_t index, num;                         // [B, H, Nq, index_stride] clean lists, [B, H, Nq] their lengths
    size_t rows;                               // backward: [B, Hkv, Nkv, group, row_words] which query blocks of which head list a key block
    size_t counters;                           // backward: zeroed together with `rows`, which it follows (see selected_sm100_backward)
    size_t stats;                              // backward: [B, H, selected_stats_rows] statistics of a query row, see selected_stat
    size_t q_order, k_order;                   // query blocks, and backward key blocks, heaviest first (not in every call)
    size_t tuned;                              // forward: what the tensor-core kernel needs
    size_t total;
};

// Statistics of the query rows, 64 rows together: 64 times minus the log-sum-exp in powers of two, then 64 times minus the sum of dout * out.  Rows that are no
// query's (behind the last one, and a block more for the tensor-core kernels' blocks) have an infinite normaliser, which makes their probabilities zero.
inline size_t selected_stats_rows(const wa_selected_params *p, int Nq) {
    return align_up(p->block_size <= 128 ? (size_t)(Nq + 1) * p->block_size : (size_t)p->Lq, 64);
}
__host__ __device__ inline long long selected_stat(long long row) { return (row >> 6) * 128 + (row & 63); }      // the sum lies 64 behind

// bf16, head_dim 128, blocks of 64 or 128 tokens.  wa_hsa_sm100.cu:
bool selected_sm100_tensors(const wa_selected_params *p);                 // q, k, v, blocks and device
bool selected_sm100_forward_supported(const wa_selected_params *p);
size_t selected_sm100_forward_bytes(const wa_selected_params *p);
bool selected_sm100_cleans(const wa_selected_params *p);                  // the call's own lists will do, which are cleaned on the way to lists of pairs
// `counts` [B, H, Nq]: lengths of those
int selected_sm100_forward(const wa_selected_params *p, const int32_t *index, const int32_t *num, int32_t *counts, void *workspace, cudaStream_t stream);
// a [B, L, H, 128] view as a map of boxes of `rows` tokens and one or both halves of the channels
int selected_sm100_map(CUtensorMap *map, const wa_tensor4 *t, int B, int L, int H, const char *name, int rows, int halves);
// wa_selected_sm100.cu:
bool selected_sm100_backward_supported(const wa_selected_params *p);
constexpr size_t SELECTED_COUNTERS = 256;      // two work counters and the failure flag
int selected_sm100_backward(const wa_selected_params *p, const int32_t *index, const int32_t *num, const uint32_t *rows, const float *stats,
                            const int32_t *q_order, const int32_t *k_order, int *counters, cudaStream_t stream);

}  // namespace wa
