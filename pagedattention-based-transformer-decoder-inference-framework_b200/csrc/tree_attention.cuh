// tree_attention.cuh -- what the kernels of attention over drafted trees share (tree_attention.cu, tree_attention_tc.cu).
#pragma once
#include "seq_common.cuh"

namespace pa {

// Row r = (node i of sequence b) of q and out; its keys are positions 0 .. ctx(b) - 1, and ctx(b) + j where bit j of its mask is set.
struct TreeParams {
    const void* q;                  // [rows, heads, dim], rows q_stride elements apart
    int64_t q_stride;
    void* out;                      // [rows, heads, dim]
    const void *k, *v;              // [total_pages * tile_size, dim]
    const float *k_scales, *v_scales;
    const int32_t *table, *beam_ids, *ctx_lens, *node_start;
    const uint32_t* mask;           // [rows, mask_words]
    int q_type, kv_type, num_beams, kv_heads, num_tiles, total_pages, mask_words, rows, num_seqs, most, heads, dim, tile_size;
    float temperature;
};

template <typename T> __device__ __forceinline__ float tree_widen(T v) { return (float)v; }
template <> __device__ __forceinline__ float tree_widen<bf16_t>(bf16_t v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float tree_widen<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T tree_narrow(float v) { return (T)v; }
template <> __device__ __forceinline__ bf16_t tree_narrow<bf16_t>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half tree_narrow<__half>(float v) { return __float2half_rn(v); }

// the sequence of a row: the last b with node_start[b] <= r
__device__ __forceinline__ int tree_seq_of(const int32_t* node_start, int num_seqs, int r) {
    int lo = 0, hi = num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(node_start + mid) <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace pa
