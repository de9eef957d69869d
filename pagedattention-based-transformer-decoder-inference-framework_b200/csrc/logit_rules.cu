// logit_rules.cu -- what a batch's requests ask of their logits before a token is taken: penalties for tokens that were there before,
// biases, and the mask of a grammar; with the greedy ids where they are wanted.
//
// Row r (of sequence b), token v, c = how often v stands in the sequence's history and, where the rows are nodes of drafted
// trees, on the way from the root to the row's node:
//     x = logits[r][v];   c > 0:  x = x > 0 ? x / repetition : x * repetition,  x -= presence;   x -= frequency c
//     x += bias[b][v];    not allowed[r][v]:  x = -inf;       id[r] = the lowest v of the largest x
// each operation rounded by itself (IEEE float, no contraction), 16-bit logits widened first and the result rounded once.
#include "seq_common.cuh"

namespace pa {
namespace rules {

constexpr int kThreads = 512, kChunk = 4096;

struct Args {
    const void* logits;
    void* out;                  // null: only ids
    int32_t* ids;               // null: only logits
    int64_t stride, out_stride;
    int rows, vocab;
    const int32_t *history, *history_start, *row_seq;
    const float *repetition, *presence, *frequency;        // per sequence; null: the value beside it
    float repetition1, presence1, frequency1;
    const int32_t *bias_ids, *bias_start;
    const float* bias;
    const uint32_t* allowed;
    int64_t allowed_stride;
    const int32_t* allowed_rows;
    const int32_t *tokens, *parents, *node_start;          // drafted trees, or null
};

template <typename T> __device__ __forceinline__ float widen(T v) { return to_f32<T>(v); }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v) { return from_f32<T>(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float adjust(float x, uint32_t c, float rep, float pres, float freq) {
    if (c) {
        x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        x = __fsub_rn(x, pres);
        x = __fsub_rn(x, __fmul_rn(freq, (float)c));
    }
    return x;
}

// One CTA per row, kChunk tokens at a time: counts and bias places in shared memory, then one pass over the chunk's logits.
template <typename T>
__global__ void __launch_bounds__(kThreads) rules_kernel(const Args a) {
    __shared__ uint32_t count[kChunk], place[kChunk];
    __shared__ float sv[kThreads / 32];
    __shared__ int si[kThreads / 32];
    const int r = blockIdx.x, b = a.row_seq ? a.row_seq[r] : r;
    const T* x = static_cast<const T*>(a.logits) + (int64_t)r * a.stride;
    T* out = a.out ? static_cast<T*>(a.out) + (int64_t)r * a.out_stride : nullptr;
    const int64_t mrow = a.allowed_rows ? a.allowed_rows[r] : r;
    const uint32_t* allowed = a.allowed && mrow >= 0 ? a.allowed + mrow * a.allowed_stride : nullptr;
    const float rep = a.repetition ? a.repetition[b] : a.repetition1, pres = a.presence ? a.presence[b] : a.presence1;
    const float freq = a.frequency ? a.frequency[b] : a.frequency1;
    float best = -INFINITY;
    int bi = 0x7fffffff;
    for (int v0 = 0; v0 < a.vocab; v0 += kChunk) {
        const int nv = min(kChunk, a.vocab - v0);
        for (int i = threadIdx.x; i < nv; i += kThreads) count[i] = place[i] = 0;
        __syncthreads();
        if (a.history)
            for (int i = a.history_start[b] + threadIdx.x; i < a.history_start[b + 1]; i += kThreads) {
                const int v = a.history[i] - v0;
                if ((unsigned)v < (unsigned)nv) atomicAdd(&count[v], 1u);
            }
        if (a.tokens && threadIdx.x == 0) {
            const int s0 = a.node_start[b];
            for (int i = r - s0; i >= 0; i = a.parents[s0 + i] < i ? a.parents[s0 + i] : -1) {
                const int v = a.tokens[s0 + i] - v0;
                if ((unsigned)v < (unsigned)nv) atomicAdd(&count[v], 1u);
            }
        }
        if (a.bias)
            for (int i = a.bias_start[b] + threadIdx.x; i < a.bias_start[b + 1]; i += kThreads) {
                const int v = a.bias_ids[i] - v0;
                if ((unsigned)v < (unsigned)nv) atomicMax(&place[v], (uint32_t)i + 1u);
            }
        __syncthreads();
        for (int i = threadIdx.x; i < nv; i += kThreads) {
            const int v = v0 + i;
            float f = adjust(widen<T>(x[v]), count[i], rep, pres, freq);
            if (place[i]) f = __fadd_rn(f, a.bias[place[i] - 1]);
            if (allowed && !((allowed[v >> 5] >> (v & 31)) & 1u)) f = -INFINITY;
            if (out) out[v] = narrow<T>(f);
            if (f > best || (f == best && v < bi)) { best = f; bi = v; }
        }
        __syncthreads();
    }
    if (!a.ids) return;
    auto join = [&](float ov, int oi) {
        if (ov > best || (ov == best && oi < bi)) { best = ov; bi = oi; }
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, bi, o));
    if ((threadIdx.x & 31) == 0) { sv[threadIdx.x >> 5] = best; si[threadIdx.x >> 5] = bi; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; ++w) join(sv[w], si[w]);
        a.ids[r] = bi == 0x7fffffff ? 0 : bi;
    }
}

}  // namespace rules
}  // namespace pa

using namespace pa;

PA_API int pa_adjust_logits(const void* d_logits, int type, int64_t stride, int rows, int vocab, void* d_out, int64_t out_stride,
                            int32_t* d_ids, const int32_t* d_row_seq, const int32_t* d_history, const int32_t* d_history_start,
                            const float* d_repetition, const float* d_presence, const float* d_frequency, float repetition, float presence,
                            float frequency, const int32_t* d_bias_ids, const float* d_bias, const int32_t* d_bias_start,
                            const int32_t* d_allowed, int64_t allowed_stride, const int32_t* d_allowed_rows, const int32_t* d_tokens,
                            const int32_t* d_parents, const int32_t* d_node_start, pa_stream_t stream) {
    using namespace pa::rules;
    PA_CHECK_ARG(rows >= 0 && vocab > 0 && stride >= vocab && (!d_out || out_stride >= vocab) && (d_out || d_ids));
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_logits && (!d_history || d_history_start) && (!d_bias || (d_bias_ids && d_bias_start)));
    PA_CHECK_ARG((!d_allowed || allowed_stride >= ((int64_t)vocab + 31) / 32) && (!d_tokens || (d_parents && d_node_start && d_row_seq)));
    const Args a{d_logits, d_out, d_ids, stride, out_stride, rows, vocab, d_history, d_history_start, d_row_seq, d_repetition, d_presence,
                 d_frequency, repetition, presence, frequency, d_bias_ids, d_bias_start, d_bias, reinterpret_cast<const uint32_t*>(d_allowed),
                 allowed_stride, d_allowed_rows, d_tokens, d_parents, d_node_start};
    cudaStream_t st = as_stream(stream);
    if (type == PA_TYPE_F32) rules_kernel<float><<<rows, kThreads, 0, st>>>(a);
    else if (type == PA_TYPE_F16) rules_kernel<__half><<<rows, kThreads, 0, st>>>(a);
    else if (type == PA_TYPE_BF16) rules_kernel<bf16_t><<<rows, kThreads, 0, st>>>(a);
    else return PA_ERR_UNSUPPORTED;
    PA_RETURN_LAUNCH_STATUS();
}
