// logit_rules.cu -- what a batch's requests ask of their logits before a token is taken: penalties for tokens that were there before,
// biases, and the mask of a grammar; with the greedy ids where they are wanted.
//
// Row r (of sequence b), token v, c = how often v stands in the sequence's history and, where the rows are nodes of drafted
// trees, on the way from the root to the row's node:
//     x = logits[r][v];   c > 0:  x = x > 0 ? x / repetition : x * repetition,  x -= presence;   x -= frequency c
//     x += bias[b][v];    not allowed[r][v]:  x = -inf;       id[r] = the lowest v of the largest x
// each operation rounded by itself (IEEE float, no contraction), 16-bit logits widened first and the result rounded once.
//
// One CTA has a chunk of one row.  A bulk copy brings the chunk into shared memory while the CTA counts the tokens of its chunk that the
// sequence's history and the node's way have (32-bit counts by integer atomics: no order) and lists the tokens that a rule touches: some
// percent of the vocabulary, scattered over it.  Those are done first, one per thread, in shared memory; then the chunk streams out
// through the mask.  (Rules in the stream took three times as long: nearly every warp has a touched token among its 128.  CTAs that stay and
// keep counts for several rows took longer too: 126 against 103 us, for their chain of small loads.)  Several small CTAs per SM cover each
// other's chain: bounds of the history, its tokens, the counts.
// Greedy ids: the largest (value, lowest index) of a chunk as one 64-bit word, joined over the chunks by an atomic maximum that nobody waits
// for; a second kernel (programmatic dependent launch) turns the words into ids and zeroes them.  (Counting the CTAs at a row, so that the last
// one does that, held every CTA's place for two trips to L2 more: 61 us for 256 x 128000 logits.)
//
// What bounds it: the instructions of a chunk, 75 % of the issue slots (512 rows x 50257 floats, ids only: 54 us, 2.0 TB/s; 100 x 100003 bfloat16,
// both results: 24 us, 1.7 TB/s), nearer to the copies where rows are written and no history is long (256 x 128000 floats: 41 us without
// rules, 6.4 TB/s; with histories of 4096 tokens, 64 biases and masks 78 us, 3.5 TB/s).  Two, four or eight rows of a tree per CTA, which would
// share the counts of their history, took 66, 62 and 70 us instead of 53: fewer CTAs cover each other.
#include <algorithm>
#include <type_traits>

#include "dynamic_smem.cuh"
#include "tcgen05_utils.cuh"
#include "seq_common.cuh"

namespace pa {
namespace rules {

constexpr int kThreads = 256, kChunk = 4096, kBiases = 512, kList = 1024;
constexpr uint32_t kNothing = 0xffffffffu;      // above every number, as ordered words: a chunk that did not come
constexpr uint32_t kBiased = 0x80000000u;

__device__ int g_errors;

struct Args {
    const void* logits;
    void* out;                  // null: only ids
    int32_t* ids;               // null: only logits
    int64_t stride, out_stride;
    int rows, vocab, chunk, chunks;                        // tokens of a chunk, chunks of a row
    int num_seqs, history_tokens, bias_entries, mask_rows;  // bounds of what the device arrays below may name
    const int32_t *history, *history_start, *row_seq;
    const float *repetition, *presence, *frequency;        // per sequence; null: the value beside it
    float repetition1, presence1, frequency1;
    const int32_t *bias_ids, *bias_start;
    const float* bias;
    const uint32_t* allowed;
    int64_t allowed_stride;
    const int32_t* allowed_rows;
    const int32_t *tokens, *node_start;                    // drafted trees, or null
    const uint32_t* path;                                  // [rows, path_words]: nodes on a row's way
    int path_words;
    unsigned long long* best;                              // [rows], zero
    uint32_t polls;                                        // of the wait for a copy
};

template <typename T> __device__ __forceinline__ float widen(T v) { return to_f32<T>(v); }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v) { return from_f32<T>(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// 16 bytes of a row
template <typename T> struct __align__(16) Word {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};
template <typename T> struct Pair { typedef float2 type; };
template <> struct Pair<__half> { typedef __half2 type; };
template <> struct Pair<bf16_t> { typedef __nv_bfloat162 type; };

// shared memory: the chunk (its ends widened to whole words), counts, the mask, for 16-bit logits a bit per touched token, a list of touched
// tokens, biases
template <typename T> __host__ __device__ constexpr int data_bytes(int chunk) { return chunk * (int)sizeof(T) + 32; }
template <typename T>
static size_t shared_bytes(const Args& a) {
    return data_bytes<T>(a.chunk) + a.chunk * 4 + (sizeof(T) < 4 ? 2 : 1) * (a.chunk / 32 + 4) * 4 + kList * 2 + (a.bias ? kBiases * 8 : 0);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rules_kernel(const Args a) {
    constexpr int N = Word<T>::N;
    constexpr bool ROUNDS = sizeof(T) < 4;              // a touched token's float may win before it is rounded, not after
    extern __shared__ __align__(16) uint8_t smem[];
    T* data = reinterpret_cast<T*>(smem);
    uint32_t *count = reinterpret_cast<uint32_t*>(smem + data_bytes<T>(a.chunk)), *mask = count + a.chunk, *touched = mask + a.chunk / 32 + 4;
    uint16_t* list = reinterpret_cast<uint16_t*>(touched + (ROUNDS ? a.chunk / 32 + 4 : 0));
    int *bias_v = reinterpret_cast<int*>(list + kList), *bias_i = bias_v + kBiases;
    __shared__ int s_listed, s_biases, s_lost, s_counted;
    __shared__ unsigned long long s_key[kThreads / 32];
    __shared__ __align__(8) uint64_t s_bar;
    const int r = blockIdx.x / a.chunks, v0 = (blockIdx.x - r * a.chunks) * a.chunk, nv = min(a.chunk, a.vocab - v0), tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.logits) + (int64_t)r * a.stride + v0;
    // ---- the chunk, from the 16-byte word that it begins in to the one that it ends in
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    const uint32_t bar = smem_u32(&s_bar);
    if (tid == 0) {
        mbar_init(bar, 1);
        mbar_fence_init();
        const uint32_t bytes = (uint32_t)((off + nv) * (int)sizeof(T) + 15) & ~15u;
        if (a.polls) {                                      // 0: a wait that is to run out
            mbar_arrive_expect_tx(bar, bytes);
            bulk_g2s_nohint(smem_u32(data), x - off, bytes, bar);
        }
        s_listed = s_biases = s_lost = s_counted = 0;
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- bounds and bits that nothing waits for yet
    const int b = a.row_seq ? __ldg(a.row_seq + r) : r;
    const bool known = (unsigned)b < (unsigned)a.num_seqs;  // no sequence of the call: no history and no biases
    int h0 = 0, h1 = 0, i0 = 0, i1 = 0, s0 = 0, s1 = 0;
    if (a.history && known) {
        h0 = max(__ldg(a.history_start + b), 0);
        h1 = min(__ldg(a.history_start + b + 1), a.history_tokens);
    }
    if (a.bias && known) {
        i0 = max(__ldg(a.bias_start + b), 0);
        i1 = min(__ldg(a.bias_start + b + 1), a.bias_entries);
    }
    if (a.tokens && known) {
        s0 = max(__ldg(a.node_start + b), 0);
        s1 = min(min(__ldg(a.node_start + b + 1), a.rows), s0 + 32 * a.path_words);
    }
    const int64_t mrow = a.allowed_rows ? __ldg(a.allowed_rows + r) : r;
    const uint32_t* allowed = a.allowed && mrow >= 0 && mrow < a.mask_rows ? a.allowed + mrow * a.allowed_stride + (v0 >> 5) : nullptr;
    const float rep = a.repetition && known ? __ldg(a.repetition + b) : a.repetition1, pres = a.presence && known ? __ldg(a.presence + b) : a.presence1;
    const float freq = a.frequency && known ? __ldg(a.frequency + b) : a.frequency1;
    if (a.history || a.tokens || a.bias)
        for (int i = tid; i < a.chunk / 4; i += kThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (ROUNDS || a.allowed) {
        const int mwords = (nv + 31) >> 5;
        for (int i = tid; i < a.chunk / 32 + 4; i += kThreads) {
            if (ROUNDS) touched[i] = 0u;
            if (a.allowed) mask[i] = i >= mwords ? 0u : allowed ? __ldg(allowed + i) : 0xffffffffu;
        }
    }
    __syncthreads();
    // ---- the touched tokens
    auto note = [&](int v) {
        if (ROUNDS) atomicOr(&touched[v >> 5], 1u << (v & 31));
        const int at = atomicAdd(&s_listed, 1);
        if (at < kList) list[at] = (uint16_t)v;
    };
    auto add = [&](int token) {
        const int v = token - v0;
        if ((unsigned)v < (unsigned)nv && atomicAdd(&count[v], 1u) == 0u) note(v);
    };
    if (a.history) {
        const int q0 = min(h1, h0 + (int)((16 - ((uintptr_t)(a.history + h0) & 15)) & 15) / 4), q1 = h1 > q0 ? q0 + ((h1 - q0) & ~3) : q0;
        if (tid < q0 - h0) add(__ldg(a.history + h0 + tid));
        if (tid >= 32 && tid - 32 < h1 - q1) add(__ldg(a.history + q1 + tid - 32));
        for (int i = q0 + 4 * tid; i < q1; i += 16 * kThreads) {
            int4 t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                t[k] = i + 4 * k * kThreads < q1 ? __ldg(reinterpret_cast<const int4*>(a.history + i + 4 * k * kThreads)) : make_int4(-1, -1, -1, -1);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned n = (unsigned)nv;
                if ((unsigned)(t[k].x - v0) < n || (unsigned)(t[k].y - v0) < n || (unsigned)(t[k].z - v0) < n || (unsigned)(t[k].w - v0) < n) {
                    add(t[k].x);
                    add(t[k].y);
                    add(t[k].z);
                    add(t[k].w);
                }
            }
        }
    }
    for (int j = tid; j < s1 - s0; j += kThreads)       // thread j has node j
        if (__ldg(a.path + (int64_t)r * a.path_words + (j >> 5)) >> (j & 31) & 1u) add(__ldg(a.tokens + s0 + j));
    if (a.bias) {
        if (a.history || a.tokens) __syncthreads();     // a token is noted once
        for (int i = i0 + tid; i < i1; i += kThreads) {
            const int v = __ldg(a.bias_ids + i) - v0;
            if ((unsigned)v >= (unsigned)nv) continue;
            if (atomicOr(&count[v], kBiased) == 0u) note(v);
            const int place = atomicAdd(&s_biases, 1);
            if (place < kBiases) {
                bias_v[place] = v;
                bias_i[place] = i;
            }
        }
    }
    __syncthreads();
    bool here = true;               // of this thread; of all, where they changed one another's tokens
    for (uint32_t polls = 0; here && !mbar_try_wait(bar, 0); ++polls) here = polls < a.polls;
    if (!here) s_lost = 1;
    // ---- their rules, in place
    auto is_allowed = [&](int i) { return !a.allowed || (mask[i >> 5] >> (i & 31) & 1u); };
    float best = -INFINITY;
    int bi = 0x7fffffff;
    auto offer = [&](float f, int i) {          // of equal ones the lowest, in whatever order they come
        if (f > best || (f == best && f > -INFINITY && i < bi)) {
            best = f;
            bi = i;
        }
    };
    if (s_listed > 0) {
        // one touched token; last(i): of the entries for its bias the last
        auto apply = [&](int i, auto last) {
            const uint32_t raw = count[i], c = raw & ~kBiased;
            if (!raw) return;
            float f = widen<T>(data[off + i]);
            if (c) {
                f = f > 0.f ? __fdiv_rn(f, rep) : __fmul_rn(f, rep);
                f = __fsub_rn(f, pres);
                f = __fsub_rn(f, __fmul_rn(freq, (float)c));
            }
            if (raw & kBiased) f = __fadd_rn(f, __ldg(a.bias + last(i)));
            if (ROUNDS && a.ids && is_allowed(i)) offer(f, i);
            data[off + i] = narrow<T>(f);
        };
        if (s_biases <= kBiases) {
            const bool kept = s_listed <= kList;        // else every token is looked at
            for (int k = tid; here && k < (kept ? s_listed : nv); k += kThreads)
                apply(kept ? list[k] : k, [&](int i) {
                    int last = -1;
                    for (int q = 0; q < s_biases; ++q)
                        if (bias_v[q] == i) last = max(last, bias_i[q]);
                    return last;
                });
        } else {
            // more entries than were kept: the last one of every token, for some tokens at a time, from a pass over the sequence's list each (16 x 128000
            // logits with as many biases 0.46 ms; a search of the list per token 146)
            for (int t0 = 0; t0 < nv; t0 += kBiases) {
                __syncthreads();
                for (int k = tid; k < kBiases; k += kThreads) bias_i[k] = -1;
                __syncthreads();
                for (int q = i0 + tid; q < i1; q += kThreads) {
                    const unsigned k = (unsigned)(__ldg(a.bias_ids + q) - v0 - t0);
                    if (k < (unsigned)kBiases) atomicMax(&bias_i[k], q);
                }
                __syncthreads();
                for (int k = tid; here && k < min(kBiases, nv - t0); k += kThreads) apply(t0 + k, [&](int i) { return bias_i[i - t0]; });
            }
        }
        __syncthreads();
        here = !s_lost;
    }
    // ---- the stream: words of the result
    T* out = a.out ? static_cast<T*>(a.out) + (int64_t)r * a.out_stride + v0 : nullptr;
    const T* edge = out ? out : x;
    const int head = min(nv, (int)((16 - ((uintptr_t)edge & 15)) & 15) / (int)sizeof(T)), words = (nv - head) / N, tail = head + words * N;
    const bool whole = (off + head) % N == 0;           // they are words of the chunk as well
    auto single = [&](int i) {                          // a place outside the words
        const T v = is_allowed(i) ? data[off + i] : narrow<T>(-INFINITY);
        if (a.ids && !(ROUNDS && (touched[i >> 5] >> (i & 31) & 1u))) offer(widen<T>(v), i);
        if (out) out[i] = v;
    };
    auto word = [&](int i) {
        Word<T> w;
        if (whole) w = *reinterpret_cast<const Word<T>*>(data + off + i);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e) w.v[e] = data[off + i + e];
        }
        if (a.allowed) {
            const uint32_t ok = __funnelshift_r(mask[i >> 5], mask[(i >> 5) + 1], i & 31);
            if constexpr (ROUNDS) {
                constexpr uint32_t NINF = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
                uint32_t* p = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const uint32_t keep = (0u - (ok >> 2 * e & 1u)) & 0xffffu | (0u - (ok >> (2 * e + 1) & 1u)) << 16;
                    p[e] = (p[e] & keep) | (NINF & ~keep);
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (!(ok >> e & 1u)) w.v[e] = narrow<T>(-INFINITY);
            }
        }
        return w;
    };
    // the numbers of a word, and the largest: touched tokens of 16-bit logits as -infinity
    auto contest = [&](Word<T> w, int i, float (&f)[N]) {
        const uint32_t t = ROUNDS ? __funnelshift_r(touched[i >> 5], touched[(i >> 5) + 1], i & 31) : 0u;
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = ROUNDS && (t >> e & 1u) ? -INFINITY : widen<T>(w.v[e]);
    };
    auto largest = [&](const Word<T>& w, int i) {
        if constexpr (ROUNDS) {
            if (!(__funnelshift_r(touched[i >> 5], touched[(i >> 5) + 1], i & 31) & ((1u << N) - 1u))) {
                typedef typename Pair<T>::type P;
                const P* p = reinterpret_cast<const P*>(&w);
                const P m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
                return fmaxf(widen<T>(m.x), widen<T>(m.y));
            }
        }
        float f[N];
        contest(w, i, f);
        float top = f[0];
#pragma unroll
        for (int e = 1; e < N; ++e) top = fmaxf(top, f[e]);
        return top;
    };
    if (!here) {                        // the copy did not come: NaN in the thread's places, and no id for the row
        if (out) {
            const T nan = narrow<T>(__int_as_float(0x7fc00000));
            if (tid < head) out[tid] = nan;
            if (tail + tid < nv) out[tail + tid] = nan;
            for (int i = head + tid * N; i < tail; i += kThreads * N)
                for (int e = 0; e < N; ++e) out[i + e] = nan;
        }
        if (a.ids) atomicMax(a.best + r, (unsigned long long)kNothing << 32);
        if (atomicExch(&s_counted, 1) == 0) atomicAdd(&g_errors, 1);
        if (a.polls) tc::tc_let_land(bar, 0);               // the CTA's shared memory outlives the copy
    } else {
        if (tid < head) single(tid);
        if (tail + tid < nv) single(tail + tid);
    }
    float wbest = -INFINITY;
    int wi = -1;                                        // the first word with the largest
    for (int i = head + tid * N; here && i < tail; i += kThreads * N) {
        const Word<T> w = word(i);
        if (out) *reinterpret_cast<Word<T>*>(out + i) = w;
        if (a.ids) {
            const float top = largest(w, i);
            if (top > wbest) {
                wbest = top;
                wi = i;
            }
        }
    }
    if (!a.ids) return;
    if (wi >= 0) {
        float f[N];
        contest(word(wi), wi, f);
#pragma unroll
        for (int e = N - 1; e >= 0; --e)
            if (f[e] == wbest) offer(wbest, wi + e);
    }
    // (value, lowest index) of the warp, then of the CTA
    const uint32_t u = __float_as_uint(best + 0.f), o = here && best > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;   // ordered as the numbers, -0 as 0
    const uint32_t top = __reduce_max_sync(0xffffffffu, o), at = __reduce_min_sync(0xffffffffu, o == top ? (uint32_t)bi : 0xffffffffu);
    if ((tid & 31) == 0) s_key[tid >> 5] = top ? (unsigned long long)top << 32 | (uint32_t)~(v0 + (int)at) : 0ull;
    __syncthreads();
    if (tid < 32) {
        unsigned long long key = tid < kThreads / 32 ? s_key[tid] : 0ull;
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
        if (tid == 0 && hi) atomicMax(a.best + r, (unsigned long long)hi << 32 | lo);
    }
}

__global__ void __launch_bounds__(128) rules_ids_kernel(unsigned long long* best, int rows, int32_t* ids) {
    const int r = blockIdx.x * 128 + threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (r >= rows) return;
    const unsigned long long key = __ldcg(best + r);
    ids[r] = key ? (int32_t)~(uint32_t)key : 0;             // (kNothing, 0): -1
    best[r] = 0ull;
}

template <typename T>
static int launch(Args a, cudaStream_t st) {
    // few rows: smaller chunks, until every SM has one (4 rows with histories of 100 K tokens: 47 us, in chunks of 4096 54; one row 6.1 us against 6.6;
    // 8 rows x 128000, which give every SM one: 8 us, in chunks of 1024 11)
    a.chunk = kChunk;
    while (a.chunk > 1024 && (int64_t)a.rows * ((a.vocab + a.chunk - 1) / a.chunk) < device_info().sm_count) a.chunk /= 2;
    a.chunks = (a.vocab + a.chunk - 1) / a.chunk;
    const int64_t ctas = (int64_t)a.rows * a.chunks;
    if (ctas > 0x7fffffff) return PA_ERR_UNSUPPORTED;
    const size_t smem = shared_bytes<T>(a);
    cudaError_t e = allow_dynamic_smem<rules_kernel<T>>(smem);
    if (e != cudaSuccess) return (int)e;
    rules_kernel<T><<<(unsigned)ctas, kThreads, smem, st>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess || !a.ids) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.rows + 127) / 128));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, rules_ids_kernel, a.best, a.rows, a.ids);
    if (e != cudaSuccess) (void)cudaMemsetAsync(a.best, 0, (size_t)a.rows * 8, st);         // as every call leaves them
    return (int)e;
}

// Whether one of `rows` rows of `width` bytes from b on, `db` apart, shares a byte with one from a on, `da` apart
static bool overlap(uintptr_t a, int64_t da, uintptr_t b, int64_t db, int rows, int64_t width) {
    const int64_t off = (int64_t)(b - a), span_a = (rows - 1) * da + width, span_b = (rows - 1) * db + width;
    if (off >= span_a || -off >= span_b) return false;
    for (int r = 0; r < rows; ++r) {
        const int64_t at = off + r * db;                    // the last row of a that begins before this one ends
        const int64_t k = std::min<int64_t>(rows - 1, at + width > 0 ? (at + width - 1) / da : -1);
        if (k >= 0 && k * da + width > at) return true;
    }
    return false;
}

}  // namespace rules

int logit_rules_errors(int* host_count) { return (int)cudaMemcpyFromSymbol(host_count, rules::g_errors, sizeof(int)); }

}  // namespace pa

using namespace pa;

PA_API size_t pa_adjust_logits_workspace_bytes(int rows) { return rows > 0 ? (size_t)rows * 8 : 0; }

PA_API int pa_adjust_logits_polls(const void* d_logits, int type, int64_t stride, int rows, int vocab, void* d_out, int64_t out_stride,
                            int32_t* d_ids, const int32_t* d_row_seq, int num_seqs, const int32_t* d_history, int history_tokens, const int32_t* d_history_start,
                            const float* d_repetition, const float* d_presence, const float* d_frequency, float repetition, float presence,
                            float frequency, const int32_t* d_bias_ids, const float* d_bias, int bias_entries, const int32_t* d_bias_start,
                            const int32_t* d_allowed, int mask_rows, int64_t allowed_stride, const int32_t* d_allowed_rows, const int32_t* d_tokens,
                            const int32_t* d_path, int path_words, const int32_t* d_node_start, void* d_workspace, size_t workspace_bytes,
                            int polls, pa_stream_t stream) {
    using namespace pa::rules;
    PA_CHECK_ARG(polls >= 0);
    PA_CHECK_ARG(rows >= 0 && vocab > 0 && stride >= vocab && (!d_out || out_stride >= vocab) && (d_out || d_ids));
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(num_seqs >= 0 && history_tokens >= 0 && bias_entries >= 0 && mask_rows >= 0);
    PA_CHECK_ARG(d_logits && (!d_history || d_history_start) && (!d_bias || (d_bias_ids && d_bias_start)));
    PA_CHECK_ARG((!d_allowed || allowed_stride >= ((int64_t)vocab + 31) / 32) && (!d_tokens || (d_path && path_words > 0 && d_node_start && d_row_seq)));
    const int64_t elem = type == PA_TYPE_F32 ? 4 : 2;
    PA_CHECK_ARG(!d_out || (d_out == d_logits && (out_stride == stride || rows == 1)) ||
                 !overlap((uintptr_t)d_logits, stride * elem, (uintptr_t)d_out, out_stride * elem, rows, vocab * elem));
    if (d_ids && (!d_workspace || (uintptr_t)d_workspace % 8 || workspace_bytes < pa_adjust_logits_workspace_bytes(rows))) return PA_ERR_WORKSPACE;
    Args a{};
    a.logits = d_logits; a.out = d_out; a.ids = d_ids; a.stride = stride; a.out_stride = out_stride; a.rows = rows; a.vocab = vocab;
    a.num_seqs = num_seqs; a.history_tokens = history_tokens; a.bias_entries = bias_entries; a.mask_rows = mask_rows;
    a.history = d_history; a.history_start = d_history_start; a.row_seq = d_row_seq;
    a.repetition = d_repetition; a.presence = d_presence; a.frequency = d_frequency;
    a.repetition1 = repetition; a.presence1 = presence; a.frequency1 = frequency;
    a.bias_ids = d_bias_ids; a.bias_start = d_bias_start; a.bias = d_bias;
    a.allowed = reinterpret_cast<const uint32_t*>(d_allowed); a.allowed_stride = allowed_stride; a.allowed_rows = d_allowed_rows;
    a.tokens = d_tokens; a.node_start = d_node_start; a.path = reinterpret_cast<const uint32_t*>(d_path); a.path_words = path_words;
    a.best = static_cast<unsigned long long*>(d_workspace);
    a.polls = (uint32_t)polls;
    cudaStream_t st = as_stream(stream);
    if (type == PA_TYPE_F32) return launch<float>(a, st);
    if (type == PA_TYPE_F16) return launch<__half>(a, st);
    if (type == PA_TYPE_BF16) return launch<bf16_t>(a, st);
    return PA_ERR_UNSUPPORTED;
}

PA_API int pa_adjust_logits(const void* d_logits, int type, int64_t stride, int rows, int vocab, void* d_out, int64_t out_stride,
                            int32_t* d_ids, const int32_t* d_row_seq, int num_seqs, const int32_t* d_history, int history_tokens, const int32_t* d_history_start,
                            const float* d_repetition, const float* d_presence, const float* d_frequency, float repetition, float presence,
                            float frequency, const int32_t* d_bias_ids, const float* d_bias, int bias_entries, const int32_t* d_bias_start,
                            const int32_t* d_allowed, int mask_rows, int64_t allowed_stride, const int32_t* d_allowed_rows, const int32_t* d_tokens,
                            const int32_t* d_path, int path_words, const int32_t* d_node_start, void* d_workspace, size_t workspace_bytes,
                            pa_stream_t stream) {
    return pa_adjust_logits_polls(d_logits, type, stride, rows, vocab, d_out, out_stride, d_ids, d_row_seq, num_seqs, d_history, history_tokens,
                                  d_history_start, d_repetition, d_presence, d_frequency, repetition, presence, frequency, d_bias_ids, d_bias,
                                  bias_entries, d_bias_start, d_allowed, mask_rows, allowed_stride, d_allowed_rows, d_tokens, d_path, path_words,
                                  d_node_start, d_workspace, workspace_bytes, tc::kPolls, stream);
}
