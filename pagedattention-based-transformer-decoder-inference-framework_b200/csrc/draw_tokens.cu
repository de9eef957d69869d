// draw_tokens.cu -- the distribution that a token is drawn from, tokens drawn from it by given numbers, and drafted tokens kept or replaced so
// that what comes out is distributed as the model's own.
//
// Row r (of sequence b), temperature T, x = its logits (NaN as -inf, +inf as the type's largest value), top = the largest:
//     w_v = exp((x_v - top) / T)                      T not above 0: only the lowest index of the largest
//     kept: #{u : x_u > x_v} < top_k;  then the w of all u with x_u > x_v below top_p of what is kept so far (the largest always);
//           then w_v >= min_p.  Tokens of one value stay or go together.
//     p_v = w_v / (sum of the kept w)
// drawn by U: the first v up to which the kept w exceed U times their sum; of several draws each leaves the others less.
// A node's children c_1, c_2, ... were drawn from q (draft probabilities), each from what the ones before it had left where they are distinct:
//     a = 0, S = 1, Q = 0;     c is kept where U_c q(c) S < max(p(c) - a q(c), 0) (1 - Q)
//     else a += S / (1 - Q), S = sum max(p - a q, 0), Q += q(c) where distinct;     none kept: drawn from max(p - a q, 0)
// (the residual p_i ~ max(p_(i-1) - q / (1 - Q), 0) of the i-th refusal is max(p - a q, 0) / S: by induction, since a refused token has none of it.)
//
// Ids have to be those of the definition: a cumulative sum that is off by e draws another token for a share of e of the numbers at each of
// up to V borders, so that weights and sums are in 64 bits (an error of 1e-12: one draw in 10^7 of 128000 tokens); floats would be off in one of a
// thousand.  2^y is 2^(j/32), from a table that the warp's lanes hold, times a polynomial of the fourth degree of the rest |r| <= 1/64 (Taylor's,
// error (r ln 2)^5 / 5! <= 1.3e-12): nine operations in 64 bits, of which an SM does 64 a cycle.
//
// A row is shared by a cluster of CTAs, whose shared memory holds it: logits come from memory once.  The least value that is kept is found
// without sorting: tokens are counted by 2048 steps of 1/64 in log2 w; with the bounds of the steps' weights the counts tell within some per cent where
// the border is; what is above is summed exactly, what is near is listed and counted again by finer steps, of floats in the end.
#include <climits>
#include <type_traits>

#include "cta_pair.cuh"
#include "dynamic_smem.cuh"
#include "pa_common.cuh"
#include "seq_common.cuh"

namespace pa {
namespace drawn {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2048, kPer = kBins / kThreads, kList = 1024, kMostRanks = 8;
constexpr uint32_t kAll = 0xffffffffu;
enum Mode { PROBS, DRAW, VERIFY };

struct Args {
    const void* logits;
    int64_t stride;
    int rows, vocab, ranks, num_seqs;
    size_t data_bytes;                                      // shared memory of a CTA's piece of the row
    const int32_t* row_seq;
    const float *temperature, *top_p, *min_p;               // per sequence; null: the value beside it
    const int32_t* top_k;
    double temperature1, top_p1, min_p1;
    int top_k1;
    float* probs;                                           // [rows][vocab], rows probs_stride apart
    int64_t probs_stride;
    int32_t* ids;                                           // [rows][count]
    float* logprobs;                                        // [rows][count], or null
    const float* uniform;                                   // [rows][count]; of nodes [rows][2]: the node's own test, the draw at it
    int count;
    const int32_t *tokens, *parents, *node_start, *draft_rows;      // nodes of drafted trees
    const void* draft;
    int64_t draft_stride;
    int draft_count, distinct;
};

template <typename T> __device__ __forceinline__ float widen(T v) { return to_f32<T>(v); }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <typename T> struct Limit;
template <> struct Limit<float> { static constexpr float most = 3.402823466e38f; };
template <> struct Limit<__half> { static constexpr float most = 65504.f; };
template <> struct Limit<bf16_t> { static constexpr float most = 3.38953139e38f; };

// NaN as -inf, +inf as the largest value, -0 as 0
template <typename T> __device__ __forceinline__ float clean(T v) {
    return fminf(fmaxf(widen<T>(v), -INFINITY), Limit<T>::most) + 0.f;
}

template <typename T> __device__ __forceinline__ T nothing() { return from_f32<T>(-INFINITY); }
template <> __device__ __forceinline__ __half nothing<__half>() { return __ushort_as_half(0xfc00); }

template <typename T> struct __align__(16) Word {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

// the same place in the shared memory of another CTA of the cluster
template <typename T> __device__ __forceinline__ const T* peer(const T* p, int rank) {
    uint64_t r;
    asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
    return reinterpret_cast<const T*>(r);
}

// ordered as the numbers (no NaN, no -0)
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Add { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Min {
    __device__ float operator()(float a, float b) const { return fminf(a, b); }
    __device__ int operator()(int a, int b) const { return min(a, b); }
};

// 2^y for y <= 0, by all lanes of a warp, lane j of which holds 2^(j/32) in `table`.  Below 2^-1022: 0.
__device__ __forceinline__ double exp2_64(double y, double table) {
    constexpr double magic = 211106232532992.0;             // 1.5 x 2^47: sums end at multiples of 1/32
    constexpr double c1 = 0.69314718055994530942, c2 = 0.24022650695910071233, c3 = 0.05550410866482157995, c4 = 0.00961812910762847716;    // ln 2 ^ k / k!
    const bool some = y > -1022.0;
    y = some ? y : 0.0;
    const double at = y + magic;
    const int n = __double2loint(at);
    const double r = y - (at - magic);
    double p = fma(r, c4, c3);
    p = fma(r, p, c2);
    p = fma(r, p, c1);
    p = fma(r, p, 1.0);
    p *= __shfl_sync(kAll, table, n & 31);
    p = __hiloint2double(__double2hiint(p) + (n >> 5 << 20), __double2loint(p));
    return some ? p : 0.0;
}

struct Shared {                     // beside the piece of the row
    uint4 hist[kBins / 4];
    float list[kList];
    double seg[kWarps];             // weights of the warps' parts of the piece, in the row's order
    double part[kWarps], part2[kWarps];
    float fpart[kWarps];
    int ipart[kWarps];
    int b_lo, b_hi, b_first, above, listed, children;
    // what the other CTAs of the cluster read
    float x_top, x_lo, x_hi, x_up;
    int x_first, x_listed;
    double x_all, x_above, x_total[2];
};
static_assert(kList >= PA_TREE_MOST_NODES, "a node's children take the place of the list");

template <typename T, typename Q, int MODE>
struct Piece {
    static constexpr int N = Word<T>::N, STRIP = 32 * N;
    const Args& a;
    Shared& sh;
    T* const data;                  // slot j is token lo + j; what is outside the row is -inf
    const int tid, warp, lane, rank, row;
    int lo, used, strips, s0, s1;   // slots that are used, strips of 32 words; this warp's are s0 .. s1 - 1
    float top, border;              // the largest; the least value that is kept
    double scale, table, min_p;
    int only;                       // the one token that is kept, or -1
    int turn = 0;                   // of x_total

    __device__ Piece(const Args& args, Shared& shared, T* piece) :
        a(args), sh(shared), data(piece), tid(threadIdx.x), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), rank((int)cluster_ctarank()),
        row((int)(blockIdx.x / args.ranks)) {}

    template <typename V, typename Op> __device__ V over_block(V v, V* parts, Op op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kAll, v, o));
        if (lane == 0) parts[warp] = v;
        __syncthreads();
        v = parts[0];
        for (int w = 1; w < kWarps; ++w) v = op(v, parts[w]);
        __syncthreads();
        return v;
    }
    template <typename V, typename Op> __device__ V over_cluster(const V* place, Op op) {     // between two cluster_sync
        V v = *peer(place, 0);
        for (int c = 1; c < a.ranks; ++c) v = op(v, *peer(place, c));
        return v;
    }
    __device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
        return v;
    }
    __device__ __forceinline__ float at(int slot) const { return sizeof(T) == 4 ? widen<T>(data[slot]) : clean<T>(data[slot]); }

    // ---- weights, by all lanes of a warp
    __device__ __forceinline__ double weight(float x) const { return exp2_64(((double)x - (double)top) * scale, table); }
    __device__ __forceinline__ double kept(float x, int v) const {
        if (only >= 0) return v == only && x > -INFINITY ? 1.0 : 0.0;
        const bool in = x >= border && x > -INFINITY;
        if (!__any_sync(kAll, in)) return 0.0;
        const double w = weight(x);
        return in && w >= min_p ? w : 0.0;
    }

    // f(x, slot) for the warp's tokens: all lanes together, word by word or (row order of lanes) token by token
    template <typename F> __device__ __forceinline__ void words(F f) const {
        for (int s = s0; s < s1; ++s) {
            const int j = s * STRIP + lane * N;
            const Word<T> w = *reinterpret_cast<const Word<T>*>(data + j);
#pragma unroll
            for (int e = 0; e < N; ++e) f(sizeof(T) == 4 ? widen<T>(w.v[e]) : clean<T>(w.v[e]), j + e);
        }
    }

    // ---- the piece into shared memory, and the row's largest
    __device__ void load() {
        const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.stride;
        const int V = a.vocab, first = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));     // tokens before the first whole word
        const int whole = (V - first) / N, w0 = (int)((int64_t)whole * rank / a.ranks), w1 = (int)((int64_t)whole * (rank + 1) / a.ranks);
        const int head = rank == 0 && first > 0, tail = rank == a.ranks - 1 && first + whole * N < V;
        used = (w1 - w0 + head + tail) * N;
        lo = first + (w0 - head) * N;
        strips = (used + STRIP - 1) / STRIP;
        s0 = strips * warp / kWarps;
        s1 = strips * (warp + 1) / kWarps;
        float m = -INFINITY;
        const Word<T>* src = reinterpret_cast<const Word<T>*>(x + first) + w0;
        Word<T>* dst = reinterpret_cast<Word<T>*>(data) + head;
#pragma unroll 4
        for (int i = tid; i < w1 - w0; i += kThreads) {
            const uint4 raw = ldg_stream_128(src + i);
            Word<T> w = *reinterpret_cast<const Word<T>*>(&raw);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float f = clean<T>(w.v[e]);
                m = fmaxf(m, f);
                if constexpr (sizeof(T) == 4) w.v[e] = f;
            }
            dst[i] = w;
        }
        auto edge = [&](int j) {                // token by token; what is not of the piece is -inf
            const int v = lo + j;
            const bool mine = v >= 0 && v < V && j < used;
            const float f = mine ? clean<T>(x[v]) : -INFINITY;
            m = fmaxf(m, f);
            if constexpr (sizeof(T) == 4) data[j] = f;
            else data[j] = mine ? x[v] : nothing<T>();
        };
        if (head && tid < N) edge(tid);
        for (int j = used - tail * N + tid; j < strips * STRIP; j += kThreads) edge(j);
        m = over_block(m, sh.fpart, Max());     // (its barriers also publish the piece)
        if (tid == 0) sh.x_top = m;
        cluster_sync();
        top = over_cluster(&sh.x_top, Max());
    }

    // ---- the least value that is kept of those from `least` on: with MASS the weights above it are below `share` of all, else fewer than
    // `share` tokens are above it.  R = [lo_x, hi_x] holds it; the first value in R is kept in any case.
    template <bool MASS> __device__ float find(double share, float least) {
        float lo_x = least, hi_x = top;
        double above_w = 0.0, limit = share;
        int above_n = 0;
        bool listed = false, halve = false;
        const float step = (float)(scale * 64.0);
        for (int level = 0; level < 128; ++level) {
            const uint32_t k_hi = key_of(hi_x), range = level ? k_hi - key_of(lo_x) : 0u;
            const int bits = 32 - __clz(range), shift = bits > 11 ? bits - 11 : 0;
            auto bin = [&](float x) {
                return level ? (int)((k_hi - key_of(x)) >> shift) : max(0, min(kBins - 1, (int)((top - x) * step)));
            };
            auto each = [&](auto f) {               // f(x) for all, or those that were listed
                if (!listed) words([&](float x, int) { f(x); });
                else for (int i = 0; i < sh.listed; i += kThreads) f(i + tid < sh.listed ? sh.list[i + tid] : -INFINITY);
            };
            auto in = [&](float x) { return x >= lo_x && x <= hi_x && x > -INFINITY; };
            int from = 0, to = 0;                   // R's steps that may hold the border
            if (halve) {                            // the bounds did not help: by halves, whose weights are summed exactly
                from = to = 1;
                cluster_sync();                     // the last sums have been read
            } else {
                for (int i = tid; i < kBins / 4; i += kThreads) sh.hist[i] = make_uint4(0, 0, 0, 0);
                if (tid == 0) {
                    sh.b_lo = sh.b_hi = -1;
                    sh.b_first = kBins;
                }
                __syncthreads();
                double all = 0.0;
                uint32_t* hist = reinterpret_cast<uint32_t*>(sh.hist);
                each([&](float x) {
                    const bool here = in(x);
                    if (here) atomicAdd(hist + bin(x), 1u);
                    if (MASS && level == 0 && __any_sync(kAll, here)) {
                        const double w = weight(x);
                        all += here ? w : 0.0;
                    }
                });
                if (MASS && level == 0) {
                    all = over_block(all, sh.part, Add());
                    if (tid == 0) sh.x_all = all;
                }
                cluster_sync();
                if (MASS && level == 0) limit = share * over_cluster(&sh.x_all, Add());
                // four steps a thread: how many tokens, and between what bounds their weights are; then of all steps above
                uint32_t n[kPer] = {0, 0, 0, 0};
                for (int c = 0; c < a.ranks; ++c) {
                    const uint4 h = *peer(sh.hist + tid, c);
                    n[0] += h.x; n[1] += h.y; n[2] += h.z; n[3] += h.w;
                }
                double least_w[kPer], most_w[kPer], least_sum = 0.0, most_sum = 0.0;
                int count = 0;
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const int b = tid * kPer + e;
                    count += n[e];
                    if (!MASS) continue;
                    if (level == 0) {               // (rounding of (top - x) * step: 2048 x 2^-22 of a step)
                        most_w[e] = n[e] * (double)exp2f(-b / 64.f) * (1.0 + 1e-5);
                        least_w[e] = b == kBins - 1 ? 0.0 : n[e] * (double)exp2f(-(b + 1) / 64.f) * (1.0 - 1e-5);
                    } else {
                        const uint64_t k0 = min((uint64_t)b << shift, (uint64_t)range), k1 = min(((uint64_t)(b + 1) << shift) - 1, (uint64_t)range);
                        most_w[e] = n[e] * weight(of_key(k_hi - (uint32_t)k0)) * (shift ? 1.0 + 1e-11 : 1.0);
                        least_w[e] = n[e] * weight(of_key(k_hi - (uint32_t)k1)) * (shift ? 1.0 - 1e-11 : 1.0);
                    }
                    most_sum += most_w[e];
                    least_sum += least_w[e];
                }
                int count_to = count;
                double least_to = least_sum, most_to = most_sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int p = __shfl_up_sync(kAll, count_to, o);
                    const double q = MASS ? __shfl_up_sync(kAll, least_to, o) : 0.0, s = MASS ? __shfl_up_sync(kAll, most_to, o) : 0.0;
                    if (lane >= o) {
                        count_to += p;
                        least_to += q;
                        most_to += s;
                    }
                }
                if (lane == 31) {
                    sh.ipart[warp] = count_to;
                    sh.part[warp] = least_to;
                    sh.part2[warp] = most_to;
                }
                __syncthreads();
                count_to -= count;
                least_to -= least_sum;
                most_to -= most_sum;
                for (int w = 0; w < warp; ++w) {
                    count_to += sh.ipart[w];
                    least_to += sh.part[w];
                    most_to += sh.part2[w];
                }
                const int before = count_to;
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const int b = tid * kPer + e;
                    if (n[e]) {
                        atomicMin(&sh.b_first, b);
                        if (MASS ? above_w + most_to < limit : above_n + count_to < limit) atomicMax(&sh.b_lo, b);
                        if (MASS ? above_w + least_to < limit : above_n + count_to < limit) atomicMax(&sh.b_hi, b);
                    }
                    count_to += n[e];
                    if (MASS) {
                        least_to += least_w[e];
                        most_to += most_w[e];
                    }
                }
                __syncthreads();
                from = max(sh.b_lo, sh.b_first);
                to = max(sh.b_hi, from);
                if (from / kPer == tid) {
                    int m = before;
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
                        if (tid * kPer + e < from) m += n[e];
                    sh.above = m;
                }
                __syncthreads();
                above_n += sh.above;
                if (level && shift == 0 && from == to) {
                    lo_x = of_key(k_hi - (uint32_t)from);
                    break;
                }
            }
            // what is above those steps, summed; the ends of what is in them, and a list of it
            const uint32_t half = key_of(lo_x) + range / 2;
            auto place = [&](float x) { return halve ? (key_of(x) > half ? 0 : 1) : bin(x); };
            double sum = 0.0;
            float least_x = INFINITY, most_x = -INFINITY, least_up = INFINITY;
            const bool listing = !listed && !halve;
            if (listing) {
                if (tid == 0) sh.listed = 0;
                __syncthreads();
            }
            each([&](float x) {
                const bool here = in(x);
                const int b = here ? place(x) : kBins;
                const bool up = b < from, near = b >= from && b <= to;
                if (MASS && __any_sync(kAll, up)) {
                    const double w = weight(x);
                    sum += up ? w : 0.0;
                    if (up) least_up = fminf(least_up, x);
                }
                if (near) {
                    least_x = fminf(least_x, x);
                    most_x = fmaxf(most_x, x);
                }
                if (listing && __any_sync(kAll, near)) {
                    const uint32_t who = __ballot_sync(kAll, near);
                    int at = 0;
                    if (lane == 0) at = atomicAdd(&sh.listed, __popc(who));
                    at = __shfl_sync(kAll, at, 0) + __popc(who & ((1u << lane) - 1u));
                    if (near && at < kList) sh.list[at] = x;
                }
            });
            if (MASS) sum = over_block(sum, sh.part, Add());
            least_x = over_block(least_x, sh.fpart, Min());
            most_x = over_block(most_x, sh.fpart, Max());
            if (halve) least_up = over_block(least_up, sh.fpart, Min());
            if (tid == 0) {
                sh.x_above = sum;
                sh.x_lo = least_x;
                sh.x_hi = most_x;
                sh.x_up = least_up;
                sh.x_listed = sh.listed;
            }
            cluster_sync();
            const double more = MASS ? over_cluster(&sh.x_above, Add()) : 0.0;
            const float lo_was = lo_x, hi_was = hi_x;
            if (halve && above_w + more >= limit) {         // the border is in the upper half
                lo_x = over_cluster(&sh.x_up, Min());
            } else {
                above_w += more;
                lo_x = over_cluster(&sh.x_lo, Min());
                hi_x = over_cluster(&sh.x_hi, Max());
                if (listing) {
                    listed = true;
                    for (int c = 0; c < a.ranks; ++c) listed = listed && *peer(&sh.x_listed, c) <= kList;
                }
            }
            if (lo_x == hi_x) break;
            // (the first count goes by steps of log2 w, the ones after it by those of floats)
            halve = MASS && level > 0 && !halve && key_of(hi_x) - key_of(lo_x) > (key_of(hi_was) - key_of(lo_was)) / 2;
        }
        cluster_sync();                 // nobody reads what comes next in its place
        return lo_x;
    }

    // ---- the rules of the row's sequence
    __device__ void rules() {
        const int b = a.row_seq ? a.row_seq[row] : row;
        const bool known = (unsigned)b < (unsigned)a.num_seqs;
        const double t = !known ? 1.0 : a.temperature ? (double)a.temperature[b] : a.temperature1;
        const double p = !known ? 1.0 : a.top_p ? (double)a.top_p[b] : a.top_p1, m = !known ? 0.0 : a.min_p ? (double)a.min_p[b] : a.min_p1;
        const int k = !known ? 0 : a.top_k ? a.top_k[b] : a.top_k1;
        only = -1;
        border = -INFINITY;
        min_p = m > 0.0 ? fmin(m, 1.0) : 0.0;
        if (!(t > 0.0)) {
            int v = INT_MAX;
            words([&](float x, int j) { if (x == top && lo + j < v && x > -INFINITY) v = lo + j; });
            v = over_block(v, sh.ipart, Min());
            if (tid == 0) sh.x_first = v;
            cluster_sync();
            only = over_cluster(&sh.x_first, Min());
            scale = 0.0;
            return;
        }
        scale = 1.4426950408889634074 / t;
        if (k > 0 && k < a.vocab) border = find<false>((double)k, -INFINITY);
        if (p < 1.0) border = find<true>(fmax(p, 0.0), border);
    }

    // ---- sums of f(x, slot) over the parts of the piece; the whole row's
    template <typename F> __device__ double sums(F f) {
        double sum = 0.0;
        words([&](float x, int j) { sum += f(x, j); });
        return join(sum);
    }
    __device__ double join(double sum) {
        sum = warp_sum64(sum);
        if (lane == 0) sh.seg[warp] = sum;
        __syncthreads();
        publish();
        cluster_sync();
        return over_cluster(&sh.x_total[turn], Add());
    }
    __device__ void publish() {
        turn ^= 1;              // two places in turn: others may still read the last one
        if (tid == 0) {
            double t = 0.0;
            for (int w = 0; w < kWarps; ++w) t += sh.seg[w];
            sh.x_total[turn] = t;
        }
    }

    // ---- the first token up to which the sums of f exceed `target`, where it is in this CTA's piece: found by its first warp; -1 elsewhere
    template <typename F> __device__ int search(double target, F f) {
        double run = 0.0, mine = 0.0;
        int owner = -1;
        for (int c = 0; c < a.ranks; ++c) {
            const double t = *peer(&sh.x_total[turn], c);
            if (t > 0.0 && (owner < 0 || run <= target)) {       // the first that exceeds, else the last that has anything
                owner = c;
                mine = run;
                if (run + t > target) break;
            }
            run += t;
        }
        if (owner != rank || warp != 0) return -1;
        run = mine;
        int part = -1;
        for (int w = 0; w < kWarps; ++w) {
            if (sh.seg[w] > 0.0) {
                part = w;
                mine = run;
                if (run + sh.seg[w] > target) break;
            }
            run += sh.seg[w];
        }
        run = mine;
        const int e0 = strips * part / kWarps, e1 = strips * (part + 1) / kWarps;
        int last = -1;
        for (int s = e0; s < e1; ++s) {
            const int j = s * STRIP + lane * N;
            double w[N], to = 0.0;
#pragma unroll
            for (int e = 0; e < N; ++e) to += w[e] = f(at(j + e), j + e);
            const double own = to;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double q = __shfl_up_sync(kAll, to, o);
                if (lane >= o) to += q;
            }
            double cum = run + to - own;
            int hit = -1, some = -1;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                cum += w[e];
                if (w[e] > 0.0) some = j + e;
                if (hit < 0 && w[e] > 0.0 && cum > target) hit = j + e;
            }
            const uint32_t who = __ballot_sync(kAll, hit >= 0);
            if (who) return __shfl_sync(kAll, hit, __ffs(who) - 1);
            last = max(last, __reduce_max_sync(kAll, some));
            run += __shfl_sync(kAll, to, 31);
        }
        return last;
    }

    // ---- what the modes do
    __device__ void probs() {
        const double total = top > -INFINITY ? sums([&](float x, int j) { return kept(x, lo + j); }) : 0.0, share = total > 0.0 ? 1.0 / total : 0.0;
        float* out = a.probs + (int64_t)row * a.probs_stride + lo;
        for (int s = s0; s < s1; ++s) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int j = s * STRIP + e * 32 + lane, v = lo + j;        // lanes on neighbouring tokens, as they are written
                const double w = share > 0.0 ? kept(at(j), v) : 0.0;
                if (v >= 0 && v < a.vocab && j < used) out[j] = (float)(w * share);
            }
        }
    }

    __device__ void draw() {
        if (!(top > -INFINITY)) {
            if (rank == 0 && tid < 32) for (int i = lane; i < a.count; i += 32) put(i, -1, 0.0);
            return;
        }
        auto f = [&](float x, int j) { return kept(x, lo + j); };
        const double whole = sums(f);
        double total = whole;
        for (int i = 0; i < a.count; ++i) {
            if (i) total = over_cluster(&sh.x_total[turn], Add());
            if (!(total > 0.0)) {
                if (rank == 0 && tid == 0) put(i, -1, 0.0);
                continue;                           // (so will all the others be)
            }
            const float u = a.uniform[(int64_t)row * a.count + i];
            const int j = search((u > 0.f ? (double)u : 0.0) * total, f);
            if (j >= 0) {
                const double w = f(at(j), j);
                if (lane == 0) put(i, lo + j, w / whole);
            }
            if (i + 1 == a.count) break;
            if (j >= 0) {                           // it leaves: its warp's part is summed anew
                __syncwarp();
                if (lane == 0) data[j] = nothing<T>();
                __syncwarp();
                int part = 0;
                while (strips * (part + 1) / kWarps <= j / STRIP) ++part;
                double sum = 0.0;
                for (int s = strips * part / kWarps; s < strips * (part + 1) / kWarps; ++s)
#pragma unroll
                    for (int e = 0; e < N; ++e) sum += f(at(s * STRIP + lane * N + e), s * STRIP + lane * N + e);
                sum = warp_sum64(sum);
                if (lane == 0) sh.seg[part] = sum;
            }
            __syncthreads();
            publish();
            cluster_sync();
        }
    }
    __device__ void put(int i, int id, double p) {
        a.ids[(int64_t)row * a.count + i] = id;
        if (a.logprobs) a.logprobs[(int64_t)row * a.count + i] = id < 0 ? -INFINITY : (float)log(p);
    }

    // (in weights: p, S and a times the sum of the kept)
    __device__ void verify() {
        if (!(top > -INFINITY)) {
            if (rank == 0 && tid == 0) put(0, -1, 0.0);
            return;
        }
        auto whole = [&](float xv, int j) { return kept(xv, lo + j); };
        const double total = sums(whole);
        const int b = a.row_seq[row], which = a.draft_rows ? a.draft_rows[row] : row;
        const bool drafted = (unsigned)which < (unsigned)a.draft_count && (unsigned)b < (unsigned)a.num_seqs;
        int32_t* child = reinterpret_cast<int32_t*>(sh.list);
        if (warp == 0) {
            int n = 0;
            if (drafted) {
                const int r0 = a.node_start[b], r1 = min(a.node_start[b + 1], a.rows);
                for (int r = row + 1; r < r1; r += 32) {
                    const bool mine = r + lane < r1 && a.parents[r + lane] == row - r0;
                    const uint32_t who = __ballot_sync(kAll, mine);
                    const int at = n + __popc(who & ((1u << lane) - 1u));
                    if (mine && at < PA_TREE_MOST_NODES) child[at] = r + lane;
                    n += __popc(who);
                }
            }
            if (lane == 0) sh.children = min(n, PA_TREE_MOST_NODES);
        }
        __syncthreads();
        const Q* q = drafted ? static_cast<const Q*>(a.draft) + (int64_t)which * a.draft_stride : nullptr;
        const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.stride;
        double taken = 0.0, S = total, gone = 0.0;
        auto rest = [&](float xv, int j) {          // what refused children have left of a token
            const double w = kept(xv, lo + j);
            return w > 0.0 ? fmax(w - taken * (double)widen<Q>(q[lo + j]), 0.0) : 0.0;
        };
        for (int i = 0; i < sh.children; ++i) {
            const int r = child[i], c = a.tokens[r];
            if ((unsigned)c >= (unsigned)a.vocab) continue;
            const double w = kept(clean<T>(x[c]), c), qc = (double)widen<Q>(q[c]);
            if ((double)a.uniform[2 * (int64_t)r] * qc * S < fmax(w - taken * qc, 0.0) * (1.0 - gone)) {
                if (rank == 0 && tid == 0) put(0, c, w / total);
                return;
            }
            taken += S / fmax(1.0 - gone, 1e-18);
            if (a.distinct) gone += qc;
            double sum = 0.0;
            for (int s = s0; s < s1; ++s)
#pragma unroll
                for (int e = 0; e < N; ++e) {       // lanes on neighbouring tokens, as q lies
                    const int j = s * STRIP + e * 32 + lane;
                    sum += rest(at(j), j);
                }
            S = join(sum);
        }
        const bool left = taken > 0.0 && S > 0.0;
        if (taken > 0.0 && !left) S = sums(whole);  // nothing is left by rounding, or where q is no distribution
        const float u = a.uniform[2 * (int64_t)row + 1];
        const double target = (u > 0.f ? (double)u : 0.0) * S;
        const int j = left ? search(target, rest) : search(target, whole);
        if (j >= 0) {
            const double w = whole(at(j), j);
            if (lane == 0) put(0, lo + j, w / total);
        }
    }
};

template <typename T, typename Q, int MODE> __global__ void __launch_bounds__(kThreads, 2) draw_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Piece<T, Q, MODE> p(a, *reinterpret_cast<Shared*>(smem + a.data_bytes), reinterpret_cast<T*>(smem));
    p.table = exp2((threadIdx.x & 31) / 32.0);
    p.load();
    if (p.top > -INFINITY) p.rules();
    if constexpr (MODE == PROBS) p.probs();
    else if constexpr (MODE == DRAW) p.draw();
    else p.verify();
    cluster_sync();                     // no CTA leaves while others read its shared memory
}

template <typename T, typename Q, int MODE> static int launch(Args a, cudaStream_t st) {
    constexpr int N = Word<T>::N;
    // the fewest CTAs whose pieces leave room for three on an SM, more while rows are few
    auto bytes = [&](int ranks) { return (((size_t)a.vocab / N / ranks + 3 + 31) / 32) * 512; };
    const size_t most = device_info().max_smem_optin - sizeof(Shared) - 1024;
    a.ranks = 1;
    while (a.ranks < kMostRanks && (bytes(a.ranks) > 56 * 1024 || (a.rows * a.ranks * 2 <= device_info().sm_count && a.vocab / a.ranks >= 4096))) a.ranks *= 2;
    a.data_bytes = bytes(a.ranks);
    if (a.data_bytes > most || (int64_t)a.rows * a.ranks > INT_MAX) return PA_ERR_UNSUPPORTED;
    const size_t smem = a.data_bytes + sizeof(Shared);
    const cudaError_t e = allow_dynamic_smem<draw_kernel<T, Q, MODE>>(smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * a.ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a.ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, draw_kernel<T, Q, MODE>, a);
}

template <int MODE> static int launch(const Args& a, int type, int draft_type, cudaStream_t st) {
    if constexpr (MODE == VERIFY) {
        auto of = [&](auto t) {
            typedef decltype(t) T;
            return draft_type == PA_TYPE_F32 ? launch<T, float, MODE>(a, st) : draft_type == PA_TYPE_F16 ? launch<T, __half, MODE>(a, st) :
                   draft_type == PA_TYPE_BF16 ? launch<T, bf16_t, MODE>(a, st) : PA_ERR_UNSUPPORTED;
        };
        return type == PA_TYPE_F32 ? of(float()) : type == PA_TYPE_F16 ? of(__half()) : type == PA_TYPE_BF16 ? of(bf16_t()) : PA_ERR_UNSUPPORTED;
    } else {
        return type == PA_TYPE_F32 ? launch<float, float, MODE>(a, st) : type == PA_TYPE_F16 ? launch<__half, float, MODE>(a, st) :
               type == PA_TYPE_BF16 ? launch<bf16_t, float, MODE>(a, st) : PA_ERR_UNSUPPORTED;
    }
}

static Args args(const void* logits, int64_t stride, int rows, int vocab, const pa_draw_rules* rules) {
    Args a{};
    a.logits = logits; a.stride = stride; a.rows = rows; a.vocab = vocab;
    a.row_seq = rules->d_row_seq; a.num_seqs = rules->num_seqs;
    a.temperature = rules->d_temperature; a.top_k = rules->d_top_k; a.top_p = rules->d_top_p; a.min_p = rules->d_min_p;
    a.temperature1 = rules->temperature; a.top_k1 = rules->top_k; a.top_p1 = rules->top_p; a.min_p1 = rules->min_p;
    return a;
}
static bool usable(const void* logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules) {
    return rows >= 0 && vocab > 0 && stride >= vocab && rules && rules->num_seqs >= 0 && (rows == 0 || logits) &&
           (uintptr_t)logits % (type == PA_TYPE_F32 ? 4 : 2) == 0;
}

}  // namespace drawn
}  // namespace pa

using namespace pa;

PA_API int pa_truncated_softmax(const void* d_logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules, float* d_probs,
                                int64_t probs_stride, pa_stream_t stream) {
    using namespace pa::drawn;
    PA_CHECK_ARG(usable(d_logits, type, stride, rows, vocab, rules) && probs_stride >= vocab);
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_probs);
    const uintptr_t in = (uintptr_t)d_logits, out = (uintptr_t)d_probs;
    const uintptr_t in_end = in + ((size_t)(rows - 1) * stride + vocab) * (type == PA_TYPE_F32 ? 4 : 2), out_end = out + ((size_t)(rows - 1) * probs_stride + vocab) * 4;
    PA_CHECK_ARG(in >= out_end || out >= in_end);
    Args a = args(d_logits, stride, rows, vocab, rules);
    a.probs = d_probs; a.probs_stride = probs_stride;
    return launch<PROBS>(a, type, 0, as_stream(stream));
}

PA_API int pa_draw_tokens(const void* d_logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules, const float* d_uniform,
                          int count, int32_t* d_ids, float* d_logprobs, pa_stream_t stream) {
    using namespace pa::drawn;
    PA_CHECK_ARG(usable(d_logits, type, stride, rows, vocab, rules) && count > 0);
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_uniform && d_ids);
    Args a = args(d_logits, stride, rows, vocab, rules);
    a.uniform = d_uniform; a.count = count; a.ids = d_ids; a.logprobs = d_logprobs;
    return launch<DRAW>(a, type, 0, as_stream(stream));
}

PA_API int pa_verify_drafts(const void* d_logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules, const float* d_uniform,
                            const int32_t* d_tokens, const int32_t* d_parents, const int32_t* d_node_start, const void* d_draft, int draft_type,
                            int64_t draft_stride, int draft_count, const int32_t* d_draft_rows, int distinct, int32_t* d_ids, float* d_logprobs,
                            pa_stream_t stream) {
    using namespace pa::drawn;
    PA_CHECK_ARG(usable(d_logits, type, stride, rows, vocab, rules) && draft_count >= 0 && (draft_count == 0 || (d_draft && draft_stride >= vocab)));
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_uniform && d_ids && d_tokens && d_parents && d_node_start && rules->d_row_seq && (d_draft_rows || draft_count >= rows));
    Args a = args(d_logits, stride, rows, vocab, rules);
    a.uniform = d_uniform; a.count = 1; a.ids = d_ids; a.logprobs = d_logprobs;
    a.tokens = d_tokens; a.parents = d_parents; a.node_start = d_node_start; a.draft = d_draft; a.draft_stride = draft_stride;
    a.draft_count = draft_count; a.draft_rows = d_draft_rows; a.distinct = distinct;
    return launch<VERIFY>(a, type, draft_type, as_stream(stream));
}
