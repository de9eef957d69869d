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

constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 1024, kPer = kBins / kThreads, kList = 256, kMany = 1024, kFew = 256, kMostRanks = 8, kMostStrips = 64;
static_assert(kFew <= kThreads && kPer % 4 == 0, "a thread for each of few, whole words of steps");
constexpr uint32_t kAll = 0xffffffffu;
constexpr float kLowest = -3.402823466e38f, kSteps = 32.f;      // steps of log2 w
enum Mode { PROBS, DRAW, VERIFY };

struct Args {
    const void* logits;
    int64_t stride;
    int rows, vocab, ranks, num_seqs;
    size_t data_bytes;                                      // shared memory of a CTA's piece of the row
    int count_shift;                                        // a step's word: tokens above it, their parts of a step below
    float parts;                                            // of a step (0: none are kept)
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
template <typename T> __device__ __forceinline__ T narrow(float v) { return from_f32<T>(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
// the largest number of a type, and how many low bits of it as a float say nothing
template <typename T> struct Limit;
template <> struct Limit<float> { static constexpr float most = 3.402823466e38f; static constexpr int spare = 0; };
template <> struct Limit<__half> { static constexpr float most = 65504.f; static constexpr int spare = 13; };
template <> struct Limit<bf16_t> { static constexpr float most = 3.38953139e38f; static constexpr int spare = 16; };

template <typename T> struct __align__(16) Word {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

// the same place in the shared memory of another CTA of the cluster
template <typename T> __device__ __forceinline__ T* peer(T* p, int rank) {
    uint64_t r;
    asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
    return reinterpret_cast<T*>(r);
}

// ordered as the numbers (no NaN; -0 as 0)
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Add {
    template <typename V> __device__ V operator()(V a, V b) const { return a + b; }
    template <typename V> __device__ static V none() { return 0; }
};
struct Max {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
    template <typename V> __device__ static V none() { return -INFINITY; }
};
struct Min {
    __device__ float operator()(float a, float b) const { return fminf(a, b); }
    __device__ int operator()(int a, int b) const { return min(a, b); }
    template <typename V> __device__ static V none() { return std::is_same<V, int>::value ? (V)INT_MAX : (V)INFINITY; }
};

// 2^y by all lanes of a warp, lane j of which holds 2^(j/32) in `table`: for y of -1022 to 0; others give some number
__device__ __forceinline__ double exp2_64(double y, double table) {
    constexpr double magic = 211106232532992.0;             // 1.5 x 2^47: sums end at multiples of 1/32
    constexpr double c1 = 0.69314718055994530942, c2 = 0.24022650695910071233, c3 = 0.05550410866482157995, c4 = 0.00961812910762847716;    // ln 2 ^ k / k!
    const double at = y + magic;
    const int n = __double2loint(at);
    const double r = y - (at - magic);
    double p = fma(r, c4, c3);
    p = fma(r, p, c2);
    p = fma(r, p, c1);
    p = fma(r, p, 1.0);
    p *= __shfl_sync(kAll, table, n & 31);
    return __hiloint2double(__double2hiint(p) + (n >> 5 << 20), __double2loint(p));
}

struct Near { float x; int slot; };
struct Verdict {                    // of the cluster's first CTA
    float up, lo;                   // what is at or above `up` is summed, what is at or above `lo` listed
    float r_lo, r_hi, border;
    double above, limit;
    int above_n, done, halve, ruled;
};

struct Shared {                     // beside the piece of the row
    union {
        uint4 hist[kBins / 4];
        float many[kMany];          // tokens that all CTAs have listed
        int32_t child[PA_TREE_MOST_NODES];
    };
    Near list[kList];
    union {
        double few_w[kFew];
        uint32_t fine[kThreads];
    };
    float few[kFew];
    double seg[kWarps];             // weights of the warps' parts of the piece, in the row's order
    double strip[kMostStrips];      // of one part's strips
    double part[kWarps], part2[kWarps];
    float fpart[kWarps], fpart2[kWarps], fpart3[kWarps];
    int ipart[kWarps];
    int b_lo, b_hi, b_first, before_n, to_n, listed, children, hit;
    // what the other CTAs of the cluster read
    Verdict verdict;
    float x_top, x_lo, x_hi, x_up;
    int x_first, x_listed;
    double x_below, x_above, x_total[2];
};

template <typename T, typename Q, int MODE>
struct Piece {
    static constexpr int N = Word<T>::N, STRIP = 32 * N;
    const Args& a;
    Shared& sh;
    T* const data;                  // slot j is token lo + j; what is outside the row is -inf
    const int tid, warp, lane, rank, row;
    int lo, used, strips, s0, s1;   // slots that are used, strips of 32 words; this warp's are s0 .. s1 - 1
    float top, border;              // the largest; the least value that is kept
    double scale, base, table;      // w = 2^(x scale + base)
    int only;                       // temperature 0: the one token that is kept, else -1
    int turn = 0;                   // of x_total
    bool left = false;              // has arrived at the last barrier

    __device__ Piece(const Args& args, Shared& shared, T* piece) :
        a(args), sh(shared), data(piece), tid(threadIdx.x), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), rank((int)cluster_ctarank()),
        row((int)(blockIdx.x / args.ranks)) {}

    template <typename V, typename Op> __device__ V over_block(V v, V* parts, Op op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kAll, v, o));
        if (lane == 0) parts[warp] = v;
        __syncthreads();
        v = parts[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) v = op(v, parts[w]);
        __syncthreads();
        return v;
    }
    // what the CTAs of the cluster have in a place: all on their way at once (between two cluster_sync)
    template <typename V> __device__ __forceinline__ void of_all(V* place, V (&v)[kMostRanks], V none) {
#pragma unroll
        for (int c = 0; c < kMostRanks; ++c) v[c] = *peer(place, min(c, a.ranks - 1));
#pragma unroll
        for (int c = 1; c < kMostRanks; ++c)
            if (c >= a.ranks) v[c] = none;
    }
    template <typename V, typename Op> __device__ __forceinline__ V over_cluster(V* place, Op op) {
        V v[kMostRanks];
        of_all(place, v, Op::template none<V>());
#pragma unroll
        for (int c = 1; c < kMostRanks; ++c) v[0] = op(v[0], v[c]);
        return v[0];
    }
    __device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
        return v;
    }
    __device__ __forceinline__ float at(int slot) const { return widen<T>(data[slot]); }

    // ---- weights, by all lanes of a warp
    __device__ __forceinline__ double weight(float x) const { return exp2_64(fma((double)x, scale, base), table); }
    __device__ __forceinline__ double kept(float x) const {
        const bool in = x >= border;
        if (!__any_sync(kAll, in)) return 0.0;
        const double w = weight(x);
        return in ? w : 0.0;
    }

    // f(x, slot) for the warp's tokens, all lanes together
    template <typename F> __device__ __forceinline__ void words(F f) const {
        for (int s = s0; s < s1; ++s) {
            const int j = s * STRIP + lane * N;
            const Word<T> w = *reinterpret_cast<const Word<T>*>(data + j);
#pragma unroll
            for (int e = 0; e < N; ++e) f(widen<T>(w.v[e]), j + e);
        }
    }
    // the weights of what is at or above `least` in a strip, or of lanes on neighbouring tokens (n of them)
    __device__ __forceinline__ double strip_sum(int s, float least) const {
        const Word<T> w = *reinterpret_cast<const Word<T>*>(data + s * STRIP + lane * N);
        float x[N], m = -INFINITY;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            x[e] = widen<T>(w.v[e]);
            m = fmaxf(m, x[e]);
        }
        if (!__any_sync(kAll, m >= least)) return 0.0;
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double v = weight(x[e]);
            sum += x[e] >= least ? v : 0.0;
        }
        return sum;
    }
    __device__ double kept_sum() {
        double sum = 0.0;
        for (int s = s0; s < s1; ++s) sum += strip_sum(s, border);
        return join(sum);
    }

    // ---- the piece into shared memory, and the row's largest (NaN is never the larger, and never at or above anything)
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
        const uint4* src = reinterpret_cast<const uint4*>(x + first) + w0;
        uint4* dst = reinterpret_cast<uint4*>(data) + head;
        constexpr int D = 8;                    // words on their way per thread
        for (int i = tid; i < w1 - w0; i += D * kThreads) {
            uint4 raw[D];
#pragma unroll
            for (int d = 0; d < D; ++d)
                if (i + d * kThreads < w1 - w0) raw[d] = ldg_stream_128(src + i + d * kThreads);
#pragma unroll
            for (int d = 0; d < D; ++d)
                if (i + d * kThreads < w1 - w0) {
                    dst[i + d * kThreads] = raw[d];
                    const Word<T> w = *reinterpret_cast<const Word<T>*>(&raw[d]);
#pragma unroll
                    for (int e = 0; e < N; ++e) m = fmaxf(m, widen<T>(w.v[e]));
                }
        }
        auto edge = [&](int j) {                // token by token; what is not of the piece is -inf
            const int v = lo + j;
            const T t = v >= 0 && v < V && j < used ? x[v] : narrow<T>(-INFINITY);
            data[j] = t;
            m = fmaxf(m, widen<T>(t));
        };
        if (head && tid < N) edge(tid);
        for (int j = used - tail * N + tid; j < strips * STRIP; j += kThreads) edge(j);
        m = over_block(m, sh.fpart, Max());     // (its barriers also publish the piece)
        if (tid == 0) sh.x_top = m;
        cluster_sync();
        top = over_cluster(&sh.x_top, Max());
        if (top == INFINITY) {                  // as the type's largest
            for (int j = tid; j < strips * STRIP; j += kThreads)
                if (at(j) == INFINITY) data[j] = narrow<T>(Limit<T>::most);
            top = Limit<T>::most;
            __syncthreads();
        }
    }

    // ---- where the border is, as far as counts tell: the steps that may hold it, of PER a thread.  counted(b): (tokens, parts); bounds(b, n, parts,
    // least, most): the weights that they have at least and at most; above, above_n: what is above the first step.  The border is where what is above it
    // reaches `limit`, or with `whole` that share of all.  Leaves the tokens above `from` in before_n, those up to `to` in to_n.
    template <bool MASS, int PER, typename C, typename B>
    __device__ void weigh(bool whole, double limit, double above, int above_n, int& from, int& to, C counted, B bounds) {
        uint32_t n[PER];
        double least_w[PER], most_w[PER], least = 0.0, most = 0.0;
        int count = 0;
        uint32_t parts[PER];
        counted(n, parts);
        if (tid == 0) {
            sh.b_lo = sh.b_hi = -1;
            sh.b_first = INT_MAX;
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            count += n[e];
            if (!MASS) continue;
            bounds(tid * PER + e, n[e], parts[e], least_w[e], most_w[e]);
            least += least_w[e];
            most += most_w[e];
        }
        int count_to = count;
        double least_to = least, most_to = most;
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
        count_to += above_n - count;
        least_to += above - least;
        most_to += above - most;
        double limit_least = limit, limit_most = limit, least_all = 0.0, most_all = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) {
                count_to += sh.ipart[w];
                least_to += sh.part[w];
                most_to += sh.part2[w];
            }
            least_all += sh.part[w];
            most_all += sh.part2[w];
        }
        if (MASS && whole) {
            limit_least *= least_all;
            limit_most *= most_all;
        }
        const int before = count_to;
        int b_first = INT_MAX, b_lo = -1, b_hi = -1;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int b = tid * PER + e;
            if (n[e]) {
                b_first = min(b_first, b);
                if (MASS ? most_to < limit_least : count_to < limit) b_lo = b;
                if (MASS ? least_to < limit_most : count_to < limit) b_hi = b;
            }
            count_to += n[e];
            if (MASS) {
                least_to += least_w[e];
                most_to += most_w[e];
            }
        }
        if (b_first < INT_MAX) atomicMin(&sh.b_first, b_first);
        if (b_lo >= 0) atomicMax(&sh.b_lo, b_lo);
        if (b_hi >= 0) atomicMax(&sh.b_hi, b_hi);
        __syncthreads();
        from = max(sh.b_lo, sh.b_first);            // the first that has any holds the largest, which is kept
        to = max(sh.b_hi, from);
        int m = before, m_to = before;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            if (tid * PER + e < from) m += n[e];
            if (tid * PER + e <= to) m_to += n[e];
        }
        if (from / PER == tid) sh.before_n = m;
        if (to / PER == tid) sh.to_n = m_to;
        __syncthreads();
    }

    // the least float whose step is below b (the steps fall while the floats grow), by a warp: 31 of them are tried at a time
    template <typename F> __device__ float edge_of(int b, F place) const {
        if (b <= 0) return INFINITY;
        uint64_t l = key_of(kLowest), h = key_of(top);          // place(h) = 0 < b; the answer is in [l, h]
        while (l < h) {
            const uint64_t d = (h - l + 31) / 32, k = min(l + d * lane, h);
            const uint32_t yes = __ballot_sync(kAll, place(of_key((uint32_t)k)) < b);
            const int i = __ffs(yes) - 1;                        // the first that is
            if (i == 0) return of_key((uint32_t)l);
            const uint64_t was = l;
            if (i > 0) {
                l = min(was + d * (i - 1) + 1, h);
                h = min(was + d * i, h);
            } else {
                l = min(was + d * 31 + 1, h);
            }
        }
        return of_key((uint32_t)h);
    }

    // the n tokens that the CTAs have listed, in this one (the first)
    __device__ void gather(int n, const int (&m)[kMostRanks]) {
        for (int t = tid; t < n; t += kThreads) {
            int c = 0, i = t;
#pragma unroll
            for (int k = 0; k < kMostRanks - 1; ++k)
                if (c == k && i >= m[k]) {
                    i -= m[k];
                    c = k + 1;
                }
            sh.many[t] = peer(sh.list + i, c)->x;
        }
        __syncthreads();
    }
    // the weights of n few tokens; the sum of those at or above `least`
    __device__ double weights_of_few(int n, float least) {
        const float x = tid < n ? sh.few[tid] : -INFINITY;
        double w = weight(x);
        w = tid < n && x >= least ? w : 0.0;
        sh.few_w[tid] = w;
        return over_block(w, sh.part, Add());
    }
    // the border among n few tokens, each of which sums (or counts) what is above it: of those at or above `least`
    template <bool MASS> __device__ float among(int n, float least, double above, int above_n, double limit) {
        const float x = tid < n ? sh.few[tid] : -INFINITY;
        double sum[4] = {above, 0.0, 0.0, 0.0};
        int count = above_n;
        if (warp * 32 < n)
            for (int i = 0; i < n; i += 4) {
                const float4 y = *reinterpret_cast<const float4*>(sh.few + i);
                const float u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (MASS) sum[e] += u[e] > x ? sh.few_w[i + e] : 0.0;
                    else count += u[e] > x;
                }
            }
        const bool in = x >= least && tid < n && (MASS ? sum[0] + sum[1] + (sum[2] + sum[3]) < limit : count < limit);
        const float low = over_block(in ? x : INFINITY, sh.fpart, Min()), most = over_block(x, sh.fpart, Max());
        return fminf(low, most);                    // the largest is kept in any case
    }
    // the border among up to kMany tokens, [l, h]: by a finer count, if they are not few; NaN: they are not, nor will they be
    template <bool MASS> __device__ float select(int n, float l, float h, double above, int above_n, double limit, int& few) {
        for (int round = 0; round < 5; ++round) {
            few = 0;
            if (l == h) return l;
            if (n <= kFew || round) {
                if (tid == 0) sh.hit = 0;
                __syncthreads();
                for (int t = tid; t < n; t += kThreads) {
                    const float x = sh.many[t];
                    if (x >= l && x <= h) {
                        const int at = atomicAdd(&sh.hit, 1);
                        if (at < kFew) sh.few[at] = x;
                    }
                }
                __syncthreads();
                few = sh.hit;
                if (few <= kFew) {
                    for (int t = few + tid; t < kFew; t += kThreads) sh.few[t] = -INFINITY;
                    __syncthreads();
                    if (MASS) weights_of_few(few, l);
                    return among<MASS>(few, l, above, above_n, limit);
                }
            }
            const uint32_t k_hi = key_of(h), range = k_hi - key_of(l);
            const int bits = 32 - __clz(range), shift = bits > 8 ? bits - 8 : 0;
            sh.fine[tid] = 0;
            __syncthreads();
            for (int t = tid; t < n; t += kThreads) {
                const float x = sh.many[t];
                if (x >= l && x <= h) atomicAdd(&sh.fine[(k_hi - key_of(x)) >> shift], 1u);
            }
            __syncthreads();
            int from, to;
            weigh<MASS, 1>(false, limit, above, above_n, from, to,
                           [&](uint32_t (&c)[1], uint32_t (&q)[1]) { c[0] = sh.fine[tid]; q[0] = 0; },
                           [&](int b, uint32_t c, uint32_t, double& least, double& most) {
                               const uint64_t k0 = min((uint64_t)b << shift, (uint64_t)range), k1 = min(((uint64_t)(b + 1) << shift) - 1, (uint64_t)range);
                               most = c * weight(of_key(k_hi - (uint32_t)k0)) * (1.0 + 1e-10);
                               least = c * weight(of_key(k_hi - (uint32_t)k1)) * (1.0 - 1e-10);
                           });
            above_n = sh.before_n;
            double sum = 0.0;
            float low = INFINITY, high = -INFINITY;
            for (int t0 = 0; t0 < n; t0 += kThreads) {
                const float x = t0 + tid < n ? sh.many[t0 + tid] : NAN;
                const int b = x >= l && x <= h ? (int)((k_hi - key_of(x)) >> shift) : INT_MAX;
                if (MASS) {
                    const double w = weight(x);
                    sum += b < from ? w : 0.0;
                }
                if (b >= from && b <= to) {
                    low = fminf(low, x);
                    high = fmaxf(high, x);
                }
            }
            if (MASS) above += over_block(sum, sh.part, Add());
            l = over_block(low, sh.fpart, Min());
            h = over_block(high, sh.fpart, Max());
        }
        return NAN;
    }

    // ---- the border: the least value that is kept of those from `least` on.  With MASS the weights above it are below `share` of all, else fewer
    // than `share` tokens are above it; the largest is kept in any case.  Where few are counted, these are also cut to share p of their weights
    // (p below 1).  Returns the value from which on sh.seg has summed all (asked for by `sums`, or MASS), the rest of it with what is listed;
    // infinity: all are listed; NaN: neither.
    template <bool MASS> __device__ float find(double share, float least, bool sums, double p, bool& ruled) {
        Verdict r;                              // R = [r_lo, r_hi] holds the border, `above` and above_n are above R
        r.r_lo = least;
        r.r_hi = top;
        r.above = 0.0;
        r.above_n = 0;
        r.limit = share;
        r.halve = 0;
        const float step = (float)(scale * kSteps), parts = a.parts;
        // steps of 1/32 in log2 w to begin with, rounded to the nearest; by floats where these would be too coarse or too fine, and afterwards
        bool first = true, by_logs = scale > 1e-6 && scale < 1e6;
        for (int level = 0; level < 128; ++level) {
            const uint32_t k_hi = key_of(r.r_hi) >> Limit<T>::spare, range = k_hi - (key_of(r.r_lo) >> Limit<T>::spare);
            const int bits = 32 - __clz(range), shift = bits > 10 ? bits - 10 : 0;
            auto by_log = [&](float x) { return fminf((top - x) * step, kBins - 1.f); };
            auto place = [&](float x) -> int {
                if (by_logs) return __float_as_int(by_log(x) + 8388608.f) & (kBins - 1);
                return (int)((k_hi - (key_of(x) >> Limit<T>::spare)) >> shift) & (kBins - 1);
            };
            if (!r.halve) {
                for (int i = tid; i < kBins / 4; i += kThreads) sh.hist[i] = make_uint4(0, 0, 0, 0);
                __syncthreads();
                const uint32_t hist = smem_u32(sh.hist), one = 1u << a.count_shift;
                for (int s = s0; s < s1; ++s) {
                    const Word<T> w = *reinterpret_cast<const Word<T>*>(data + s * STRIP + lane * N);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float x = widen<T>(w.v[e]);
                        uint32_t at = hist, add = one;
                        if (by_logs) {
                            const float d = by_log(x), up = d + 8388608.f;
                            at += (__float_as_uint(up) & (kBins - 1)) * 4;
                            if (MASS) add += __float_as_uint(fmaf(d - (up - 8388608.f), parts, 8388608.f + 0.5f * parts)) & 0x7fffffu;
                        } else {
                            at += place(x) * 4;
                        }
                        if (x >= r.r_lo && x <= r.r_hi) asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(at), "r"(add) : "memory");
                    }
                }
                cluster_sync();
                if (rank == 0) {
                    int from, to;
                    auto counted = [&](uint32_t (&n)[kPer], uint32_t (&q)[kPer]) {
                        uint4 h[kMostRanks];
                        of_all(sh.hist + tid, h, make_uint4(0, 0, 0, 0));
#pragma unroll
                        for (int e = 0; e < kPer; ++e) n[e] = q[e] = 0;
#pragma unroll
                        for (int c = 0; c < kMostRanks; ++c) {
                            const uint32_t w[4] = {h[c].x, h[c].y, h[c].z, h[c].w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                n[k] += w[k] >> a.count_shift;
                                q[k] += w[k] & (one - 1u);
                            }
                        }
                    };
                    // d of a step's tokens: b + what their parts say, within half a part; w = 2^(-d/32) falls by at most a 6e-5th of itself more than
                    // evenly between the ends of a step, and (top - x) step is rounded by 1024 x 2^-22 of a step
                    const float half = parts > 0.f ? 0.5f / parts : 0.5f;
                    auto by_step = [&](int b, uint32_t n, uint32_t q, double& l, double& m) {
                        const float mean = parts > 0.f && n ? (__fdividef((float)q, (float)n) - 0.5f * parts) * (2.f * half) : 0.f;
                        m = n * (double)exp2f((half - mean - b) * (1.f / kSteps)) * (1.0 + 8e-5);
                        l = b == kBins - 1 ? 0.0 : n * (double)exp2f((-half - mean - b) * (1.f / kSteps)) * (1.0 - 2e-5);
                    };
                    auto by_float = [&](int b, uint32_t n, uint32_t, double& l, double& m) {
                        const uint64_t k0 = min((uint64_t)b << shift, (uint64_t)range), k1 = min(((uint64_t)(b + 1) << shift) - 1, (uint64_t)range);
                        const double w0 = weight(of_spared(k_hi - (uint32_t)k0)), w1 = weight(of_spared(k_hi - (uint32_t)k1));
                        m = n * w0 * (shift ? 1.0 + 1e-10 : 1.0);
                        l = n * w1 * (shift ? 1.0 - 1e-10 : 1.0);
                    };
                    if (by_logs) weigh<MASS, kPer>(first, r.limit, r.above, r.above_n, from, to, counted, by_step);
                    else weigh<MASS, kPer>(first, r.limit, r.above, r.above_n, from, to, counted, by_float);
                    const bool all_few = !MASS && first && sh.to_n <= kFew;         // all that can be kept are few: listed, not summed
                    if (by_logs) {
                        if (warp == 0) {
                            const float e = all_few ? INFINITY : edge_of(from, place);
                            if (lane == 0) sh.verdict.up = e;
                        } else if (warp == 1) {
                            const float e = to == kBins - 1 ? r.r_lo : fmaxf(edge_of(to + 1, place), r.r_lo);
                            if (lane == 0) sh.verdict.lo = e;
                        }
                    } else if (tid == 0) {
                        const uint64_t k = (uint64_t)(to + 1) << shift;
                        sh.verdict.up = all_few ? INFINITY : from == 0 ? above_of(r.r_hi) : of_spared(k_hi - (uint32_t)(((uint64_t)from << shift) - 1));
                        sh.verdict.lo = k > range ? r.r_lo : fmaxf(of_spared(k_hi - (uint32_t)k + 1), r.r_lo);
                    }
                    if (tid == 0) sh.verdict.above_n = all_few ? 0 : sh.before_n;
                }
            } else {                                        // the bounds did not help: by halves, whose weights are summed
                cluster_sync();                             // the last verdict has been read
                if (rank == 0 && tid == 0) {
                    sh.verdict.up = of_spared(k_hi - range / 2);
                    sh.verdict.lo = r.r_lo;
                    sh.verdict.above_n = r.above_n;
                }
            }
            cluster_sync();
            const float up = peer(&sh.verdict, 0)->up, near = peer(&sh.verdict, 0)->lo;
            const int above_n = peer(&sh.verdict, 0)->above_n;
            // ---- what is above those steps, summed (with what is not, the first time: a share is of all); what is in them, listed
            if (tid == 0) sh.listed = 0;
            __syncthreads();
            double sum = 0.0, below = 0.0;
            float least_x = INFINITY, most_x = -INFINITY, least_up = INFINITY;
            const float floor = MASS && first ? least : near;
            for (int s = s0; s < s1; ++s) {
                const int j = s * STRIP + lane * N;
                const Word<T> w = *reinterpret_cast<const Word<T>*>(data + j);
                float x[N], m = -INFINITY;
                uint32_t mine = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    x[e] = widen<T>(w.v[e]);
                    m = fmaxf(m, x[e]);
                }
                if (!__any_sync(kAll, m >= floor)) continue;
                if (MASS && first) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const double v = weight(x[e]);
                        sum += x[e] >= up ? v : 0.0;
                        below += x[e] >= floor && !(x[e] >= up) ? v : 0.0;
                    }
                } else if ((MASS || sums) && __any_sync(kAll, m >= up)) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const double v = weight(x[e]);
                        sum += x[e] >= up ? v : 0.0;
                        if (r.halve && x[e] >= up && x[e] <= r.r_hi) least_up = fminf(least_up, x[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < N; ++e) mine |= (uint32_t)(x[e] >= near && !(x[e] >= up)) << e;
                if (mine) {
                    int at = atomicAdd(&sh.listed, __popc(mine));
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (mine >> e & 1u) {
                            least_x = fminf(least_x, x[e]);
                            most_x = fmaxf(most_x, x[e]);
                            if (at < kList) sh.list[at] = Near{x[e], j + e};
                            ++at;
                        }
                }
                __syncwarp();
            }
            sum = warp_sum64(sum);
            if (MASS && first) below = warp_sum64(below);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                least_x = fminf(least_x, __shfl_xor_sync(kAll, least_x, o));
                most_x = fmaxf(most_x, __shfl_xor_sync(kAll, most_x, o));
                if (r.halve) least_up = fminf(least_up, __shfl_xor_sync(kAll, least_up, o));
            }
            if (lane == 0) {
                sh.seg[warp] = sum;
                sh.part[warp] = below;
                sh.fpart[warp] = least_x;
                sh.fpart2[warp] = most_x;
                sh.fpart3[warp] = least_up;
            }
            __syncthreads();
            if (tid == 0) {
                sum = below = 0.0;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    sum += sh.seg[w];
                    below += sh.part[w];
                    least_x = fminf(least_x, sh.fpart[w]);
                    most_x = fmaxf(most_x, sh.fpart2[w]);
                    least_up = fminf(least_up, sh.fpart3[w]);
                }
                sh.x_above = sum;
                sh.x_below = below;
                sh.x_lo = least_x;
                sh.x_hi = most_x;
                sh.x_up = least_up;
                sh.x_listed = sh.listed;
            }
            cluster_sync();
            // ---- not many are left, or all alike: the border; else once more
            if (rank == 0) {
                int listed[kMostRanks], n = 0, most = 0;
                of_all(&sh.x_listed, listed, 0);
#pragma unroll
                for (int c = 0; c < kMostRanks; ++c) {
                    n += listed[c];
                    most = max(most, listed[c]);
                }
                const double above = MASS ? over_cluster(&sh.x_above, Add()) : 0.0;
                const double limit = MASS && first ? share * (above + over_cluster(&sh.x_below, Add())) : r.limit;
                const float l = over_cluster(&sh.x_lo, Min()), h = over_cluster(&sh.x_hi, Max()), u = r.halve ? over_cluster(&sh.x_up, Min()) : 0.f;
                const bool upper = MASS && r.halve && above >= limit;            // the border is in the upper half
                const bool many = !upper && n <= kMany && most <= kList, rules_too = !MASS && up == INFINITY && many && n <= kFew;
                float found = NAN;
                if (l == h && !upper && !rules_too) found = l;
                else if (many) {
                    int few;
                    gather(n, listed);
                    found = select<MASS>(n, l, h, above, above_n, limit, few);
                    if (rules_too && p < 1.0) {
                        if (few == 0) {                     // (all alike)
                            sh.few[tid] = tid < n ? sh.many[tid] : -INFINITY;
                            __syncthreads();
                        }
                        const double all = weights_of_few(n, found);
                        found = among<true>(n, found, 0.0, 0, p * all);
                    }
                }
                if (tid == 0) {
                    Verdict& v = sh.verdict;
                    v.border = found;
                    v.done = found == found;
                    v.ruled = rules_too;
                    v.r_lo = upper ? u : l;
                    v.r_hi = upper ? r.r_hi : h;
                    v.above = upper ? r.above : above;
                    v.above_n = above_n;
                    v.limit = limit;
                    v.halve = MASS && !by_logs && !r.halve && !v.done &&
                              key_of(v.r_hi) - key_of(v.r_lo) > (key_of(r.r_hi) - key_of(r.r_lo)) / 2;
                }
            }
            cluster_sync();
            const Verdict v = *peer(&sh.verdict, 0);
            border = v.border;
            ruled = v.ruled;
            if (v.done) {
                if (!(MASS || sums || up == INFINITY)) return NAN;
                return sh.listed > kList ? NAN : up;
            }
            r.r_lo = v.r_lo;
            r.r_hi = v.r_hi;
            r.above = v.above;
            r.above_n = v.above_n;
            r.limit = v.limit;
            r.halve = v.halve;
            by_logs = first = false;
        }
        return NAN;
    }
    // the listed tokens that are kept, to the parts that they are in
    __device__ void add_listed() {
        double more = 0.0;
        for (int i = 0; i < sh.listed; i += 32) {
            const Near one = i + lane < sh.listed ? sh.list[i + lane] : Near{-INFINITY, 0};
            const bool mine = one.x >= border && one.slot >= s0 * STRIP && one.slot < s1 * STRIP;
            if (__any_sync(kAll, mine)) {
                const double w = weight(one.x);
                more += mine ? w : 0.0;
            }
        }
        more = warp_sum64(more);
        if (lane == 0) sh.seg[warp] += more;
    }
    __device__ __forceinline__ float of_spared(uint32_t k) const {             // the least float of a key without its spare bits
        const uint32_t full = k << Limit<T>::spare;
        // (negative numbers have ones in their spare bits as keys)
        return of_key(full & 0x80000000u ? full : full | ((1u << Limit<T>::spare) - 1u));
    }
    __device__ __forceinline__ float above_of(float x) const { return of_key(key_of(x) + 1u); }

    // ---- the rules of the row's sequence: the border, and the sums of what is kept.  The total
    __device__ double rules() {
        const int b = a.row_seq ? a.row_seq[row] : row;
        const bool known = (unsigned)b < (unsigned)a.num_seqs;
        const double t = !known ? 1.0 : a.temperature ? (double)a.temperature[b] : a.temperature1;
        const double p = !known ? 1.0 : a.top_p ? (double)a.top_p[b] : a.top_p1, m = !known ? 0.0 : a.min_p ? (double)a.min_p[b] : a.min_p1;
        const int k = !known ? 0 : a.top_k ? a.top_k[b] : a.top_k1;
        only = -1;
        if (!(t > 0.0)) {
            int v = INT_MAX;
            words([&](float x, int j) { if (x == top) v = min(v, lo + j); });
            v = over_block(v, sh.ipart, Min());
            if (tid == 0) sh.x_first = v;
            cluster_sync();
            only = over_cluster(&sh.x_first, Min());
            words([&](float x, int j) { if (x == top && lo + j != only) data[j] = narrow<T>(-INFINITY); });
            __syncwarp();
            border = top;
            scale = base = 0.0;
            return kept_sum();
        }
        scale = 1.4426950408889634074 / t;
        base = -(double)top * scale;
        border = at_least((double)top - 1021.0 / scale);                // what has no weight in 64 bits
        const float least = !(m > 0.0) ? kLowest : m >= 1.0 ? (t < INFINITY ? top : kLowest) : at_least((double)top + t * log(m));      // w >= m
        float from = NAN;
        bool ruled = false;
        if (k > 0 && k < a.vocab) from = find<false>((double)k, border, !(p < 1.0), p, ruled);
        if (p < 1.0 && !ruled) from = find<true>(fmax(p, 0.0), border, true, 1.0, ruled);
        border = fmaxf(border, least);
        if (!(from >= border)) return kept_sum();       // no sums, or of more than is kept
        add_listed();
        return joined();
    }
    __device__ __forceinline__ float at_least(double x) const { return x >= (double)kLowest ? __double2float_ru(x) : kLowest; }

    // ---- the parts' sums, and the whole row's
    __device__ double join(double sum) {
        sum = warp_sum64(sum);
        if (lane == 0) sh.seg[warp] = sum;
        return joined();
    }
    __device__ double joined() {
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

    // ---- the first token up to which the sums of f(slot) exceed `target`, as a slot of the CTA whose piece has it; -1 in the others
    template <typename F> __device__ int search(double target, bool last, F f) {
        double t[kMostRanks], run = 0.0, mine = 0.0;
        of_all(&sh.x_total[turn], t, 0.0);
        if (last) {             // nothing of the others is read any more
            cluster_arrive();
            left = true;
        }
        int owner = -1;
        bool open = true;
#pragma unroll
        for (int c = 0; c < kMostRanks; ++c) {              // the first that exceeds it, else (by rounding) the last that has anything
            if (open && t[c] > 0.0) {
                owner = c;
                mine = run;
                open = !(run + t[c] > target);
            }
            run += t[c];
        }
        if (owner != rank) return -1;
        run = mine;
        int part = 0;
        open = true;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (open && sh.seg[w] > 0.0) {
                part = w;
                mine = run;
                open = !(run + sh.seg[w] > target);
            }
            run += sh.seg[w];
        }
        const int e0 = strips * part / kWarps, n = strips * (part + 1) / kWarps - e0;       // at most kMostStrips
        for (int i = warp; i < n; i += kWarps) {
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < N; ++e) sum += f((e0 + i) * STRIP + lane * N + e);
            sum = warp_sum64(sum);
            if (lane == 0) sh.strip[i] = sum;
        }
        __syncthreads();
        if (warp == 0) {
            run = mine;
            int at = 0;
            open = true;
            for (int i = 0; i < n; ++i) {
                const double w = sh.strip[i];
                if (open && w > 0.0) {
                    at = i;
                    mine = run;
                    open = !(run + w > target);
                }
                run += w;
            }
            const int j = (e0 + at) * STRIP + lane * N;
            double w[N], to = 0.0;
#pragma unroll
            for (int e = 0; e < N; ++e) to += w[e] = f(j + e);
            const double own = to;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double q = __shfl_up_sync(kAll, to, o);
                if (lane >= o) to += q;
            }
            double cum = mine + to - own;
            int hit = -1, end = -1;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                cum += w[e];
                if (w[e] > 0.0) {
                    end = j + e;
                    if (hit < 0 && cum > target) hit = j + e;
                }
            }
            const uint32_t who = __ballot_sync(kAll, hit >= 0);
            hit = who ? __shfl_sync(kAll, hit, __ffs(who) - 1) : __reduce_max_sync(kAll, end);
            if (lane == 0) sh.hit = hit;
        }
        __syncthreads();
        return sh.hit;
    }

    // ---- what the modes do
    __device__ void probs() {
        const double total = top > -INFINITY ? rules() : 0.0, share = total > 0.0 ? 1.0 / total : 0.0;
        if (!(total > 0.0)) border = INFINITY;
        float* out = a.probs + (int64_t)row * a.probs_stride + lo;
        for (int s = s0; s < s1; ++s) {
            const int j = s * STRIP + lane;                 // lanes on neighbouring tokens, as they are written
            float x[N], m = -INFINITY, y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                x[e] = at(j + e * 32);
                m = fmaxf(m, x[e]);
                y[e] = 0.f;
            }
            if (__any_sync(kAll, m >= border)) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const double w = weight(x[e]);
                    y[e] = x[e] >= border ? (float)(w * share) : 0.f;
                }
            }
            if (lo + s * STRIP >= 0 && (s + 1) * STRIP <= used && lo + (s + 1) * STRIP <= a.vocab) {
#pragma unroll
                for (int e = 0; e < N; ++e) out[j + e * 32] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (lo + j + e * 32 >= 0 && lo + j + e * 32 < a.vocab && j + e * 32 < used) out[j + e * 32] = y[e];
            }
        }
    }

    __device__ void draw() {
        if (!(top > -INFINITY)) {
            if (rank == 0 && tid < 32) for (int i = lane; i < a.count; i += 32) put(i, -1, 0.0);
            return;
        }
        auto f = [&](int j) { return kept(at(j)); };
        const double whole = rules();
        double total = whole;
        for (int i = 0; i < a.count; ++i) {
            if (i) total = over_cluster(&sh.x_total[turn], Add());
            if (!(total > 0.0)) {
                if (rank == 0 && tid == 0) put(i, -1, 0.0);
                continue;                           // (so will all the others be)
            }
            const float u = a.uniform[(int64_t)row * a.count + i];
            const int j = search((u > 0.f ? (double)u : 0.0) * total, i + 1 == a.count, f);
            if (j >= 0 && warp == 0) {
                const double w = kept(at(j));
                if (lane == 0) put(i, lo + j, w / whole);
            }
            if (i + 1 == a.count) break;
            if (j >= 0) {                           // it leaves: its warp's part is summed anew
                __syncthreads();
                if (tid == 0) data[j] = narrow<T>(-INFINITY);
                __syncthreads();
                if (j >= s0 * STRIP && j < s1 * STRIP) {
                    double sum = 0.0;
                    for (int s = s0; s < s1; ++s) sum += strip_sum(s, border);
                    sum = warp_sum64(sum);
                    if (lane == 0) sh.seg[warp] = sum;
                }
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
        const double total = rules();
        const int b = a.row_seq[row], which = a.draft_rows ? a.draft_rows[row] : row;
        const bool drafted = (unsigned)which < (unsigned)a.draft_count && (unsigned)b < (unsigned)a.num_seqs;
        if (warp == 0) {
            int n = 0;
            if (drafted) {
                const int r0 = a.node_start[b], r1 = min(a.node_start[b + 1], a.rows);
                for (int r = row + 1; r < r1; r += 32) {
                    const bool mine = r + lane < r1 && a.parents[r + lane] == row - r0;
                    const uint32_t who = __ballot_sync(kAll, mine);
                    const int at = n + __popc(who & ((1u << lane) - 1u));
                    if (mine && at < PA_TREE_MOST_NODES) sh.child[at] = r + lane;
                    n += __popc(who);
                }
            }
            if (lane == 0) sh.children = min(n, PA_TREE_MOST_NODES);
        }
        __syncthreads();
        const Q* q = drafted ? static_cast<const Q*>(a.draft) + (int64_t)which * a.draft_stride : nullptr;
        const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.stride;
        double taken = 0.0, S = total, gone = 0.0;
        for (int i = 0; i < sh.children; ++i) {
            const int r = sh.child[i], c = a.tokens[r];
            if ((unsigned)c >= (unsigned)a.vocab) continue;
            const float xc = widen<T>(x[c]);
            const double w = kept(only >= 0 && c != only ? -INFINITY : fminf(xc, xc == xc ? Limit<T>::most : -INFINITY)), qc = (double)widen<Q>(q[c]);
            if ((double)a.uniform[2 * (int64_t)r] * qc * S < fmax(w - taken * qc, 0.0) * (1.0 - gone)) {
                if (rank == 0 && tid == 0) put(0, c, w / total);
                return;
            }
            taken += S / fmax(1.0 - gone, 1e-18);
            if (a.distinct) gone += qc;
            double sum = 0.0;
            for (int s = s0; s < s1; ++s) {
                const int j = s * STRIP + lane;     // lanes on neighbouring tokens, as q lies
                float xs[N], qs[N], m = -INFINITY;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    xs[e] = at(j + e * 32);
                    m = fmaxf(m, xs[e]);
                }
                if (!__any_sync(kAll, m >= border)) continue;
#pragma unroll
                for (int e = 0; e < N; ++e) qs[e] = xs[e] >= border ? widen<Q>(q[lo + j + e * 32]) : 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const double v = weight(xs[e]) - taken * (double)qs[e];
                    sum += xs[e] >= border && v > 0.0 ? v : 0.0;
                }
            }
            S = join(sum);
        }
        const bool some = taken > 0.0 && S > 0.0;
        if (taken > 0.0 && !some) S = kept_sum();   // nothing is left by rounding, or where q is no distribution
        const float u = a.uniform[2 * (int64_t)row + 1];
        const int j = search((u > 0.f ? (double)u : 0.0) * S, true, [&](int slot) {
            const double w = kept(at(slot));
            return some && w > 0.0 ? fmax(w - taken * (double)widen<Q>(q[lo + slot]), 0.0) : w;
        });
        if (j >= 0 && warp == 0) {
            const double w = kept(at(j));
            if (lane == 0) put(0, lo + j, w / total);
        }
    }
};

template <typename T, typename Q, int MODE> __global__ void __launch_bounds__(kThreads, 3) draw_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Piece<T, Q, MODE> p(a, *reinterpret_cast<Shared*>(smem + a.data_bytes), reinterpret_cast<T*>(smem));
    p.table = exp2((threadIdx.x & 31) / 32.0);
    p.load();
    if constexpr (MODE == PROBS) p.probs();
    else if constexpr (MODE == DRAW) p.draw();
    else p.verify();
    if (!p.left) cluster_arrive();      // no CTA leaves while others read its shared memory
    cluster_wait();
}

template <typename T, typename Q, int MODE> static int launch(Args a, cudaStream_t st) {
    constexpr int N = Word<T>::N;
    // the fewest CTAs whose pieces leave room for three on an SM, more while rows are few
    auto bytes = [&](int ranks) { return (((size_t)a.vocab / N / ranks + 3 + 31) / 32) * 512; };
    const size_t most = device_info().max_smem_optin - sizeof(Shared) - 1024;
    a.ranks = 1;
    while (a.ranks < kMostRanks && (bytes(a.ranks) > 56 * 1024 || (a.rows * a.ranks * 2 <= device_info().sm_count && a.vocab / a.ranks >= 4096))) a.ranks *= 2;
    a.data_bytes = bytes(a.ranks);
    int counts = 1;                     // bits for a CTA's tokens; parts of a step, whose sums must fit beside them
    while (((size_t)1 << counts) <= a.data_bytes / sizeof(T)) ++counts;
    a.count_shift = 32 - counts;
    a.parts = 2 * counts < 32 ? (float)(1 << (32 - 2 * counts < 8 ? 32 - 2 * counts : 8)) : 0.f;
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
