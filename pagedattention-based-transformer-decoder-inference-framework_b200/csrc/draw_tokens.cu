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
// thousand.  2^y is 2^(j/32), from a table of which every lane of a warp holds one, times a polynomial of the fourth degree of the rest |r| <= 1/64
// (Taylor's, error (r ln 2)^5 / 5! <= 1.3e-12): nine operations in 64 bits, of which an SM does 64 a cycle.  With the conversion of the logit and
// the table's word a weight takes 9.4 cycles of an SM for 32 tokens (8.2 with the table in shared memory, which is better where all of a row is
// summed; 10.3 with the conversion by whole numbers): 35 us for 256 rows of 128000, against 20 for reading them.
//
// Rows are read in chunks of up to 64 strips (8192 tokens) by CTAs that know nothing of each other, from memory once and, as far as L2 holds them
// (256 rows of 128000 floats, 131 MB, are more than that), from there once more:
//   count   (where a rule needs it) every chunk's largest logit, and its tokens by 1024 steps of 1/32 in log2 w
//   range   (a CTA a row) the least value that is kept lies in one or two of these steps: found from bounds of their weights, without sorting
//   sum     the weights of what is above those steps, in 64 bits, and a list of what is in them
//   finish  (a cluster of CTAs a row) the border among the listed tokens, the sums of the chunks, the tokens that the numbers draw; verification
//   write   probabilities
// Rows that this does not settle are searched by finish itself, by finer steps: 30 us more for one row of 128000, 1 to 1.4 a row for 256.  These are rows
// with more tokens next to the border than the lists hold (logits that lie closer than a step); a share of what a top_k of more than kFew leaves; and
// rows whose largest logit lies outside the grid of the steps, which is one of x itself, so that chunks need not know it: |top| of 2840 T (4096 where T
// is above 1.4) and more, infinity too, and T outside 1.4e-6 to 1.4e6.
//
// 256 rows of 128000 float logits, rules of their own, replayed: 102 us (the first form, a cluster of CTAs a row that read it four times: 352; one that
// kept it in shared memory: 152, better below 64 rows (one row 25 us against 31), but an SM waits there while one CTA of the cluster
// looks for the border).  Each kernel begins while the one before ends (programmatic launches), which hides their 4 us each.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "cta_pair.cuh"
#include "dynamic_smem.cuh"
#include "pa_common.cuh"
#include "seq_common.cuh"

namespace pa {
namespace drawn {

constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 1024, kPer = kBins / kThreads, kList = 1024, kMany = 2048, kFew = 256, kOwn = 256, kMostRanks = 8, kElsewhere = -2;
constexpr int kWords = 8, kMostChunkStrips = kWords * kWarps, kMostStrips = 512, kMostChunks = 512, kGroup = 8192;       // a group of rows has so many chunks
static_assert(kFew == kThreads && kPer == 4, "a thread for each of few; a word of steps a thread");
constexpr int kMostRows = 1 << 30;          // (so that a row's number and a little more fit 31 bits)
constexpr int kCountShift = 18;             // a step's word: a chunk's tokens (up to 8192) from here on, the sum of their parts below
constexpr uint32_t kAll = 0xffffffffu;
constexpr float kLowest = -3.402823466e38f, kSteps = 32.f, kLogitSteps = 32.f;      // steps of log2 w, or of a logit where these are smaller
constexpr int kParts = 16;                                      // of a step, by which its tokens' mean is known
constexpr float kMagic = 12582912.f;                            // 1.5 x 2^23: sums end at whole numbers
enum Mode { PROBS, DRAW, VERIFY };

struct Near { float x; int token; };
struct Chunk {
    double above, whole;            // sums of the weights at or above `up`, and of all
    float top, lo, hi;              // the largest logit; the ends of what is listed
    int listed, first;              // how many, the lowest of them
};
struct Row {                        // what range and finish leave
    float top, up, lo, border;      // (up may be no number: nothing is at or above it)
    float floor;                    // what has a weight in 64 bits
    int above_n, settled, only, all;
    double scale, share;
};

struct Rest {                       // a node whose last child was refused
    double taken, out, total;       // a, Q, the sum of the kept
    int child;                      // the next one
};

struct Args {
    const void* logits;
    int64_t stride;
    int rows, vocab, ranks, num_seqs;
    int row0, group, chunks, chunk_strips;                  // of the group of rows; chunks of a row, strips of a chunk
    int ranked;                                             // whether a rule may need an order (top_k, top_p, min_p)
    uint32_t* hist;                                         // workspace: [chunks of the group][kBins]
    Near* list;                                             // [chunks][kList]
    Chunk* chunk;
    Row* row;
    Rest* rest;
    double* rest_sum;                                       // [chunks]
    int32_t *open, *opened;                                 // of every round, how many rows are open, and which
    int round;
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
    int draft_count, distinct, most_children;
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
struct Most { __device__ int operator()(int a, int b) const { return max(a, b); } };
struct Max {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
    template <typename V> __device__ static V none() { return -INFINITY; }
};
struct Min {
    __device__ float operator()(float a, float b) const { return fminf(a, b); }
    __device__ int operator()(int a, int b) const { return min(a, b); }
    template <typename V> __device__ static V none() { return std::is_same<V, int>::value ? (V)INT_MAX : (V)INFINITY; }
};

__device__ const double kTable[32] = {     // 2^(j/32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};
__constant__ double kPoly[4] = {0.69314718055994530942, 0.24022650695910071233, 0.05550410866482157995, 0.00961812910762847716};        // ln 2 ^ k / k!
// 2^y = p s for y = d scale of -1022 to 0 (others give some numbers): s = 2^(n/32), from table(n) = 2^(j/32) less j 2^-5 in its exponent's place, j = the
// low five bits of n, so that n can be added there as it is.  The largest logit is taken away before the scaling (d is exact, or off by 2^-53 of itself): a
// difference of two products would be off by 2^-53 of the larger, which small temperatures and large logits make more than all of y
template <typename F> __device__ __forceinline__ double2 exp2_parts(double d, double scale, F table) {
    constexpr double magic = 211106232532992.0;             // 1.5 x 2^47: sums end at multiples of 1/32
    const double at = fma(d, scale, magic);
    const int n = __double2loint(at);
    const double r = fma(d, scale, magic - at), t = table(n);
    double p = fma(r, kPoly[3], kPoly[2]);
    p = fma(r, p, kPoly[1]);
    p = fma(r, p, kPoly[0]);
    p = fma(r, p, 1.0);
    return make_double2(p, __hiloint2double((int)((unsigned)__double2hiint(t) + ((unsigned)n << 15)), __double2loint(t)));
}
__device__ __forceinline__ double table_entry(int j) { return __hiloint2double(__double2hiint(kTable[j]) - (j << 15), __double2loint(kTable[j])); }
// by all lanes of a warp, lane j of which holds entry j
__device__ __forceinline__ double exp2_64(double d, double scale, double table) {
    const double2 w = exp2_parts(d, scale, [&](int n) { return __shfl_sync(kAll, table, n); });
    return w.x * w.y;
}

__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// the rules of a row's sequence
struct Rules {
    double t, p, m, scale;
    float fine;                     // parts of a logit
    int k;
    __device__ Rules(const Args& a, int row) {
        const int b = a.row_seq ? a.row_seq[row] : row;
        const bool known = (unsigned)b < (unsigned)a.num_seqs;
        t = !known ? 1.0 : a.temperature ? (double)a.temperature[b] : a.temperature1;
        p = !known ? 1.0 : a.top_p ? (double)a.top_p[b] : a.top_p1;
        m = !known ? 0.0 : a.min_p ? (double)a.min_p[b] : a.min_p1;
        k = !known ? 0 : a.top_k ? a.top_k[b] : a.top_k1;
        if (k >= a.vocab || k < 0) k = 0;
        scale = greedy() ? 0.0 : fmin(1.4426950408889634074 / t, 1e300);        // (a number, that 0 times it is 0: floats differ by 1e-45 or not at all)
        fine = fmaxf((float)(scale * kSteps), kLogitSteps) * kParts;
    }
    __device__ bool greedy() const { return !(t > 0.0); }
    __device__ bool counts() const { return (k > 0 || p < 1.0) && !greedy() && scale > 1e-6 && scale < 1e6; }
    __device__ static float at_least(double x) { return x >= (double)kLowest ? __double2float_ru(x) : kLowest; }
    // from where on a token has a weight in 64 bits, and one of at least m
    __device__ float floor(float top) const { return at_least((double)top - 1021.0 / scale); }
    __device__ float least(float top) const {
        return !(m > 0.0) ? kLowest : m >= 1.0 ? (t < INFINITY ? top : kLowest) : at_least((double)top + t * log(m));
    }
};
// Steps on a grid that all chunks share, each of kParts: the bits of a float that is the nearest part above kMagic, so that differences of bits are
// differences of parts (up to 2^22 of them; what lies further down differs by more).  `first` ends the step of the largest.
__device__ __forceinline__ uint32_t on_grid(float x, float fine) { return __float_as_uint(fmaf(x, fine, kMagic)); }
__device__ __forceinline__ uint32_t below(uint32_t first, float x, float fine) { return min(first - on_grid(x, fine), (uint32_t)(kBins * kParts - 1)); }

// a row as strips of 32 words of 16 bytes from the word that it begins in; what is outside it is -inf
template <typename T> struct View {
    static constexpr int N = Word<T>::N, STRIP = 32 * N;
    const T* x;
    int V, off, strips;
    __device__ View(const Args& a, int row) : x(static_cast<const T*>(a.logits) + (int64_t)row * a.stride), V(a.vocab) {
        off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
        strips = (V + off + STRIP - 1) / STRIP;
    }
    __device__ __forceinline__ int token(int s, int lane) const { return s * STRIP + lane * N - off; }         // the first of a lane's word
    // whether n strips are whole (for all lanes alike: loads that wait on no branch of their own are on their way together)
    __device__ __forceinline__ bool whole(int s, int n) const { return token(s, 0) >= 0 && token(s + n, 0) <= V; }
    __device__ __forceinline__ Word<T> load_whole(int s, int lane) const {
        const uint4 raw = ldg_stream_128(x + token(s, lane));
        return *reinterpret_cast<const Word<T>*>(&raw);
    }
    __device__ __forceinline__ Word<T> load(int s, int lane) const {
        const int v = token(s, lane);
        Word<T> w;
        if (whole(s, 1)) w = load_whole(s, lane);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e) w.v[e] = v + e >= 0 && v + e < V ? x[v + e] : narrow<T>(-INFINITY);
        }
        return w;
    }
    // f(word, strip, first token of the lane's word) for the strips from s on, `step` apart, several on their way at once
    template <int SOME, typename F> __device__ __forceinline__ void each(int s, int s1, int step, int lane, F f) const {
        for (; s < s1; s += SOME * step) {
            Word<T> w[SOME];
            if (s + (SOME - 1) * step < s1 && whole(s, (SOME - 1) * step + 1)) {
#pragma unroll
                for (int k = 0; k < SOME; ++k) w[k] = load_whole(s + k * step, lane);
            } else {
#pragma unroll
                for (int k = 0; k < SOME; ++k)
                    if (s + k * step < s1) w[k] = load(s + k * step, lane);
            }
#pragma unroll
            for (int k = 0; k < SOME; ++k)
                if (s + k * step < s1) f(w[k], s + k * step, token(s + k * step, lane));
        }
    }
    __device__ __forceinline__ float at(int v) const { return v >= 0 && v < V ? widen<T>(x[v]) : -INFINITY; }
};
// +inf as the type's largest (NaN never is at or above anything, what is made of it does not count)
template <typename T> __device__ __forceinline__ float finite(float x) { return fminf(x, Limit<T>::most); }

// what a block of kThreads does together
struct Block {
    const int tid, warp, lane;
    double table;                   // the lane's entry
    double scale = 0.0, largest = 0.0;      // w = 2^((x - largest) scale)
    __device__ Block() : tid(threadIdx.x), warp(threadIdx.x >> 5), lane(threadIdx.x & 31) { table = table_entry(threadIdx.x & 31); }
    __device__ __forceinline__ void relative_to(float top, double s) {
        scale = s;
        largest = top;
    }
    template <typename T> __device__ __forceinline__ double weight(float x) const { return exp2_64((double)finite<T>(x) - largest, scale, table); }
    template <typename V, typename Op> __device__ V over(V v, V* parts, Op op) {
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
    __device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
        return v;
    }
};

// a chunk's words, all on their way at once, into shared memory, where each is its thread's own; the largest that the thread has
template <typename T> __device__ __forceinline__ float load_chunk(const View<T>& view, int s0, int s1, int warp, int lane, Word<T>* words) {
    constexpr int N = Word<T>::N;
    const T* from = view.x + view.token(s0 + warp, lane);
    Word<T>* to = words + warp * 32 + lane;
    if (view.whole(s0, s1 - s0)) {
#pragma unroll 4
        for (int s = s0 + warp; s < s1; s += kWarps, from += kWarps * View<T>::STRIP, to += kWarps * 32)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
    } else {
        for (int s = s0 + warp; s < s1; s += kWarps) words[(s - s0) * 32 + lane] = view.load(s, lane);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    float m = -INFINITY;
#pragma unroll 2
    for (int s = s0 + warp; s < s1; s += kWarps) {
        const Word<T> w = words[(s - s0) * 32 + lane];
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, widen<T>(w.v[e]));
    }
    return m;
}
// ------------------------------------------------------------------------------------------------------------------- count
// Bound by shared memory's additions, then by memory: 256 x 128000 floats in 32 us (4.1 TB/s), 57 % of the issue slots.  A warp's additions to one word
// go one after the other, so that steps are fine enough (1/32) for a warp's logits to fall into different ones; a step's tokens and parts go in one word.
template <typename T> __global__ void __launch_bounds__(kThreads, 6) count_kernel(const __grid_constant__ Args a) {
    constexpr int N = Word<T>::N;
    __shared__ Word<T> s_words[kMostChunkStrips * 4 / N * 32];
    __shared__ uint4 s_hist[kBins / 4];
    __shared__ float s_part[kWarps], s_fine;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, local = blockIdx.x / a.chunks, c = blockIdx.x - local * a.chunks, row = a.row0 + local;
    let_next_start();
    const View<T> view(a, row);
    if (tid == 0) {                     // (one thread: its divisions take as long as a word of every other)
        const Rules r(a, row);
        s_fine = r.counts() ? r.fine : 0.f;
    }
    const int s0 = c * a.chunk_strips, s1 = min(s0 + a.chunk_strips, view.strips);
    s_hist[tid] = make_uint4(0, 0, 0, 0);
    const float m0 = load_chunk<T>(view, s0, s1, warp, lane, s_words);
    float m = m0;
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
    if (lane == 0) s_part[warp] = m;
    __syncthreads();
    m = s_part[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) m = fmaxf(m, s_part[i]);
    m = finite<T>(m);
    const float fine = s_fine;
    if (fine > 0.f && m > -INFINITY) {
        const uint32_t first = on_grid(m, fine) | (kParts - 1), one = 1u << kCountShift, hist = smem_u32(s_hist);
#pragma unroll 2
        for (int s = s0 + warp; s < s1; s += kWarps) {
            const Word<T> w = s_words[(s - s0) * 32 + lane];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float x = widen<T>(w.v[e]);
                const uint32_t d = below(first, x, fine);
                asm volatile("{\n\t.reg .pred p;\n\tsetp.gt.f32 p, %2, %3;\n\t@p red.shared.add.u32 [%0], %1;\n\t}"
                             ::"r"(hist + (d / kParts) * 4), "r"(one | (d % kParts)), "f"(x), "f"(-INFINITY) : "memory");
            }
        }
        __syncthreads();
        reinterpret_cast<uint4*>(a.hist + (int64_t)blockIdx.x * kBins)[tid] = s_hist[tid];
    }
    if (tid == 0) a.chunk[blockIdx.x].top = m;
}

// ------------------------------------------------------------------------------------------------------------------- range
struct WeighShared {
    double part[kWarps], part2[kWarps];
    float fpart[kWarps];
    int ipart[kWarps], b_lo, b_hi, b_first, before_n, to_n;
};
struct Weigher : Block {
    WeighShared& sh;
    __device__ Weigher(WeighShared& s) : sh(s) {}

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
    template <typename F> __device__ float edge_of(int b, float top, F place) const {
        if (b <= 0) return NAN;                     // nothing is at or above it, nor infinity
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
};

// A chain of dependent steps in one CTA a row (chunks' counts, two scans, the searches for the steps' ends): 15 us for 256 rows, 7 for one.  A kernel of its
// own, or, for few rows, the beginning of sum.  By the last of the row's CTAs in count it is slower (124 us against 103 for the whole call: nothing of
// it is done ahead, and count has 40 registers).
struct Steps {
    alignas(16) uint32_t n[kBins];      // (read four at a time)
    alignas(16) uint32_t q[kBins];
};
struct RangeShared : WeighShared {
    float top[kWarps], edge[2], tops[kMostChunks];
};
// by all threads of a CTA, when count has ended
__device__ __forceinline__ Row range_of(const Args& a, int local, const Rules& r, Steps& steps, RangeShared& sh) {
    Weigher b(sh);
    const int tid = b.tid;
    uint32_t *const s_n = steps.n, *const s_q = steps.q;
    float *const s_tops = sh.tops, *const s_edge = sh.edge;
    for (int i = tid; i < kBins; i += kThreads) s_n[i] = s_q[i] = 0;
    const Chunk* chunk = a.chunk + (int64_t)local * a.chunks;
    float top = -INFINITY;
    for (int c = tid; c < a.chunks; c += kThreads) top = fmaxf(top, s_tops[c] = __ldcg(&chunk[c].top));
    top = b.over(top, sh.top, Max());
    Row out{};
    out.top = top;
    out.settled = 1;
    out.only = -1;
    b.relative_to(top, r.scale);
    const float floor = r.greedy() ? top : r.floor(top), least = r.greedy() ? top : r.least(top);
    out.up = out.lo = fmaxf(floor, least);              // nothing but min_p
    if (r.greedy()) out.up = NAN;
    const float t0 = top * r.fine;
    if (top > -INFINITY && (r.k > 0 || r.p < 1.0) && !r.greedy()) {
        if (!r.counts() || !(fabsf(t0) < 2097152.f)) out.settled = 0;
        else {
            const uint32_t g0 = on_grid(top, r.fine) | (kParts - 1), one = 1u << kCountShift;
            const float log2_w = (float)(r.scale / r.fine), end = __uint_as_float(g0) - kMagic - t0, err = 0.5f + (fabsf(t0) + kBins * kParts) * 1.3e-7f;
            constexpr int SOME = 8;                     // chunks whose words are on their way at once
            for (int c0 = 0; c0 < a.chunks; c0 += SOME) {
                uint32_t h[SOME][kPer];
                int off[SOME];
#pragma unroll
                for (int k = 0; k < SOME; ++k) {
                    const float m = c0 + k < a.chunks ? s_tops[c0 + k] : -INFINITY;
                    off[k] = (int)(min(g0 - (on_grid(m, r.fine) | (kParts - 1)), (uint32_t)(kBins * kParts - 1)) / kParts);
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        h[k][i] = m > -INFINITY ? __ldcg(a.hist + ((int64_t)local * a.chunks + c0 + k) * kBins + tid + i * kThreads) : 0u;
                }
#pragma unroll
                for (int k = 0; k < SOME; ++k)
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (h[k][i]) {
                            const int at = min(tid + i * kThreads + off[k], kBins - 1);
                            atomicAdd(s_n + at, h[k][i] >> kCountShift);
                            atomicAdd(s_q + at, h[k][i] & (one - 1u));
                        }
            }
            __syncthreads();
            auto counted = [&](uint32_t (&n)[kPer], uint32_t (&q)[kPer]) {
#pragma unroll
                for (int i = 0; i < kPer; i += 4) {
                    const uint4 u = reinterpret_cast<const uint4*>(s_n)[tid * (kPer / 4) + i / 4], v = reinterpret_cast<const uint4*>(s_q)[tid * (kPer / 4) + i / 4];
                    n[i] = u.x; n[i + 1] = u.y; n[i + 2] = u.z; n[i + 3] = u.w;
                    q[i] = v.x; q[i + 1] = v.y; q[i + 2] = v.z; q[i + 3] = v.w;
                }
            };
            // a token lies by d parts below the end of the first step, on the mean as many as the parts say, within half of one and the rounding of
            // its product (err); w falls by at most a 6e-5th of itself more than evenly between the ends of a step
            auto bounds = [&](int i, uint32_t n, uint32_t q, double& l, double& m) {
                const float mean = end - i * kParts - (n ? __fdividef((float)q, (float)n) : 0.f);
                m = n * (double)exp2f((mean + err) * log2_w) * (1.0 + 8e-5);
                l = i == kBins - 1 ? 0.0 : n * (double)exp2f((mean - err) * log2_w) * (1.0 - 2e-5);
            };
            auto place = [&](float x) { return (int)(below(g0, x, r.fine) / kParts); };
            int from = 0, to = 0;
            bool few = false;
            if (r.k > 0) {
                b.weigh<false, kPer>(false, (double)r.k, 0.0, 0, from, to, counted, bounds);
                few = sh.to_n <= kFew;                  // all that can be kept are few: listed, not summed
                if (!few && r.p < 1.0) out.settled = 0; // (a share of many: of those from a border that is not known yet)
            } else {
                b.weigh<true, kPer>(true, r.p, 0.0, 0, from, to, counted, bounds);
            }
            if (b.warp < 2) {
                const float e = b.warp == 0 ? (few ? NAN : b.edge_of(from, top, place)) : (to == kBins - 1 ? floor : b.edge_of(to + 1, top, place));
                if (b.lane == 0) s_edge[b.warp] = e;
            }
            __syncthreads();
            out.up = s_edge[0];
            out.lo = fmaxf(s_edge[1], floor);
            out.above_n = few ? 0 : sh.before_n;
            if (least >= out.up) out.up = out.lo = least;           // min_p keeps less: its border is the border
        }
    }
    out.all = out.settled && !r.greedy() && r.p < 1.0 && !(r.k > 0) && !(out.lo >= out.up);
    out.floor = floor;
    out.scale = r.scale;
    return out;
}
template <typename T> __global__ void __launch_bounds__(kThreads) range_kernel(const __grid_constant__ Args a) {
    __shared__ Steps steps;
    __shared__ RangeShared sh;
    let_next_start();
    const Rules r(a, a.row0 + (int)blockIdx.x);
    wait_for_last();
    const Row out = range_of(a, blockIdx.x, r, steps, sh);
    if (threadIdx.x == 0) a.row[blockIdx.x] = out;
}

// --------------------------------------------------------------------------------------------------------------------- sum
// Bound by instructions (60 % of the issue slots, 18 to 36 % of the 64-bit pipe) where all of a row is summed (a share is asked for, or temperatures alone), else by reading: 40 us for
// 256 rows with rules of their own, 58 for 384 of 16-bit logits.  Words of which nothing is kept are passed over by whole warps.
template <typename T, bool RANGES> __global__ void __launch_bounds__(kThreads, 4) sum_kernel(const __grid_constant__ Args a) {
    constexpr int N = Word<T>::N;
    __shared__ Word<T> s_words[kMostChunkStrips * 4 / N * 32];
    __shared__ union {
        Near list[kList];
        Steps steps;
    } s_near;
    Near* const s_list = s_near.list;
    __shared__ double s_above[kWarps], s_whole[kWarps];
    __shared__ float s_lo[kWarps], s_hi[kWarps], s_top[kWarps];
    __shared__ int s_listed, s_first;
    Block b;
    const int tid = b.tid, warp = b.warp, lane = b.lane, local = blockIdx.x / a.chunks, c = blockIdx.x - local * a.chunks, row = a.row0 + local;
    let_next_start();
    const View<T> view(a, row);
    __shared__ Row s_row;
    __shared__ double s_table[32];
    if (tid < 32) s_table[tid] = b.table;
    auto exp2_s = [&](float x) { return exp2_parts((double)x - b.largest, b.scale, [&](int n) { return s_table[n & 31]; }); };
    const int s0 = c * a.chunk_strips, s1 = min(s0 + a.chunk_strips, view.strips);
    if (tid == 0) {
        s_listed = 0;
        s_first = INT_MAX;
        if (blockIdx.x == 0 && a.open) {
            for (int i = 0; i <= a.round; ++i) a.open[i] = 0;           // (here: how many rounds there may be)
        }
        if (a.ranked && !RANGES) {
            wait_for_last();
            s_row = a.row[local];
            if (!s_row.settled) s_row.up = s_row.lo = NAN;
        }
    }
    const float mine_top = load_chunk<T>(view, s0, s1, warp, lane, s_words);
    if constexpr (RANGES) {             // every CTA for itself
        __shared__ RangeShared sh;
        const Rules r(a, row);
        wait_for_last();
        Row out = range_of(a, local, r, s_near.steps, sh);
        if (tid == 0) {
            if (c == 0) a.row[local] = out;
            if (!out.settled) out.up = out.lo = NAN;
            s_row = out;
        }
    }
    if (!a.ranked) {                    // temperatures alone: relative to the chunk's own largest
        const float m = finite<T>(b.over(mine_top, s_top, Max()));
        if (tid == 0) {
            const Rules r(a, row);
            s_row.top = m;
            s_row.scale = r.scale;
            s_row.floor = s_row.up = s_row.lo = r.floor(m);
            if (r.greedy()) s_row.up = NAN, s_row.lo = m;
            s_row.all = 0;
        }
    }
    __syncthreads();
    const float up = s_row.up, lo = s_row.lo, top = s_row.top, floor = s_row.all ? s_row.floor : lo;
    const bool all = s_row.all, lists = !(lo >= up), plain = up == s_row.floor && (top - up) * s_row.scale > 900.0;        // also what is below; whether any is listed; whether all is above
    b.relative_to(top, s_row.scale);
    double above = 0.0, whole = 0.0;
    float least_x = INFINITY, most_x = -INFINITY;
    // (a warp without a token that has a weight sums nothing: below, what has none counts as a little)
    if (top > -INFINITY && !(plain && !__any_sync(kAll, mine_top >= floor))) {
        for (int s = s0 + warp; s < s1; s += kWarps) {
            const Word<T> w = s_words[(s - s0) * 32 + lane];
            float x[N];
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = widen<T>(w.v[e]);
            uint32_t mine = 0;
            if (plain) {                // (what has no weight, or is no number, as 2^-900 or less)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const double2 v = exp2_s(finite<T>(fmaxf(x[e], floor)));
                    above = fma(v.x, v.y, above);
                }
                continue;
            }
            if (all) {                  // (no infinity: range has left such rows to finish)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const double2 u = exp2_s(fmaxf(x[e], floor));
                    const double v = u.x * u.y;
                    whole += v;
                    above += x[e] >= up ? v : 0.0;
                    mine |= (uint32_t)(x[e] >= lo && !(x[e] >= up)) << e;
                }
            } else {
                float m = x[0];
#pragma unroll
                for (int e = 1; e < N; ++e) m = fmaxf(m, x[e]);
                if (!__any_sync(kAll, m >= floor)) continue;
                if (up == up && __any_sync(kAll, m >= up)) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const double v = b.weight<T>(x[e]);
                        above += x[e] >= up ? v : 0.0;
                    }
                }
                if (lists) {
#pragma unroll
                    for (int e = 0; e < N; ++e) mine |= (uint32_t)(x[e] >= lo && !(x[e] >= up)) << e;
                }
            }
            if (!lists) continue;
            if (mine) {
                int at = atomicAdd(&s_listed, __popc(mine));
                const int v = view.token(s, lane);
                atomicMin(&s_first, v + __ffs(mine) - 1);
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (mine >> e & 1u) {
                        const float y = finite<T>(x[e]);
                        least_x = fminf(least_x, y);
                        most_x = fmaxf(most_x, y);
                        if (at < kList) s_list[at] = Near{y, v + e};
                        ++at;
                    }
            }
            __syncwarp();
        }
    }
    above = b.warp_sum(above);
    if (all) whole = b.warp_sum(whole);
    if (lists)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            least_x = fminf(least_x, __shfl_xor_sync(kAll, least_x, o));
            most_x = fmaxf(most_x, __shfl_xor_sync(kAll, most_x, o));
        }
    if (lane == 0) {
        s_above[warp] = above;
        s_whole[warp] = whole;
        s_lo[warp] = least_x;
        s_hi[warp] = most_x;
    }
    __syncthreads();
    const int listed = s_listed;
    for (int i = tid; i < min(listed, kList); i += kThreads) a.list[(int64_t)blockIdx.x * kList + i] = s_list[i];
    if (tid == 0) {
        Chunk out{};
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            out.above += s_above[i];
            out.whole += s_whole[i];
            least_x = fminf(least_x, s_lo[i]);
            most_x = fmaxf(most_x, s_hi[i]);
        }
        out.lo = least_x;
        out.hi = most_x;
        out.listed = listed;
        out.first = s_first;
        Chunk* const to = a.chunk + blockIdx.x;
        if (!a.ranked) to->top = top;           // (else count's, which the row's other CTAs may still read)
        to->above = out.above;
        to->whole = out.whole;
        to->lo = out.lo;
        to->hi = out.hi;
        to->listed = out.listed;
        to->first = out.first;
    }
}

// ------------------------------------------------------------------------------------------------------------------ finish
template <typename Q> __device__ __forceinline__ const Q* draft_row(const Args& a, int row) {       // (of a node that has one)
    return static_cast<const Q*>(a.draft) + (int64_t)(a.draft_rows ? a.draft_rows[row] : row) * a.draft_stride;
}

struct Verdict {                    // of the cluster's first CTA
    float up, lo;                   // what is at or above `up` is summed, what is at or above `lo` listed
    float r_lo, r_hi, border, top;
    double above, limit, total;
    int above_n, done, halve, only, settled;
};

struct Shared : WeighShared {
    union {
        uint4 hist[kBins / 4];
        float many[kMany];          // listed tokens of the row
        int32_t child[PA_TREE_MOST_NODES];
    };
    union {
        Near list[kOwn];
        double strip[kMostStrips];  // sums of a part's strips
    };
    union {
        double few_w[kFew];
        uint32_t fine[kThreads];
    };
    alignas(16) float few[kFew];
    double chunk[kMostChunks];      // sums of the chunks, in the row's order
    int first[kMostChunks + 1];     // listed tokens of the chunks before
    double seg[kWarps];             // or of the warps' parts of this CTA's share of the row
    float fpart2[kWarps], fpart3[kWarps];
    int listed, children, hit;
    // what the other CTAs of the cluster read
    Verdict verdict;
    float x_lo, x_hi, x_up;
    int x_listed;
    double x_below, x_above, x_total[2];
};

template <typename T, typename Q, int MODE>
struct Finish : Weigher {
    static constexpr int N = Word<T>::N, STRIP = 32 * N, FEW = N > 4 ? 2 : 4;           // (strips on their way at once)
    const Args& a;
    Shared& sh;
    const int rank, local, row;
    const View<T> view;
    uint32_t* const gone;           // a bit per token that was drawn (where several are drawn)
    int s0, s1;                     // strips of this warp's part
    float top, border;              // the largest; the least value that is kept
    int only = -1;                  // temperature 0: the one token that is kept
    int turn = 0;                   // of x_total
    bool by_chunks = true;          // the sums are the chunks', in the first CTA
    bool left = false;              // has arrived at the last barrier

    __device__ Finish(const Args& args, Shared& shared, uint32_t* bits, int of_group) :
        Weigher(shared), a(args), sh(shared), rank((int)cluster_ctarank()), local(of_group), row(args.row0 + local), view(args, row), gone(bits) {
        const int parts = a.ranks * kWarps, part = rank * kWarps + warp;
        s0 = (int)((int64_t)view.strips * part / parts);
        s1 = (int)((int64_t)view.strips * (part + 1) / parts);
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

    // ---- weights, by all lanes of a warp
    __device__ __forceinline__ double weight(float x) const { return Block::weight<T>(x); }
    __device__ __forceinline__ double kept(float x, int v) const {
        bool in = x >= border && (only < 0 || v == only);
        if (gone && in) in = !(gone[v >> 5] >> (v & 31) & 1u);
        if (!__any_sync(kAll, in)) return 0.0;
        const double w = weight(x);
        return in ? w : 0.0;
    }
    // the weights of a word's tokens, v and on
    __device__ __forceinline__ void kept_of(const Word<T>& x, int v, double (&w)[N]) const {
        uint32_t in = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) in |= (uint32_t)(widen<T>(x.v[e]) >= border) << e;
        if (only >= 0) in &= only >= v && only < v + N ? 1u << (only - v) : 0u;
        if (gone && in)
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (in >> e & 1u) in &= ~((gone[(v + e) >> 5] >> ((v + e) & 31) & 1u) << e);
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = 0.0;
        if (!__any_sync(kAll, in != 0)) return;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double u = weight(widen<T>(x.v[e]));
            w[e] = in >> e & 1u ? u : 0.0;
        }
    }
    __device__ __forceinline__ double word_sum(const Word<T>& x, int v) const {
        double w[N], sum = 0.0;
        kept_of(x, v, w);
#pragma unroll
        for (int e = 0; e < N; ++e) sum += w[e];
        return sum;
    }
    __device__ double kept_sum() {
        double sum = 0.0;
        view.template each<FEW>(s0, s1, 1, lane, [&](const Word<T>& x, int, int v) { sum += word_sum(x, v); });
        return join(sum);
    }
    // ---- the parts' sums, and the whole row's
    __device__ double join(double sum) {
        sum = warp_sum(sum);
        if (lane == 0) sh.seg[warp] = sum;
        return joined();
    }
    __device__ double joined() {
        by_chunks = false;
        __syncthreads();
        publish();
        cluster_sync();
        return over_cluster(&sh.x_total[turn], Add());
    }
    __device__ void publish() {
        turn ^= 1;              // two places in turn: others may still read the last one
        if (tid == 0) {
            double t = 0.0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) t += sh.seg[w];
            sh.x_total[turn] = t;
        }
    }

    // the weights of n few tokens; the sum of those at or above `least`
    __device__ double weights_of_few(int n, float least) {
        const float x = tid < n ? sh.few[tid] : -INFINITY;
        double w = weight(x);
        w = tid < n && x >= least ? w : 0.0;
        sh.few_w[tid] = w;
        return over(w, sh.part, Add());
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
        const float low = over(in ? x : INFINITY, sh.fpart, Min()), most = over(x, sh.fpart, Max());
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
            if (MASS) above += over(sum, sh.part, Add());
            l = over(low, sh.fpart, Min());
            h = over(high, sh.fpart, Max());
        }
        return NAN;
    }

    // ---- the border: the least value that is kept of those from `least` on.  With MASS the weights above it are below `share` of all, else fewer
    // than `share` tokens are above it; the largest is kept in any case.  By steps of floats, 1024 at a time; what is above those that may hold it
    // is summed exactly.  Returns the value from which on sh.seg has summed all (asked for by `sums`, or MASS), the rest of it with what is listed;
    // NaN: it has not.
    template <bool MASS> __device__ float find(double share, float least, bool sums) {
        Verdict r{};                            // R = [r_lo, r_hi] holds the border, `above` and above_n are above R
        r.r_lo = least;
        r.r_hi = top;
        r.limit = share;
        bool first = true;
        for (int level = 0; level < 128; ++level) {
            const uint32_t k_hi = key_of(r.r_hi) >> Limit<T>::spare, range = k_hi - (key_of(r.r_lo) >> Limit<T>::spare);
            const int bits = 32 - __clz(range), shift = bits > 10 ? bits - 10 : 0;
            cluster_sync();                     // the last verdict, and this CTA's counts, have been read
            if (!r.halve) {
                sh.hist[tid] = make_uint4(0, 0, 0, 0);
                __syncthreads();
                const uint32_t hist = smem_u32(sh.hist);
                view.template each<FEW>(s0, s1, 1, lane, [&](const Word<T>& w, int, int) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float x = finite<T>(widen<T>(w.v[e]));
                        const uint32_t b = ((k_hi - (key_of(x) >> Limit<T>::spare)) >> shift) & (kBins - 1);
                        if (widen<T>(w.v[e]) >= r.r_lo && x <= r.r_hi) asm volatile("red.shared.add.u32 [%0], 1;" ::"r"(hist + 4 * b) : "memory");
                    }
                });
                cluster_sync();
                if (rank == 0) {
                    int from, to;
                    auto counted = [&](uint32_t (&n)[4], uint32_t (&q)[4]) {
                        uint4 h[kMostRanks];
                        of_all(sh.hist + tid, h, make_uint4(0, 0, 0, 0));
#pragma unroll
                        for (int c = 1; c < kMostRanks; ++c) {
                            h[0].x += h[c].x; h[0].y += h[c].y; h[0].z += h[c].z; h[0].w += h[c].w;
                        }
                        n[0] = h[0].x; n[1] = h[0].y; n[2] = h[0].z; n[3] = h[0].w;
                        q[0] = q[1] = q[2] = q[3] = 0;
                    };
                    auto bounds = [&](int b, uint32_t n, uint32_t, double& l, double& m) {
                        const uint64_t k0 = min((uint64_t)b << shift, (uint64_t)range), k1 = min(((uint64_t)(b + 1) << shift) - 1, (uint64_t)range);
                        // (the least value need not be one of the type, whose next one below has no weight in 64 bits, nor any number for it)
                        m = n * weight(fmaxf(of_spared(k_hi - (uint32_t)k0), r.r_lo)) * (1.0 + 1e-10);
                        l = n * weight(fmaxf(of_spared(k_hi - (uint32_t)k1), r.r_lo)) * (1.0 - 1e-10);
                    };
                    weigh<MASS, 4>(first, r.limit, r.above, r.above_n, from, to, counted, bounds);
                    if (tid == 0) {
                        const uint64_t k = (uint64_t)(to + 1) << shift;
                        sh.verdict.up = from == 0 ? (r.r_hi < Limit<T>::most ? of_key(key_of(r.r_hi) + 1u) : NAN) : of_spared(k_hi - (uint32_t)(((uint64_t)from << shift) - 1));
                        sh.verdict.lo = k > range ? r.r_lo : fmaxf(of_spared(k_hi - (uint32_t)k + 1), r.r_lo);
                        sh.verdict.above_n = sh.before_n;
                    }
                }
            } else if (rank == 0 && tid == 0) {             // the bounds did not help: by halves, whose weights are summed
                sh.verdict.up = of_spared(k_hi - range / 2);
                sh.verdict.lo = r.r_lo;
                sh.verdict.above_n = r.above_n;
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
            view.template each<FEW>(s0, s1, 1, lane, [&](const Word<T>& w, int, int v) {
                float x[N], m = -INFINITY;
                uint32_t mine = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    x[e] = widen<T>(w.v[e]);
                    m = fmaxf(m, x[e]);
                }
                if (!__any_sync(kAll, m >= floor)) return;
                if ((MASS && first) || ((MASS || sums) && __any_sync(kAll, m >= up))) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const double u = weight(x[e]);
                        sum += x[e] >= up ? u : 0.0;
                        if (MASS && first) below += x[e] >= floor && !(x[e] >= up) ? u : 0.0;
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
                            const float y = finite<T>(x[e]);
                            least_x = fminf(least_x, y);
                            most_x = fmaxf(most_x, y);
                            if (at < kOwn) sh.list[at] = Near{y, v + e};
                            ++at;
                        }
                }
                __syncwarp();
            });
            sum = warp_sum(sum);
            below = warp_sum(below);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                least_x = fminf(least_x, __shfl_xor_sync(kAll, least_x, o));
                most_x = fmaxf(most_x, __shfl_xor_sync(kAll, most_x, o));
                least_up = fminf(least_up, __shfl_xor_sync(kAll, least_up, o));
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
                const float l = over_cluster(&sh.x_lo, Min()), h = over_cluster(&sh.x_hi, Max()), u = over_cluster(&sh.x_up, Min());
                const bool upper = MASS && r.halve && above >= limit;            // the border is in the upper half
                float found = NAN;
                if (l == h && !upper) found = l;
                else if (!upper && n <= kMany && most <= kOwn) {
                    int few, from = 0;
#pragma unroll
                    for (int c = 0; c < kMostRanks; ++c) {
                        if (tid < listed[c]) sh.many[from + tid] = peer(sh.list + tid, min(c, a.ranks - 1))->x;
                        from += listed[c];
                    }
                    __syncthreads();
                    found = select<MASS>(n, l, h, above, above_n, limit, few);
                }
                if (tid == 0) {
                    Verdict& v = sh.verdict;
                    v.border = found;
                    v.done = found == found;
                    v.r_lo = upper ? u : l;
                    v.r_hi = upper ? r.r_hi : h;
                    v.above = upper ? r.above : above;
                    v.above_n = above_n;
                    v.limit = limit;
                    v.halve = MASS && !r.halve && !v.done && key_of(v.r_hi) - key_of(v.r_lo) > (key_of(r.r_hi) - key_of(r.r_lo)) / 2;
                }
            }
            cluster_sync();
            r = *peer(&sh.verdict, 0);
            border = r.border;
            if (r.done) return (MASS || sums) && sh.listed <= kOwn ? up : NAN;
            first = false;
        }
        return NAN;
    }
    __device__ __forceinline__ float of_spared(uint32_t k) const {             // the least float of a key without its spare bits
        const uint32_t full = k << Limit<T>::spare;
        return of_key(full & 0x80000000u ? full : full | ((1u << Limit<T>::spare) - 1u));      // (negative numbers have ones there as keys)
    }
    // the listed tokens that are kept, to the parts that they are in
    __device__ void add_listed() {
        const int v0 = view.token(s0, 0), v1 = view.token(s1, 0);
        double more = 0.0;
        for (int i = 0; i < sh.listed; i += 32) {
            const Near one = i + lane < sh.listed ? sh.list[i + lane] : Near{-INFINITY, 0};
            const bool mine = one.x >= border && one.token >= v0 && one.token < v1;
            if (__any_sync(kAll, mine)) {
                const double w = weight(one.x);
                more += mine ? w : 0.0;
            }
        }
        more = warp_sum(more);
        if (lane == 0) sh.seg[warp] += more;
    }
    // ---- the border and the sums: from what the kernels before have left, or, where that does not settle it, from the row
    __device__ double rules() {
        const Rules r(a, row);
        wait_for_last();
        if (rank == 0) settle(r);
        cluster_sync();
        const Verdict v = *peer(&sh.verdict, 0);
        top = v.top;
        border = v.border;
        only = v.only;
        relative_to(top, r.scale);
        if (!(top > -INFINITY) || v.settled) return v.total;
        border = r.floor(top);
        float from = NAN;
        if (r.k > 0) from = find<false>((double)r.k, border, !(r.p < 1.0));
        if (r.p < 1.0) from = find<true>(fmax(r.p, 0.0), border, true);
        border = fmaxf(border, r.least(top));
        if (!(from >= border)) return kept_sum();       // no sums, or of more than is kept
        add_listed();
        return joined();
    }
    // (by the first CTA)
    __device__ void settle(const Rules& r) {
        const Chunk* chunk = a.chunk + (int64_t)local * a.chunks;
        const Near* list = a.list + (int64_t)local * a.chunks * kList;
        Row in{};
        if (a.ranked) in = a.row[local];
        float m = -INFINITY, l = INFINITY, h = -INFINITY;
        int n = 0, most = 0, first = INT_MAX;
        double above = 0.0, all = 0.0;
        for (int c = tid; c < a.chunks; c += kThreads) {
            const Chunk one = chunk[c];
            m = fmaxf(m, one.top);
            l = fminf(l, one.lo);
            h = fmaxf(h, one.hi);
            n += one.listed;
            most = max(most, one.listed);
            above += one.above;
            all += one.whole;
            sh.chunk[c] = one.above;
            sh.first[c] = one.listed;
        }
        m = over(m, sh.fpart, Max());
        top = m;
        relative_to(top, r.scale);
        double total = 0.0;
        float found = INFINITY;
        bool settled = true;
        if (!(m > -INFINITY)) {
            // every logit is -inf: nothing is kept
        } else if (r.greedy()) {                        // the lowest of the largest
            for (int c = tid; c < a.chunks; c += kThreads)
                if (chunk[c].top == m && chunk[c].listed) first = min(first, chunk[c].first);
            first = over(first, sh.ipart, Min());
            for (int c = tid; c < a.chunks; c += kThreads) {
                const int v = (c * a.chunk_strips) * STRIP - view.off;
                sh.chunk[c] = first >= v && first < v + a.chunk_strips * STRIP ? 1.0 : 0.0;
            }
            found = m;
            total = 1.0;
        } else if (!a.ranked) {
            found = r.floor(m);
            for (int c0 = 0; c0 < a.chunks; c0 += kThreads) {       // from the chunk's largest to the row's
                const float t = c0 + tid < a.chunks ? chunk[c0 + tid].top : m;
                const double u = weight(fmaxf(t, found)), w = t >= found ? u : 0.0;         // (by all lanes: weights need a warp)
                if (c0 + tid < a.chunks) total += sh.chunk[c0 + tid] *= w;
            }
            total = over(total, sh.part, Add());
        } else if (!in.settled) {
            settled = false;
        } else {
            n = over(n, sh.ipart, Add());
            most = over(most, sh.ipart, Most());
            l = over(l, sh.fpart, Min());
            h = over(h, sh.fpart, Max());
            above = over(above, sh.part, Add());
            all = over(all, sh.part, Add());
            const float least = r.least(m);
            if (n == 0) found = in.up;                  // only min_p: all of it is summed
            else {
                const bool both = r.k > 0 && r.p < 1.0;          // (a count, of which all are listed; a share of it comes next)
                if (l == h) found = l;
                else if (most <= kList) {
                    starts();
                    auto listed = [&](int i) {                  // the i-th listed token
                        int c = 0, end = a.chunks - 1;          // in the last chunk that begins at or before it
                        while (c < end) {
                            const int mid = (c + end + 1) >> 1;
                            if (sh.first[mid] <= i) c = mid;
                            else end = mid - 1;
                        }
                        return list[c * kList + i - sh.first[c]].x;
                    };
                    const double limit = r.k > 0 ? (double)r.k : r.p * all;
                    int count = n, above_n = in.above_n, some;
                    float low = l, high = h;
                    if (n <= kMany) {
                        for (int i = tid; i < n; i += kThreads) sh.many[i] = listed(i);
                        __syncthreads();
                    } else if (r.k > 0) {
                        count = narrow_listed<false>(n, low, high, above, above_n, limit, listed);
                    } else {
                        count = narrow_listed<true>(n, low, high, above, above_n, limit, listed);
                    }
                    if (count > kMany) found = NAN;
                    else if (r.k > 0) found = select<false>(count, low, high, 0.0, above_n, limit, some);
                    else found = select<true>(count, low, high, above, 0, limit, some);
                    if (both && found == found) {
                        const double counted = weights_of_few(n, found);
                        found = among<true>(n, found, 0.0, 0, r.p * counted);
                    }
                } else found = NAN;
                found = fmaxf(found, found == found ? least : found);
            }
            settled = found == found;
            if (settled) {                              // what is listed and kept, to its chunk
                if (l == h) {                           // (all alike)
                    const double w = weight(l);
                    for (int c = tid; c < a.chunks; c += kThreads)
                        if (found <= l) sh.chunk[c] += chunk[c].listed * w;
                } else if (n > 0) {
                    for (int c = warp; c < a.chunks; c += kWarps) {
                        double sum = 0.0;
                        for (int i = sh.first[c]; i < sh.first[c + 1]; i += 32) {
                            const float x = i + lane >= sh.first[c + 1] ? -INFINITY : n <= kMany ? sh.many[i + lane] : list[c * kList + i + lane - sh.first[c]].x;
                            if (__any_sync(kAll, x >= found)) {
                                const double w = weight(x);
                                sum += x >= found ? w : 0.0;
                            }
                        }
                        sum = warp_sum(sum);
                        if (lane == 0) sh.chunk[c] += sum;
                    }
                }
                __syncthreads();
                for (int c = tid; c < a.chunks; c += kThreads) total += sh.chunk[c];
                total = over(total, sh.part, Add());
            }
        }
        __syncthreads();
        if (tid == 0) {
            Verdict& v = sh.verdict;
            v.top = m;
            v.border = found;
            v.only = r.greedy() && m > -INFINITY ? first : -1;
            v.total = total;
            v.settled = settled;
        }
    }
    // Of n listed tokens, [l, h], more than select takes: counted by 1024 steps of floats; those of the steps that may hold the border go to sh.many.
    // How many these are; [l, h], above and above_n become theirs
    template <bool MASS, typename F> __device__ int narrow_listed(int n, float& l, float& h, double& above, int& above_n, double limit, F listed) {
        const uint32_t k_hi = key_of(h), range = k_hi - key_of(l);
        const int bits = 32 - __clz(range), shift = bits > 10 ? bits - 10 : 0;
        sh.hist[tid] = make_uint4(0, 0, 0, 0);
        if (tid == 0) sh.hit = 0;
        __syncthreads();
        uint32_t* hist = reinterpret_cast<uint32_t*>(sh.hist);
        for (int i = tid; i < n; i += kThreads) atomicAdd(hist + ((k_hi - key_of(listed(i))) >> shift), 1u);
        __syncthreads();
        int from, to;
        weigh<MASS, kPer>(false, limit, above, above_n, from, to,
                          [&](uint32_t (&c)[kPer], uint32_t (&q)[kPer]) {
                              const uint4 u = sh.hist[tid];
                              c[0] = u.x; c[1] = u.y; c[2] = u.z; c[3] = u.w;
                              q[0] = q[1] = q[2] = q[3] = 0;
                          },
                          [&](int b, uint32_t c, uint32_t, double& least, double& most) {
                              const uint64_t k0 = min((uint64_t)b << shift, (uint64_t)range), k1 = min(((uint64_t)(b + 1) << shift) - 1, (uint64_t)range);
                              most = c * weight(of_key(k_hi - (uint32_t)k0)) * (1.0 + 1e-10);
                              least = c * weight(of_key(k_hi - (uint32_t)k1)) * (1.0 - 1e-10);
                          });
        above_n = sh.before_n;
        double sum = 0.0;
        float low = INFINITY, high = -INFINITY;
        for (int i0 = 0; i0 < n; i0 += kThreads) {
            const float x = i0 + tid < n ? listed(i0 + tid) : NAN;
            const int b = x == x ? (int)((k_hi - key_of(x)) >> shift) : INT_MAX;
            if (MASS) {
                const double w = weight(x);
                sum += b < from ? w : 0.0;
            }
            if (b >= from && b <= to) {
                low = fminf(low, x);
                high = fmaxf(high, x);
                const int at = atomicAdd(&sh.hit, 1);
                if (at < kMany) sh.many[at] = x;        // (the counts there have been read)
            }
        }
        if (MASS) above += over(sum, sh.part, Add());
        l = over(low, sh.fpart, Min());
        h = over(high, sh.fpart, Max());
        const int some = sh.hit;
        __syncthreads();                            // (select counts there anew)
        return some;
    }
    // sh.first: from the chunks' numbers of listed tokens to where they begin
    __device__ void starts() {
        __syncthreads();
        if (warp == 0) {
            constexpr int EACH = kMostChunks / 32;
            int n[EACH], sum = 0;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int c = lane * EACH + e;
                n[e] = c < a.chunks ? sh.first[c] : 0;
                sum += n[e];
            }
            int to = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int p = __shfl_up_sync(kAll, to, o);
                if (lane >= o) to += p;
            }
            to -= sum;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int c = lane * EACH + e;
                if (c <= a.chunks) sh.first[c] = to;
                to += n[e];
            }
            if (lane == 31 && a.chunks == kMostChunks) sh.first[kMostChunks] = to;
        }
        __syncthreads();
    }

    // by a warp: the first of n sums up to which they exceed `target` (else, by rounding, the last that is anything), and what is before it
    __device__ __forceinline__ int locate(const double* t, int n, double target, double& before) const {
        const int each = (n + 31) / 32, i0 = min(lane * each, n), i1 = min(i0 + each, n);
        double own = 0.0;
        for (int i = i0; i < i1; ++i) own += t[i];
        double to = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double q = __shfl_up_sync(kAll, to, o);
            if (lane >= o) to += q;
        }
        const double from = before + (to - own);
        int hit = -1;
        double run = from, at = from;
        bool open = true;
        for (int i = i0; i < i1; ++i) {
            if (open && t[i] > 0.0) {
                hit = i;
                at = run;
                open = !(run + t[i] > target);
            }
            run += t[i];
        }
        const uint32_t over = __ballot_sync(kAll, !open), some = __ballot_sync(kAll, hit >= 0);
        const int who = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : 0;
        before = __shfl_sync(kAll, at, who);
        return max(__shfl_sync(kAll, hit, who), 0);
    }

    // ---- the first token up to which the sums of f(x, token) exceed `target` (-1: none has any), or kElsewhere in the CTAs that it is not in.  `part` is where it is
    // (f of a word's tokens: their weights)
    template <typename F> __device__ int search(double target, bool last, int& part, F f) {
        double run = 0.0, mine = 0.0;
        bool open = true;               // the first that exceeds it, else (by rounding) the last that has anything
        int owner = 0;
        if (!by_chunks) {
            double t[kMostRanks];
            of_all(&sh.x_total[turn], t, 0.0);
#pragma unroll
            for (int c = 0; c < kMostRanks; ++c) {
                if (open && t[c] > 0.0) {
                    owner = c;
                    mine = run;
                    open = !(run + t[c] > target);
                }
                run += t[c];
            }
        }
        if (last && a.ranks > 1) {      // nothing of the others is read any more
            cluster_arrive();
            left = true;
        }
        if (owner != rank) return kElsewhere;
        part = locate(by_chunks ? sh.chunk : sh.seg, by_chunks ? a.chunks : kWarps, target, mine);
        const int of = rank * kWarps + part, all = a.ranks * kWarps;
        const int e0 = by_chunks ? part * a.chunk_strips : (int)((int64_t)view.strips * of / all);
        const int n = (by_chunks ? min(e0 + a.chunk_strips, view.strips) : (int)((int64_t)view.strips * (of + 1) / all)) - e0;
        view.template each<FEW>(e0 + warp, e0 + n, kWarps, lane, [&](const Word<T>& x, int s, int v) {
            double w[N], sum = 0.0;
            f(x, v, w);
#pragma unroll
            for (int e = 0; e < N; ++e) sum += w[e];
            sum = warp_sum(sum);
            if (lane == 0) sh.strip[s - e0] = sum;
        });
        __syncthreads();
        if (warp == 0) {
            const int at = locate(sh.strip, n, target, mine);
            const int v = view.token(e0 + at, lane);
            double w[N], to = 0.0;
            f(view.load(e0 + at, lane), v, w);
#pragma unroll
            for (int e = 0; e < N; ++e) to += w[e];
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
                    end = v + e;
                    if (hit < 0 && cum > target) hit = v + e;
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
        const double total = rules();
        if (rank == 0 && tid == 0) {
            Row& out = a.row[local];
            out.top = top;
            out.border = total > 0.0 ? border : INFINITY;
            out.only = only;
            out.share = total > 0.0 ? 1.0 / total : 0.0;
        }
    }

    __device__ void draw() {
        const double whole = rules();
        if (by_chunks && rank != 0) return;
        double total = whole;
        auto f = [&](const Word<T>& x, int v, double (&w)[N]) { kept_of(x, v, w); };
        for (int i = 0; i < a.count; ++i) {
            if (!(total > 0.0)) {
                if (rank == 0 && tid == 0) put(i, -1, 0.0);
                continue;                           // (so will all the others be)
            }
            const float u = a.uniform[(int64_t)row * a.count + i];
            int part = 0;
            const int v = search((u > 0.f ? (double)u : 0.0) * total, !by_chunks && i + 1 == a.count, part, f);
            if (v != kElsewhere && warp == 0) {
                const double w = kept(view.at(v), v);
                if (lane == 0) put(i, v, w / whole);
            }
            if (i + 1 == a.count) break;
            if (v >= 0) {                           // it leaves: its part is summed anew
                __syncthreads();
                if (tid == 0) gone[v >> 5] |= 1u << (v & 31);
                __syncthreads();
                const int of = rank * kWarps + part, all = a.ranks * kWarps;
                const int e0 = by_chunks ? part * a.chunk_strips : (int)((int64_t)view.strips * of / all);
                const int e1 = by_chunks ? min(e0 + a.chunk_strips, view.strips) : (int)((int64_t)view.strips * (of + 1) / all);
                const int own = (v + view.off) / STRIP;         // its strip has changed
                if (warp == 0) {
                    const double t = warp_sum(word_sum(view.load(own, lane), view.token(own, lane)));
                    if (lane == 0) sh.strip[own - e0] = t;
                }
                __syncthreads();
                double sum = 0.0;
                for (int s = tid; s < e1 - e0; s += kThreads) sum += sh.strip[s];
                sum = over(sum, sh.part, Add());
                if (tid == 0) (by_chunks ? sh.chunk[part] : sh.seg[part]) = sum;
            }
            __syncthreads();
            if (by_chunks) {
                total = 0.0;
                for (int c = tid; c < a.chunks; c += kThreads) total += sh.chunk[c];
                total = over(total, sh.part, Add());
            } else {
                publish();
                cluster_sync();
                total = over_cluster(&sh.x_total[turn], Add());
            }
        }
    }
    __device__ void put(int i, int id, double p) {
        a.ids[(int64_t)row * a.count + i] = id;
        if (a.logprobs) a.logprobs[(int64_t)row * a.count + i] = id < 0 ? -INFINITY : (float)log(p);
    }

    // ---- verification, in weights: p, S and a times the sum of the kept.  A node's tests go on until a child is kept, or refused: then what it
    // leaves is summed by chunks (rest_kernel) before the next one
    __device__ void children() {
        const int b = a.row_seq[row], which = a.draft_rows ? a.draft_rows[row] : row;
        const bool drafted = (unsigned)which < (unsigned)a.draft_count && (unsigned)b < (unsigned)a.num_seqs;
        __syncthreads();
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
            if (lane == 0) sh.children = min(n, a.most_children);       // (of more there would be no round)
        }
        __syncthreads();
    }
    // true: the node's id is given, or a refused child's rest has to be summed (a.rest); false: no child is left
    __device__ bool tests(Rest st, double S) {
        const Q* q = draft_row<Q>(a, row);
        for (int i = st.child; i < sh.children; ++i) {
            const int r = sh.child[i], c = a.tokens[r];
            if ((unsigned)c >= (unsigned)a.vocab) continue;
            const double w = kept(view.at(c), c), qc = (double)widen<Q>(q[c]);
            if ((double)a.uniform[2 * (int64_t)r] * qc * S < fmax(fma(-st.taken, qc, w), 0.0) * (1.0 - st.out)) {
                if (rank == 0 && tid == 0) put(0, c, w / st.total);
                return true;
            }
            st.taken += S / fmax(1.0 - st.out, 1e-18);
            if (a.distinct) st.out += qc;
            st.child = i + 1;
            if (rank == 0 && tid == 0) {
                a.rest[local] = st;
                a.opened[(int64_t)a.round * a.group + atomicAdd(a.open + a.round, 1)] = local;      // (their order changes nothing)
            }
            return true;
        }
        return false;
    }
    __device__ void draw_from(double S, double taken, double total) {
        const Q* q = draft_row<Q>(a, row);
        const float u = a.uniform[2 * (int64_t)row + 1];
        int part;
        const int v = search((u > 0.f ? (double)u : 0.0) * S, true, part, [&](const Word<T>& x, int token, double (&w)[N]) {
            float y[N];
            if (taken > 0.0)            // (of places outside the row, whose weights are 0, any)
#pragma unroll
                for (int e = 0; e < N; ++e) y[e] = widen<Q>(q[min(max(token + e, 0), view.V - 1)]);
            kept_of(x, token, w);
            if (taken > 0.0)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const double u = fma(-taken, (double)y[e], w[e]);
                    w[e] = u > 0.0 ? u : 0.0;
                }
        });
        if (v != kElsewhere && warp == 0) {
            const double w = kept(view.at(v), v);
            if (lane == 0) put(0, v, w / total);
        }
    }
    __device__ void verify() {
        const double total = rules();
        Rest st{};
        st.total = total;
        if (rank == 0 && tid == 0) {
            Row& out = a.row[local];
            out.top = top;
            out.border = border;
            out.only = only;
            out.scale = scale;
            if (!(total > 0.0)) put(0, -1, 0.0);
        }
        if (!(total > 0.0)) return;
        children();
        if (!tests(st, total)) draw_from(total, 0.0, total);
    }
    __device__ void go_on() {
        const Rest st = a.rest[local];
        const Row in = a.row[local];
        top = in.top;
        border = in.border;
        only = in.only;
        relative_to(top, in.scale);
        const double* sums = a.rest_sum + (int64_t)local * a.chunks;
        double S = 0.0;
        for (int c = tid; c < a.chunks; c += kThreads) S += sh.chunk[c] = sums[c];
        S = over(S, sh.part, Add());
        children();
        if (S > 0.0 && tests(st, S)) return;
        if (S > 0.0) draw_from(S, st.taken, st.total);
        else draw_from(kept_sum(), 0.0, st.total);          // nothing is left by rounding, or where q is no distribution: p
    }
};

// Again dependent steps: 27 us for 256 rows, 10 for one.  Two CTAs an SM (191 registers without the bound: one; 112 us against 103 for the whole call)
template <typename T, typename Q, int MODE> __global__ void __launch_bounds__(kThreads, 2) finish_kernel(const __grid_constant__ Args a) {
    __shared__ Shared sh;
    extern __shared__ uint32_t bits[];
    if (MODE == DRAW && a.count > 1) {
        for (int i = threadIdx.x; i < (a.vocab + 31) / 32; i += kThreads) bits[i] = 0;
        __syncthreads();
    }
    let_next_start();
    Finish<T, Q, MODE> p(a, sh, MODE == DRAW && a.count > 1 ? bits : nullptr, (int)(blockIdx.x / a.ranks));
    if constexpr (MODE == PROBS) p.probs();
    else if constexpr (MODE == DRAW) p.draw();
    else p.verify();
    if (!p.left) cluster_arrive();      // no CTA leaves while others read its shared memory
    cluster_wait();
}

// -------------------------------------------------------------------------------------------------------------------- rest
// What refused children have left of a chunk: max(w - taken q, 0).  Words of the logits, and of q where it lies alike, several on their way at once.  A launch
// for every child that a node may have, of the rows whose last test has failed: 64 chains of six, 16-bit, 39 us (by the CTA that
// tests, a row took 60 to 100); without such a row 3
template <typename T, typename Q> __global__ void __launch_bounds__(kThreads, 3) rest_kernel(const __grid_constant__ Args a) {
    constexpr int N = Word<T>::N, QN = 16 / (int)sizeof(Q), SOME = sizeof(T) < 4 ? 2 : 4;
    __shared__ double s_part[kWarps];
    Block b;
    const int lane = b.lane;
    let_next_start();
    wait_for_last();
    const int all = a.open[a.round - 1] * a.chunks;
    for (int i = blockIdx.x; i < all; i += gridDim.x) {
        const int local = a.opened[(int64_t)(a.round - 1) * a.group + i / a.chunks], c = i % a.chunks, row = a.row0 + local;
        const Rest st = a.rest[local];
        const View<T> view(a, row);
        const Row r = a.row[local];
        b.relative_to(r.top, r.scale);
        const Q* q = draft_row<Q>(a, row);
        const int s0 = c * a.chunk_strips, s1 = min(s0 + a.chunk_strips, view.strips);
        const bool alike = ((uintptr_t)(q - view.off) & 15) == 0;
        double sum = 0.0;
        auto add = [&](const Word<T>& x, int v, const float (&y)[N]) {
            float m = -INFINITY;
#pragma unroll
            for (int e = 0; e < N; ++e) m = fmaxf(m, widen<T>(x.v[e]));
            if (!__any_sync(kAll, m >= r.border)) return;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float z = widen<T>(x.v[e]);
                const double u = fma(-st.taken, (double)y[e], b.weight<T>(z));         // (rounded alike wherever it is taken)
                if (z >= r.border && (r.only < 0 || v + e == r.only) && u > 0.0) sum += u;
            }
        };
        for (int s = s0 + b.warp; s < s1; s += SOME * kWarps) {
            if (alike && s + (SOME - 1) * kWarps < s1 && view.whole(s, (SOME - 1) * kWarps + 1)) {
                Word<T> x[SOME];
                float y[SOME][N];
#pragma unroll
                for (int k = 0; k < SOME; ++k) x[k] = view.load_whole(s + k * kWarps, lane);
#pragma unroll
                for (int k = 0; k < SOME; ++k) {
                    const int v = view.token(s + k * kWarps, lane);
                    if constexpr (QN <= N) {
#pragma unroll
                        for (int e = 0; e < N; e += QN) {
                            const uint4 raw = ldg_stream_128(q + v + e);
#pragma unroll
                            for (int i = 0; i < QN; ++i) y[k][e + i] = widen<Q>(reinterpret_cast<const Q*>(&raw)[i]);
                        }
                    } else {                            // (eight of q to a word of its own, four of the logits)
                        const uint2 raw = ldg_stream_64(q + v);
#pragma unroll
                        for (int i = 0; i < N; ++i) y[k][i] = widen<Q>(reinterpret_cast<const Q*>(&raw)[i]);
                    }
                }
#pragma unroll
                for (int k = 0; k < SOME; ++k) add(x[k], view.token(s + k * kWarps, lane), y[k]);
            } else {
                for (int k = 0; k < SOME && s + k * kWarps < s1; ++k) {
                    const int v = view.token(s + k * kWarps, lane);
                    float y[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] = v + e >= 0 && v + e < view.V ? widen<Q>(q[v + e]) : 0.f;
                    add(view.load(s + k * kWarps, lane), v, y);
                }
            }
        }
        sum = b.over(sum, s_part, Add());
        if (b.tid == 0) a.rest_sum[(int64_t)local * a.chunks + c] = sum;
    }
}

// Where a node's tests go on after that
template <typename T, typename Q> __global__ void __launch_bounds__(kThreads, 2) go_on_kernel(const __grid_constant__ Args a) {
    __shared__ Shared sh;
    let_next_start();
    wait_for_last();
    const int i = blockIdx.x;           // of the rows that are open, which a list has
    if (i >= a.open[a.round - 1]) return;
    Finish<T, Q, VERIFY> p(a, sh, nullptr, a.opened[(int64_t)(a.round - 1) * a.group + i]);
    p.go_on();
}

// ------------------------------------------------------------------------------------------------------------------- write
// 64 x 50257: 15 us, for 13 MB from L2 and as many written; weights are formed anew, which costs less than keeping them in 64 bits
template <typename T> __global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ Args a) {
    constexpr int N = Word<T>::N, STRIP = 32 * N;
    Block b;
    const int local = blockIdx.x / a.chunks, c = blockIdx.x - local * a.chunks, row = a.row0 + local;
    const View<T> view(a, row);
    const Rules rules(a, row);
    const int s0 = c * a.chunk_strips, s1 = min(s0 + a.chunk_strips, view.strips);
    wait_for_last();
    const Row r = a.row[local];
    b.relative_to(r.top, rules.scale);
    float* out = a.probs + (int64_t)row * a.probs_stride;
#pragma unroll 2
    for (int s = s0 + b.warp; s < s1; s += kWarps) {
        const int v = s * STRIP + b.lane - view.off;                // lanes on neighbouring tokens, as they are written
        float x[N], y[N], m = -INFINITY;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            x[e] = view.at(v + e * 32);
            if (r.only >= 0 && v + e * 32 != r.only) x[e] = -INFINITY;
            m = fmaxf(m, x[e]);
            y[e] = 0.f;
        }
        if (__any_sync(kAll, m >= r.border))
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const double w = b.weight<T>(x[e]);
                y[e] = x[e] >= r.border ? (float)(w * r.share) : 0.f;
            }
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (v + e * 32 >= 0 && v + e * 32 < a.vocab) out[v + e * 32] = y[e];
    }
}

// ------------------------------------------------------------------------------------------------------------------ launch
// Chunks of 8192 tokens, of 4096 where there are fewer of these than SMs (16 rows of 50257 are 112 or 208 CTAs)
struct Cut {
    int chunks, chunk_strips, group;        // of a row; rows that go together
};
static Cut cut_of(int type, int rows, int vocab) {
    const int words = type == PA_TYPE_F32 ? 4 : 8, strips = (vocab + words - 1 + 32 * words - 1) / (32 * words);        // of a row that begins inside a word
    Cut c;
    c.chunk_strips = type == PA_TYPE_F32 ? 64 : 32;
    auto chunks = [&] { return (strips + c.chunk_strips - 1) / c.chunk_strips; };
    while (c.chunk_strips > (type == PA_TYPE_F32 ? 32 : 16) && (int64_t)rows * chunks() < device_info().sm_count) c.chunk_strips /= 2;
    c.chunks = chunks();
    c.group = std::min(rows, std::max(1, kGroup / c.chunks));
    return c;
}
static size_t row_bytes(const Cut& c) { return (size_t)c.chunks * (kBins * 4 + kList * sizeof(Near) + sizeof(Chunk) + sizeof(double)) + sizeof(Row) + sizeof(Rest); }
static size_t round_bytes(const Cut& c) { return ((size_t)c.group + 1) * 4; }

template <auto Kernel> static cudaError_t start(const Args& a, unsigned ctas, unsigned cluster, size_t smem, bool first, cudaStream_t st) {
    const cudaError_t e = smem ? allow_dynamic_smem<Kernel>(smem) : cudaSuccess;
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (cluster) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = cluster;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    if (!first) {                   // the first kernel begins when all before it have ended, the others while theirs does
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, Kernel, a);
}

template <typename T, typename Q, int MODE> static int launch(Args a, int type, int most_children, void* workspace, cudaStream_t st) {
    if ((size_t)a.vocab * sizeof(T) > PA_DRAW_MOST_ROW_BYTES) return PA_ERR_UNSUPPORTED;
    const Cut c = cut_of(type, a.rows, a.vocab);
    a.chunks = c.chunks;
    a.chunk_strips = c.chunk_strips;
    a.ranked = a.top_k || a.top_k1 > 0 || a.top_p || a.top_p1 < 1.0 || a.min_p || a.min_p1 > 0.0;
    a.ranks = 1;
    while (a.ranks < kMostRanks && (int64_t)a.rows * a.ranks <= device_info().sm_count) a.ranks *= 2;
    uint8_t* at = static_cast<uint8_t*>(workspace);
    const size_t n = (size_t)c.group * c.chunks;
    a.hist = reinterpret_cast<uint32_t*>(at);
    at += n * kBins * 4;
    a.list = reinterpret_cast<Near*>(at);
    at += n * kList * sizeof(Near);
    a.chunk = reinterpret_cast<Chunk*>(at);
    at += n * sizeof(Chunk);
    a.rest_sum = reinterpret_cast<double*>(at);
    at += n * sizeof(double);
    a.rest = reinterpret_cast<Rest*>(at);
    at += c.group * sizeof(Rest);
    a.row = reinterpret_cast<Row*>(at);
    at += c.group * sizeof(Row);
    if (MODE == VERIFY) {
        a.open = reinterpret_cast<int32_t*>(at);
        a.opened = a.open + most_children + 1;
    }
    a.group = c.group;
    a.round = a.most_children = most_children;
    const int rows = a.rows;
    for (int r = 0; r < rows; r += c.group) {
        a.row0 = r;
        const unsigned some = (unsigned)std::min(c.group, rows - r), ctas = some * (unsigned)c.chunks;
        cudaError_t e = cudaSuccess;
        // up to two CTAs for an SM: each finds its row's range by itself, a launch less, and nothing else would run there meanwhile (one row of 50257, 13
        // CTAs: 32.9 -> 30.9 us; 33 x 32001 half, 264 CTAs: 31.8 -> 30; where there are more it takes longer: 64 x 50257, 448 CTAs: 50.9 -> 53.1)
        const bool at_once = a.ranked && ctas <= 2u * (unsigned)std::max(0, device_info().sm_count);
        if (a.ranked) {
            e = start<count_kernel<T>>(a, ctas, 0, 0, true, st);
            if (e == cudaSuccess && !at_once) e = start<range_kernel<T>>(a, some, 0, 0, false, st);
        }
        if (e == cudaSuccess) e = at_once ? start<sum_kernel<T, true>>(a, ctas, 0, 0, false, st) : start<sum_kernel<T, false>>(a, ctas, 0, 0, !a.ranked, st);
        Args f = a;
        f.round = 0;
        if (e == cudaSuccess) e = start<finish_kernel<T, Q, MODE>>(f, some * a.ranks, a.ranks, MODE == DRAW && a.count > 1 ? (size_t)(a.vocab + 31) / 32 * 4 : 0, false, st);
        if (e == cudaSuccess && MODE == PROBS) e = start<write_kernel<T>>(a, ctas, 0, 0, false, st);
        if constexpr (MODE == VERIFY) {
            f.ranks = 1;                // (few nodes come so far)
            const unsigned sms = (unsigned)std::max(1, device_info().sm_count);
            for (f.round = 1; f.round <= most_children && e == cudaSuccess; ++f.round) {
                e = start<rest_kernel<T, Q>>(f, std::min(ctas, 16 * sms), 0, 0, false, st);
                if (e == cudaSuccess) e = start<go_on_kernel<T, Q>>(f, some, 0, 0, false, st);
            }
        }
        if (e != cudaSuccess) return (int)e;
    }
    return PA_OK;
}

template <int MODE> static int launch(const Args& a, int type, int draft_type, int most_children, void* workspace, cudaStream_t st) {
    if constexpr (MODE == VERIFY) {
        auto of = [&](auto t) {
            typedef decltype(t) T;
            return draft_type == PA_TYPE_F32 ? launch<T, float, MODE>(a, type, most_children, workspace, st) : draft_type == PA_TYPE_F16 ? launch<T, __half, MODE>(a, type, most_children, workspace, st) :
                   draft_type == PA_TYPE_BF16 ? launch<T, bf16_t, MODE>(a, type, most_children, workspace, st) : PA_ERR_UNSUPPORTED;
        };
        return type == PA_TYPE_F32 ? of(float()) : type == PA_TYPE_F16 ? of(__half()) : type == PA_TYPE_BF16 ? of(bf16_t()) : PA_ERR_UNSUPPORTED;
    } else {
        return type == PA_TYPE_F32 ? launch<float, float, MODE>(a, type, most_children, workspace, st) : type == PA_TYPE_F16 ? launch<__half, float, MODE>(a, type, most_children, workspace, st) :
               type == PA_TYPE_BF16 ? launch<bf16_t, float, MODE>(a, type, most_children, workspace, st) : PA_ERR_UNSUPPORTED;
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
static bool holds(const void* workspace, size_t bytes, size_t need) { return workspace && (uintptr_t)workspace % 16 == 0 && bytes >= need; }
static bool usable(const void* logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules) {
    return rows >= 0 && rows <= kMostRows && vocab > 0 && stride >= vocab && rules && rules->num_seqs >= 0 && (rows == 0 || logits) &&
           (uintptr_t)logits % (type == PA_TYPE_F32 ? 4 : 2) == 0;
}

}  // namespace drawn
}  // namespace pa

using namespace pa;

PA_API size_t pa_draw_workspace_bytes(int type, int rows, int vocab, int most_children) {
    if (rows <= 0 || vocab <= 0 || most_children < 0 || type < PA_TYPE_F32 || type > PA_TYPE_BF16) return 0;
    if ((size_t)vocab * (type == PA_TYPE_F32 ? 4 : 2) > PA_DRAW_MOST_ROW_BYTES) return 0;
    const drawn::Cut c = drawn::cut_of(type, rows, vocab);
    return drawn::row_bytes(c) * c.group + drawn::round_bytes(c) * ((size_t)most_children + 1);
}

PA_API int pa_truncated_softmax(const void* d_logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules, float* d_probs,
                                int64_t probs_stride, void* d_workspace, size_t workspace_bytes, pa_stream_t stream) {
    using namespace pa::drawn;
    PA_CHECK_ARG(usable(d_logits, type, stride, rows, vocab, rules) && probs_stride >= vocab);
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_probs);
    const uintptr_t in = (uintptr_t)d_logits, out = (uintptr_t)d_probs;
    const uintptr_t in_end = in + ((size_t)(rows - 1) * stride + vocab) * (type == PA_TYPE_F32 ? 4 : 2), out_end = out + ((size_t)(rows - 1) * probs_stride + vocab) * 4;
    PA_CHECK_ARG(in >= out_end || out >= in_end);
    Args a = args(d_logits, stride, rows, vocab, rules);
    a.probs = d_probs; a.probs_stride = probs_stride;
    if (!holds(d_workspace, workspace_bytes, pa_draw_workspace_bytes(type, rows, vocab, 0))) return PA_ERR_WORKSPACE;
    return launch<PROBS>(a, type, 0, 0, d_workspace, as_stream(stream));
}

PA_API int pa_draw_tokens(const void* d_logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules, const float* d_uniform,
                          int count, int32_t* d_ids, float* d_logprobs, void* d_workspace, size_t workspace_bytes, pa_stream_t stream) {
    using namespace pa::drawn;
    PA_CHECK_ARG(usable(d_logits, type, stride, rows, vocab, rules) && count > 0);
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_uniform && d_ids);
    Args a = args(d_logits, stride, rows, vocab, rules);
    a.uniform = d_uniform; a.count = count; a.ids = d_ids; a.logprobs = d_logprobs;
    if (!holds(d_workspace, workspace_bytes, pa_draw_workspace_bytes(type, rows, vocab, 0))) return PA_ERR_WORKSPACE;
    return launch<DRAW>(a, type, 0, 0, d_workspace, as_stream(stream));
}

PA_API int pa_verify_drafts(const void* d_logits, int type, int64_t stride, int rows, int vocab, const pa_draw_rules* rules, const float* d_uniform,
                            const int32_t* d_tokens, const int32_t* d_parents, const int32_t* d_node_start, int most_children, const void* d_draft, int draft_type,
                            int64_t draft_stride, int draft_count, const int32_t* d_draft_rows, int distinct, int32_t* d_ids, float* d_logprobs,
                            void* d_workspace, size_t workspace_bytes, pa_stream_t stream) {
    using namespace pa::drawn;
    PA_CHECK_ARG(usable(d_logits, type, stride, rows, vocab, rules) && draft_count >= 0 && most_children >= 0 && most_children < PA_TREE_MOST_NODES && (draft_count == 0 || (d_draft && draft_stride >= vocab && (uintptr_t)d_draft % (draft_type == PA_TYPE_F32 ? 4 : 2) == 0)));
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_uniform && d_ids && d_tokens && d_parents && d_node_start && rules->d_row_seq && (d_draft_rows || draft_count >= rows));
    Args a = args(d_logits, stride, rows, vocab, rules);
    a.uniform = d_uniform; a.count = 1; a.ids = d_ids; a.logprobs = d_logprobs;
    a.tokens = d_tokens; a.parents = d_parents; a.node_start = d_node_start; a.draft = d_draft; a.draft_stride = draft_stride;
    a.draft_count = draft_count; a.draft_rows = d_draft_rows; a.distinct = distinct;
    if (!holds(d_workspace, workspace_bytes, pa_draw_workspace_bytes(type, rows, vocab, most_children))) return PA_ERR_WORKSPACE;
    return launch<VERIFY>(a, type, draft_type, most_children, d_workspace, as_stream(stream));
}
