// tree_terms.cu -- attention of drafted trees on the 5th-generation tensor cores with factors in several terms: float queries over half pages, and
// int8 pages (tree_attention.cuh has the work list, tree_stream.cu the join).
//
// Keys are the rows of the products, query rows (and their terms) the columns: a tile is 128 keys whatever the number of query rows, and
// staged keys and values are the A operands as they stand in their pages.
//     S^T = K Q^T      [128 keys x terms R],   O^T = V^T P^T   [D x terms R],   R = 16, 32 or 64 query rows of a block
//   half pages    two terms of half each for a query (its row scaled by a power of two first) and for a weight: 22 bits of every factor
//   int8 pages    kind::i8 with signed digits: a query row as 23-bit integers relative to its largest (three digits), the weights times their
//                 values' scales as 31-bit ones (four) relative to the largest possible, where a tile's values have scales alike; where they
//                 have not, relative to the row's largest in the tile, so that a key which a row does not see, or hardly weighs, takes no bits from
//                 the others.  Products and their sums are exact integers, no byte is converted
// A row's reference moves only when a score exceeds it by more than 2^8 (int8: 2^7), which the terms leave room for: after a piece's first tile
// hardly ever.  (So the formula's 1e-6 stands beside a sum that may be up to 2^8 times the one relative to the largest score: 1e-6 of a result.)
// The sums of a tile leave the tensor cores as they are and are added up in float registers (the tensor cores cut where float rounds: over a
// long context that would add up).  A row's terms are neighbours in P^T, whose rows are keys: a thread stores four query rows at once.
//   warps 0-7    softmax, one thread per key and half of the rows (blocks of 16 rows: warps 0-3 and all rows, two CTAs an SM): its scores, one vote
//                per tile whether a row's reference has to move (then the maxima by warp and through shared memory), weights to shared memory
//                as the MN-major B operand
//   next four    one thread per value column: the tile's sums into its R float sums, rescaled where a reference moved
//   next         issues  S^T of tile t + 1  and  O^T of tile t;  scores and sums are double-buffered in TMEM
//   next         TMA boxes of 16 keys into a ring (int8: and the rows' scales), page ids a tile ahead
//   last two     the next piece's queries into the K-major B operand, their factors and masks
//
// What bounds it: the latency of a tile's chain (scores, vote, weights, products, sums) at one or two softmax warps for each quarter of an SM, and
// of a piece's beginning and end, some 6 us.  12 sequences of 4K keys, 32 heads: half pages and 32 float rows 152 us, 5.3 TB/s; int8 pages and 16
// float rows 87 us, 4.8 TB/s; 48 sequences of 1 to 2K keys, int8 pages 128 us, 3.5 TB/s (values' scales that differ by more than 8 in every tile:
// 255); 16 sequences of 4K keys, 128 rows a kv head (blocks of 64) 134 us, 257 TFLOP/s of the formula's operations.  Rows as the columns of the products keep the tile at 128 keys for any number of rows: as rows
// they would fill 128 lanes with 16.  Digits and terms instead of tf32 or a conversion to half: int8 pages stay as they are, and float results keep
// 22 bits.  Reading a tile's maximum before its exponentials for every tile took 223 us where votes on 2^8 took 192 (before the shares counted
// beginnings and ends).  Instructions are what its caches are short of: a branch more in the softmax, never taken, took 14 of 107 us where pieces are
// short.
#include "tcgen05_utils.cuh"
#include "tree_pieces.cuh"

namespace pa {
namespace tterms {

using namespace tc;

constexpr int KT = 128, kNotes = 32;
constexpr float kDigits = 8.3e6f, kDigits4 = 2.1e9f;      // the largest number of three and of four signed digits, and some to spare
// Scales (1 / scale of a value) of a tile are alike within a factor of 8.  They are taken relative to 1.25 times the largest of the last such tile as long
// as they lie within a factor of 16 below: weights have 24 bits at that scale and 20 at the far end.
constexpr float kAlike = 8.f, kRoom = 1.25f, kLeast = 1.f / 16.f;

__device__ int g_errors;

// I8: int8 pages.  R: query rows of a block.  Blocks of 16 rows need so little that two CTAs share an SM and cover each other's beginnings and ends
template <int D, bool I8, int R> struct Shape {
    static constexpr int HALVES = R == 16 ? 1 : 2, CTAS = R == 16 ? 2 : 1, SOFTMAX = 128 * HALVES;     // threads
    static constexpr int W_SUMS = 4 * HALVES, W_MMA = W_SUMS + 4, W_PROD = W_MMA + 1, W_LOAD = W_PROD + 1, THREADS = (W_LOAD + 2) * 32;
    static constexpr int TERMS = I8 ? 3 : 2, N = TERMS * R;         // columns of the scores: term by term
    static constexpr int NO = I8 ? 4 * R : 2 * R;                   // columns of the sums: row by row
    static constexpr int TILE = KT * D * (I8 ? 1 : 2), SCALES = I8 ? KT * 8 : 0, SLOT = TILE + SCALES;     // of keys or values; both scales of a tile come with its values
    static constexpr int Q_BYTES = N * 128 * (I8 ? 1 : D / 64), P_BYTES = KT * 128 * (R == 64 ? 2 : 1);
    static constexpr int Q_BUFS = Q_BYTES > 16384 ? 1 : 2;
    static constexpr int FREE = (CTAS == 2 ? 106 : 200) * 1024 - Q_BUFS * Q_BYTES;
    static constexpr int RING = (FREE - 2 * P_BYTES) / SLOT < 12 ? (FREE - 2 * P_BYTES) / SLOT : 12;       // weights are double-buffered
    static constexpr int COLS = 2 * N + 2 * NO, TMEM = COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr int NBAR = 2 * RING + 16;      // full, empty [ring]; s_full, p_full, o_full, o_empty, q_ready, q_free [2]; piece_done [4]
    static constexpr int FLOATS = 2 * R /*factors*/ + 2 * R /*references, thresholds*/ + 4 * R /*corrections*/ + 4 * R /*maxima*/ +
                                  4 * 5 * R /*sums, references at the end*/ + 2 * R /*what becomes of the sums*/ + (I8 ? 8 * R : 0) /*units, largest products*/ + 28;
    static size_t smem(int seqs, int mask_words) {
        return (size_t)RING * SLOT + Q_BUFS * Q_BYTES + 2 * P_BYTES + NBAR * 8 + FLOATS * 4 + 2 * R * mask_words * 4 + kNotes * 4 + 64 + (seqs + 1) * 4 + 1024;
    }
};

__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// kind::i8: c = S32 (2) [4,6), a and b signed (1) [7,10) [10,13), the rest as for kind::f16
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N, int a_mn_major, int b_mn_major) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn_major << 15) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
}
template <int N> __device__ __forceinline__ void tmem_ldn(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 8) tmem_ld8(taddr, r);
    else tmem_ld16(taddr, r);
}
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// three signed digits of x, the lowest in the lowest byte: x = d0 + 256 d1 + 65536 d2
__device__ __forceinline__ uint32_t digits(int x) { return (uint32_t)(x + 0x808080) ^ 0x808080u; }
// their sums of products: the upper one is below 2^22 (128 x 127 x 127), so that a float's mantissa holds it
__device__ __forceinline__ float from_digits(uint32_t d0, uint32_t d1, uint32_t d2) {
    const float hi = __uint_as_float(d2 + 0x4b400000u) - 12582912.f;
    return fmaf(hi, 65536.f, (float)((int)d1 * 256 + (int)d0));
}
// and of four
__device__ __forceinline__ uint32_t digits4(int x) { return (uint32_t)(x + 0x80808080) ^ 0x80808080u; }
__device__ __forceinline__ float from_digits4(uint32_t d0, uint32_t d1, uint32_t d2, uint32_t d3) {
    return fmaf((float)((int)d3 * 256 + (int)d2), 65536.f, (float)((int)d1 * 256 + (int)d0));
}

// Weights of a tile whose values have scales that are not alike, by all softmax threads, each a key's RH rows from h0 on: from floats in the place of the digits
// (a word a row, see the softmax) to digits relative to the row's largest product of weight and scale; units: what the rows' sums are times.  A product that
// is not finite makes its row's sums NaN.  Row by row through shared memory and out of line, since instructions are what the kernel's caches are short of
// (48 sequences of 1 to 2K keys: 128 us, inline and in registers 138, without any of this 123).
template <int R, int RH, int SOFTMAX>
__device__ __noinline__ void digits_apart(uint32_t pb, int h0, float vsc, uint32_t* s_top, float* units) {
    const int lane = threadIdx.x & 31, kk = threadIdx.x & 127, quarter = threadIdx.x >> 5 & 3;
    auto group_sync = [&] { asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX) : "memory"); };
    auto word = [&](int r) { return pb + (((h0 + r) >> 2 ^ (kk & 7)) << 4) + (r & 3) * 4; };
#pragma unroll 1
    for (int r = 0; r < RH; ++r) {
        float e;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(e) : "r"(word(r)) : "memory");
        e = e != 0.f ? e * vsc : 0.f;
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(word(r)), "f"(e) : "memory");
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(e) & 0x7fffffffu);
        if (lane == 0) s_top[quarter * R + h0 + r] = top;
    }
    group_sync();
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        const uint32_t top = max(max(s_top[r], s_top[R + r]), max(s_top[2 * R + r], s_top[3 * R + r]));
        const bool finite = top < 0x7f800000u;
        const float most = fmaxf(__uint_as_float(top), 1e-28f);
        units[r] = finite ? __fdiv_rn(most, kDigits4) : __int_as_float(0x7fc00000);
        s_top[r] = __float_as_uint(finite ? __fdiv_rn(kDigits4, most) : 0.f);
    }
    group_sync();
#pragma unroll 1
    for (int r = 0; r < RH; ++r) {
        float y;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(word(r)) : "memory");
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(word(r)), "r"(digits4(__float2int_rn(y * __uint_as_float(s_top[h0 + r])))) : "memory");
    }
}

template <int D, bool I8, int R, typename Q>
__global__ void __launch_bounds__(Shape<D, I8, R>::THREADS, Shape<D, I8, R>::CTAS) tree_terms_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeWork a) {
    typedef Shape<D, I8, R> C;
    constexpr int N = C::N, TERMS = C::TERMS, RING = C::RING, CB = I8 ? 1 : D / 64, RH = R / C::HALVES;       // CB: column blocks of a tile
    constexpr int W_SUMS = C::W_SUMS, W_MMA = C::W_MMA, W_PROD = C::W_PROD, W_LOAD = C::W_LOAD, kSoftmax = C::SOFTMAX;
    constexpr float kRaise = I8 ? 7.f : 8.f, kShift = I8 ? 0.f : 7.f;      // half weights times 2^7: up to 2^15; int8: up to 2^7, a bit more for the rest
    constexpr float kWeight = kDigits4 / 128.f;                  // int8: integers of a weight
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const TreeParams& p = a.p;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_sm = base + RING * C::TILE, p_sm = q_sm + C::Q_BUFS * C::Q_BYTES, sc_sm = p_sm + 2 * C::P_BYTES, bar0 = sc_sm + RING * C::SCALES;
    auto kv_full = [&](int s) { return bar0 + s * 8; };
    auto kv_empty = [&](int s) { return bar0 + (RING + s) * 8; };
    auto s_full = [&](int i) { return bar0 + (2 * RING + i) * 8; };
    auto p_full = [&](int i) { return bar0 + (2 * RING + 2 + i) * 8; };
    auto o_full = [&](int i) { return bar0 + (2 * RING + 4 + i) * 8; };
    auto o_empty = [&](int i) { return bar0 + (2 * RING + 6 + i) * 8; };
    auto q_ready = [&](uint32_t piece) { return bar0 + (2 * RING + 8 + piece % C::Q_BUFS) * 8; };
    auto q_free = [&](uint32_t piece) { return bar0 + (2 * RING + 10 + piece % C::Q_BUFS) * 8; };
    auto q_phase = [&](uint32_t piece) { return piece / C::Q_BUFS & 1u; };
    auto piece_done = [&](uint32_t piece) { return bar0 + (2 * RING + 12 + (piece & 3)) * 8; };
    const uint32_t tmem_slot = bar0 + C::NBAR * 8, fail_sm = tmem_slot + 8, meta_sm = fail_sm + 8;
    // factors of the scores [2 pieces], references (less kShift) and whether rows have one, corrections of the last four tiles, maxima
    // by warp, sums by warp and references of the last four pieces, a piece's rows of the output and what their sums are
    // multiplied by; int8: what the last four tiles' sums are times, largest products of weights and scales by warp;
    // the unit of the scales and what gives integers of it, bits of the largest and the smallest scale by warp;
    // whether references moved in the last four tiles, whether the last four pieces are computed by rows,
    // whether a row has no reference yet
    float* fl = reinterpret_cast<float*>(smem_raw + (meta_sm + kNotes * 4 - smem_u32(smem_raw)));
    float *s_fe = fl, *s_ref = fl + 2 * R, *s_set = fl + 3 * R, *s_corr = fl + 4 * R, *s_max = fl + 8 * R, *s_end = fl + 12 * R, *s_unit = fl + 34 * R;
    uint32_t *s_top = reinterpret_cast<uint32_t*>(s_unit + (I8 ? 4 * R : 0)), *s_big = s_top + (I8 ? 4 * R : 0), *s_small = s_big + 4;
    float* s_scale = reinterpret_cast<float*>(s_small + 4);
    int2* s_fin = reinterpret_cast<int2*>(fl + 32 * R);
    int *s_moved = reinterpret_cast<int*>(s_scale + 8), *s_odd = s_moved + 4, *s_pending = s_odd + 4, *pre = s_pending + 4;
    uint32_t* s_mask = reinterpret_cast<uint32_t*>(pre + p.num_seqs + 1);      // [2 pieces][R][mask_words]
    auto failed = [&] { return tc_failed(fail_sm); };
    auto wait = [&](uint32_t bar, uint32_t parity) { tc_wait(bar, parity, fail_sm, a.polls); };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.group;
    if (threadIdx.x == 0) {
        for (int s = 0; s < RING; ++s) {
            mbar_init(kv_full(s), I8 ? 33 : 1);     // int8: a warp's copies of scales, too
            mbar_init(kv_empty(s), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(p_full(i), kSoftmax);
            mbar_init(o_full(i), 1);
            mbar_init(o_empty(i), 128);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(q_ready(i), 64);
            mbar_init(q_free(i), 1 + kSoftmax / 32);
        }
        for (uint32_t i = 0; i < 4; ++i) mbar_init(piece_done(i), kSoftmax / 32);
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(fail_sm), "r"(0u) : "memory");
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmV));
    }
    if (warp == W_MMA) tmem_alloc(tmem_slot, C::TMEM);
    shares::count_units(pre, p.num_seqs, [&](int b) { return tree_seq(p, b, a.block, a.unit).units(a.extra); });
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
    // columns of TMEM: scores [2][N], sums [2][NO]
    auto s_col = [&](int i) { return tmem_base + i * N; };
    auto o_col = [&](int i) { return tmem_base + 2 * N + i * C::NO; };
    TreeWalk w(a, pre);
    // Tiles go through the ring in the order of their products: K(0), K(1), V(0), K(2), V(1), ..., K(n - 1), V(n - 2), V(n - 1); the ring's
    // count `at` runs on through the pieces, as do the tiles' parities
    auto k_at = [&](uint32_t at, int i) { return at + (uint32_t)(i == 0 ? 0 : 2 * i - 1); };
    auto v_at = [&](uint32_t at, int i, int nt) { return at + (uint32_t)(i + 1 < nt ? 2 * i + 2 : 2 * nt - 1); };
    auto slot_of = [&](uint32_t c) { return (int)(c % RING); };
    auto phase_of = [&](uint32_t c) { return c / RING & 1u; };
    uint32_t at = 0, n = 0, pieces = 0;     // requests to the ring, tiles, pieces so far

    if (warp == W_PROD) {
        uint32_t c = 0, tiles = 0;          // requests and tiles of keys so far
        bool ok = a.polls > 0;              // 0: nothing is requested, so that all waits run out
        if (w.f >= w.f_hi && lane == 0) a.notes[blockIdx.x] = TreeNote{};
        auto request = [&](const CUtensorMap* map, bool scales, int rows) {         // lane u < 8: of unit u
            const int s = (int)(c % RING);
            wait(kv_empty(s), (c / RING & 1u) ^ 1u);
            if (__any_sync(0xffffffffu, failed())) {
                ok = false;
                return;
            }
            const uint32_t st = base + s * C::TILE;
            if (elect_one()) mbar_arrive_expect_tx(kv_full(s), C::TILE);
            int r[8];
#pragma unroll
            for (int uu = 0; uu < 8; ++uu) {
                r[uu] = __shfl_sync(0xffffffffu, rows, uu);
                if (r[uu] < 0) r[uu] = a.total_rows;    // no page: zeros, and its scores are masked
            }
            if (elect_one())
#pragma unroll
                for (int uu = 0; uu < 8; ++uu)
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) tma_load_2d(st + cb * 16384 + uu * 2048, map, cb * 64, r[uu], kv_full(s));
            __syncwarp();
            if (I8 && scales) {                         // a lane: 16 bytes of a unit's 64, of keys and of values
                const int row = __shfl_sync(0xffffffffu, rows, lane >> 2);
                if (row >= 0) {
                    const uint32_t to = sc_sm + s * C::SCALES + lane * 16;
                    cp_async_16(to, p.k_scales + row + (lane & 3) * 4, true);
                    cp_async_16(to + 512, p.v_scales + row + (lane & 3) * 4, true);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(kv_full(s)) : "memory");
            } else if (I8) {
                mbar_arrive(kv_full(s));
            }
            ++c;
        };
        TreePages pages(p);
        while (ok && w.next()) {
            pages.open(w, 8);
            int rows = -1, before = -1;
#pragma unroll 1
            for (int i = w.i0; i <= w.i1 && ok; ++i) {              // K(i) and V(i - 1)
                if (i < w.i1) {
                    rows = pages.lane_row((i - w.i0) * 8);
                    const uint32_t mapped = __ballot_sync(0xffffffffu, rows >= 0) & 255u;
                    if (lane == 0) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(meta_sm + tiles % kNotes * 4), "r"(mapped) : "memory");
                    __syncwarp();
                    ++tiles;
                }
#pragma unroll 1
                for (int v = i < w.i1 ? 0 : 1; v < (i > w.i0 ? 2 : 1) && ok; ++v) request(v ? &tmV : &tmK, v, v ? before : rows);
                before = rows;
            }
        }
        if (failed())           // let the copies in flight land before the CTA's shared memory goes away
            for (uint32_t i = c > RING ? c - RING : 0; i < c; ++i) tc_let_land(kv_full((int)(i % RING)), i / RING & 1u);
    } else if (warp == W_MMA) {
        constexpr uint32_t kIdescS = I8 ? idesc_i8(128, N, 0, 0) : idesc_f16(128, N, 0, 0, 0);
        constexpr uint32_t kIdescO = I8 ? idesc_i8(128, C::NO, 1, 1) : idesc_f16(128, C::NO, 1, 1, 0);
        while (w.next()) {
            const int nt = w.i1 - w.i0;
            auto issue_S = [&](int i) {
                const int s = slot_of(k_at(at, i)), sb = (int)(n + i) & 1;
                wait(kv_full(s), phase_of(k_at(at, i)));
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t st = base + s * C::TILE, qb = q_sm + pieces % C::Q_BUFS * C::Q_BYTES;
                    if constexpr (I8) {
#pragma unroll
                        for (int ks = 0; ks < D / 32; ++ks)
                            umma_i8(s_col(sb), make_desc(st + ks * 32, 16, 1024), make_desc(qb + ks * 32, 16, 1024), kIdescS, ks > 0 ? 1u : 0u);
                    } else {
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks)
                            umma_f16(s_col(sb), make_desc(st + (ks >> 2) * 16384 + (ks & 3) * 32, 16, 1024),
                                     make_desc(qb + (ks >> 2) * (N * 128) + (ks & 3) * 32, 16, 1024), kIdescS, ks > 0 ? 1u : 0u);
                    }
                    umma_commit(s_full(sb));
                    umma_commit(kv_empty(s));
                    if (i + 1 == nt) umma_commit(q_free(pieces));
                }
                __syncwarp();
            };
            wait(q_ready(pieces), q_phase(pieces));
            issue_S(0);
            for (int i = 0; i < nt; ++i) {
                if (i + 1 < nt) issue_S(i + 1);
                const uint32_t t = n + i;
                const int s = slot_of(v_at(at, i, nt)), sb = (int)t & 1, nvalid = min(KT, w.sq.keys - (w.i0 + i) * KT);
                const uint32_t st = base + s * C::TILE;
                wait(kv_full(s), phase_of(v_at(at, i, nt)));
                if (!I8 && (nvalid & 15)) {         // value rows past the last key may hold anything (0 x NaN = NaN): zeros
                    const int r1 = (nvalid + 15) & ~15;
                    for (int idx = lane; idx < (r1 - nvalid) * (D / 8); idx += 32) {
                        const int r = nvalid + idx / (D / 8), c = idx % (D / 8);
                        const uint32_t addr = st + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(addr), "r"(0u) : "memory");
                    }
                    fence_proxy_async();
                    __syncwarp();
                }
                wait(p_full(sb), t >> 1 & 1u);
                wait(o_empty(sb), (t >> 1 & 1u) ^ 1u);          // the sums of tile t - 2 are taken
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t pb = p_sm + sb * C::P_BYTES;
                    if constexpr (I8) {
                        const int ksteps = (nvalid + 31) >> 5;
                        for (int ks = 0; ks < ksteps; ++ks)
                            umma_i8(o_col(sb), make_desc(st + ks * 32 * 128, 16, 1024), make_desc(pb + ks * 32 * 128, 16, 1024), kIdescO, ks > 0 ? 1u : 0u);
                    } else {
                        const int ksteps = (nvalid + 15) >> 4;
                        for (int ks = 0; ks < ksteps; ++ks)     // 64 value columns twice where there are no more
                            umma_f16(o_col(sb), make_desc(st + ks * 2048, D == 128 ? 16384 : 0, 1024),
                                     make_desc(pb + ks * 2048, 16384, 1024), kIdescO, ks > 0 ? 1u : 0u);
                    }
                    umma_commit(o_full(sb));
                    umma_commit(kv_empty(s));
                }
                __syncwarp();
            }
            at += 2 * nt;
            n += nt;
            ++pieces;
        }
    } else if (warp >= W_LOAD) {
        // ---- queries: half of the rows a warp, one row at a time over its lanes, up to 16 rows under way together
        constexpr int PER = D / 32, HALF = R / 2, LB = HALF < 16 ? HALF : 16;       // columns of a lane, rows of a warp, rows under way
        const float f0 = 1.4426950408889634f / p.temperature;
        const int c0 = lane * PER, mine = (warp - W_LOAD) * HALF + lane;            // the row that this lane knows about
        while (w.next()) {
            const int all = w.sq.n * G, buf = (int)(pieces % C::Q_BUFS), rr = w.rr0 + mine, div = rr / G;
            const uint32_t qb = q_sm + buf * C::Q_BYTES;
            const int node = lane < HALF && rr < all ? w.sq.r0 + div : -1, head = w.g * G + rr - div * G;
            const int64_t own = node >= 0 ? (int64_t)node * p.q_stride + (int64_t)head * D : -1;
            const uint32_t mask0 = node >= 0 ? __ldg(p.mask + (int64_t)node * p.mask_words) : 0u;
#pragma unroll 1
            for (int b0 = 0; b0 < HALF; b0 += LB) {
                float x[LB][PER], big[LB];
#pragma unroll
                for (int k = 0; k < LB; ++k) {
                    const int64_t from = __shfl_sync(0xffffffffu, own, b0 + k);
                    const Q* q = static_cast<const Q*>(p.q) + from + c0;
                    if constexpr (sizeof(Q) == 4 && PER == 4) {
                        const float4 v = from >= 0 ? __ldg(reinterpret_cast<const float4*>(q)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        x[k][0] = v.x; x[k][1] = v.y; x[k][PER - 2] = v.z; x[k][PER - 1] = v.w;
                    } else if constexpr (sizeof(Q) == 4) {
                        const float2 v = from >= 0 ? __ldg(reinterpret_cast<const float2*>(q)) : make_float2(0.f, 0.f);
                        x[k][0] = v.x; x[k][1] = v.y;
                    } else {
                        const uint2 v = from >= 0 ? __ldg(reinterpret_cast<const uint2*>(q)) : make_uint2(0u, 0u);
                        const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
                        x[k][0] = lo.x; x[k][1] = lo.y; x[k][PER - 2] = hi.x; x[k][PER - 1] = hi.y;
                    }
                }
                if (b0 == 0) wait(q_free(pieces), q_phase(pieces) ^ 1u);        // their place is read; the rows are on their way by then
#pragma unroll
                for (int k = 0; k < LB; ++k) {
                    big[k] = 0.f;
#pragma unroll
                    for (int c = 0; c < PER; ++c) big[k] = fmaxf(big[k], fabsf(x[k][c]));
                }
#pragma unroll
                for (int k = 0; k < LB; ++k) big[k] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big[k])));
#pragma unroll
                for (int k = 0; k < LB; ++k) {
                    const int r = (warp - W_LOAD) * HALF + b0 + k;
                    if constexpr (I8) {
                        // a row with numbers that are not finite: no digits, and its scores are not finite through their factor
                        bool odd = false;
#pragma unroll
                        for (int c = 0; c < PER; ++c) odd |= !(fabsf(x[k][c]) < INFINITY);
                        odd = __any_sync(0xffffffffu, odd);
                        const float up = big[k] > 0.f && !odd ? __fdividef(kDigits, big[k]) : 0.f;
                        uint32_t z[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) z[c] = digits(__float2int_rn(x[k][c < PER ? c : 0] * up));
#pragma unroll
                        for (int t = 0; t < 3; ++t) {
                            const int row = t * R + r;
                            const uint32_t sel = (uint32_t)t | (uint32_t)(4 + t) << 4;
                            const uint32_t word = __byte_perm(__byte_perm(z[0], z[1], sel), __byte_perm(z[2], z[3], sel), 0x5410);
                            asm volatile("st.shared.u32 [%0], %1;" ::"r"(qb + row * 128 + (((c0 >> 4) ^ (row & 7)) << 4) + (c0 & 15)), "r"(word) : "memory");
                        }
                        if (lane == 0) s_fe[buf * R + r] = odd ? __int_as_float(0x7fc00000) : up > 0.f ? __fdiv_rn(f0, up) : 0.f;
                    } else {
                        // the row's largest between 2^10 and 2^11: halves hold hi, and lo down to 2^-35 of it
                        const int e = max(-100, min(100, 137 - (int)(__float_as_uint(big[k]) >> 23)));
                        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                        uint32_t v[2][PER / 2];
#pragma unroll
                        for (int c = 0; c < PER; c += 2) {
                            v[0][c / 2] = pack_half2(x[k][c] * up, x[k][c + 1] * up);
                            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&v[0][c / 2]));
                            v[1][c / 2] = pack_half2(x[k][c] * up - back.x, x[k][c + 1] * up - back.y);
                        }
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int row = t * R + r;
                            const uint32_t addr = qb + (c0 >> 6) * (N * 128) + row * 128 + ((((c0 & 63) >> 3) ^ (row & 7)) << 4) + (c0 & 7) * 2;
                            if constexpr (PER == 4)
                                asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(v[t][0]), "r"(v[t][PER / 2 - 1]) : "memory");
                            else
                                asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v[t][0]) : "memory");
                        }
                        if (lane == 0) s_fe[buf * R + r] = f0 * __uint_as_float((uint32_t)(127 - e) << 23);
                    }
                }
            }
            if (lane < HALF) {
                uint32_t* mask = s_mask + (buf * R + mine) * p.mask_words;
                mask[0] = mask0;
                for (int x = 1; x < p.mask_words; ++x) mask[x] = node >= 0 ? __ldg(p.mask + (int64_t)node * p.mask_words + x) : 0u;
            }
            fence_proxy_async();
            mbar_arrive_cnt(q_ready(pieces));
            ++pieces;
            // (these warps come to the share's end whatever runs out: the join goes by the note)
            if (w.f >= w.f_hi && threadIdx.x == W_LOAD * 32) a.notes[blockIdx.x] = tree_note(a, w.sq, w.g, w.rr0, w.i0, w.i1, w.item_at(), w.total, w.ns, w.slot);
        }
    } else if (warp < W_SUMS) {
        // ---- softmax: one thread per key and half of the rows
        const int kk = threadIdx.x & 127, quarter = warp & 3, h0 = (warp >> 2) * RH;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        auto group_sync = [&] { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmax) : "memory"); };
        auto group_any = [&](bool x) {
            int any;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\t"
                "setp.ne.b32 p, %1, 0;\n\t"
                "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
                "selp.b32 %0, 1, 0, q;\n\t}"
                : "=r"(any) : "r"((int)x), "n"(kSoftmax) : "memory");
            return any != 0;
        };
        auto four = [&](const float* f) { return *reinterpret_cast<const float4*>(f); };
        auto fresh = [&] {                  // no references yet
            if (threadIdx.x < R) s_ref[threadIdx.x] = s_set[threadIdx.x] = 0.f;
            if (threadIdx.x == 0) *s_pending = 1;
            if (I8 && threadIdx.x == 0) s_scale[0] = s_scale[1] = 0.f;
        };
        fresh();
        while (w.next()) {
            const int nt = w.i1 - w.i0, buf = (int)(pieces % C::Q_BUFS);
            wait(q_ready(pieces), q_phase(pieces));
            group_sync();                   // fresh references
            const float* fes = s_fe + buf * R + h0;
            float l[RH];
#pragma unroll
            for (int r = 0; r < RH; ++r) l[r] = 0.f;
            bool odd = false;
#pragma unroll 1
            for (int i = 0; i < nt; ++i) {
                const uint32_t t = n + i;
                const int sb = (int)t & 1, ring4 = (int)t & 3, kp = (w.i0 + i) * KT + kk;
                const bool drafts = (w.i0 + i + 1) * KT > w.sq.ctx;
                wait(s_full(sb), t >> 1 & 1u);
                tc_fence_after();
                uint32_t mapped;            // the producer's note about this tile, older than the scores
                asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(mapped) : "r"(meta_sm + t % kNotes * 4) : "memory");
                const bool here = kp < w.sq.keys && (mapped >> (kk >> 4) & 1u);
                float ksc = 1.f, vsc = 0.f;
                if (I8) {
                    const uint32_t c = v_at(at, i, nt), sc = sc_sm + slot_of(c) * C::SCALES + kk * 4;
                    wait(kv_full(slot_of(c)), phase_of(c));
                    float ks, vs;
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks) : "r"(sc) : "memory");
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vs) : "r"(sc + 512) : "memory");
                    ksc = here ? __frcp_rn(ks) : 1.f;
                    vsc = here ? __frcp_rn(vs) : 0.f;
                } else if (drafts) {        // values that are not finite (rows past the last key: zeros, or looked at in vain)
                    const uint32_t c = v_at(at, i, nt);
                    wait(kv_full(slot_of(c)), phase_of(c));
                    if (kp < w.sq.keys && h0 == 0) {
                        const uint32_t vt = base + slot_of(c) * C::TILE + kk * 128;
#pragma unroll
                        for (int x = 0; x < D / 8; ++x) {
                            const uint4 v = lds_128(vt + (x >> 3) * 16384 + ((x & 7) << 4));
                            const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) odd |= (q[e] & 0x7c00u) == 0x7c00u || (q[e] >> 16 & 0x7c00u) == 0x7c00u;
                        }
                    }
                }
                // ---- scores, less their references; does one exceed its own?
                constexpr int CH = C::HALVES == 1 || RH < 16 ? 8 : 16;
                const int bit = kp - w.sq.ctx;              // of the rows' masks, where it is not negative
                const bool masked = drafts && here && bit >= 0, hidden = !here || (masked && (bit >> 5) >= p.mask_words);
                float s[RH];
                // a value's scale that lies outside the range of the unit (or is not finite) is a reason, too
                const float by = I8 ? s_scale[0] : 0.f;
                const bool strange = I8 && here && !(fabsf(vsc) <= by && fabsf(vsc) >= kLeast * by);
                bool over = false;
#pragma unroll
                for (int c = 0; c < RH / CH; ++c) {
                    uint32_t x[TERMS][CH];
#pragma unroll
                    for (int term = 0; term < TERMS; ++term) tmem_ldn<CH>(s_col(sb) + lane_base + term * R + h0 + c * CH, x[term]);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < CH; j += 4) {
                        const int r = c * CH + j;
                        const float4 fe = four(fes + r), ref = four(s_ref + h0 + r);
                        const float f[4] = {fe.x, fe.y, fe.z, fe.w}, o[4] = {ref.x, ref.y, ref.z, ref.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v;
                            if constexpr (I8) v = fmaf(from_digits(x[0][j + e], x[1][j + e], x[TERMS - 1][j + e]), f[e] * ksc, -o[e]);
                            else v = fmaf(__uint_as_float(x[0][j + e]) + __uint_as_float(x[1][j + e]), f[e], -o[e]);
                            s[r + e] = hidden ? -INFINITY : v;
                            over |= s[r + e] > kRaise + kShift;
                        }
                    }
                }
                if (drafts) {
                    const uint32_t* mw = s_mask + (buf * R + h0) * p.mask_words + (masked && !hidden ? bit >> 5 : 0);
                    over = false;
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        if (masked && !(mw[r * p.mask_words] >> (bit & 31) & 1u)) s[r] = -INFINITY;
                        over |= s[r] > kRaise + kShift;
                    }
                }
                const bool any = group_any(over || strange || *s_pending);
                if (threadIdx.x == 0) s_moved[ring4] = any;
                const uint32_t pb = p_sm + (uint32_t)(sb * C::P_BYTES) + kk * 128;
                if (I8 && threadIdx.x < R) s_unit[ring4 * R + threadIdx.x] = by * (1.f / kWeight);
                if (any) {
                    if (I8) {
                        const uint32_t bits = __float_as_uint(vsc) & 0x7fffffffu;       // what is not a number is above infinity
                        const uint32_t most = __reduce_max_sync(0xffffffffu, bits), least = __reduce_min_sync(0xffffffffu, here ? bits : 0x7f7fffffu);
                        if (lane == 0) {                                                // both halves the same
                            s_big[quarter] = most;
                            s_small[quarter] = least;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        const uint32_t top = __reduce_max_sync(0xffffffffu, ordered(s[r] == s[r] ? s[r] : -INFINITY));
                        if (lane == 0) s_max[quarter * R + h0 + r] = unordered(top);
                    }
                    group_sync();
                    if (threadIdx.x < R) {
                        const int r = threadIdx.x;
                        const float top = fmaxf(fmaxf(s_max[r], s_max[R + r]), fmaxf(s_max[2 * R + r], s_max[3 * R + r]));
                        const bool has = s_set[r] != 0.f, raise = has ? top > kRaise + kShift : top > -INFINITY;
                        const float by = raise ? top - kShift : 0.f;
                        s_corr[ring4 * R + r] = has ? exp2f(-by) : 1.f;         // a first reference has no sums to correct
                        s_max[r] = by;
                        s_ref[r] += by;
                        if (raise) s_set[r] = 1.f;
                        else if (!has && w.rr0 + r < w.sq.n * G) s_moved[ring4] = 2;        // still none
                    }
                    float big = 0.f;            // int8: the tile's largest scale, if all are alike; infinity, if they are not
                    if constexpr (I8) {
                        const uint4 b4 = *reinterpret_cast<const uint4*>(s_big), s4 = *reinterpret_cast<const uint4*>(s_small);
                        big = __uint_as_float(max(max(b4.x, b4.y), max(b4.z, b4.w)));
                        if (!(big < 1e36f && (big == 0.f || big > 1e-28f) && big <= kAlike * __uint_as_float(min(min(s4.x, s4.y), min(s4.z, s4.w))))) big = INFINITY;
                        if (threadIdx.x == 0 && big > 0.f && big < INFINITY) {
                            s_scale[0] = kRoom * big;
                            s_scale[1] = __fdiv_rn(kWeight, kRoom * big);
                        }
                    }
                    group_sync();
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        l[r] *= s_corr[ring4 * R + h0 + r];
                        s[r] -= s_max[h0 + r];
                    }
                    if (threadIdx.x == 0) *s_pending = s_moved[ring4] == 2;
                    if constexpr (I8) {
                        if (big < INFINITY) {
                            if (threadIdx.x < R) s_unit[ring4 * R + threadIdx.x] = s_scale[0] * (1.f / kWeight);
                        } else {
#pragma unroll
                            for (int r = 0; r < RH; r += 4) {
                                float e[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    e[k] = fast_exp2(s[r + k]);
                                    l[r + k] += e[k];
                                }
                                asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(pb + (((h0 + r) >> 2 ^ (kk & 7)) << 4)), "f"(e[0]), "f"(e[1]), "f"(e[2]),
                                             "f"(e[3]) : "memory");
                            }
                            digits_apart<R, RH, kSoftmax>(pb, h0, vsc, s_top, s_unit + ring4 * R);
                            fence_proxy_async();
                            tc_fence_before();
                            mbar_arrive_cnt(p_full(sb));
                            continue;
                        }
                    }
                }
                // ---- weights
                const float unit = I8 ? vsc * s_scale[1] : 0.f;            // per value's scale, as integers: weights are 2^7 at most
#pragma unroll
                for (int r = 0; r < RH; r += 4) {
                    float e[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        e[k] = fast_exp2(s[r + k]);
                        l[r + k] += e[k];
                    }
                    uint32_t v[4];
                    if constexpr (I8) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = digits4(__float2int_rn(e[k] * unit));
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            v[2 * k] = pack_half2(e[2 * k], e[2 * k + 1]);
                            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&v[2 * k]));
                            v[2 * k + 1] = pack_half2(e[2 * k] - back.x, e[2 * k + 1] - back.y);
                        }
                    }
                    const int c = (h0 + r) >> 2;
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(pb + (c >> 3) * 16384 + (((c & 7) ^ (kk & 7)) << 4)), "r"(v[0]), "r"(v[1]),
                                 "r"(v[2]), "r"(v[3]) : "memory");
                }
                fence_proxy_async();
                tc_fence_before();
                mbar_arrive_cnt(p_full(sb));
            }
            n += nt;
            at += 2 * nt;
            // ---- the piece's end: sums over the warps' keys, references, whether it has to be computed by rows
            odd = group_any(odd);           // everyone is through with the references, too
            float* end = s_end + (pieces & 3) * 5 * R;
#pragma unroll
            for (int r = 0; r < RH; ++r) {
                const float sum = warp_sum(l[r]);
                if (lane == 0) end[quarter * R + h0 + r] = sum;
            }
            if (threadIdx.x < R) end[4 * R + threadIdx.x] = s_set[threadIdx.x] != 0.f ? s_ref[threadIdx.x] + kShift : -INFINITY;
            if (threadIdx.x == 0) s_odd[pieces & 3] = odd;
            fresh();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_cnt(piece_done(pieces));
                mbar_arrive_cnt(q_free(pieces));
            }
            if (!I8 && odd) tree_piece_by_rows<D, Q, __half>(a, w, warp * (R / W_SUMS), R / W_SUMS);
            ++pieces;
        }
    } else {
        // ---- sums: one thread per value column (64 columns: the upper half of the threads has them a second time)
        const int d = threadIdx.x - kSoftmax;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        while (w.next()) {
            const int nt = w.i1 - w.i0;
            float o[R];
#pragma unroll
            for (int r = 0; r < R; ++r) o[r] = 0.f;
#pragma unroll 1
            for (int i = 0; i < nt; ++i) {
                const uint32_t t = n + i;
                const int sb = (int)t & 1, ring4 = (int)t & 3;
                wait(o_full(sb), t >> 1 & 1u);
                tc_fence_after();
                if (s_moved[ring4])
#pragma unroll
                    for (int r = 0; r < R; ++r) o[r] *= s_corr[ring4 * R + r];
#pragma unroll
                for (int c = 0; c < C::NO / 32; ++c) {
                    uint32_t x[32];
                    tmem_ld32(o_col(sb) + lane_base + c * 32, x);
                    float unit[8] = {};         // int8: of the rows' digits
                    if constexpr (I8) {
                        const float4* u = reinterpret_cast<const float4*>(s_unit + ring4 * R + c * 8);
                        const float4 a = u[0], b = u[1];
                        unit[0] = a.x; unit[1] = a.y; unit[2] = a.z; unit[3] = a.w;
                        unit[4] = b.x; unit[5] = b.y; unit[6] = b.z; unit[7] = b.w;
                    }
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if constexpr (I8) {                 // a row's digits
                            const int r = c * 8 + j / 4;
                            o[r] = fmaf(from_digits4(x[j], x[j + 1], x[j + 2], x[j + 3]), unit[j / 4], o[r]);
                        } else {                            // two rows' large terms, and their small ones
                            const int r = c * 16 + j / 2;
                            o[r] += __uint_as_float(x[j]) + __uint_as_float(x[j + 2]);
                            o[r + 1] += __uint_as_float(x[j + 1]) + __uint_as_float(x[j + 3]);
                        }
                    }
                }
                tc_fence_before();
                mbar_arrive_cnt(o_empty(sb));
            }
            n += nt;
            wait(piece_done(pieces), pieces >> 2 & 1u);
            const float* end = s_end + (pieces & 3) * 5 * R;
            // a wait ran out: what the others left here may be of another piece
            const bool lost = failed(), skip = !I8 && !lost && s_odd[pieces & 3];
            constexpr float scale = I8 ? 1.f : 1.f / 128.f;     // 2^-kShift
            const float bad = lost ? __int_as_float(0x7fc00000) : 0.f;
            if (d < R) {
                const float sum = (end[d] + end[R + d] + end[2 * R + d] + end[3 * R + d]) * scale, ref = end[4 * R + d];
                const int rr = w.rr0 + d, node = rr / G;
                const bool row = rr < w.sq.n * G && !skip;
                s_fin[d] = make_int2(row ? (w.slot < 0 ? (w.sq.r0 + node) * p.heads + w.g * G + rr - node * G : d) : -1,
                                     __float_as_int((w.slot < 0 ? __fdiv_rn(scale, sum + 1e-6f) : scale * a.p_scale) + bad));
                if (w.slot >= 0 && row)
                    *reinterpret_cast<float4*>(a.part + (w.slot * a.block + d) * (D + 4) + D) = make_float4(ref + bad, sum * a.p_scale + bad, ref, 0.f);
            }
            ++pieces;
            asm volatile("bar.sync 3, 128;" ::: "memory");
            if (!skip && d < D) {
                float* part = a.part + w.slot * a.block * (D + 4) + d;
                Q* out = static_cast<Q*>(p.out) + d;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int2 f = s_fin[r];
                    const float x = o[r] * __int_as_float(f.y);
                    if (f.x < 0) continue;
                    if (w.slot < 0) out[(int64_t)f.x * D] = tree_narrow<Q>(x);
                    else part[r * (D + 4)] = x;
                }
            }
            asm volatile("bar.sync 3, 128;" ::: "memory");      // s_fin is read
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        if (failed()) {
            __nanosleep(1000000);       // products in flight write TMEM for microseconds at most
            if (lane == 0) atomicAdd(&g_errors, 1);
        }
        tmem_dealloc(tmem_base, C::TMEM);
    }
}

// [rows][D] bytes, boxes of 16 rows, SWIZZLE_128B
static bool make_byte_map(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t cols) {
    EncodeTiledFn fn = encode_fn();
    if (!fn || rows == 0) return false;
    cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols};
    cuuint32_t box[2] = {(cuuint32_t)cols, 16}, estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool I8, int R, typename Q>
static int launch(const TreeWork& a, cudaStream_t st) {
    const TreeParams& p = a.p;
    typedef Shape<D, I8, R> C;
    static_assert(C::COLS <= 512 && C::RING >= 3, "TMEM or shared memory");
    const size_t smem = C::smem(p.num_seqs, p.mask_words);
    if (smem > (size_t)device_info().max_smem_optin) return PA_ERR_UNSUPPORTED;
    auto kern = tree_terms_kernel<D, I8, R, Q>;
    const cudaError_t e = allow_dynamic_smem<tree_terms_kernel<D, I8, R, Q>>(smem);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap k, v;
    const bool ok = I8 ? make_byte_map(&k, p.k, a.total_rows, D) && make_byte_map(&v, p.v, a.total_rows, D)
                       : make_bf16_map(&k, p.k, a.total_rows, D, D, 16) && make_bf16_map(&v, p.v, a.total_rows, D, D, 16);     // boxes move bits
    if (!ok) return PA_ERR_UNSUPPORTED;
    kern<<<a.workers, C::THREADS, smem, st>>>(k, v, a);
    PA_RETURN_LAUNCH_STATUS();
}

}  // namespace tterms

int tree_terms_workers(int block) { return device_info().sm_count * (block == 16 ? 2 : 1); }

// Rows of a block, 0 where this kernel does not serve or the streaming one is faster.  us, this kernel against the streaming one: int8 pages, 16
// rows: 1000 keys 112 against 214, 4K keys 87 against 204, ragged 128 against 216, 100 keys 38 against 52; half pages, 32 float rows: 4K keys 153
// against 292, 1000 keys 186 against 305, 90 keys 96 against 71 (the host does not know how long contexts are); 16 float rows 205 against 209, and
// of 64 columns 65 against 58: from 17 on.  int8 rows of 64 bytes have no tile here.  Blocks: int8, 256 rows in 32s 332, in 16s 365, 16 rows in a
// block of 32 (ragged) 229 instead of 128; half, 128 rows in 64s 133, in 32s 196; 32 rows in a block of 64 177 instead of 153.
int tree_terms_block(const TreeParams& p) {
    const int G = p.heads / p.kv_heads, rows = p.most * G;
    const bool half = p.q_type == PA_TYPE_F32 && p.kv_type == PA_TYPE_F16, bytes = p.kv_type == PA_TYPE_I8 && p.dim == 128;
    if ((!half && !bytes) || (p.dim != 64 && p.dim != 128) || p.tile_size % 16 || p.num_seqs > kTreeMostSeqs) return 0;
    if ((int64_t)p.total_pages * p.tile_size >= 0x7fffff00ll || ((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.k_scales | (uintptr_t)p.v_scales) % 16) return 0;
    if (half && rows <= 16) return 0;
    if ((uintptr_t)p.q % 16 || p.q_stride % 4) return 0;
    const int block = bytes ? (rows <= 16 ? 16 : 32) : rows <= 32 ? 32 : 64;
    const int64_t steps = ((int64_t)p.num_tiles * p.tile_size + tterms::KT - 1) / tterms::KT;
    return ((int64_t)p.rows * G / block + p.num_seqs) * (steps + kTreeTermsExtra) < 0x7fffffff ? block : 0;     // the list's sums are 32 bits
}

int tree_terms_launch(const TreeWork& a, cudaStream_t st) {
    using namespace tterms;
    const TreeParams& p = a.p;
    if (p.kv_type == PA_TYPE_I8) {
        if (p.q_type == PA_TYPE_F32) return a.block == 16 ? launch<128, true, 16, float>(a, st) : launch<128, true, 32, float>(a, st);
        return a.block == 16 ? launch<128, true, 16, __half>(a, st) : launch<128, true, 32, __half>(a, st);
    }
    if (p.dim == 64) return a.block == 32 ? launch<64, false, 32, float>(a, st) : launch<64, false, 64, float>(a, st);
    return a.block == 32 ? launch<128, false, 32, float>(a, st) : launch<128, false, 64, float>(a, st);
}

int tree_terms_errors(int* host_count) { return (int)cudaMemcpyFromSymbol(host_count, tterms::g_errors, sizeof(int)); }

}  // namespace pa
