// tree_stream.cu -- attention of drafted trees for few query rows: every warp streams keys and values of its own (tree_attention.cuh has
// the work list; the join of pieces is here too).
//
// A warp is a worker with an equal share of the list of 16-key units.  It keeps a ring of its own (16-bit pools: TMA boxes of 16 keys
// x 64 columns, SWIZZLE_128B; int8 pools: bulk copies of 16 rows and their scales), holds 16 or 32 query rows as fragments of mma.sync
// m16n8k16 products, and walks   S = Q K^T,  softmax with a running maximum and sum in float,  O += P V   unit by unit.
//
//   float queries   two terms of half each for q (a row scaled by a power of two first) and for the weights: 22 bits of every factor, float
//                   sums; twice the products, which the copies still cover
//   int8 pools      bytes become halves in registers (1024 + 128 + b as a half, minus 1152: exact); the order of the summed columns and
//                   keys is free as long as both factors have it, so every lane reads 16 bytes of a row at a time; a
//                   key's scale goes to its scores, a value's to its weights, which a row's power of two then brings between 2^14 and 2^15
//                   unit by unit: halves hold the largest product of weight and 1 / scale, whatever it is, and all others to 2^-39 of it
//
// What bounds it: 16-bit pages of 128 columns the copies (32 sequences of 2K keys, 32 heads, 8 rows a head: 189 us, 5.7 TB/s; float queries, 16
// rows: 207 us, 5.3 TB/s), narrower ones and int8 pages the chain of a unit, wait, products, softmax, products, that one to four warps of an SM's
// quarter cover for each other (16 sequences of 4K keys, 12 heads of 64, float queries: 58 us, 3.5 TB/s; instructions issue half of the time; int8
// pages: 72 us, 1.5 TB/s, of which the scaling of the weights takes 2.5).  Softmax weights of 16-bit queries enter the second product in the pages' type,
// since both factors of one are of a type (2.3e-3 of a bfloat16 result where rounding it alone takes 1.7e-3); their sum is of the float ones.  Keys
// come by the warp because few rows give no tile to share, and units of 16 because a page is that long; a smaller unit is the finest cut of a long
// context (one sequence of 333 keys, 12 heads: 14.0 us, of which 5 are the join and its launch).
//
// A value that is not finite in a drafted row does not reach the rows that do not see it: a unit of drafted keys with such values takes
// them out of the product and adds them for the rows that see them.
#include <algorithm>

#include "f32x2.cuh"
#include "mma_utils.cuh"
#include "tcgen05_utils.cuh"
#include "tree_attention.cuh"

namespace pa {
namespace tstream {

constexpr int kUnit = 16;
enum { F32 = PA_TYPE_F32, F16 = PA_TYPE_F16, BF16 = PA_TYPE_BF16, I8 = PA_TYPE_I8 };

__device__ int g_errors;

template <int D, int KT> __host__ __device__ constexpr int stage_bytes() { return KT == I8 ? 2 * kUnit * D + 2 * kUnit * 4 : 2 * kUnit * D * 2; }
template <int D, int W, int KT> __host__ __device__ constexpr int stages() { return W == 16 ? (KT == I8 ? 5 : 3) : KT == I8 ? (D == 128 ? 5 : 8) : D == 128 ? 3 : 6; }

template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF) mma_bf16_16816(d, a, b0, b1);
    else mma_16816_full(d, a[0], a[1], a[2], a[3], b0, b1);
}
// the product alone: d = a b
template <bool BF>
__device__ __forceinline__ void mma_from_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// to += x * by[row], two at a time
__device__ __forceinline__ void add_four_times(float (&to)[4], const float (&x)[4], const float (&by)[2]) {
#pragma unroll
    for (int c = 0; c < 4; c += 2)
        f32x2::unpack2(f32x2::fma2(f32x2::pack2(x[c], x[c + 1]), f32x2::pack2(by[c >> 1], by[c >> 1]), f32x2::pack2(to[c], to[c + 1])), to[c], to[c + 1]);
}
// to += x, two at a time
__device__ __forceinline__ void add_four(float (&to)[4], const float (&x)[4]) {
#pragma unroll
    for (int c = 0; c < 4; c += 2) f32x2::unpack2(f32x2::add2(f32x2::pack2(to[c], to[c + 1]), f32x2::pack2(x[c], x[c + 1])), to[c], to[c + 1]);
}
template <bool BF> __device__ __forceinline__ uint32_t pack(float x, float y) {
    if constexpr (BF) return pack_bf16x2(x, y);
    else return pack_half2(x, y);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// two halves from two bytes of w (already ^ 0x80): those that sel names, beside 0x64 as the upper byte of each
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t w, uint32_t sel) {
    const uint32_t u = __byte_perm(w, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));     // 1152
    return *reinterpret_cast<const uint32_t*>(&h);
}
// byte j of x and of y
__device__ __forceinline__ uint32_t byte_of_both(uint32_t x, uint32_t y, int j) {
    const uint32_t w = __byte_perm(x, y, (uint32_t)j | (uint32_t)(4 + j) << 4);
    return bytes_to_half2(w, 0x5140);
}

template <int D, int MT, int QT, int KT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 1) tree_stream_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                                     const TreeWork a) {
    constexpr bool BF = KT == BF16, TWO = QT == F32;
    constexpr int ST = stages<D, kWarps, KT>(), STAGE = stage_bytes<D, KT>(), NT = D / 8, KS = D / 16, TERMS = TWO ? 2 : 1, CB = D / 64;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ int fail_word;
    const TreeParams& p = a.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lr = lane >> 2, lc = lane & 3;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = base + warp * ST * STAGE, bar0 = base + kWarps * ST * STAGE + warp * ST * 8;
    int* pre = reinterpret_cast<int*>(smem_raw + (base - smem_u32(smem_raw)) + kWarps * ST * (STAGE + 8));
    const uint32_t fail_sm = smem_u32(&fail_word);
    if (lane == 0) {
        for (int s = 0; s < ST; ++s) mbar_init(bar0 + s * 8, 1);
        mbar_fence_init();
    }
    if (threadIdx.x == 0) fail_word = 0;
    int* cut = pre + p.num_seqs + 1;
    shares::count_units(pre, p.num_seqs, [&](int b) { return tree_seq(p, b, MT * 16, kUnit).units(0); });
    shares::count_units(cut, p.num_seqs, [&](int b) { return tree_seq(p, b, MT * 16, kUnit).units(a.extra); });
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int w = warp * gridDim.x + blockIdx.x, G = p.heads / p.kv_heads;
    // the list is cut with what items take to begin and end (`cut`), and walked by its units of keys (`pre`)
    const int64_t total = (int64_t)cut[p.num_seqs] * p.kv_heads;
    const int64_t ns = shares::count(total, a.workers, a.least);
    auto unit_at = [&](int64_t c) -> int64_t {
        if (c >= total) return (int64_t)pre[p.num_seqs] * p.kv_heads;
        const int b = shares::find_token(cut, p.num_seqs, c, p.kv_heads);
        const TreeSeq q = tree_seq(p, b, MT * 16, kUnit);
        const int64_t rem = c - (int64_t)cut[b] * p.kv_heads;
        const int each = q.steps + a.extra, item = (int)(rem / each);
        return (int64_t)pre[b] * p.kv_heads + (int64_t)item * q.steps + (a.whole ? 0 : max((int)(rem - (int64_t)item * each) - a.extra, 0));
    };
    const int64_t at = w < ns ? unit_at(total * (w + (lane & 1)) / ns) : 0;         // even lanes: the beginning, odd ones: the end
    const int64_t f_lo = __shfl_sync(0xffffffffu, at, 0), f_hi = __shfl_sync(0xffffffffu, at, 1);
    if (f_lo >= f_hi) {
        if (lane == 0) a.notes[w] = TreeNote{};
        return;
    }

    // ---- the copies: unit f's rows in the pools, 32 units at a time
    auto rows_of = [&](int64_t f) -> int {
        if (f >= f_hi) return -1;
        const int b = shares::find_token(pre, p.num_seqs, f, p.kv_heads);
        const TreeSeq q = tree_seq(p, b, MT * 16, kUnit);
        const int64_t rem = f - (int64_t)pre[b] * p.kv_heads;
        const int g = (int)(rem / q.units(0)), j = (int)(rem % q.steps) * kUnit, t = j / p.tile_size;
        const int row = p.beam_ids ? __ldg(p.beam_ids + b) : b;
        if ((unsigned)row >= (unsigned)p.num_beams || t >= p.num_tiles) return -1;
        const int page = __ldg(p.table + ((int64_t)row * p.kv_heads + g) * p.num_tiles + t);
        return (unsigned)page < (unsigned)p.total_pages ? page * p.tile_size + (j - t * p.tile_size) : -1;
    };
    int rows_cur = rows_of(f_lo + lane), rows_nxt = rows_of(f_lo + 32 + lane);
    int64_t f_is = f_lo;                // next unit to request
    int is_stage = 0;
    uint32_t mapped = 0;                // bit s: the unit in stage s has a page
    auto issue = [&] {
        if (f_is >= f_hi) return;
        const int o = (int)(f_is - f_lo);
        if (o && (o & 31) == 0) {
            rows_cur = rows_nxt;
            rows_nxt = rows_of(f_is + 32 + lane);
        }
        const int row = __shfl_sync(0xffffffffu, rows_cur, o & 31);
        mapped = row >= 0 ? mapped | 1u << is_stage : mapped & ~(1u << is_stage);
        if (a.polls && elect_one()) {   // 0: a wait that is to run out
            const uint32_t st = ring + is_stage * STAGE, bar = bar0 + is_stage * 8;
            if (row < 0) {
                mbar_arrive(bar);       // nothing to fetch
            } else {
                mbar_arrive_expect_tx(bar, STAGE);
                if constexpr (KT == I8) {
                    bulk_g2s_nohint(st, static_cast<const int8_t*>(p.k) + (int64_t)row * D, kUnit * D, bar);
                    bulk_g2s_nohint(st + 2 * kUnit * D, p.k_scales + row, kUnit * 4, bar);
                    bulk_g2s_nohint(st + kUnit * D, static_cast<const int8_t*>(p.v) + (int64_t)row * D, kUnit * D, bar);
                    bulk_g2s_nohint(st + 2 * kUnit * D + kUnit * 4, p.v_scales + row, kUnit * 4, bar);
                } else {
#pragma unroll
                    for (int b = 0; b < CB; ++b) tma_load_2d(st + b * 2048, &tmK, b * 64, row, bar);
#pragma unroll
                    for (int b = 0; b < CB; ++b) tma_load_2d(st + (CB + b) * 2048, &tmV, b * 64, row, bar);
                }
            }
        }
        __syncwarp();
        ++f_is;
        if (++is_stage == ST) is_stage = 0;
    };
#pragma unroll
    for (int s = 0; s < ST; ++s) issue();

    // ---- the item at hand
    int b = shares::find_token(pre, p.num_seqs, f_lo, p.kv_heads);
    TreeSeq sq = tree_seq(p, b, MT * 16, kUnit);
    int item, u;                        // item within the sequence (kv head, block), unit within the item
    {
        const int64_t rem = f_lo - (int64_t)pre[b] * p.kv_heads;
        item = (int)(rem / sq.steps);
        u = (int)(rem % sq.steps);
    }
    int u0 = u;                         // the piece at hand begins with it
    uint32_t qf[MT][TERMS][KS][4];
    float o[MT][NT][4], m[MT][2], l[MT][2], fe[MT][2], top[MT][2];     // reference, sum, factor of the scores, largest score
    int node[MT][2];                    // of a row, -1: no row
    // columns of a lane's part of the A and B fragments of step ks, and of its part of the results' tile j
    auto qcol = [&](int ks, int hf) { return KT == I8 ? (ks >> 2) * 64 + lc * 16 + (ks & 3) * 4 + hf * 2 : ks * 16 + hf * 8 + 2 * lc; };
    auto ocol = [&](int j, int e) { return KT == I8 ? (2 * lc + e) * (D / 8) + j : j * 8 + 2 * lc + e; };
    auto open_item = [&] {
        const int g = item / sq.blocks, rr0 = item % sq.blocks * (MT * 16);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int rr = rr0 + mt * 16 + lr + 8 * i;
                node[mt][i] = rr < sq.n * G ? rr / G : -1;
                m[mt][i] = top[mt][i] = -INFINITY;
                l[mt][i] = 0.f;
                const int64_t at = node[mt][i] >= 0 ? (int64_t)(sq.r0 + rr / G) * p.q_stride + (int64_t)(g * G + rr % G) * D : 0;
                fe[mt][i] = 1.4426950408889634f / p.temperature;
                if constexpr (!TWO) {
                    const uint16_t* q = static_cast<const uint16_t*>(p.q) + at;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf)
                            qf[mt][0][ks][2 * hf + i] = node[mt][i] >= 0 ? __ldg(reinterpret_cast<const uint32_t*>(q + qcol(ks, hf))) : 0u;
                } else {
                    const float* q = static_cast<const float*>(p.q) + at;
                    float2 x[KS][2];
                    float big = 0.f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            x[ks][hf] = node[mt][i] >= 0 ? __ldg(reinterpret_cast<const float2*>(q + qcol(ks, hf))) : make_float2(0.f, 0.f);
                            big = fmaxf(big, fmaxf(fabsf(x[ks][hf].x), fabsf(x[ks][hf].y)));
                        }
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    // the row's largest between 2^10 and 2^11: halves hold hi, and lo down to 2^-35 of it
                    const int e = big > 0.f && big < INFINITY ? max(-100, min(100, 10 - ilogbf(big))) : 0;
                    const float up = exp2f((float)e);
                    fe[mt][i] *= exp2f((float)-e);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const float vx = x[ks][hf].x * up, vy = x[ks][hf].y * up;
                            const uint32_t hi = pack_half2(vx, vy);
                            const float2 back = unpack_half2(hi);
                            qf[mt][0][ks][2 * hf + i] = hi;
                            qf[mt][TERMS - 1][ks][2 * hf + i] = pack_half2(vx - back.x, vy - back.y);
                        }
                }
            }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[mt][n][c] = 0.f;
    };
    // to_end: the piece ends its item
    auto close_item = [&](bool to_end) {
        const int g = item / sq.blocks, rr0 = item % sq.blocks * (MT * 16);
        const int64_t f_item = (int64_t)pre[b] * p.kv_heads + (int64_t)item * sq.steps;
        const int64_t slot = 2 * (int64_t)w + (f_item > f_lo ? 1 : 0);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float s = l[mt][i] + __shfl_xor_sync(0xffffffffu, l[mt][i], 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                if (node[mt][i] < 0) continue;
                const int rl = mt * 16 + lr + 8 * i, rr = rr0 + rl;
                if (u0 == 0 && to_end) {
                    const float eps = 1e-6f * kTreeStreamScale * (TWO && m[mt][i] != -INFINITY ? fast_exp2(top[mt][i] - m[mt][i]) : 1.f);
                    const float inv = 1.f / (s + eps);
                    const int64_t at = ((int64_t)(sq.r0 + rr / G) * p.heads + g * G + rr % G) * D;
                    if constexpr (KT == I8) {
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int n = 0; n < NT; n += 2) {
                                const float x = o[mt][n][2 * i + e] * inv, y = o[mt][n + 1][2 * i + e] * inv;
                                if constexpr (TWO) *reinterpret_cast<float2*>(static_cast<float*>(p.out) + at + ocol(n, e)) = make_float2(x, y);
                                else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + at + ocol(n, e)) = pack<BF>(x, y);
                            }
                    } else {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const float x = o[mt][n][2 * i] * inv, y = o[mt][n][2 * i + 1] * inv;
                            if constexpr (TWO) *reinterpret_cast<float2*>(static_cast<float*>(p.out) + at + ocol(n, 0)) = make_float2(x, y);
                            else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + at + ocol(n, 0)) = pack<BF>(x, y);
                        }
                    }
                } else {
                    float* dst = a.part + (slot * (MT * 16) + rl) * (D + 4);
                    if (lc == 0) *reinterpret_cast<float4*>(dst + D) = make_float4(m[mt][i], s, TWO ? top[mt][i] : m[mt][i], 0.f);
                    if constexpr (KT == I8) {
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int n = 0; n < NT; n += 2)
                                *reinterpret_cast<float2*>(dst + ocol(n, e)) = make_float2(o[mt][n][2 * i + e], o[mt][n + 1][2 * i + e]);
                    } else {
#pragma unroll
                        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(dst + ocol(n, 0)) = make_float2(o[mt][n][2 * i], o[mt][n][2 * i + 1]);
                    }
                }
            }
    };
    auto next_item = [&] {
        u = u0 = 0;
        if (++item == p.kv_heads * sq.blocks) {
            item = 0;
            do ++b; while (pre[b + 1] == pre[b]);       // a sequence without nodes has no items
            sq = tree_seq(p, b, MT * 16, kUnit);
        }
        open_item();
    };
    open_item();
    int stage = 0;
    uint32_t phase = 0;
    int64_t f = f_lo;
    for (; f < f_hi; ++f) {
        if (u == sq.steps) {
            close_item(true);
            next_item();
        }
        const uint32_t ks_sm = ring + stage * STAGE, vs_sm = ks_sm + (KT == I8 ? kUnit * D : CB * 2048);
        if (!__all_sync(0xffffffffu, tc::tc_wait(bar0 + stage * 8, phase, fail_sm, a.polls))) break;
        if (mapped >> stage & 1u) {
            const int j0 = u * kUnit, valid = min(kUnit, sq.keys - j0);
            const bool drafts = j0 + kUnit > sq.ctx;
            // which of the unit's keys a row sees
            uint32_t vis[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    vis[mt][i] = node[mt][i] >= 0 ? 0xffffu : 0u;
                    if (drafts && node[mt][i] >= 0) {
                        const uint32_t* mw = p.mask + (int64_t)(sq.r0 + node[mt][i]) * p.mask_words;
                        vis[mt][i] = tree_visible(j0 - sq.ctx, p.mask_words, [&](int x) { return __ldg(mw + x); }) & ((1u << valid) - 1u);
                    }
                }
            if (KT != I8 && valid < kUnit) {    // value rows past the last key may hold anything (0 x NaN = NaN)
                for (int i = lane; i < (kUnit - valid) * (D / 8); i += 32) {
                    const int r = valid + i / (D / 8), c = i % (D / 8);
                    asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vs_sm + (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4)),
                                 "r"(0u) : "memory");
                }
                fence_proxy_async();
                __syncwarp();
            }
            // The tensor cores' own sums are cut, not rounded: float queries sum the large terms over two steps there at most, and the
            // rest in float; the small terms (2^-11 of the large ones) may be summed up there
            float s[MT][2][4], s_lo[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[mt][n][c] = s_lo[mt][n][c] = 0.f;
            auto add_to = [&](float (&to)[4], const uint32_t (&q0)[4], const uint32_t (&q1)[4], uint32_t b00, uint32_t b01, uint32_t b10, uint32_t b11) {
                float t[4];
                mma_from_zero<BF>(t, q0, b00, b01);
                mma<BF>(t, q1, b10, b11);
                add_four(to, t);
            };
            if constexpr (KT == I8) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        const uint4 v = lds_128(ks_sm + (n * 8 + lr) * D + cb * 64 + lc * 16);
                        const uint32_t wd[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
#pragma unroll
                        for (int k = 0; k < 4; k += 2) {
                            const uint32_t b00 = bytes_to_half2(wd[k], 0x4140), b01 = bytes_to_half2(wd[k], 0x4342);
                            const uint32_t b10 = bytes_to_half2(wd[k + 1], 0x4140), b11 = bytes_to_half2(wd[k + 1], 0x4342);
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                if constexpr (TWO) {
                                    mma<BF>(s_lo[mt][n], qf[mt][1][cb * 4 + k], b00, b01);
                                    mma<BF>(s_lo[mt][n], qf[mt][1][cb * 4 + k + 1], b10, b11);
                                    add_to(s[mt][n], qf[mt][0][cb * 4 + k], qf[mt][0][cb * 4 + k + 1], b00, b01, b10, b11);
                                } else {
                                    mma<BF>(s[mt][n], qf[mt][0][cb * 4 + k], b00, b01);
                                    mma<BF>(s[mt][n], qf[mt][0][cb * 4 + k + 1], b10, b11);
                                }
                            }
                        }
                    }
            } else {
                const int r = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                for (int ks = 0; ks < KS; ks += 2) {
                    uint32_t b[2][4];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int c = ((ks + k) & 3) * 2 + ((lane >> 3) & 1);
                        ldsm_x4(ks_sm + (ks >> 2) * 2048 + r * 128 + ((c ^ (r & 7)) << 4), b[k][0], b[k][1], b[k][2], b[k][3]);
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            if constexpr (TWO) {
                                mma<BF>(s_lo[mt][n], qf[mt][1][ks], b[0][2 * n], b[0][2 * n + 1]);
                                mma<BF>(s_lo[mt][n], qf[mt][1][ks + 1], b[1][2 * n], b[1][2 * n + 1]);
                                add_to(s[mt][n], qf[mt][0][ks], qf[mt][0][ks + 1], b[0][2 * n], b[0][2 * n + 1], b[1][2 * n], b[1][2 * n + 1]);
                            } else {
                                mma<BF>(s[mt][n], qf[mt][0][ks], b[0][2 * n], b[0][2 * n + 1]);
                                mma<BF>(s[mt][n], qf[mt][0][ks + 1], b[1][2 * n], b[1][2 * n + 1]);
                            }
                        }
                }
            }
            if constexpr (TWO) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[mt][n][c] += s_lo[mt][n][c];
            }
            float ksc[4] = {1.f, 1.f, 1.f, 1.f}, vsc[4] = {1.f, 1.f, 1.f, 1.f};      // of the lane's keys 2 lc, 2 lc + 1, 2 lc + 8, 2 lc + 9
            if constexpr (KT == I8) {
                const uint32_t sc = ks_sm + 2 * kUnit * D + 8 * lc;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint2 kk = lds_64(sc + 32 * x), vv = lds_64(sc + 64 + 32 * x);
                    ksc[2 * x] = __frcp_rn(__uint_as_float(kk.x));
                    ksc[2 * x + 1] = __frcp_rn(__uint_as_float(kk.y));
                    vsc[2 * x] = __frcp_rn(__uint_as_float(vv.x));
                    vsc[2 * x + 1] = __frcp_rn(__uint_as_float(vv.y));
                }
            }
            uint32_t pf[MT][TERMS][4];
            float down[MT][2];              // int8: what a row's products are times
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int i = c >> 1, k = n * 8 + 2 * lc + (c & 1);
                        float x = s[mt][n][c] * fe[mt][i];
                        if constexpr (KT == I8) x *= ksc[2 * n + (c & 1)];
                        s[mt][n][c] = vis[mt][i] >> k & 1u ? x : -INFINITY;
                        mx[i] = fmaxf(mx[i], s[mt][n][c]);
                    }
                float ref[2], corr[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                    mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                    if constexpr (TWO) top[mt][i] = fmaxf(top[mt][i], mx[i]);
                    // the reference moves only when a score exceeds it by more than 2^8: most units rescale nothing
                    const bool raise = mx[i] > m[mt][i] + 8.f || m[mt][i] == -INFINITY;
                    const float mn = raise ? mx[i] : m[mt][i];
                    corr[i] = raise && m[mt][i] != -INFINITY ? fast_exp2(m[mt][i] - mn) : 1.f;
                    m[mt][i] = mn;
                    ref[i] = (mn == -INFINITY ? 0.f : mn) - 7.f;        // weights times kTreeStreamScale
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        l[mt][i] *= corr[i];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            o[mt][n][2 * i] *= corr[i];
                            o[mt][n][2 * i + 1] *= corr[i];
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float e = fast_exp2(s[mt][n][c] - ref[c >> 1]);
                        l[mt][c >> 1] += e;
                        if constexpr (KT == I8) e = e != 0.f ? e * vsc[2 * n + (c & 1)] : 0.f;      // a key that nobody sees may have any scale
                        s[mt][n][c] = e;
                    }
                if constexpr (KT == I8) {       // a row's largest between 2^14 and 2^15, see above
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float big = fmaxf(fmaxf(fabsf(s[mt][0][2 * i]), fabsf(s[mt][0][2 * i + 1])), fmaxf(fabsf(s[mt][1][2 * i]), fabsf(s[mt][1][2 * i + 1])));
                        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                        const uint32_t e = max(__float_as_uint(big) >> 23, 15u);
                        const float up = __uint_as_float((268u - e) << 23);
                        down[mt][i] = __uint_as_float((e - 14u) << 23);
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c) s[mt][n][2 * i + c] *= up;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = s[mt][j >> 1][2 * (j & 1)], y = s[mt][j >> 1][2 * (j & 1) + 1];
                    pf[mt][0][j] = pack<BF>(x, y);
                    if constexpr (TWO) {
                        const float2 back = unpack_half2(pf[mt][0][j]);
                        pf[mt][TERMS - 1][j] = pack_half2(x - back.x, y - back.y);
                    }
                }
            }
            auto weigh = [&](int mt, int n, uint32_t b0, uint32_t b1) {
                if constexpr (TWO || KT == I8) {
                    float t[4];
                    mma_from_zero<BF>(t, pf[mt][TERMS - 1], b0, b1);
                    if constexpr (TWO) mma<BF>(t, pf[mt][0], b0, b1);
                    if constexpr (KT == I8) add_four_times(o[mt][n], t, down[mt]);
                    else add_four(o[mt][n], t);
                } else {
                    mma<BF>(o[mt][n], pf[mt][0], b0, b1);
                }
            };
            if constexpr (KT == I8) {
                constexpr int W = D / 32;       // words of a lane's part of a value row
                uint32_t vw[4][W];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t at = vs_sm + (2 * lc + (k & 1) + (k >> 1) * 8) * D + lr * (D / 8);
                    if constexpr (W == 4) {
                        const uint4 v = lds_128(at);
                        vw[k][0] = v.x; vw[k][1] = v.y; vw[k][W - 2] = v.z; vw[k][W - 1] = v.w;
                    } else {
                        const uint2 v = lds_64(at);
                        vw[k][0] = v.x; vw[k][1] = v.y;
                    }
#pragma unroll
                    for (int x = 0; x < W; ++x) vw[k][x] ^= 0x80808080u;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t b0 = byte_of_both(vw[0][n >> 2], vw[1][n >> 2], n & 3), b1 = byte_of_both(vw[2][n >> 2], vw[3][n >> 2], n & 3);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) weigh(mt, n, b0, b1);
                }
            } else {
                const int vr = (lane & 7) + ((lane >> 3) & 1) * 8;
                auto load_values = [&](int np, uint32_t (&v)[4]) {
                    ldsm_x4_trans(vs_sm + (np >> 2) * 2048 + vr * 128 + ((((np & 3) * 2 + (lane >> 4)) ^ (vr & 7)) << 4), v[0], v[1], v[2], v[3]);
                };
                bool odd = false;
                if (drafts) {           // a drafted row that is not finite may be hidden from some
                    uint32_t any = 0;
#pragma unroll
                    for (int np = 0; np < NT / 2; ++np) {
                        uint32_t v[4];
                        load_values(np, v);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
                            any |= (uint32_t)((v[x] & E) == E) | (uint32_t)((v[x] >> 16 & E) == E);
                        }
                    }
                    odd = __any_sync(0xffffffffu, any != 0);
                }
                if (odd) {
                    // rows that see such a key meet it here, value by value; the product below finds a zero in its place
                    for (int k = 0; k < valid; ++k) {
                        const int from = (lane & ~3) | ((k & 7) >> 1);      // the lane with this key's weights
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            float pk[2];
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const float x0 = k < 8 ? s[mt][0][2 * i] : s[mt][1][2 * i], x1 = k < 8 ? s[mt][0][2 * i + 1] : s[mt][1][2 * i + 1];
                                pk[i] = __shfl_sync(0xffffffffu, k & 1 ? x1 : x0, from);
                            }
                            for (int n = 0; n < NT; ++n) {
                                uint32_t v;
                                const int c = n & 7;
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(vs_sm + (n >> 3) * 2048 + k * 128 + ((c ^ (k & 7)) << 4) + 4 * lc) : "memory");
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint16_t h = (uint16_t)(e ? v >> 16 : v);
                                    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
                                    if ((h & E) != E) continue;
                                    const float x = BF ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
#pragma unroll
                                    for (int i = 0; i < 2; ++i)
                                        if (vis[mt][i] >> k & 1u) {
#pragma unroll
                                            for (int nn = 0; nn < NT; ++nn)         // registers: no index that is not known
                                                if (nn == n) o[mt][nn][2 * i + e] += pk[i] * x;
                                        }
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int np = 0; np < NT / 2; ++np) {
                    uint32_t v[4];
                    load_values(np, v);
                    if (odd) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
                            v[x] = ((v[x] & E) == E ? 0u : v[x] & 0xffffu) | ((v[x] >> 16 & E) == E ? 0u : v[x] & 0xffff0000u);
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        weigh(mt, 2 * np, v[0], v[1]);
                        weigh(mt, 2 * np + 1, v[2], v[3]);
                    }
                }
            }
        }
        __syncwarp();                   // every lane has read the stage
        issue();                        // refills it
        ++u;
        if (++stage == ST) {
            stage = 0;
            phase ^= 1u;
        }
    }
    if (f < f_hi) {                     // a wait ran out: the copies that were requested land, and the pieces from here on are NaN
        for (int64_t i = a.polls ? f : f_is; i < f_is; ++i) {
            const int at = stage + (int)(i - f);
            tc::tc_let_land(bar0 + at % ST * 8, at < ST ? phase : phase ^ 1u);
        }
        if (lane == 0) atomicAdd(&g_errors, 1);
        const float nan = __int_as_float(0x7fc00000);
        auto spoil = [&] {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) l[mt][0] = l[mt][1] = nan;
        };
        for (f += sq.steps - u; f < f_hi; f += sq.steps) {
            spoil();
            close_item(true);
            next_item();
        }
        spoil();
        u = (int)(sq.steps - (f - f_hi));
    }
    close_item(u == sq.steps);
    if (lane == 0) {
        const int64_t f_item = (int64_t)pre[b] * p.kv_heads + (int64_t)item * sq.steps;
        const int64_t c_item = (int64_t)cut[b] * p.kv_heads + (int64_t)item * (sq.steps + a.extra);
        a.notes[w] = tree_note(a, sq, item / sq.blocks, item % sq.blocks * (MT * 16), u0, u, c_item, total, ns, 2 * (int64_t)w + (f_item > f_lo ? 1 : 0));
    }
}

// The rows of items whose keys were in several shares.  blockIdx.x: the share that noted the item (where items are few and their pieces many,
// the number of the note among all), blockIdx.y: its share of the item's rows.  A warp has RW rows at a time, or SPLIT warps one row whose pieces they
// share; a lane has D / 32 neighbouring columns.  Pieces come in order, FLIGHT of a warp at a time with the loads of all its rows in flight, under a running
// maximum.  It is bound by trips to L2: waiting for the shares, note, pieces.  (One row a warp and a CTA for every eight of them took 19 of 128 us
// behind 32 sequences of 128 rows and 8 kv heads.)
constexpr int kJoinWarps = 8;
template <typename Q, int NV, int SPLIT, int RW>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_join_kernel(const TreeWork a) {
    constexpr int D = NV * 32, LD = D + 4, ROWS = kJoinWarps / SPLIT * RW, FLIGHT = SPLIT > 1 ? 8 : RW == 1 ? 4 : 8 / RW;
    __shared__ float s_acc[SPLIT > 1 ? kJoinWarps : 1][D], s_ml[SPLIT > 1 ? kJoinWarps : 1][3];
    const TreeParams& p = a.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = p.group;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int w0 = blockIdx.x;
    int4 n0, n1;
    if constexpr (SPLIT > 1) {
        __shared__ int s_count[kJoinWarps], s_found;
        __shared__ int4 s_note[2];
        const int per = (a.workers + kJoinWarps * 32 - 1) / (kJoinWarps * 32);
        uint32_t noted = 0;             // a thread has `per` shares, at most 32 (a trip to L2 each, eight under way at a time)
        for (int i0 = 0; i0 < per; i0 += 8) {
            int rows[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int w = threadIdx.x * per + i0 + i;
                rows[i] = i0 + i < per && w < a.workers ? __ldcg(&a.notes[w].rows) : 0;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) noted |= rows[i] > 0 ? 1u << (i0 + i) : 0u;
        }
        // the first note of a thread comes along: one is all that most have
        const int4* mine0 = reinterpret_cast<const int4*>(a.notes + threadIdx.x * per + max(__ffs(noted) - 1, 0));
        int4 a0 = make_int4(0, 0, 0, 0), a1 = a0;
        if (noted) {
            a0 = __ldcg(mine0);
            a1 = __ldcg(mine0 + 1);
        }
        const int mine = __popc(noted);
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        if (lane == 31) s_count[warp] = before;
        if (threadIdx.x == 0) s_found = -1;
        __syncthreads();
        before -= mine;
        for (int k = 0; k < warp; ++k) before += s_count[k];
        if ((int)blockIdx.x >= before && (int)blockIdx.x < before + mine) {
            const int left = blockIdx.x - before;
            for (int k = left; k > 0; --k) noted &= noted - 1;
            const int w = threadIdx.x * per + __ffs(noted) - 1;
            if (left > 0) {
                a0 = __ldcg(reinterpret_cast<const int4*>(a.notes + w));
                a1 = __ldcg(reinterpret_cast<const int4*>(a.notes + w) + 1);
            }
            s_found = w;
            s_note[0] = a0;
            s_note[1] = a1;
        }
        __syncthreads();
        w0 = s_found;
        if (w0 < 0) return;
        n0 = s_note[0];
        n1 = s_note[1];
    } else {
        const int4* note = reinterpret_cast<const int4*>(a.notes + w0);
        n0 = __ldcg(note);
        n1 = __ldcg(note + 1);
    }
    const int w1 = n1.x;
    const int64_t step = (int64_t)2 * a.block * LD;
    const float *rest = a.part + (int64_t)2 * w0 * a.block * LD, *first = a.part + (int64_t)n1.y * a.block * LD;       // share w's piece, w > w0; the first
#pragma unroll 1
    for (int r0 = blockIdx.y * ROWS; r0 < n0.x; r0 += gridDim.y * ROWS) {
        const int rl = r0 + warp / SPLIT * RW;          // the warp's rows: rl .. rl + RW - 1
        float mx[RW], top[RW], l[RW], acc[RW][NV];
#pragma unroll
        for (int x = 0; x < RW; ++x) {
            mx[x] = top[x] = -INFINITY;
            l[x] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) acc[x][i] = 0.f;
        }
#pragma unroll 1
        for (int w = w0 + warp % SPLIT; rl < n0.x && w <= w1; w += FLIGHT * SPLIT) {
            float4 ml[FLIGHT][RW];
            float v[FLIGHT][RW][NV];
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k)
#pragma unroll
                for (int x = 0; x < RW; ++x) {
                    const int wk = w + k * SPLIT;
                    ml[k][x] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
                    if (wk > w1 || rl + x >= n0.x) continue;
                    const float* s = (wk == w0 ? first : rest + (wk - w0) * step) + (rl + x) * LD;
                    ml[k][x] = __ldcg(reinterpret_cast<const float4*>(s + D));
                    if constexpr (NV == 4) {
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(s) + lane);
                        v[k][x][0] = y.x; v[k][x][1] = y.y; v[k][x][NV - 2] = y.z; v[k][x][NV - 1] = y.w;
                    } else {
                        const float2 y = __ldcg(reinterpret_cast<const float2*>(s) + lane);
                        v[k][x][0] = y.x; v[k][x][1] = y.y;
                    }
                }
#pragma unroll
            for (int x = 0; x < RW; ++x) {
                float mn = mx[x];
#pragma unroll
                for (int k = 0; k < FLIGHT; ++k) {
                    mn = fmaxf(mn, ml[k][x].x);
                    top[x] = fmaxf(top[x], ml[k][x].z);
                }
                const float ref = mn == -INFINITY ? 0.f : mn, f = exp2f(mx[x] - ref);
                mx[x] = mn;
                l[x] *= f;
#pragma unroll
                for (int i = 0; i < NV; ++i) acc[x][i] *= f;
#pragma unroll
                for (int k = 0; k < FLIGHT; ++k) {
                    if (ml[k][x].x == -INFINITY && ml[k][x].y == 0.f) continue;       // no piece, or it saw nothing: 0 x infinity = NaN
                    const float c = exp2f(ml[k][x].x - ref);
                    l[x] = fmaf(c, ml[k][x].y, l[x]);
#pragma unroll
                    for (int i = 0; i < NV; ++i) acc[x][i] = fmaf(c, v[k][x][i], acc[x][i]);
                }
            }
        }
        if constexpr (SPLIT > 1) {                      // RW is 1
#pragma unroll
            for (int i = 0; i < NV; ++i) s_acc[warp][lane * NV + i] = acc[0][i];
            if (lane == 0) {
                s_ml[warp][0] = mx[0];
                s_ml[warp][1] = l[0];
                s_ml[warp][2] = top[0];
            }
            __syncthreads();
            if (warp % SPLIT == 0) {
                float all = -INFINITY;
#pragma unroll
                for (int k = 0; k < SPLIT; ++k) {
                    all = fmaxf(all, s_ml[warp + k][0]);
                    top[0] = fmaxf(top[0], s_ml[warp + k][2]);
                }
                l[0] = 0.f;
                mx[0] = all;
                const float ref = all == -INFINITY ? 0.f : all;
#pragma unroll
                for (int i = 0; i < NV; ++i) acc[0][i] = 0.f;
#pragma unroll
                for (int k = 0; k < SPLIT; ++k) {
                    const float m = s_ml[warp + k][0];
                    if (m == -INFINITY && s_ml[warp + k][1] == 0.f) continue;
                    const float c = exp2f(m - ref);
                    l[0] = fmaf(c, s_ml[warp + k][1], l[0]);
#pragma unroll
                    for (int i = 0; i < NV; ++i) acc[0][i] = fmaf(c, s_acc[warp + k][lane * NV + i], acc[0][i]);
                }
            }
            __syncthreads();
            if (warp % SPLIT) continue;
        }
#pragma unroll
        for (int x = 0; x < RW; ++x) {
            if (rl + x >= n0.x) continue;
            const int rr = n0.w + rl + x;
            const float inv = 1.f / (l[x] + 1e-6f * a.p_scale * (mx[x] == -INFINITY ? 1.f : exp2f(top[x] - mx[x])));     // the formula's sum is relative to the largest score
            Q* out = static_cast<Q*>(p.out) + ((int64_t)(n0.y + rr / G) * p.heads + n0.z * G + rr % G) * D + lane * NV;
#pragma unroll
            for (int i = 0; i < NV; i += 2) {
                if constexpr (sizeof(Q) == 4) {
                    *reinterpret_cast<float2*>(out + i) = make_float2(acc[x][i] * inv, acc[x][i + 1] * inv);
                } else {
                    Q two[2] = {tree_narrow<Q>(acc[x][i] * inv), tree_narrow<Q>(acc[x][i + 1] * inv)};
                    *reinterpret_cast<uint32_t*>(out + i) = *reinterpret_cast<uint32_t*>(two);
                }
            }
        }
    }
}

template <int D, int MT, int QT, int KT, int kWarps>
static int launch(const TreeWork& a, cudaStream_t st) {
    const TreeParams& p = a.p;
    constexpr int ST = stages<D, kWarps, KT>(), STAGE = stage_bytes<D, KT>();
    const size_t smem = (size_t)kWarps * ST * (STAGE + 8) + 2 * (p.num_seqs + 1) * 4 + 1024;
    auto kern = tree_stream_kernel<D, MT, QT, KT, kWarps>;
    const cudaError_t e = allow_dynamic_smem<tree_stream_kernel<D, MT, QT, KT, kWarps>>(smem);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap k{}, v{};
    if constexpr (KT != I8) {           // boxes move bits: one map type for both 16-bit types
        if (!tc::make_bf16_map(&k, p.k, a.total_rows, D, D, 16) || !tc::make_bf16_map(&v, p.v, a.total_rows, D, D, 16)) return PA_ERR_UNSUPPORTED;
    }
    kern<<<device_info().sm_count, kWarps * 32, smem, st>>>(k, v, a);
    PA_RETURN_LAUNCH_STATUS();
}

}  // namespace tstream

namespace tstream {

template <typename Q, int NV, int SPLIT, int RW>
static int join(const TreeWork& a, int64_t items, cudaStream_t st) {
    const int64_t rows = std::min<int64_t>((int64_t)a.p.most * a.p.group, a.block), groups = (rows * SPLIT + kJoinWarps * RW - 1) / (kJoinWarps * RW);
    const int64_t x = SPLIT > 1 ? items : a.workers, most = SPLIT == 1 && RW == 1 ? groups : 4 * device_info().sm_count / x;      // a few CTAs an SM walk the rest
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)x, (unsigned)std::max<int64_t>(1, std::min(groups, most)));
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // resident before the shares' kernel ends
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, tree_join_kernel<Q, NV, SPLIT, RW>, a);
}

}  // namespace tstream

int tree_join_launch(const TreeWork& a, cudaStream_t st) {
    using namespace tstream;
    const TreeParams& p = a.p;
    // pieces of an item, were all items alike: from 16 (64) on a row's pieces are shared by four (eight) warps
    const int64_t items = tree_items(p, a.block);
    const int split = a.workers > 32 * kJoinWarps * 32 ? 1 : a.workers >= 64 * items ? 8 : a.workers >= 16 * items ? 4 : 1;
#define PA_TJN(Q, NV)                                                                                                  \
    return split == 8 ? join<Q, NV, 8, 1>(a, items, st) : split == 4 ? join<Q, NV, 4, 1>(a, items, st)                 \
         : a.block <= 32 ? join<Q, NV, 1, 1>(a, items, st) : join<Q, NV, 1, 4>(a, items, st);
#define PA_TJ(QT, Q)                                                                                                   \
    if (p.q_type == QT) {                                                                                              \
        if (p.dim == 64) PA_TJN(Q, 2)                                                                                  \
        PA_TJN(Q, 4)                                                                                                   \
    }
    PA_TJ(F32, float) PA_TJ(F16, __half) PA_TJ(BF16, bf16_t)
#undef PA_TJ
#undef PA_TJN
    return PA_ERR_UNSUPPORTED;
}

// Warps of a CTA.  16 rows of 64 columns leave registers for 16 warps, which cover each other's waits (16 sequences of 4K keys, 12 heads, float
// queries: 59 us, with 8 warps 67); where a warp would have a unit or two all the same, a warp alone is through sooner with more registers and the
// join finds room beside 8 warps (one sequence of 333 keys: 14.5 us, with 16 warps 16.8).
int tree_stream_warps(const TreeParams& p, int block) {
    const int64_t units = p.kv_heads * ((int64_t)p.rows * (p.heads / p.kv_heads) / block + p.num_seqs) * (((int64_t)p.num_tiles * p.tile_size + tstream::kUnit - 1) / tstream::kUnit);
    return p.dim == 64 && block == 16 && units >= 4 * 16 * (int64_t)device_info().sm_count ? 16 : 8;
}

// Rows of a block, 0 where these kernels do not serve.  Float queries have twice the fragments: 16 rows of them fill the registers.
int tree_stream_block(const TreeParams& p) {
    using tstream::kUnit;
    if ((p.dim != 64 && p.dim != 128) || p.tile_size % 16 || p.num_seqs > kTreeMostSeqs || p.kv_type == PA_TYPE_F32) return 0;
    if ((int64_t)p.total_pages * p.tile_size >= 0x7fffff00ll || ((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.k_scales | (uintptr_t)p.v_scales) % 16) return 0;
    if ((uintptr_t)p.q % 8 || (uintptr_t)p.out % 8 || p.q_stride % 2) return 0;
    const int G = p.heads / p.kv_heads, block = p.q_type == PA_TYPE_F32 || p.most * G <= 16 ? 16 : 32;
    const int64_t steps = ((int64_t)p.num_tiles * p.tile_size + kUnit - 1) / kUnit;
    return ((int64_t)p.rows * G / block + p.num_seqs) * (steps + kTreeStreamExtra) < 0x7fffffff ? block : 0;     // the list's sums are 32 bits
}

int tree_stream_launch(const TreeWork& a, cudaStream_t st) {
    using namespace tstream;
    const TreeParams& p = a.p;
    const int warps = a.workers / device_info().sm_count;
#define PA_TS(D, MT, QT, KT, W) if (p.dim == D && a.block == MT * 16 && p.q_type == QT && p.kv_type == KT && warps == W) return launch<D, MT, QT, KT, W>(a, st);
#define PA_TSD(MT, QT, KT) PA_TS(64, MT, QT, KT, 8) PA_TS(128, MT, QT, KT, 8)
    PA_TS(64, 1, F32, F16, 16) PA_TS(64, 1, F32, I8, 16)
    PA_TS(64, 1, F16, F16, 16) PA_TS(64, 1, F16, I8, 16) PA_TS(64, 1, BF16, BF16, 16)
    PA_TSD(1, F32, F16) PA_TSD(1, F32, I8)
    PA_TSD(1, F16, F16) PA_TSD(1, F16, I8) PA_TSD(1, BF16, BF16)
    PA_TSD(2, F16, F16) PA_TSD(2, F16, I8) PA_TSD(2, BF16, BF16)
#undef PA_TSD
#undef PA_TS
    return PA_ERR_UNSUPPORTED;
}

int tree_stream_errors(int* host_count) { return (int)cudaMemcpyFromSymbol(host_count, tstream::g_errors, sizeof(int)); }

}  // namespace pa
