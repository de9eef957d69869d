// tree_pieces.cuh -- what the tcgen05 kernels of attention over drafted trees share (tree_tc.cu, tree_terms.cu): the walk over the pieces of a
// CTA's share, and a piece computed row by row.
#pragma once
#include "tree_attention.cuh"

namespace pa {

// Pieces of a CTA's share, in order.  Every role walks them for itself, from the first one, which is found before the roles part: that takes
// divisions, and the roles' instructions share the SM's caches.
struct TreeWalk {
    const TreeWork& a;
    const int* pre;
    int64_t f, f_hi;
    int b, rb;                          // sequence, block within the kv head
    TreeSeq sq;
    int g, rr0, i0, i1;                 // the piece: kv head, first row, steps [i0, i1)
    int u, pieces;                      // its first unit within the item; pieces before it
    int64_t slot;                       // of its partial sums, -1: it is a whole item
    int64_t total, ns;
    __device__ __forceinline__ TreeWalk(const TreeWork& w, const int* pre_) : a(w), pre(pre_), pieces(-1) {
        total = (int64_t)pre[w.p.num_seqs] * w.p.kv_heads;
        ns = shares::count(total, w.workers, w.least);
        f = blockIdx.x < ns ? total * blockIdx.x / ns : 0;
        f_hi = blockIdx.x < ns ? total * (blockIdx.x + 1) / ns : 0;
        if (f >= f_hi) return;
        b = shares::find_token(pre, w.p.num_seqs, f, w.p.kv_heads);
        sq = tree_seq(w.p, b, w.block, w.unit);
        const int64_t rem = f - (int64_t)pre[b] * w.p.kv_heads;
        const int each = sq.steps + w.extra, item = (int)(rem / each);
        u = (int)(rem - (int64_t)item * each);
        g = item / sq.blocks;
        rb = item - g * sq.blocks;
        if (w.whole) {                      // both ends back to where their items begin
            f -= u;
            u = 0;
            if (f_hi < total) {
                const int b1 = shares::find_token(pre, w.p.num_seqs, f_hi, w.p.kv_heads);
                f_hi -= (f_hi - (int64_t)pre[b1] * w.p.kv_heads) % (tree_seq(w.p, b1, w.block, w.unit).steps + w.extra);
            }
            if (f >= f_hi) return;
        }
        if (u + (f_hi - f) <= w.extra) f = f_hi;            // no step of the item is this share's
    }
    __device__ __forceinline__ bool next() {
        if (f >= f_hi) return false;
        if (++pieces > 0) {                 // the pieces behind the first begin their items
            u = 0;
            if (++rb == sq.blocks) {
                rb = 0;
                if (++g == a.p.kv_heads) {
                    g = 0;
                    do ++b; while (pre[b + 1] == pre[b]);       // a sequence without nodes has no items
                    sq = tree_seq(a.p, b, a.block, a.unit);
                }
            }
        }
        rr0 = rb * a.block;
        const int64_t left = f_hi - f;
        const int all = sq.steps + a.extra, end = left < all - u ? u + (int)left : all;
        i0 = max(u - a.extra, 0);
        i1 = end - a.extra;
        slot = i0 == 0 && i1 == sq.steps ? -1 : 2 * (int64_t)blockIdx.x + (pieces > 0 ? 1 : 0);
        f += end - u;
        if (f_hi - f <= a.extra) f = f_hi;                  // nothing but units before the steps of the next item
        return true;
    }
    // where the item that the share's last piece began stands in the list
    __device__ __forceinline__ int64_t item_at() const { return f_hi - a.extra - i1; }
};

// The pool rows of a piece's 16-key units, by a whole warp: 32 of them looked up at a time, the next 32 on their way (every lane divides and waits
// for one unit; one thread that did it for all was slower than the products).
struct TreePages {
    const TreeParams& p;
    const int32_t* trow;                // of the piece's sequence and kv head, null: out of range
    int keys, u0, cur, nxt;
    __device__ __forceinline__ explicit TreePages(const TreeParams& params) : p(params) {}
    __device__ __forceinline__ int look_up(int u) const {
        const int t0 = u * 16, t = t0 / p.tile_size;
        const int page = trow && t0 < keys && t < p.num_tiles ? __ldg(trow + t) : -1;
        return (unsigned)page < (unsigned)p.total_pages ? page * p.tile_size + (t0 - t * p.tile_size) : -1;
    }
    __device__ __forceinline__ void open(const TreeWalk& w, int units_per_step) {
        const int row = p.beam_ids ? __ldg(p.beam_ids + w.b) : w.b, lane = threadIdx.x & 31;
        trow = (unsigned)row < (unsigned)p.num_beams ? p.table + ((int64_t)row * p.kv_heads + w.g) * p.num_tiles : nullptr;
        keys = w.sq.keys;
        u0 = w.i0 * units_per_step;
        cur = look_up(u0 + lane);
        nxt = look_up(u0 + 32 + lane);
    }
    // lane k: the row of the k-th unit from `at`
    __device__ __forceinline__ int lane_row(int at) {
        if (at && (at & 31) == 0) {
            cur = nxt;
            nxt = look_up(u0 + at + 32 + (threadIdx.x & 31));
        }
        return __shfl_sync(0xffffffffu, cur, ((at & 31) + (threadIdx.x & 31)) & 31);
    }
    // rows of the N units from `at` (a multiple of N, counted from the piece's first; in rising order), -1: no page; returns which have one
    template <int N>
    __device__ __forceinline__ uint32_t rows(int at, int (&r)[N]) {
        if (at && (at & 31) == 0) {
            cur = nxt;
            nxt = look_up(u0 + at + 32 + (threadIdx.x & 31));
        }
        uint32_t mapped = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            r[k] = __shfl_sync(0xffffffffu, cur, (at & 31) + k);
            mapped |= (r[k] >= 0 ? 1u : 0u) << k;
        }
        return mapped;
    }
};

// Row by row, keys [k0, k1) that the row sees and no others (see above): by a warp, lanes over columns
template <int D, typename Q, typename KV>
__device__ __noinline__ void tree_piece_by_rows(const TreeWork& a, const TreeWalk& w, int row_in_block, int rows) {
    constexpr int NC = D / 32;
    const TreeParams& p = a.p;
    const int lane = threadIdx.x & 31, G = p.group;
    const int trow = p.beam_ids ? __ldg(p.beam_ids + w.b) : w.b;
    const float fe = 1.4426950408889634f / p.temperature;
    for (int x = 0; x < rows; ++x) {
        const int rr = w.rr0 + row_in_block + x;
        if (rr >= w.sq.n * G) break;
        const int node = rr / G, h = w.g * G + rr % G, r = w.sq.r0 + node;
        const Q* q = static_cast<const Q*>(p.q) + (int64_t)r * p.q_stride + (int64_t)h * D;
        const uint32_t* mask = p.mask + (int64_t)r * p.mask_words;
        float qf[NC], o[NC], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qf[c] = tree_widen<Q>(q[lane + 32 * c]);
            o[c] = 0.f;
        }
        for (int t = w.i0 * a.unit; t < min(w.i1 * a.unit, w.sq.keys); ++t) {
            const int j = t - w.sq.ctx;
            if (j >= 0 && (j >= p.mask_words * 32 || !((__ldg(mask + (j >> 5)) >> (j & 31)) & 1u))) continue;
            const int tile = t / p.tile_size;
            if ((unsigned)trow >= (unsigned)p.num_beams || tile >= p.num_tiles) continue;
            const int page = __ldg(p.table + ((int64_t)trow * p.kv_heads + w.g) * p.num_tiles + tile);
            if ((unsigned)page >= (unsigned)p.total_pages) continue;
            const int64_t at = ((int64_t)page * p.tile_size + (t - tile * p.tile_size)) * D + lane;
            float s = 0.f, v[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = fmaf(qf[c], tree_widen<KV>(static_cast<const KV*>(p.k)[at + 32 * c]), s);
                v[c] = tree_widen<KV>(static_cast<const KV*>(p.v)[at + 32 * c]);
            }
            s = warp_sum(s) * fe;
            const float mn = fmaxf(m, s);
            const float f = m == mn ? 1.f : fast_exp2(m - mn), e = s == mn ? 1.f : fast_exp2(s - mn);
            m = mn;
            l = l * f + e;
#pragma unroll
            for (int c = 0; c < NC; ++c) o[c] = fmaf(e, v[c], o[c] * f);
        }
        if (w.slot < 0) {
            Q* out = static_cast<Q*>(p.out) + ((int64_t)r * p.heads + h) * D;
#pragma unroll
            for (int c = 0; c < NC; ++c) out[lane + 32 * c] = tree_narrow<Q>(o[c] / (l + 1e-6f));
        } else {
            float* dst = a.part + (w.slot * a.block + row_in_block + x) * (D + 4);
#pragma unroll
            for (int c = 0; c < NC; ++c) dst[lane + 32 * c] = o[c] * a.p_scale;
            if (lane == 0) *reinterpret_cast<float4*>(dst + D) = make_float4(m, l * a.p_scale, m, 0.f);
        }
    }
}

}  // namespace pa
