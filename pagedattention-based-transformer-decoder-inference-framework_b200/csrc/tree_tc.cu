// tree_tc.cu -- attention of drafted trees with many query rows on the 5th-generation tensor cores (tcgen05.mma kind::f16, operands of one
// 16-bit type, float accumulators in TMEM); tree_attention.cuh has the work list, tree_stream.cu the join.
//
// One CTA = NQ tiles of 128 query rows (node, head of the group) of one kv head, which share every staged key and value.  Persistent over
// its share of the list: barriers and ring run on from piece to piece.  Keys come in tiles of 64:
//   warps 0-3 (4-7)  softmax of query tile 0 (1), one thread per row = TMEM lane: its 64 scores, the mask of its node where the tile has
//                    drafted keys, running reference and sum in float, P back to TMEM over the scores it came from
//   next NQ warps    one elected thread each:  S = Q K^T of tile i + 1  and  O += P V  of tile i (A operand from TMEM)
//   last warp        TMA boxes of 16 keys x 64 columns into a ring, SWIZZLE_128B, page ids a tile ahead
// The reference of a row is raised only when a score exceeds it by more than 2^8; weights are 2^(s - reference + 7), so that halves
// hold them down to 2^-31 of the largest.  They enter the second product in the values' type, since its factors have one type (bfloat16: 2.3e-3 from
// float64, where rounding the result alone takes 1.7e-3); their sum is taken of the float ones.
//
// What bounds it: the hand-over between tensor pipe and exponentials, one thread per row as in prefill attention (131072 keys, 64 nodes, 16 heads on
// 4: 89 us, 3.0 TB/s, 770 TFLOP/s; the tensor pipe is busy 42 % of the time), with fewer rows the copies (12 sequences of 4K keys, 32 heads, 64 rows a head: 156 us, 5.2
// TB/s), and where contexts are short what a piece takes to begin and end, some 7 us (60 keys: 72 us for 1536 pieces on 296 CTAs).  So the next
// piece's queries come as boxes under the last products of this one, and results leave through shared memory: 93 us before.  A CTA per 128 rows, two
// an SM, covers one's softmax with the other's products; 256 rows in one CTA share what is staged, which pays where a kv head has more than 128 of
// them.
//
// Drafted rows whose values are not finite may be hidden from some rows, and zero times them is no zero: the softmax threads look
// through the values of tiles with drafted keys, and a piece that has such values is computed again row by row, from the keys that
// each row sees alone.
#include "softmax_tile.cuh"
#include "tcgen05_utils.cuh"
#include "tree_pieces.cuh"

namespace pa {
namespace ttc {

using namespace tc;

constexpr int QT = 128, KT = 64;
constexpr float kShift = 7.f;           // weights times 2^7

__device__ int g_errors;

__host__ __device__ constexpr int q_bytes(int D) { return D * QT * 2; }
// the ring: tiles of keys and of values, each of 64 rows
__host__ __device__ constexpr int tile_bytes(int D) { return D * KT * 2; }
__host__ __device__ constexpr int ring_for(int D, int nq) { return nq == 2 ? (D == 128 ? 8 : 18) : D == 128 ? 4 : 10; }
constexpr int kNotes = 32;              // of the producer on its tiles; more than it can be ahead
__host__ __device__ constexpr int threads_for(int nq) { return (5 * nq + 1) * 32; }
// full, empty [ring]; per query tile s_full, p_full, o_full [2], q_ready
__host__ __device__ constexpr int nbar_for(int D, int nq) { return 2 * ring_for(D, nq) + 7 * nq; }
constexpr int kStage = 2048;            // of a warp: 32 columns of its rows' results
constexpr size_t smem_for(int D, int nq, int seqs) {
    return (size_t)nq * q_bytes(D) + ring_for(D, nq) * tile_bytes(D) + nq * 4 * kStage + nbar_for(D, nq) * 8 + 64 + kNotes * 4 + (seqs + 1) * 4 + 1024;
}

template <bool BF> struct Elem { typedef __half T; };
template <> struct Elem<true> { typedef bf16_t T; };

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
                 "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}

// q_boxes: tmQ has boxes of a query tile, else the softmax warps gather its rows
template <int D, int NQ, bool BF>
__global__ void __launch_bounds__(threads_for(NQ), NQ == 1 ? 2 : 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmQ,
               const bool q_boxes, const TreeWork a) {
    typedef typename Elem<BF>::T T;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    constexpr int RING = ring_for(D, NQ), NBAR = nbar_for(D, NQ), TMEM_COLS = NQ * 256, KB = D / 64;
    constexpr int Q_BYTES = q_bytes(D), TILE = tile_bytes(D);
    constexpr int W_MMA = 4 * NQ, W_PROD = 5 * NQ;
    const TreeParams& p = a.p;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t kv_sm = base + NQ * Q_BYTES, stage_sm = kv_sm + RING * TILE, bar0 = stage_sm + NQ * 4 * kStage;
    auto kv_full = [&](int s) { return bar0 + s * 8; };
    auto kv_empty = [&](int s) { return bar0 + (RING + s) * 8; };
    auto s_full = [&](int x, int i) { return bar0 + (2 * RING + 7 * x + i) * 8; };
    auto p_full = [&](int x, int i) { return bar0 + (2 * RING + 7 * x + 2 + i) * 8; };
    auto o_full = [&](int x, int i) { return bar0 + (2 * RING + 7 * x + 4 + i) * 8; };
    auto q_ready = [&](int x) { return bar0 + (2 * RING + 7 * x + 6) * 8; };
    const uint32_t tmem_slot = bar0 + NBAR * 8, fail_sm = tmem_slot + 8, odd_sm = fail_sm + 4, meta_sm = odd_sm + 8;
    int* pre = reinterpret_cast<int*>(smem_raw + (meta_sm + kNotes * 4 - smem_u32(smem_raw)));
    auto failed = [&] { return tc_failed(fail_sm); };
    auto wait = [&](uint32_t bar, uint32_t parity) { tc_wait(bar, parity, fail_sm, a.polls); };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.group;
    if (threadIdx.x == 0) {
        for (int s = 0; s < RING; ++s) {
            mbar_init(kv_full(s), 1);
            mbar_init(kv_empty(s), NQ);
        }
        for (int x = 0; x < NQ; ++x) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(s_full(x, i), 1);
                mbar_init(p_full(x, i), QT);
                mbar_init(o_full(x, i), 1);
            }
            mbar_init(q_ready(x), 1);
        }
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(fail_sm), "r"(0u) : "memory");
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(odd_sm), "r"(0u) : "memory");
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(odd_sm + 4), "r"(0u) : "memory");
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmV));
    }
    if (warp == W_MMA) tmem_alloc(tmem_slot, TMEM_COLS);
    shares::count_units(pre, p.num_seqs, [&](int b) { return tree_seq(p, b, a.block, a.unit).units(a.extra); });
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
    TreeWalk w(a, pre);
    // Tiles go through the ring in the order of their products: K(0), K(1), V(0), K(2), V(1), ..., K(n - 1), V(n - 2), V(n - 1); the ring's
    // count `at` runs on through the pieces
    auto k_at = [&](uint32_t at, int i) { return at + (uint32_t)(i == 0 ? 0 : 2 * i - 1); };
    auto v_at = [&](uint32_t at, int i, int nt) { return at + (uint32_t)(i + 1 < nt ? 2 * i + 2 : 2 * nt - 1); };
    auto slot_of = [&](uint32_t c) { return (int)(c % RING); };
    auto phase_of = [&](uint32_t c) { return c / RING & 1u; };
    // which query tiles of a piece have rows
    auto rows_of = [&](const TreeWalk& piece, int x) { return piece.rr0 + x * QT < piece.sq.n * G; };
    auto has_rows = [&](int x) { return rows_of(w, x); };

    if (warp == W_PROD) {
        uint32_t c = 0, tiles = 0;          // requests and tiles of keys so far
        bool ok = a.polls > 0;              // 0: nothing is requested, so that all waits run out
        if (w.f >= w.f_hi && lane == 0) a.notes[blockIdx.x] = TreeNote{};
        auto request = [&](const CUtensorMap* map, const int (&r)[4]) {
            const int s = (int)(c % RING);
            wait(kv_empty(s), (c / RING & 1u) ^ 1u);
            if (__any_sync(0xffffffffu, failed())) {
                ok = false;
                return;
            }
            if (elect_one()) {
                const uint32_t st = kv_sm + s * TILE;
                mbar_arrive_expect_tx(kv_full(s), TILE);
#pragma unroll
                for (int uu = 0; uu < 4; ++uu)
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)     // no page: zeros, and its scores are masked
                        tma_load_2d(st + kb * 8192 + uu * 2048, map, kb * 64, r[uu] >= 0 ? r[uu] : a.total_rows, kv_full(s));
            }
            __syncwarp();
            ++c;
        };
        TreePages pages(p);
        while (w.next()) {                  // to the end, also where a wait ran out: the join goes by the last piece's note
            if (w.f >= w.f_hi && lane == 0) a.notes[blockIdx.x] = tree_note(a, w.sq, w.g, w.rr0, w.i0, w.i1, w.item_at(), w.total, w.ns, w.slot);
            if (!ok) continue;
            pages.open(w, 4);
            int r[4] = {-1, -1, -1, -1}, prev[4] = {-1, -1, -1, -1};
            for (int i = w.i0; i <= w.i1 && ok; ++i) {              // K(i) and V(i - 1)
                if (i < w.i1) {
                    const uint32_t mapped = pages.rows<4>((i - w.i0) * 4, r);
                    if (lane == 0) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(meta_sm + tiles % kNotes * 4), "r"(mapped) : "memory");
                    __syncwarp();
                    ++tiles;
                    request(&tmK, r);
                }
                if (i > w.i0 && ok) request(&tmV, prev);
#pragma unroll
                for (int uu = 0; uu < 4; ++uu) prev[uu] = r[uu];
            }
        }
        if (failed())           // let the copies in flight land before the CTA's shared memory goes away
            for (uint32_t i = c > RING ? c - RING : 0; i < c; ++i) tc_let_land(kv_full((int)(i % RING)), i / RING & 1u);
    } else if (warp >= W_MMA) {
        constexpr uint32_t kIdescS = idesc_f16(QT, KT, 0, 0, BF), kIdescO = idesc_f16(QT, D, 0, 1, BF);
        const int x = warp - W_MMA;
        int n = 0, qn = 0, asked = 0;       // key tiles and pieces of this query tile so far; its boxes asked for
        uint32_t at = 0;
        // the queries of the piece after this one, as soon as the products with this one's are done; rows behind the sequence's are others' or
        // zeros, and nobody looks at what becomes of them
        TreeWalk ahead = w;
        auto fetch_q = [&] {
            if (!q_boxes || !a.polls || !ahead.next() || !rows_of(ahead, x) || __any_sync(0xffffffffu, failed())) return;
            ++asked;
            if (elect_one()) {
                mbar_arrive_expect_tx(q_ready(x), Q_BYTES);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                    tma_load_3d(base + x * Q_BYTES + kb * (QT * 128), &tmQ, kb * 64, ahead.g * G, ahead.sq.r0 + (ahead.rr0 + x * QT) / G, q_ready(x));
            }
            __syncwarp();
        };
        fetch_q();
        while (w.next()) {
            const bool mine = has_rows(x);
            if (!mine) fetch_q();
            auto issue_S = [&](int i) {     // every issuer waits for every tile: its arrival at the empty barrier belongs to THIS use of it
                const int s = slot_of(k_at(at, i));
                wait(kv_full(s), phase_of(k_at(at, i)));
                tc_fence_after();
                if (mine && elect_one()) {
                    const uint32_t st = kv_sm + s * TILE, qx = base + x * Q_BYTES;
                    const int sb = (n + i) & 1;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint64_t da = make_desc(qx + (ks >> 2) * (QT * 128) + (ks & 3) * 32, 16, 1024);
                        const uint64_t db = make_desc(st + (ks >> 2) * (KT * 128) + (ks & 3) * 32, 16, 1024);
                        umma_f16(tmem_base + x * 2 * KT + sb * KT, da, db, kIdescS, ks > 0 ? 1u : 0u);
                    }
                    umma_commit(s_full(x, sb));
                }
                __syncwarp();
                if (elect_one()) umma_commit(kv_empty(s));
                __syncwarp();
            };
            const int nt = w.i1 - w.i0;
            if (mine) wait(q_ready(x), (uint32_t)qn & 1u);
            issue_S(0);
            for (int i = 0; i < nt; ++i) {
                if (i + 1 < nt) issue_S(i + 1);
                const int s = slot_of(v_at(at, i, nt));
                wait(kv_full(s), phase_of(v_at(at, i, nt)));
                if (mine) {
                    const uint32_t st = kv_sm + s * TILE;
                    const int sb = (n + i) & 1, nvalid = min(KT, w.sq.keys - (w.i0 + i) * KT);
                    if (nvalid & 15) {
                        // value rows past the last key may hold anything (0 x NaN = NaN): zeros (both issuers write the same)
                        const int r1 = (nvalid + 15) & ~15;
                        for (int idx = lane; idx < (r1 - nvalid) * (D / 8); idx += 32) {
                            const int r = nvalid + idx / (D / 8), c = idx % (D / 8);
                            const uint32_t addr = st + (c >> 3) * 8192 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(addr), "r"(0u) : "memory");
                        }
                        fence_proxy_async();
                        __syncwarp();
                    }
                    // every row's thread has also read the last piece's O by the time it hands over a piece's first P
                    wait(p_full(x, sb), (uint32_t)((n + i) >> 1) & 1u);
                    tc_fence_after();
                    if (elect_one()) {
                        const int ksteps = (nvalid + 15) >> 4;
                        for (int ks = 0; ks < ksteps; ++ks) {
                            const uint32_t ta = tmem_base + x * 2 * KT + sb * KT + ks * 8;
                            const uint64_t db = make_desc(st + ks * 2048, 8192, 1024);
                            umma_f16_ts(tmem_base + NQ * 2 * KT + x * D, ta, db, kIdescO, (i > 0 || ks > 0) ? 1u : 0u);
                        }
                        umma_commit(o_full(x, sb));
                    }
                    __syncwarp();
                }
                if (elect_one()) umma_commit(kv_empty(s));
                __syncwarp();
                if (mine && i + 1 == nt) fetch_q();         // (its scores were read: the products with the queries are done)
            }
            at += 2 * nt;
            if (mine) {
                n += nt;
                ++qn;
            }
        }
        if (failed() && asked > 0) tc_let_land(q_ready(x), (uint32_t)(asked - 1) & 1u);
    } else {
        // ---- softmax: one thread per query row
        const int x = warp >> 2, qtr = warp & 3, row_in_block = x * QT + qtr * 32;
        const uint32_t lane_base = (uint32_t)(qtr * 32) << 16;
        const uint32_t s_addr = tmem_base + lane_base + x * 2 * KT;
        const uint32_t o_addr = tmem_base + lane_base + NQ * 2 * KT + x * D;
        const float f0 = 1.4426950408889634f / p.temperature, fe = fmaxf(fabsf(f0), 1e-30f);
        const bool flip = f0 < 0.f;
        auto group_sync = [&] {
            if (x == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
            else asm volatile("bar.sync 2, 128;" ::: "memory");
        };
        // P.V(t) is complete.  Unambiguous without consuming every phase: S(n) follows P.V(n - 2) on the pipe, so by the time a
        // thread works on tile n the barrier of P.V(n - 1) is in the phase asked for or just past it.
        auto pv_done = [&](int t) { wait(o_full(x, t & 1), (uint32_t)((t >> 1) & 1)); };
        int n = 0;
        uint32_t tiles = 0;                 // of keys, of all pieces
        uint32_t at = 0;
        while (w.next()) {
            const int nt = w.i1 - w.i0, all = w.sq.n * G;
            if (!has_rows(x)) {
                at += 2 * nt;
                tiles += nt;
                continue;
            }
            const int rr = w.rr0 + row_in_block + lane, rows = min(32, all - w.rr0 - row_in_block);       // rows of this warp, may be negative
            const int div = rr / G, node = rr < all ? div : -1, head = w.g * G + rr - div * G;
            if (!q_boxes && rows > 0) {
                // the warp's query rows into the swizzled K-major A tile, whose last products this thread has seen complete
                const uint32_t qx = base + x * Q_BYTES;
                constexpr int CH = D / 8, PER = 8;      // 16-byte pieces of a row; loads in flight per lane
                const int64_t own = node >= 0 ? (int64_t)(w.sq.r0 + node) * p.q_stride + (int64_t)head * D : 0;      // one division a row
#pragma unroll 1
                for (int c0 = 0; c0 < 32 * CH; c0 += 32 * PER) {
                    uint4 v[PER];
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        const int idx = c0 + j * 32 + lane, r = idx / CH, c = idx % CH;
                        const int64_t from = __shfl_sync(0xffffffffu, own, r);
                        v[j] = make_uint4(0u, 0u, 0u, 0u);
                        if (r < rows) v[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + from) + c);
                    }
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        const int idx = c0 + j * 32 + lane, r = idx / CH, c = idx % CH, at = qtr * 32 + r;
                        const uint32_t addr = qx + (c >> 3) * (QT * 128) + at * 128 + (((c & 7) ^ (at & 7)) << 4);
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v[j].x), "r"(v[j].y), "r"(v[j].z), "r"(v[j].w) : "memory");
                    }
                }
            }
            if (!q_boxes) {
                fence_proxy_async();
                group_sync();
                if (qtr == 0 && lane == 0) mbar_arrive_cnt(q_ready(x));
            }
            const uint32_t* mask = p.mask + (int64_t)(w.sq.r0 + max(node, 0)) * p.mask_words;
            float m_ref = -INFINITY, l_run = 0.f;
            bool odd = false;
#pragma unroll 1
            for (int i = 0; i < nt; ++i) {
                const int sb = (n + i) & 1, kp0 = (w.i0 + i) * KT;
                const bool drafts = kp0 + KT > w.sq.ctx;
                wait(s_full(x, sb), (uint32_t)((n + i) >> 1) & 1u);
                tc_fence_after();
                if (drafts) {       // values that are not finite (the keys past the last one were looked at or are zeros)
                    const uint32_t c = v_at(at, i, nt);
                    wait(kv_full(slot_of(c)), phase_of(c));
                    const uint32_t vt = kv_sm + slot_of(c) * TILE;
                    const int mine = threadIdx.x & 127, r = mine >> 1;
                    if (kp0 + r < w.sq.keys) {
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            const uint4 v = lds_128(vt + ((mine & 1) * (D / 16) + c) / 8 * 8192 + r * 128 + ((((mine & 1) * (D / 16) + c) & 7) << 4));
                            constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
                            const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) odd |= (q[e] & E) == E || (q[e] >> 16 & E) == E;
                        }
                    }
                }
                if (rows <= 0) {    // nothing of this warp's: it only keeps the barriers' count
                    mbar_arrive_cnt(p_full(x, sb));
                    continue;
                }
                uint32_t mapped;    // the producer's note about this tile, older than the scores
                asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(mapped) : "r"(meta_sm + (tiles + i) % kNotes * 4) : "memory");
                uint32_t sr[2][32];
                tmem_ld32(s_addr + sb * KT, sr[0]);
                tmem_ld32(s_addr + sb * KT + 32, sr[1]);
                tmem_wait_ld();
                if (flip) {
#pragma unroll
                    for (int k = 0; k < KT; ++k) sr[k >> 5][k & 31] ^= 0x80000000u;
                }
                const bool full = !drafts && mapped == 15u;
                if (!full) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int k0 = kp0 + 32 * hf, valid = w.sq.keys - k0;
                        uint32_t vis = 0xffffffffu;
                        if (drafts) {
                            vis = tree_visible(k0 - w.sq.ctx, p.mask_words, [&](int j) { return __ldg(mask + j); });
                            if (valid < 32) vis &= valid > 0 ? (1u << valid) - 1u : 0u;
                        }
                        if (!(mapped >> 2 * hf & 1u)) vis &= 0xffff0000u;
                        if (!(mapped >> 2 * hf & 2u)) vis &= 0x0000ffffu;
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(vis >> k & 1u)) sr[hf][k] = 0xff800000u;
                    }
                }
                // A row's reference rarely moves, so a tile that all rows of the warp see whole takes the exponentials with the one at
                // hand, without waiting for the maximum, and the scores' first half is on its way to TMEM under the second's exponentials
                auto pack = [](float lo, float hi) {
                    if constexpr (BF) return pack_bf16x2(lo, hi);
                    else return pack_half2(lo, hi);
                };
                uint32_t w0[16], w1[16];
                uint64_t acc[2] = {0ull, 0ull};
                if (__all_sync(0xffffffffu, full && m_ref > -INFINITY)) {
                    smx::exp_half(sr[0], fe, m_ref - kShift, w0, acc, pack);
                    tmem_st16(s_addr + sb * KT, w0);
                    const float mx = smx::row_max(sr) * fe;
                    smx::exp_half(sr[1], fe, m_ref - kShift, w1, acc, pack);
                    if (!__any_sync(0xffffffffu, mx > m_ref + 8.f)) {
                        tmem_st16(s_addr + sb * KT + 16, w1);
                        l_run += smx::sum_of(acc);
                        tmem_wait_st();
                        tc_fence_before();
                        mbar_arrive_cnt(p_full(x, sb));
                        continue;
                    }
                    acc[0] = acc[1] = 0ull;
                    tmem_wait_st();
                }
                const float mx = smx::row_max(sr) * fe;
                const bool raise = mx > m_ref + 8.f || (m_ref == -INFINITY && mx > -INFINITY);
                const float m_new = raise ? mx : m_ref;
                const float corr = raise && m_ref != -INFINITY ? fast_exp2(m_ref - m_new) : 1.f;
                m_ref = m_new;
                smx::exp_half(sr[0], fe, m_ref - kShift, w0, acc, pack);
                smx::exp_half(sr[1], fe, m_ref - kShift, w1, acc, pack);
                const bool dead = m_ref == -INFINITY;       // nothing visible yet: the exponents above are NaN
                if (__any_sync(0xffffffffu, corr != 1.f)) {
                    if (i > 0) pv_done(n + i - 1);
                    tc_fence_after();
#pragma unroll
                    for (int c4 = 0; c4 < D / 32; ++c4) {
                        uint32_t orr[32];
                        tmem_ld32(o_addr + c4 * 32, orr);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) orr[j] = __float_as_uint(__uint_as_float(orr[j]) * corr);
                        tmem_st32(o_addr + c4 * 32, orr);
                    }
                    l_run *= corr;
                }
                if (dead) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) w0[k] = w1[k] = 0u;
                } else {
                    l_run += smx::sum_of(acc);
                }
                tmem_st16(s_addr + sb * KT, w0);
                tmem_st16(s_addr + sb * KT + 16, w1);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive_cnt(p_full(x, sb));
            }
            n += nt;
            at += 2 * nt;
            tiles += nt;
            pv_done(n - 1);
            tc_fence_after();
            if (w.i1 * KT > w.sq.ctx) {         // the piece had drafted keys
                if (odd) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(odd_sm + 4 * x), "r"(1u) : "memory");
                group_sync();
                uint32_t any;
                asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(any) : "r"(odd_sm + 4 * x) : "memory");
                group_sync();
                odd = any != 0;
                if (odd && qtr == 0 && lane == 0) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(odd_sm + 4 * x), "r"(0u) : "memory");
            }
            if (odd && !failed()) {
                tree_piece_by_rows<D, T, T>(a, w, row_in_block, 32);
                continue;
            }
            if (rows <= 0) continue;
            // a share's own piece: every thread its row; a whole item: 32 columns of the warp's rows at a time through shared memory, so that
            // four lanes write 64 bytes of a row (each lane its own row: 32 half sectors a store, half of a short piece's time)
            float inv = 1.f / (l_run + 1e-6f * 128.f);
            if (m_ref == -INFINITY) inv = 0.f;              // saw nothing
            if (failed()) inv = m_ref = l_run = __int_as_float(0x7fc00000);
            const int64_t own_row = node >= 0 ? ((int64_t)(w.sq.r0 + node) * p.heads + head) * D : -1;
            int64_t out_row[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) out_row[j] = __shfl_sync(0xffffffffu, own_row, 8 * j + (lane >> 2));
            const uint32_t stage = stage_sm + warp * kStage;
            float* part = a.part + (w.slot * a.block + row_in_block + lane) * (D + 4);
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + c0, o);
                tmem_wait_ld();
                if (w.slot < 0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float lo = m_ref == -INFINITY ? 0.f : __uint_as_float(o[j * 8 + 2 * e]) * inv;
                            const float hi = m_ref == -INFINITY ? 0.f : __uint_as_float(o[j * 8 + 2 * e + 1]) * inv;
                            if constexpr (BF) v[e] = pack_bf16x2(lo, hi);
                            else v[e] = pack_half2(lo, hi);
                        }
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)), "r"(v[0]), "r"(v[1]),
                                     "r"(v[2]), "r"(v[3]) : "memory");
                    }
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = 8 * j + (lane >> 2);
                        const uint4 v = lds_128(stage + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) << 4));
                        if (out_row[j] >= 0) reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_row[j] + c0)[lane & 3] = v;
                    }
                } else if (node >= 0) {
                    const float k = a.p_scale / 128.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = m_ref == -INFINITY ? 0.f : __uint_as_float(o[4 * j + e]) * k;
                        reinterpret_cast<float4*>(part + c0)[j] = make_float4(v[0], v[1], v[2], v[3]);
                    }
                }
                __syncwarp();
            }
            if (node >= 0 && w.slot >= 0) *reinterpret_cast<float4*>(part + D) = make_float4(m_ref, l_run * (a.p_scale / 128.f), m_ref, 0.f);
        }
        tc_fence_before();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        if (failed()) {
            __nanosleep(1000000);       // products in flight write TMEM for microseconds at most
            if (lane == 0) atomicAdd(&g_errors, 1);
        }
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// [rows][heads][dim], box = (128 / G) rows x G heads x 64 columns
static bool make_q_map(CUtensorMap* map, const TreeParams& p, int G) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)p.dim, (cuuint64_t)p.heads, (cuuint64_t)p.rows}, strides[2] = {(cuuint64_t)p.dim * 2, (cuuint64_t)p.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(QT / G)}, estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NQ, bool BF>
static int launch(const TreeWork& a, cudaStream_t st) {
    const TreeParams& p = a.p;
    const size_t smem = smem_for(D, NQ, p.num_seqs);
    if (smem > (size_t)device_info().max_smem_optin) return PA_ERR_UNSUPPORTED;
    auto kern = tree_tc_kernel<D, NQ, BF>;
    const cudaError_t e = allow_dynamic_smem<tree_tc_kernel<D, NQ, BF>>(smem);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap k, v, q{};              // boxes move bits: one map type for both 16-bit types
    if (!make_bf16_map(&k, p.k, a.total_rows, D, D, 16) || !make_bf16_map(&v, p.v, a.total_rows, D, D, 16)) return PA_ERR_UNSUPPORTED;
    // queries: boxes of 128 rows = 128 / G nodes' heads of a group
    const int G = p.heads / p.kv_heads;
    const bool q_boxes = QT % G == 0 && make_q_map(&q, p, G);
    kern<<<a.workers, threads_for(NQ), smem, st>>>(k, v, q, q_boxes, a);
    PA_RETURN_LAUNCH_STATUS();
}

}  // namespace ttc

int tree_tc_workers(int block) { return device_info().sm_count * (block == 128 ? 2 : 1); }

// Rows of a block, 0 where this kernel does not serve or the streaming one is faster.  us, this kernel against the streaming one: 64 rows a head (32
// sequences, 4K keys, 8 kv heads) 113 against 235, 32 rows 106 against 132, 16 rows 104 against 106, 8 rows and 32 kv heads of 2K keys 191 against 189, ragged
// contexts 168 against 161: from 17 on.  Blocks of 128 rows against 256: 128 rows a head 126 against 142, 64 rows 113 against 135; 160 rows (2K
// keys) 121 against 99, 256 rows 130 against 112; 384 rows 102 against 104, 448 rows 80 against 83, 800 rows 45 against 47.
int tree_tc_block(const TreeParams& p) {
    const int G = p.heads / p.kv_heads, rows = p.most * G;
    if (!((p.q_type == PA_TYPE_F16 && p.kv_type == PA_TYPE_F16) || (p.q_type == PA_TYPE_BF16 && p.kv_type == PA_TYPE_BF16)) || rows <= 16) return 0;
    if ((p.dim != 64 && p.dim != 128) || p.tile_size % 16 || p.num_seqs > kTreeMostSeqs) return 0;
    if ((int64_t)p.total_pages * p.tile_size >= 0x7fffff00ll || ((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.q | (uintptr_t)p.out) % 16 || p.q_stride % 8) return 0;
    const int block = rows <= 128 || rows > 256 ? 128 : 256;
    const int64_t steps = ((int64_t)p.num_tiles * p.tile_size + ttc::KT - 1) / ttc::KT;
    return ((int64_t)p.rows * G / block + p.num_seqs) * (steps + kTreeTcExtra) < 0x7fffffff ? block : 0;     // the list's sums are 32 bits
}

int tree_tc_launch(const TreeWork& a, cudaStream_t st) {
    using namespace ttc;
    const bool bf = a.p.q_type == PA_TYPE_BF16;
    if (a.p.dim == 64) {
        if (a.block == 128) return bf ? launch<64, 1, true>(a, st) : launch<64, 1, false>(a, st);
        return bf ? launch<64, 2, true>(a, st) : launch<64, 2, false>(a, st);
    }
    if (a.block == 128) return bf ? launch<128, 1, true>(a, st) : launch<128, 1, false>(a, st);
    return bf ? launch<128, 2, true>(a, st) : launch<128, 2, false>(a, st);
}

int tree_tc_errors(int* host_count) { return (int)cudaMemcpyFromSymbol(host_count, ttc::g_errors, sizeof(int)); }

}  // namespace pa
