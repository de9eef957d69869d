// tree_accept.cu -- the end of a step that verified trees of drafted tokens: which drafted tokens the model chose itself, and the move
// of their K/V rows to the places they have as accepted tokens.
//
// A sequence's nodes are numbered parents first; node i's rows stand at position ctx + i of the caches.  From node 0 the walk goes to the
// child whose token is the one chosen at the node (of several the lowest), as long as there is one:
//     path[0] = 0,  path[d + 1] = min { j : parent[j] = path[d], token[j] = ids[path[d]] }
// and row path[d] of every layer moves to position ctx + d.  path[d] >= d and the path rises, so place d may be the source of an
// earlier row of the path, never of a later one: rows in path order, a batch of them read before any of it is written, need no copy.
//
// One warp per (sequence, layer, kv head, keys or values); every CTA walks its sequence's tree for itself (32 candidates at a time from shared
// memory), so that one launch does it all.  What bounds it: latency, two dependent trips to memory (page, row) and the launch (24 sequences of 32
// nodes, 16 layers of 8 kv heads: 11.5 us; one sequence, 12 layers: 4.1 us).
#include "pa_common.cuh"

namespace pa {
namespace accept {

constexpr int kThreads = 128, kBatch = 4;

// of a launch: as many as its arguments hold (issuing 64 caches' addresses takes longer than 16's)
template <int MOST> struct Caches {
    void* p[MOST][4];                   // keys, values, their scales (or null)
    const int32_t* table[MOST];
};

struct Args {
    const int32_t *ids, *tokens, *parents, *node_start, *ctx_lens, *beam_ids;
    int num_seqs, most, depth, num_beams, kv_heads, num_tiles, total_pages, tile_size, bytes[2], num_caches;
    int32_t *counts, *out_tokens, *nodes, *new_lens;       // null: an earlier launch of the call wrote them
};

// rows [path[d]] -> [d] of one (layer, kv head, pool), U bytes at a time
template <typename U>
__device__ __forceinline__ void move_rows(uint8_t* pool, int row_bytes, const int32_t* trow, const Args& a, int ctx, const int* path, int n) {
    const int lane = threadIdx.x & 31, per = row_bytes / (int)sizeof(U);
    const int64_t cap = (int64_t)a.num_tiles * a.tile_size;
    auto row_of = [&](int64_t pos) -> int64_t {            // row of the pool, or -1
        if (pos >= cap) return -1;
        const int t = (int)(pos / a.tile_size), page = __ldg(trow + t);
        return (unsigned)page < (unsigned)a.total_pages ? (int64_t)page * a.tile_size + (pos - (int64_t)t * a.tile_size) : -1;
    };
    const int64_t total = (int64_t)n * per;
    for (int64_t i0 = 0; i0 < total; i0 += 32 * kBatch) {
        U v[kBatch];
        U* to[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int64_t i = i0 + k * 32 + lane;
            to[k] = nullptr;
            if (i >= total) continue;
            const int d = (int)(i / per), c = (int)(i % per);
            if (path[d] == d) continue;
            const int64_t src = row_of((int64_t)ctx + path[d]), dst = row_of((int64_t)ctx + d);
            if (src < 0 || dst < 0) continue;
            v[k] = reinterpret_cast<const U*>(pool + src * row_bytes)[c];
            to[k] = reinterpret_cast<U*>(pool + dst * row_bytes) + c;
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (to[k]) *to[k] = v[k];
        __syncwarp();
    }
}

template <int MOST>
__global__ void __launch_bounds__(kThreads) tree_accept_kernel(const Args a, const __grid_constant__ Caches<MOST> caches) {
    extern __shared__ int sm[];
    __shared__ int s_len;
    const int b = blockIdx.x, r0 = a.node_start[b], n = min(a.node_start[b + 1] - r0, a.most);
    int *ids = sm, *tokens = sm + a.most, *parents = sm + 2 * a.most, *path = sm + 3 * a.most;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        ids[i] = a.ids[r0 + i];
        tokens[i] = a.tokens[r0 + i];
        parents[i] = a.parents[r0 + i];
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        int len = 0, cur = n > 0 ? 0 : -1;
        while (cur >= 0) {                      // the path rises: at most n steps
            if (lane == 0) path[len] = cur;
            ++len;
            const int want = ids[cur];
            int next = -1;
            for (int j0 = cur + 1; j0 < n && next < 0; j0 += 32) {
                const int j = j0 + lane;
                const uint32_t hit = __ballot_sync(0xffffffffu, j < n && parents[j] == cur && tokens[j] == want);
                if (hit) next = j0 + __ffs(hit) - 1;
            }
            cur = next;
        }
        if (lane == 0) s_len = len;
    }
    __syncthreads();
    const int len = s_len, ctx = max(a.ctx_lens[b], 0);
    if (blockIdx.y == 0 && a.counts) {
        if (threadIdx.x == 0) {
            a.counts[b] = len;
            a.new_lens[b] = a.ctx_lens[b] + len;
        }
        for (int d = threadIdx.x; d < a.depth; d += kThreads) {
            a.out_tokens[(int64_t)b * a.depth + d] = d < len ? ids[path[d]] : -1;
            a.nodes[(int64_t)b * a.depth + d] = d < len ? path[d] : -1;
        }
    }
    const int row = a.beam_ids ? a.beam_ids[b] : b;
    if ((unsigned)row >= (unsigned)a.num_beams) return;
    int first = 0;
    while (first < len && path[first] == first) ++first;   // in place already
    if (first == len) return;
    const int items = a.num_caches * a.kv_heads * 2;
    for (int w = blockIdx.y * (kThreads / 32) + warp; w < items; w += gridDim.y * (kThreads / 32)) {
        const int kv = w & 1, g = (w >> 1) % a.kv_heads, c = (w >> 1) / a.kv_heads, bytes = a.bytes[kv];
        const int32_t* trow = caches.table[c] + ((int64_t)row * a.kv_heads + g) * a.num_tiles;
        uint8_t* pool = static_cast<uint8_t*>(caches.p[c][kv]);
        if (pool && bytes > 0) {
            if (((uintptr_t)pool | (uintptr_t)bytes) % 16 == 0) move_rows<uint4>(pool, bytes, trow, a, ctx, path, len);
            else if (((uintptr_t)pool | (uintptr_t)bytes) % 4 == 0) move_rows<uint32_t>(pool, bytes, trow, a, ctx, path, len);
            else move_rows<uint8_t>(pool, bytes, trow, a, ctx, path, len);
        }
        uint8_t* scales = static_cast<uint8_t*>(caches.p[c][2 + kv]);
        if (scales) move_rows<uint32_t>(scales, 4, trow, a, ctx, path, len);
    }
}

// caches c0 .. of the call; the first launch also writes what was accepted
template <int MOST>
static cudaError_t launch(Args a, void* const* caches, int c0, int num_caches, cudaStream_t st) {
    Caches<MOST> cs;
    a.num_caches = num_caches - c0 < MOST ? num_caches - c0 : MOST;
    if (c0 > 0) a.counts = nullptr;
    for (int c = 0; c < a.num_caches; ++c) {
        for (int k = 0; k < 4; ++k) cs.p[c][k] = caches[5 * (c0 + c) + k];
        cs.table[c] = static_cast<const int32_t*>(caches[5 * (c0 + c) + 4]);
    }
    const int items = a.num_caches * a.kv_heads * 2, per = kThreads / 32;
    const int y = items <= per ? 1 : (items + per - 1) / per;
    tree_accept_kernel<MOST><<<dim3((unsigned)a.num_seqs, (unsigned)(y < 65535 ? y : 65535)), kThreads, (size_t)4 * a.most * sizeof(int), st>>>(a, cs);
    return cudaGetLastError();
}

}  // namespace accept
}  // namespace pa

using namespace pa;

PA_API int pa_tree_accept(const int32_t* d_ids, const int32_t* d_tokens, const int32_t* d_parents, const int32_t* d_node_start, int num_seqs,
                          int most_nodes, int depth, const int32_t* d_ctx_lens, const int32_t* d_beam_ids, int num_beams, int kv_heads,
                          int num_tiles, int total_pages, int tile_size, int key_bytes, int value_bytes, int num_caches, void* const* caches,
                          int32_t* d_counts, int32_t* d_out_tokens, int32_t* d_nodes, int32_t* d_new_lens, pa_stream_t stream) {
    using namespace pa::accept;
    PA_CHECK_ARG(num_seqs >= 0 && most_nodes >= 0 && depth >= 0 && num_caches >= 0);
    if (num_seqs == 0) return PA_OK;
    PA_CHECK_ARG(d_ids && d_tokens && d_parents && d_node_start && d_ctx_lens && d_counts && d_out_tokens && d_nodes && d_new_lens);
    PA_CHECK_ARG(num_caches == 0 || (caches && num_beams > 0 && kv_heads > 0 && num_tiles > 0 && total_pages > 0 && tile_size > 0 &&
                                     key_bytes > 0 && value_bytes >= 0));
    if (most_nodes > PA_TREE_MOST_NODES) return PA_ERR_UNSUPPORTED;
    Args a{d_ids, d_tokens, d_parents, d_node_start, d_ctx_lens, d_beam_ids, num_seqs, most_nodes, depth, num_beams, kv_heads, num_tiles,
           total_pages, tile_size, {key_bytes, value_bytes}, 0, d_counts, d_out_tokens, d_nodes, d_new_lens};
    for (int c = 0; c < num_caches; ++c) PA_CHECK_ARG(caches[5 * c] && caches[5 * c + 4]);
    for (int c0 = 0; c0 == 0 || c0 < num_caches; c0 += 64) {
        const cudaError_t e = num_caches - c0 <= 16 ? launch<16>(a, caches, c0, num_caches, as_stream(stream)) : launch<64>(a, caches, c0, num_caches, as_stream(stream));
        if (e != cudaSuccess) return (int)e;
    }
    return PA_OK;
}
