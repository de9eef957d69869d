// tree_attention.cu -- attention of drafted tokens that stand in trees: every row sees its sequence's cached context and, of the drafted
// rows behind it, its own ancestors and itself.
//
//     s[t] = q . K[t] / temperature,   p = exp(s - max s) / (sum exp(s - max s) + 1e-6),   out = sum p[t] V[t]
// over t < ctx and t = ctx + j with bit j of the row's mask set; keys on unmapped pages contribute nothing, a row that sees nothing
// is zero.
//
// The form for every page size, head size up to 256 and element type: one CTA per (row, head), its warps take the keys in turns, a lane holds dim /
// 32 columns; softmax with a running maximum and sum in float, joined over the warps at the end.  It reads a sequence's keys and values once per row
// and is bound by that and by the chain from key to key: 16 sequences of 4096 keys, 12 float heads of 64 columns, float pages, 8 nodes 1.8 ms, 224
// GB/s of the bytes there are.  The kernels of tree_stream.cu, tree_tc.cu and tree_terms.cu take half, bfloat16 and int8 pages of 16 rows (or
// multiples), head sizes 64 and 128 and up to 1024 sequences.
#include "tcgen05_utils.cuh"
#include "tree_attention.cuh"

namespace pa {
namespace tree {

constexpr int kWarps = 8, kMostCols = 8;

template <typename Q, typename KV>
__global__ void __launch_bounds__(kWarps * 32) tree_rows_kernel(const TreeParams p) {
    __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][kMostCols * 32];
    const int r = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = tree_seq_of(p.node_start, p.num_seqs, r);
    const int r0 = p.node_start[b], n = min(p.node_start[b + 1], p.rows) - r0, ctx = max(p.ctx_lens[b], 0);
    const int row = p.beam_ids ? p.beam_ids[b] : b, g = h / (p.heads / p.kv_heads);
    const int32_t* trow = p.table + ((int64_t)row * p.kv_heads + g) * p.num_tiles;
    const uint32_t* mask = p.mask + (int64_t)r * p.mask_words;
    const Q* q = static_cast<const Q*>(p.q) + (int64_t)r * p.q_stride + (int64_t)h * p.dim;
    float qf[kMostCols], o[kMostCols];
#pragma unroll
    for (int c = 0; c < kMostCols; ++c) {
        qf[c] = lane + 32 * c < p.dim ? tree_widen<Q>(q[lane + 32 * c]) : 0.f;
        o[c] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int64_t keys = (unsigned)row < (unsigned)p.num_beams ? min((int64_t)ctx + n, (int64_t)p.num_tiles * p.tile_size) : 0;
    for (int64_t t = warp; t < keys; t += kWarps) {
        if (t >= ctx) {
            const int j = (int)(t - ctx);
            if (j >= p.mask_words * 32 || !((__ldg(mask + (j >> 5)) >> (j & 31)) & 1u)) continue;
        }
        const int tile = (int)(t / p.tile_size), page = __ldg(trow + tile);
        if ((unsigned)page >= (unsigned)p.total_pages) continue;
        const int64_t at = (int64_t)page * p.tile_size + (t - (int64_t)tile * p.tile_size);
        const KV *k = static_cast<const KV*>(p.k) + at * p.dim, *v = static_cast<const KV*>(p.v) + at * p.dim;
        float s = 0.f, vf[kMostCols];
#pragma unroll
        for (int c = 0; c < kMostCols; ++c) {
            const bool in = lane + 32 * c < p.dim;
            s = fmaf(qf[c], in ? tree_widen<KV>(k[lane + 32 * c]) : 0.f, s);
            vf[c] = in ? tree_widen<KV>(v[lane + 32 * c]) : 0.f;
        }
        s = warp_sum(s);
        float vs = 1.f;
        if (p.k_scales) {
            s /= __ldg(p.k_scales + at);
            vs = 1.f / __ldg(p.v_scales + at);
        }
        s /= p.temperature;
        const float mn = fmaxf(m, s);
        const float f = m == mn ? 1.f : expf(m - mn), e = s == mn ? 1.f : expf(s - mn);
        m = mn;
        l = l * f + e;
#pragma unroll
        for (int c = 0; c < kMostCols; ++c) o[c] = fmaf(e * vs, vf[c], o[c] * f);
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int c = 0; c < kMostCols; ++c) s_o[warp][lane + 32 * c] = o[c];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
    float f[kWarps];
    for (int w = 0; w < kWarps; ++w) {
        f[w] = s_l[w] > 0.f ? expf(s_m[w] - M) : 0.f;
        L += s_l[w] * f[w];
    }
    Q* out = static_cast<Q*>(p.out) + ((int64_t)r * p.heads + h) * p.dim;
    for (int c = threadIdx.x; c < p.dim; c += kWarps * 32) {
        float x = 0.f;
        for (int w = 0; w < kWarps; ++w) x = fmaf(s_o[w][c], f[w], x);
        out[c] = tree_narrow<Q>(x / (L + 1e-6f));
    }
}

template <typename Q, typename KV>
static int launch_rows(const TreeParams& p, cudaStream_t st) {
    if (p.dim > kMostCols * 32 || p.heads > 65535) return PA_ERR_UNSUPPORTED;
    tree_rows_kernel<Q, KV><<<dim3((unsigned)p.rows, (unsigned)p.heads), kWarps * 32, 0, st>>>(p);
    PA_RETURN_LAUNCH_STATUS();
}

}  // namespace tree
}  // namespace pa

using namespace pa;

PA_API size_t pa_tree_attention_workspace_bytes(int rows, int num_seqs, int most_nodes, int heads, int kv_heads, int head_dim) {
    if (rows <= 0 || num_seqs <= 0 || num_seqs > kTreeMostSeqs || heads <= 0 || kv_heads <= 0 || heads % kv_heads || (head_dim != 64 && head_dim != 128))
        return 0;
    // whichever kernel serves: it goes by the types too
    size_t most = 0;
    for (int block : {16, 32, 64, 128, 256}) {
        const size_t n = tree_work_bytes(num_seqs, block <= 32 ? (head_dim == 64 && block == 16 ? 16 : 8) * device_info().sm_count : block == 64 ? tree_terms_workers(block) : tree_tc_workers(block), block, head_dim);
        if (n > most) most = n;
    }
    return most;
}

PA_API int pa_tree_attention_polls(const void* d_q, int64_t q_stride, int q_type, void* d_out, const void* d_k_pool, const void* d_v_pool,
                             const float* d_k_scales, const float* d_v_scales, int kv_type, const int32_t* d_table, int num_beams, int kv_heads,
                             int num_tiles, int total_pages, const int32_t* d_beam_ids, const int32_t* d_ctx_lens, const int32_t* d_node_start,
                             const int32_t* d_mask, int mask_words, int rows, int num_seqs, int most_nodes, int heads, int head_dim,
                             int tile_size, float temperature, void* d_workspace, size_t workspace_bytes, int polls, pa_stream_t stream) {
    using namespace pa::tree;
    PA_CHECK_ARG(polls >= 0);
    PA_CHECK_ARG(rows >= 0 && num_seqs >= 0 && most_nodes >= 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && head_dim > 0);
    PA_CHECK_ARG(num_beams > 0 && num_tiles > 0 && total_pages > 0 && tile_size > 0 && temperature != 0.f && (num_seqs > 0 || rows == 0));
    if (rows == 0) return PA_OK;
    PA_CHECK_ARG(d_q && d_out && d_k_pool && d_v_pool && d_table && d_ctx_lens && d_node_start && d_mask);
    PA_CHECK_ARG(q_stride >= (int64_t)heads * head_dim && mask_words > 0 && (int64_t)mask_words * 32 >= most_nodes);
    PA_CHECK_ARG((kv_type == PA_TYPE_I8) == (d_k_scales != nullptr) && (kv_type == PA_TYPE_I8) == (d_v_scales != nullptr));
    const bool pair = q_type == PA_TYPE_F32    ? kv_type == PA_TYPE_F16 || kv_type == PA_TYPE_I8 || kv_type == PA_TYPE_F32
                      : q_type == PA_TYPE_F16 ? kv_type == PA_TYPE_F16 || kv_type == PA_TYPE_I8
                                              : q_type == PA_TYPE_BF16 && kv_type == PA_TYPE_BF16;
    if (most_nodes > PA_TREE_MOST_NODES || !pair) return PA_ERR_UNSUPPORTED;
    const TreeParams p{d_q, q_stride, d_out, d_k_pool, d_v_pool, d_k_scales, d_v_scales, d_table, d_beam_ids, d_ctx_lens, d_node_start,
                       reinterpret_cast<const uint32_t*>(d_mask), q_type, kv_type, num_beams, kv_heads, num_tiles, total_pages, mask_words,
                       rows, num_seqs, most_nodes, heads, head_dim, tile_size, temperature, heads / kv_heads};
    cudaStream_t st = as_stream(stream);
    struct Form {
        int block, workers, unit, extra;
        int (*launch)(const TreeWork&, cudaStream_t);
    };
    Form f{tree_tc_block(p), 0, 64, kTreeTcExtra, tree_tc_launch};
    f.workers = tree_tc_workers(f.block);
    if (!f.block) {
        f = Form{tree_terms_block(p), 0, 128, kTreeTermsExtra, tree_terms_launch};
        f.workers = tree_terms_workers(f.block);
    }
    if (!f.block) {
        f = Form{tree_stream_block(p), 0, 16, kTreeStreamExtra, tree_stream_launch};
        if (f.block) f.workers = tree_stream_warps(p, f.block) * device_info().sm_count;
    }
    if (f.block) {
        if (!d_workspace || (uintptr_t)d_workspace % 16 || workspace_bytes < tree_work_bytes(num_seqs, f.workers, f.block, head_dim)) return PA_ERR_WORKSPACE;
        const bool whole = (int64_t)num_tiles * tile_size <= (f.unit == 16 ? kTreeWholeStream : kTreeWhole) && tree_items(p, f.block) <= f.workers;
        const TreeWork w{p, f.workers, kTreeLeast, f.block, f.unit, total_pages * tile_size, f.extra, whole, kTreeStreamScale, (uint32_t)polls, static_cast<TreeNote*>(d_workspace),
                         reinterpret_cast<float*>(static_cast<TreeNote*>(d_workspace) + f.workers)};
        int rc = f.launch(w, st);
        if (rc == PA_OK && !whole) rc = tree_join_launch(w, st);
        if (rc != PA_ERR_UNSUPPORTED) return rc;
    }
#define PA_TREE(QT, QC, KT, KC) if (q_type == QT && kv_type == KT) return launch_rows<QC, KC>(p, st);
    PA_TREE(PA_TYPE_F32, float, PA_TYPE_F16, __half)
    PA_TREE(PA_TYPE_F32, float, PA_TYPE_I8, int8_t)
    PA_TREE(PA_TYPE_F32, float, PA_TYPE_F32, float)
    PA_TREE(PA_TYPE_F16, __half, PA_TYPE_F16, __half)
    PA_TREE(PA_TYPE_F16, __half, PA_TYPE_I8, int8_t)
    PA_TREE(PA_TYPE_BF16, bf16_t, PA_TYPE_BF16, bf16_t)
#undef PA_TREE
    return PA_ERR_UNSUPPORTED;
}

PA_API int pa_tree_attention(const void* d_q, int64_t q_stride, int q_type, void* d_out, const void* d_k_pool, const void* d_v_pool,
                             const float* d_k_scales, const float* d_v_scales, int kv_type, const int32_t* d_table, int num_beams, int kv_heads,
                             int num_tiles, int total_pages, const int32_t* d_beam_ids, const int32_t* d_ctx_lens, const int32_t* d_node_start,
                             const int32_t* d_mask, int mask_words, int rows, int num_seqs, int most_nodes, int heads, int head_dim,
                             int tile_size, float temperature, void* d_workspace, size_t workspace_bytes, pa_stream_t stream) {
    return pa_tree_attention_polls(d_q, q_stride, q_type, d_out, d_k_pool, d_v_pool, d_k_scales, d_v_scales, kv_type, d_table, num_beams, kv_heads,
                                   num_tiles, total_pages, d_beam_ids, d_ctx_lens, d_node_start, d_mask, mask_words, rows, num_seqs, most_nodes, heads,
                                   head_dim, tile_size, temperature, d_workspace, workspace_bytes, tc::kPolls, stream);
}
