// tree_attention.cuh -- what the kernels of attention over drafted trees share (tree_attention.cu, tree_stream.cu,
// tree_tc.cu, tree_terms.cu).
//
// The rows of a sequence that share a kv head are its nodes' query heads: row rr = node * G + head of the group, G = heads / kv_heads.
// An item is a block of `block` such rows of one (sequence, kv head) with the keys that its sequence has, in steps of `unit` keys.  The
// list of all items' steps, sequence by sequence, kv head by kv head, block by block, `extra` units before each item's, is cut into equal
// contiguous shares (decode_shares.cuh: their number follows from the lengths and the workers of the call).  A cut before an item's steps
// is one at its beginning.  A share that holds all of an item writes its rows' results; otherwise
// it leaves reference, sum and weighted sums of its piece in a slot, and a second kernel joins the pieces: the share in which such an
// item begins notes it (TreeNote); the item's first piece is in slot 2 w + 1 of that share w unless the share begins with it, every other one
// is the beginning of its share, in slot 2 w.
#pragma once
#include "decode_shares.cuh"
#include "dynamic_smem.cuh"
#include "seq_common.cuh"

namespace pa {

// Row r = (node i of sequence b) of q and out; its keys are positions 0 .. ctx(b) - 1, and ctx(b) + j where bit j of its mask is set.
struct TreeParams {
    const void* q;                  // [rows, heads, dim], rows q_stride elements apart
    int64_t q_stride;
    void* out;                      // [rows, heads, dim]
    const void *k, *v;              // [total_pages * tile_size, dim]
    const float *k_scales, *v_scales;
    const int32_t *table, *beam_ids, *ctx_lens, *node_start;
    const uint32_t* mask;           // [rows, mask_words]
    int q_type, kv_type, num_beams, kv_heads, num_tiles, total_pages, mask_words, rows, num_seqs, most, heads, dim, tile_size;
    float temperature;
    int group;                      // heads / kv_heads
};

template <typename T> __device__ __forceinline__ float tree_widen(T v) { return (float)v; }
template <> __device__ __forceinline__ float tree_widen<bf16_t>(bf16_t v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float tree_widen<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T tree_narrow(float v) { return (T)v; }
template <> __device__ __forceinline__ bf16_t tree_narrow<bf16_t>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half tree_narrow<__half>(float v) { return __float2half_rn(v); }

// the sequence of a row: the last b with node_start[b] <= r
__device__ __forceinline__ int tree_seq_of(const int32_t* node_start, int num_seqs, int r) {
    int lo = 0, hi = num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(node_start + mid) <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---- the shares
constexpr int kTreeMostSeqs = 1024;     // sequences that the streaming kernels take: their step counts stand in shared memory
constexpr int kTreeLeast = 2;           // units of a share, where there are that many
// Beginning and ending an item takes as long as this many steps (of 64 and 128 keys; 16 in the streaming kernel); where shares are cut by steps
// alone, the ones with many short items end last.  48 sequences of 1 to 2048 keys, 32 heads: 32 bf16 rows 331 -> 188 us (5 units: 192, 3: 210), int8 pages
// 182 -> 131 us (3: 137, 8: 131), 32 float rows 312 -> 200 us (8: 196),
// 8 bf16 rows 188 -> 161 us (8: 164, 16: 168).
constexpr int kTreeTcExtra = 8, kTreeTermsExtra = 6, kTreeStreamExtra = 4;

// Items are left whole, and nothing is joined, where the page table has room for no more than this many keys and every worker has an item at most: a
// warp that streams 16 keys at a time passes 6 such units in the time of the join, the tcgen05 kernels 512 keys.  us, whole against cut: 2 sequences of 57 keys, 16 rows,
// 9.9 against 12.8; 4 of 181 in the streaming kernel 23.9 against 15.7; 45 of up to 309 on tcgen05 18 against 25, 9 of 116 18 against 24; 4 of 554 20 against 16.
constexpr int kTreeWholeStream = 96, kTreeWhole = 512;

struct TreeSeq {
    int r0, n, ctx, keys, blocks, steps;
    __device__ __forceinline__ int units(int extra) const { return steps > 0 ? blocks * (steps + extra) : 0; }     // of one kv head
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int b, int block, int unit) {
    TreeSeq s;
    s.r0 = max(__ldg(p.node_start + b), 0);
    s.n = max(min(__ldg(p.node_start + b + 1), p.rows) - s.r0, 0);
    s.ctx = max(__ldg(p.ctx_lens + b), 0);
    const int64_t cap = min((int64_t)p.num_tiles * p.tile_size, (int64_t)0x7fffff00);
    s.keys = s.n > 0 ? (int)min((int64_t)s.ctx + s.n, cap) : 0;
    s.blocks = (s.n * p.group + block - 1) >> (31 - __clz(block));      // powers of two, both
    s.steps = (s.keys + unit - 1) >> (31 - __clz(unit));
    return s;
}
// Bits 0 .. width - 1: which of the keys at ctx + off .. a row sees (off < 0: the first -off are context).  word: of the row's mask
template <typename W>
__device__ __forceinline__ uint32_t tree_visible(int off, int words, W word) {
    if (off <= -32) return 0xffffffffu;
    if (off < 0) return ((1u << -off) - 1u) | (word(0) << -off);
    const int i = off >> 5;
    const uint32_t lo = i < words ? word(i) : 0u, hi = i + 1 < words ? word(i + 1) : 0u;
    return __funnelshift_r(lo, hi, off & 31);
}

// The item that begins in a share and does not end there
struct __align__(16) TreeNote {
    int rows;                           // of the item's block; 0: there is none
    int first_row, g, rr0;              // the sequence's first row, kv head, the block's first row within the group
    int last;                           // the share in which it ends
    int slot;                           // of its first piece
    int pad[2];
};

struct TreeWork {
    TreeParams p;
    int workers, least, block, unit, total_rows;
    int extra;                          // units before an item's steps in the list: what beginning and ending an item costs
    bool whole;                         // shares end with items: no item is cut, and nothing is joined
    float p_scale;                      // the partial sums are times this (softmax weights enter products so that small halves keep their bits)
    uint32_t polls;                     // of a wait
    TreeNote* notes;                    // [workers]
    float* part;                        // [2 * workers][block][dim + 4]: weighted sums, reference (log2), sum, largest score, -
};

static inline size_t tree_work_bytes(int num_seqs, int workers, int block, int dim) {
    (void)num_seqs;
    return (size_t)workers * sizeof(TreeNote) + (size_t)2 * workers * block * (dim + 4) * sizeof(float);
}
// by one thread of a worker: what it notes of the last piece of its share, steps [i0, i1) of an item that begins at unit f_item of the list
__device__ __forceinline__ TreeNote tree_note(const TreeWork& a, const TreeSeq& s, int g, int rr0, int i0, int i1, int64_t f_item, int64_t total, int64_t ns, int64_t slot) {
    TreeNote t{};
    if (i0 == 0 && i1 < s.steps) {
        t.rows = min(a.block, s.n * a.p.group - rr0);
        t.first_row = s.r0;
        t.g = g;
        t.rr0 = rr0;
        t.last = (int)(((f_item + a.extra + s.steps) * ns - 1) / total);
        t.slot = (int)slot;
    }
    return t;
}

// items of a call, at most
static inline int64_t tree_items(const TreeParams& p, int block) {
    return p.kv_heads * (((int64_t)p.rows * p.group + (int64_t)p.num_seqs * (block - 1)) / block);
}

// tree_stream.cu: few query rows; the join of pieces
constexpr float kTreeStreamScale = 128.f;
int tree_stream_warps(const TreeParams& p, int block);          // workers of an SM
int tree_stream_block(const TreeParams& p);                     // rows of a block, 0: not served
int tree_stream_launch(const TreeWork& w, cudaStream_t st);
int tree_join_launch(const TreeWork& w, cudaStream_t st);
// tree_tc.cu: many query rows of 16-bit types
int tree_tc_workers(int block);
int tree_tc_block(const TreeParams& p);
int tree_tc_launch(const TreeWork& w, cudaStream_t st);
// tree_terms.cu: float queries over half pages, int8 pages
int tree_terms_workers(int block);
int tree_terms_block(const TreeParams& p);
int tree_terms_launch(const TreeWork& w, cudaStream_t st);

}  // namespace pa
