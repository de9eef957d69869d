// device_pages.cu -- pages of a table handed out and taken back on the GPU, and the places of new rows.
//
// Sequence b (table row b) holds pages for its first held[b] tiles, of every head.  Room for n rows behind its first `length` tokens:
//     held' = max(held, ceil((length + n) / tile));   row i of them: position length + i, slot of head h: page(b, h, position / tile) tile + position % tile
// New pages come from the end of the free list, sequence by sequence, tile by tile, head by head: the order that the host hands them out in.  What is
// beyond ceil(length / tile) goes back in reverse, so that it undoes what took it.
//
// Integers and few bytes: the floor is a launch and two dependent trips to memory.  Every CTA sums the sequences' tiles by itself (a scan in shared
// memory), because waiting for another CTA's sums would take as long; then the CTAs share the table's entries and the rows.  Nobody writes what
// others still read: counts and held tiles change by the CTA that is the last to have read them (an ordered count, 2 us where there are several).
// Replayed, a take and the release that undoes it: one sequence and 8 rows 8 us; 128 of up to 8192 tokens and 2614 rows 14; 32 prompts, 164435 rows of 32
// heads 25 (4.4 is the floor of all bytes, 3.2 of it the slots): there the slots' addresses, a thread for a head of neighbouring rows (35 with a thread a slot).
#include <climits>

#include "dynamic_smem.cuh"
#include "pa_common.cuh"

namespace pa {
namespace pages {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMostSeqs = 16384, kRows = 64, kMostRows = 1 << 30;

struct Args {
    int32_t* table;             // [beams][heads][tiles]
    int32_t *free, *held, *state;       // state: pages in the free list, calls that found too few, CTAs that have read
    const int32_t *lengths, *start;     // start null: pages go back
    int seqs, rows, heads, tiles, tile, total;
    int32_t *row_seq, *positions, *slots;
};
enum { FREE, REFUSED, READ };

// Tiles that sequence b holds afterwards; -1: more than the table has
__device__ __forceinline__ int wanted(const Args& a, int b, int held) {
    const int64_t n = a.start ? a.start[b + 1] - a.start[b] : 0, end = (int64_t)max(a.lengths[b], 0) + max(n, (int64_t)0), t = (end + a.tile - 1) / a.tile;
    if (!a.start) return (int)min(t, (int64_t)held);
    return t > a.tiles ? -1 : max((int)t, held);
}

template <bool TAKE> __global__ void __launch_bounds__(kThreads) pages_kernel(const __grid_constant__ Args a) {
    extern __shared__ int32_t smem[];
    int32_t* first = smem;                              // [seqs + 1] tiles that change of the sequences before
    int32_t* from = smem + a.seqs + 1;                  // [seqs] the lowest of them
    __shared__ int64_t s_sum[kWarps], s_run;
    __shared__ int s_bad, s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        s_run = 0;
        s_bad = 0;
    }
    __syncthreads();
    for (int b0 = 0; b0 < a.seqs; b0 += kThreads) {
        const int b = b0 + tid;
        int64_t n = 0;
        if (b < a.seqs) {
            const int held = a.held[b], to = wanted(a, b, held);
            if (to < 0) s_bad = 1;
            else n = TAKE ? to - held : held - to;
            from[b] = TAKE ? held : to;
        }
        int64_t sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t p = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += p;
        }
        if (lane == 31) s_sum[warp] = sum;
        __syncthreads();
        int64_t before = s_run;
        for (int w = 0; w < warp; ++w) before += s_sum[w];
        if (b < a.seqs) first[b] = (int32_t)min(before + sum - n, (int64_t)INT_MAX);
        __syncthreads();
        if (tid == 0)
            for (int w = 0; w < kWarps; ++w) s_run += s_sum[w];
        __syncthreads();
    }
    const int count = a.state[FREE];
    const int64_t all = s_run * a.heads;
    const bool fits = !s_bad && (TAKE ? all <= count : count + all <= a.total);
    const int entries = fits ? (int)all : 0;
    if (tid == 0) first[a.seqs] = fits ? (int)s_run : 0;
    __syncthreads();
    // (all of this CTA's threads have what they read; who comes last changes it, when its own share is done)
    if (tid == 0) {
        int arrived = 0;
        if (gridDim.x > 1) asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(arrived) : "l"(a.state + READ) : "memory");
        s_last = arrived == (int)gridDim.x - 1;
    }
    auto sequence = [&](const int32_t* starts, int at) {        // the last sequence that begins at or before `at`
        int lo = 0, hi = a.seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (starts[mid] <= at) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    // ---- the table: neighbouring threads on neighbouring tiles of a head
    if (entries) {
        const int64_t step = (int64_t)gridDim.x * kThreads;
#pragma unroll 2
        for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < entries; i += step) {
            const int b = sequence(first, (int)(i / a.heads)), base = first[b], n = first[b + 1] - base;
            const int own = (int)(i - (int64_t)base * a.heads), h = own / n, t = own - h * n;
            int32_t* entry = a.table + ((int64_t)b * a.heads + h) * a.tiles + from[b] + t;
            const int64_t nth = (int64_t)(base + t) * a.heads + h;
            if (TAKE) *entry = a.free[count - 1 - nth];
            else {
                a.free[count + entries - 1 - nth] = *entry;
                *entry = -1;
            }
        }
    }
    // ---- the rows, some at a time: their sequences, where their pages stand and their places in these; then their slots, a thread for a head of
    // some neighbouring rows, which looks up a page once for the rows of a tile
    if (TAKE) {
        __shared__ int64_t r_page[kRows];           // in the table, or counted down from -1 in the free list
        __shared__ int r_at[kRows];                 // (-1: no page)
        const int groups = max(1, kThreads / a.heads), each = (kRows + groups - 1) / groups, g = tid / a.heads, h0 = tid - g * a.heads;
        for (int r0 = blockIdx.x * kRows; r0 < a.rows; r0 += gridDim.x * kRows) {
            const int n = min(kRows, a.rows - r0);
            __syncthreads();
            if (tid < n) {
                const int r = r0 + tid, b = sequence(a.start, r), s0 = a.start[b];
                const bool in = r >= s0 && r < a.start[b + 1];
                const int pos = in ? max(a.lengths[b], 0) + r - s0 : -1, t = pos / a.tile, own = t - from[b];
                a.row_seq[r] = in ? b : -1;
                a.positions[r] = pos;
                r_at[tid] = pos >= 0 && t < a.tiles ? pos - t * a.tile : -1;
                r_page[tid] = fits && own >= 0 && own < first[b + 1] - first[b] ? -(int64_t)(count - 1 - (first[b] + own) * a.heads) - 1 : (int64_t)b * a.heads * a.tiles + t;
            }
            __syncthreads();
            if (g >= groups) continue;
            for (int h = h0; h < a.heads; h += kThreads) {
                int64_t last = LLONG_MIN;
                int page = -1;
                int32_t* out = a.slots + ((int64_t)r0 + g * each) * a.heads + h;
                for (int r = g * each; r < min(n, (g + 1) * each); ++r, out += a.heads) {
                    const int at = r_at[r];
                    if (at >= 0 && r_page[r] != last) {
                        last = r_page[r];
                        page = last < 0 ? a.free[-(last + 1) - h] : a.table[last + (int64_t)h * a.tiles];
                        if ((unsigned)page >= (unsigned)a.total) page = -1;
                    }
                    *out = at >= 0 && page >= 0 ? page * a.tile + at : -1;
                }
            }
        }
    }
    __syncthreads();
    if (s_last) {
        if (fits)
            for (int b = tid; b < a.seqs; b += kThreads) a.held[b] = TAKE ? wanted(a, b, from[b]) : from[b];
        if (tid == 0) {
            a.state[READ] = 0;
            if (fits) a.state[FREE] = count + (TAKE ? -entries : entries);
            else a.state[REFUSED] += 1;
        }
    }
}

template <bool TAKE> static int launch(const Args& a, int64_t ctas, int64_t most, cudaStream_t st) {
    const size_t smem = (size_t)(2 * a.seqs + 1) * 4;
    const cudaError_t e = allow_dynamic_smem<pages_kernel<TAKE>>(smem);
    if (e != cudaSuccess) return (int)e;
    pages_kernel<TAKE><<<(unsigned)(ctas < 1 ? 1 : ctas > most ? most : ctas), kThreads, smem, st>>>(a);
    PA_RETURN_LAUNCH_STATUS();
}

static bool usable(const Args& a) {
    return a.seqs >= 0 && a.heads > 0 && a.tiles > 0 && a.tile > 0 && a.total >= 0 && (int64_t)a.total * a.tile <= INT_MAX &&
           (a.seqs == 0 || (a.table && a.free && a.held && a.state && a.lengths));
}

}  // namespace pages
}  // namespace pa

using namespace pa;

PA_API int pa_take_pages(int32_t* d_table, int num_beams, int num_heads, int num_tiles, int tile_size, int total_pages, int32_t* d_free, int32_t* d_held,
                         int32_t* d_state, const int32_t* d_lengths, const int32_t* d_start, int num_seqs, int rows, int32_t* d_row_seq,
                         int32_t* d_positions, int32_t* d_slots, pa_stream_t stream) {
    using namespace pa::pages;
    const Args a{d_table, d_free, d_held, d_state, d_lengths, d_start, num_seqs, rows, num_heads, num_tiles, tile_size, total_pages, d_row_seq, d_positions, d_slots};
    PA_CHECK_ARG(usable(a) && rows >= 0 && rows <= kMostRows && num_seqs <= num_beams && (num_seqs == 0 || d_start) && (rows == 0 || (num_seqs > 0 && d_row_seq && d_positions && d_slots)));
    if (num_seqs == 0) return PA_OK;
    if (num_seqs > kMostSeqs) return PA_ERR_UNSUPPORTED;
    return launch<true>(a, ((int64_t)rows * num_heads + 4 * kThreads - 1) / (4 * kThreads), 4 * (int64_t)device_info().sm_count, as_stream(stream));
}

PA_API int pa_release_pages(int32_t* d_table, int num_beams, int num_heads, int num_tiles, int tile_size, int total_pages, int32_t* d_free, int32_t* d_held,
                            int32_t* d_state, const int32_t* d_lengths, int num_seqs, pa_stream_t stream) {
    using namespace pa::pages;
    const Args a{d_table, d_free, d_held, d_state, d_lengths, nullptr, num_seqs, 0, num_heads, num_tiles, tile_size, total_pages, nullptr, nullptr, nullptr};
    PA_CHECK_ARG(usable(a) && num_seqs <= num_beams);
    if (num_seqs == 0) return PA_OK;
    if (num_seqs > kMostSeqs) return PA_ERR_UNSUPPORTED;
    // (how much goes back the host does not know: as many CTAs as a whole table keeps busy)
    return launch<false>(a, (int64_t)num_seqs * num_heads * num_tiles / (8 * kThreads), 3 * (int64_t)device_info().sm_count, as_stream(stream));
}
