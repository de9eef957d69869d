// draft_tree.cu -- the arrays of a batch of drafted trees, on the host: every step of a model that verifies drafts makes new ones.
#include <cstring>

#include "seq_common.cuh"

PA_API int pa_draft_trees(const int64_t* parents, const int32_t* node_start, int num_seqs, int mask_words, int32_t* row_seq, int32_t* row_parents,
                          int32_t* depths, int32_t* nodes, int32_t* mask, int32_t* longest) {
    PA_CHECK_ARG(num_seqs >= 0 && mask_words > 0 && node_start && longest);
    *longest = 0;
    for (int b = 0; b < num_seqs; ++b) {
        const int r0 = node_start[b], n = node_start[b + 1] - r0;
        PA_CHECK_ARG(r0 >= 0 && n >= 0 && n <= PA_TREE_MOST_NODES && n <= 32 * mask_words && (n == 0 || (parents && row_seq && row_parents && depths && nodes && mask)));
        for (int i = 0; i < n; ++i) {
            const int64_t up = parents[r0 + i], r = r0 + i;
            PA_CHECK_ARG(i == 0 ? up == -1 : up >= 0 && up < i);
            int32_t* words = mask + r * mask_words;
            if (i == 0) std::memset(words, 0, sizeof(int32_t) * mask_words);
            else std::memcpy(words, mask + (r0 + up) * mask_words, sizeof(int32_t) * mask_words);
            words[i >> 5] |= (int32_t)(1u << (i & 31));
            row_seq[r] = b;
            row_parents[r] = (int32_t)up;
            nodes[r] = i;
            depths[r] = i == 0 ? 0 : depths[r0 + up] + 1;
            if (depths[r] >= *longest) *longest = depths[r] + 1;
        }
    }
    return PA_OK;
}
