// Waits of the attention block's kernels by their number in the status word, and what one that ran out leaves behind.
#pragma once

#define IT_SITE_EVICT_MOVE 71                    // k_evict_move: rows that another block still has to read

static inline const char* it_ops_after_timeout(int site) {
    return site == IT_SITE_EVICT_MOVE ? "its caches are moved in part, its weights and kept slots are those of the finished move" : "its outputs are NaN";
}
