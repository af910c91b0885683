// Stable grouping of integer indices (the order behind cvhrf_group_rows and
// cvhrf_table_gradient): a chunked LSD radix sort without waits between blocks.
#pragma once
#include "common.cuh"

namespace cvhrf {

constexpr long long kGroupMaxEntries = (1ll << 30) - 1;

// Words (u32) of scratch for group_sort.
size_t group_sort_words(long long n);

// Sorts n indices (4 or 8 bytes each) stably by value.  An index outside [0, rows) is left
// out; with keep_outside it counts as the value `rows` and so comes last.  On return
// *keys / *entries (inside scratch) hold the sorted values and the entries they came from;
// *count_dev (a device u32 inside scratch) is how many there are.  touched (rows bytes, may be
// null): 1 for the values that occur, 0 for the others.
int group_sort(const void* index, int index_bytes, long long n, long long rows, bool keep_outside, uint32_t* scratch,
               uint8_t* touched, cudaStream_t st, const uint32_t** keys, const uint32_t** entries,
               const uint32_t** count_dev);

}  // namespace cvhrf
