// paged_index.hpp — where a sequence's position lies in a cache of pages (plain
// integer arithmetic, for the kernels and for a host test).
#pragma once

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define AXF_HD __host__ __device__ __forceinline__
#else
#define AXF_HD inline
#endif

namespace axf {

// Row of the pool's layer that holds position pos of the sequence with this
// table row, or -1: past the table, or an entry that is no page.  64-bit: a
// layer of a 288 GB cache has more rows than 32 bits of value offsets reach.
AXF_HD long kv_row(int pos, const int* table, int table_ld, int n_pages, int page_shift) {
    const int col = pos >> page_shift;
    if (pos < 0 || col >= table_ld) return -1;
    const int page = table[col];
    if (page < 0 || page >= n_pages) return -1;
    return ((long)page << page_shift) + (pos & ((1 << page_shift) - 1));
}

// Rows a sequence is taken to hold: len cut to what its table can name.
AXF_HD int kv_len(int len, int table_ld, int page_shift) {
    const long cap = (long)table_ld << page_shift;
    return len < 0 ? 0 : (len < cap ? len : (int)cap);
}

}  // namespace axf
