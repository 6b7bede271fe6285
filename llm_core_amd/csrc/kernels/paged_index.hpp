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

// The table's entry for a position, for kv_row_of.  The nearest column's outside the
// table (table_ld >= 1), so that no branch keeps a caller's lookups apart.
AXF_HD int kv_page(int pos, const int* table, int table_ld, int page_shift) {
    const int col = pos >> page_shift;  // -1 or less before the sequence
    return table[col < 0 ? 0 : (col < table_ld ? col : table_ld - 1)];
}

// Row of the pool's layer that holds position pos with the entry kv_page gave, or -1:
// past the table, or an entry that is no page.  64-bit: a layer of a 288 GB cache has
// more rows than 32 bits of value offsets reach.
AXF_HD long kv_row_of(int pos, int page, int table_ld, int n_pages, int page_shift) {
    const int col = pos >> page_shift;
    const bool there = (unsigned)col < (unsigned)table_ld && (unsigned)page < (unsigned)n_pages;
    const long row = ((long)page << page_shift) + (pos & ((1 << page_shift) - 1));
    return there ? row : -1;
}

AXF_HD long kv_row(int pos, const int* table, int table_ld, int n_pages, int page_shift) {
    return kv_row_of(pos, kv_page(pos, table, table_ld, page_shift), table_ld, n_pages, page_shift);
}

// Rows a sequence is taken to hold: len cut to what its table can name.
AXF_HD int kv_len(int len, int table_ld, int page_shift) {
    const long cap = (long)table_ld << page_shift;
    return len < 0 ? 0 : (len < cap ? len : (int)cap);
}

}  // namespace axf
