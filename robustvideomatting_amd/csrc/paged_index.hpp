// Where a position of a stream lives in a paged cache.  Plain C++ on both sides, so that the bounds can be checked on the host.
#pragma once
#include <stdint.h>
#ifndef RVM_HD
#ifdef __HIPCC__
#define RVM_HD __host__ __device__ __forceinline__
#else
#define RVM_HD inline
#endif
#endif
// Position of the i-th new token (i >= 0) of a stream of `length` tokens; past the last int, that int
RVM_HD int paged_position(int length, int i) {
    const int64_t pos = (int64_t)length + i;
    return pos > INT32_MAX ? INT32_MAX : (int)pos;
}
// Keys that a pass over a stream up to `pos` looks at: those up to it, or up to the first one past the table (which is lost)
RVM_HD unsigned paged_keys(int width, int page_shift, int pos) {
    const unsigned keys = (unsigned)pos + 1, held = (unsigned)width << page_shift;
    return keys <= held ? keys : held + 1;
}
// Page of position `pos` (>= 0) of stream s, or -1 where the table has none: a column past its end, a page number outside
// the pool.  The table is read in bounds whatever the caller's lengths hold.
RVM_HD int page_of(const int* table, int width, int pages, int page_shift, int s, int pos) {
    const int col = pos >> page_shift;
    if (pos < 0 || col >= width) return -1;
    const int pg = table[(int64_t)s * width + col];
    return (unsigned)pg < (unsigned)pages ? pg : -1;
}
