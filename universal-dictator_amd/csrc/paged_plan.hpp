// Page lists and launch plans of the windowed attention kernels, in plain C++ (window.hip, prefill.hip
// and a CPU test include it).
//
// A query row with range [lo, hi) sees the keys [0, min(sinks, lo)) (the sinks) and [lo, hi) (its window);
// an empty range (lo >= hi) sees nothing.  The rows that one workgroup serves see pages of two stretches:
// those of the sinks and those of the union of their windows.  The kernels walk the two as one list, so a
// long context costs what its window costs, and table entries in between (pages given back) are not read.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define UD_HD __host__ __device__ __forceinline__
#else
#define UD_HD inline
#endif

namespace ud {

constexpr int KPAGE = 16;                          // keys per page

struct PageList {
    int sink;                                      // pages of the sinks that are not window pages
    int first;                                     // first page of the windows
    int count;                                     // pages in all
};

// lo, hi: lowest start and highest end of the rows' non-empty ranges, 0 <= lo < hi <= 16 max_blocks (lo >= hi: no
// row sees a key).
UD_HD PageList page_list(int lo, int hi, int sinks) {
    PageList p{0, 0, 0};
    if (lo >= hi) return p;
    p.first = lo / KPAGE;
    const int s = sinks < lo ? sinks : lo;
    const int pages = s / KPAGE + (s % KPAGE != 0);    // no sum that could pass INT_MAX
    p.sink = pages < p.first ? pages : p.first;
    p.count = p.sink + (hi - 1) / KPAGE - p.first + 1;
    return p;
}

// The logical page (entry of the block table) at position u of the list.
UD_HD int page_at(const PageList& p, int u) { return u < p.sink ? u : u - p.sink + p.first; }

// Most pages of a list whose rows' windows span at most `span` keys.
UD_HD int64_t max_pages(int64_t span, int64_t sinks) {
    return (span + KPAGE - 2) / KPAGE + 1 + (sinks + KPAGE - 1) / KPAGE;
}

// Splits of the page lists over workgroups: split s takes pages [s pages, (s + 1) pages) of its list, the
// last one all that follow (a span larger than the caller said costs balance, not keys).
struct SplitPlan {
    int splits;
    int pages;
};

constexpr int MAX_SPLITS = 256;

// want: splits wanted; step: pages that a workgroup takes at a time, which a split is a multiple of.
inline SplitPlan split_plan(int64_t want, int64_t pages, int64_t step) {
    if (want > MAX_SPLITS) want = MAX_SPLITS;
    if (want < 1) want = 1;
    const int64_t each = ((pages + want - 1) / want + step - 1) / step * step;
    return SplitPlan{(int)((pages + each - 1) / each), (int)each};
}

}  // namespace ud
