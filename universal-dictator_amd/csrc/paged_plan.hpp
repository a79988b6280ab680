// Page lists and launch plans of the windowed attention kernels, in plain C++ (window.hip, prefill.hip
// and a CPU test include it).
//
// A query row with range [lo, hi) sees the keys [0, min(sinks, lo)) (the sinks) and [lo, hi) (its window);
// an empty range (lo >= hi) sees nothing.  The rows that one workgroup serves see pages of two stretches:
// those of the sinks and those of the union of their windows.  The kernels walk the two as one list, so a
// long context costs what its window costs, and table entries in between (pages given back) are not read.
#pragma once
#include <stdint.h>

#include <algorithm>

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

// Windowed attention (window.hip).
//
// Waves of a workgroup, and workgroups: one round of eight waves per CU (512 workgroups of 4 waves, 256 of 8), not quite full
// rather than just beyond, but at least three quarters of it.  A workgroup's first rows arrive some 3 us after its start (its
// ranges, its table entries, its pages) and its waves are joined at its end, so few, long ones pay while the chip is full.
// us at 512 / 1,024 / 2,048 of 4 waves wanted, 32/8 heads of 128: 1 x 60,000 keys bf16 50.6 / 52.4 / 57.4, MXFP4 21.9 / 24.9 /
// 30.0; 64 x 4,096 bf16 184 / 191 / 194, MXFP4 57.6 / 64.6 / 66.2; 64 x 1,000 bf16 51.0 / 56.8 / 59.5.
// Beyond or below a round, 4,000 keys: 12 sequences (96 units) 576 -> 480 workgroups bf16 47.8 -> 43.2 us; 50 (400) 800 ->
// 400 162 -> 146, MXFP4 61.5 -> 51.9; but 33 (264) 528 -> 264 117 -> 132.
// 8 waves, 16-bit pages of up to 16 rows: the grid is one round, or a sequence has 2,048 keys and more.  They halve the longest
// workgroup of unequal contexts, and half as many splits are joined; of short ones too many start and end with the CU to
// themselves.  4 -> 8 waves, bf16, us: 24 x 1,000 25.3 -> 22.1, 24 x 4 queries of 500-8,000 114 -> 104, 8 x 1,000-30,000 111 ->
// 104, 64 x 512-8,192 231 -> 224, 400 x 100-3,000 452 -> 436, 64 x 4,096 182.4 -> 181.9, but 12 x 4 of 300-8,192 57 -> 61;
// where 4 stay: 40 x 2,000 67 -> 74, 64 x 1,000 51 -> 55, 200 x 500 80 -> 96.  MXFP4 (its waves are busy, and three
// workgroups of 4 fit a CU): 64 x 4,096 56 -> 60, 200 x 300-2,000 65 -> 93.
// By length (rank_of_layer), up to 64 sequences of 2,048 keys and more in more workgroups than CUs: 16-bit pages (a workgroup
// of 8 waves to a CU) longest first, MXFP4 (two of 4 waves to a CU) the second 256 workgroups shortest first.  In the order given
// -> by length, us: 64 x 512-8,192 bf16 224 -> 196, MXFP4 75.2 -> 66.8; 40 x 1,000-6,000 bf16 126 -> 110; 64 x 4 queries of
// 500-8,000 MXFP4 77 -> 69; what it costs where all are alike: 64 x 4,096 bf16 181.4 -> 182.6, 40 x 3,000 107 -> 108.5; where the
// order given stays: 64 x 1,000 bf16 50.8 -> 53.3, 12 x 4 of 300-8,192 MXFP4 (5 splits) 26 -> 30.
// A workgroup's waves take 2 pages each at a time (MXFP4: 4), of which a split is a multiple.
struct WindowPlan {
    SplitPlan split;
    int waves;                                     // of a workgroup
    int tiles, groups;                             // tiles of 16 rows of a workgroup, workgroups for a kv head's rows
    int layer;                                     // 0: sequences in the order given; else by length (rank_of_layer)
};
// rows: query rows of a kv head, 1 .. 64.
inline WindowPlan window_plan(bool fp4, int64_t rows, int32_t n, int32_t kv_heads, int32_t n_sinks, int32_t max_span) {
    // (a window that does not start with a page has one more: the last split takes it)
    const int64_t pages = std::max<int64_t>(1, ((int64_t)max_span + KPAGE - 1) / KPAGE + ((int64_t)n_sinks + KPAGE - 1) / KPAGE);
    const int64_t units = (int64_t)n * kv_heads;
    const int waves = !fp4 && rows <= 16 && (units <= 256 || pages >= 128) ? 8 : 4;
    const int tiles = rows <= 16 ? 1 : 2, groups = (int)((rows + 16 * tiles - 1) / (16 * tiles));
    const int64_t round = 2048 / waves;
    int64_t want = round / units;
    if (want * units < round * 3 / 4) want++;
    const SplitPlan split = split_plan(want, pages, waves * (fp4 ? 4 : 2));
    const bool by_length = n <= 64 && units > 256 && split.splits == 1 && pages >= 128;
    return WindowPlan{split, waves, tiles, groups, !by_length ? 0 : fp4 ? std::max(1, 256 / (kv_heads * groups)) : n};
}
// Splits that a workspace has to hold, whatever the rows and the page format: 4 waves over 16-bit pages are the finest of all
// plans (8 waves want half a round, which is never more splits, of twice the step; MXFP4 the same round, of twice the step).
inline int window_most_splits(int32_t n, int32_t kv_heads, int32_t n_sinks, int32_t max_span) {
    return window_plan(false, 64, n, kv_heads, n_sinks, max_span).split.splits;
}
// A sequence's place in the order by length: the longer, then the later one first (at most 64 sequences).
UD_HD int length_key(int length, int seq) {
    const int most = (1 << 25) - 1;
    return (length < 0 ? 0 : length > most ? most : length) << 6 | seq;
}
// The rank of the sequence that layer z of the workgroups takes: z of the descending order up to `layer`, then from the
// shortest back, so that workgroups that share a CU make up for each other.
UD_HD int rank_of_layer(int z, int layer, int n) { return z < layer ? z : n - 1 - (z - layer); }

// Prompts (prefill.hip).
//
// Blocks of 128 query rows of the longest sequence, and splits of their keys.
// - At most 256 workgroups (one per CU; two fit): split until there are 512, down to 8 tiles of 64 keys each.
// - Above: split up to 2,048, so that the unequal workgroups of unequal sequences fill each other's gaps, but not below 64
//   tiles, since every split of a row costs its fp32 partial, written and read (520 bytes at D = 128).
// us, 32/8 heads of 128, bf16, one split -> this rule: 16 rows behind 16,000 keys 310 -> 26 (31 splits), 512 rows 322 -> 162
// (4); 512 behind 2,000 58 -> 42 (4); 6 x 37-563 rows behind 4,000-12,000 368 -> 320, MXFP4 377 -> 309 (3); 8 x 64-500 behind
// 2,700-8,000 283 -> 263, MXFP4 285 -> 253 (2).  Where it keeps one split, two lose: a causal prompt of 2,000 rows 58 -> 85,
// of 4,000 169 -> 232.
inline int64_t prefill_blocks(int64_t max_rows, int64_t group) { return (max_rows * group + 127) / 128; }
inline int prefill_splits(int64_t n, int64_t kv_heads, int64_t blocks, int64_t n_sinks, int64_t max_span) {
    const int64_t units = n * kv_heads * blocks, tiles = (max_pages(max_span, n_sinks) + 3) / 4;
    const int64_t want = ((units <= 256 ? 512 : 2048) + units - 1) / units, most = tiles / (units <= 256 ? 8 : 64);
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), MAX_SPLITS));
}

}  // namespace ud
