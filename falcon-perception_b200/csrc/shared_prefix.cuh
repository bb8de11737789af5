// What the two halves of shared-prefix decode attention agree on: rows, groups, and how the prefixes' key tiles are shared out.
#pragma once

#include <cuda.h>
#include "common.cuh"

namespace fpkv {

// The batch as the kernels see it.
struct RowParams {
    const int64_t* page_table;
    const int64_t* p2l;
    const int64_t* batch_idx;
    const void* pos;
    const int4* groups;                        // {first row, rows, shared pages, 0}
    const int* row_group;
    int32_t* status;
    int B, Hq, H, n_rep, n_groups, n_pages, max_batch, pos_is_64;
    int rows_per_tile;                         // batch rows of a query tile of the prefix part
};

struct PrefixParams {
    RowParams rows;
    float2* ml;                                // partials [slot][128 rows] (m, l): maximum and sum in base 2
    float* acc;                                // [slot][D/4][128 rows][4]
    int4* segments;                            // [max_segments] for the merge: {first batch row, query rows | stored head << 8, first slot,
                                               // partials | group << 16}, all zero past the last
    int max_segments;
    int rows_per_plane, q_box_rows;
    float scale_log2;
};

constexpr int kPrefixTileRows = 128;

int prefix_ctas();
bool prefix_supported(const PoolView& pv);
// Tensor map of one layer's K and V planes: `rows` token rows at a time, 64-element column groups one behind the other.
bool encode_rows(CUtensorMap* map, const PoolView& pv, int layer, int rows);
int launch_prefix(const PoolView& pv, int layer, const void* q, long long q_stride_b, long long q_stride_h, PrefixParams prm, cudaStream_t stream);

// Visible keys of a row and its slot; a slot or position out of range gives none.
__device__ __forceinline__ int row_keys(const RowParams& p, int b, int* slot, bool report) {
    const long long s = p.batch_idx[b];
    const long long at = p.pos_is_64 ? reinterpret_cast<const int64_t*>(p.pos)[b] : (long long)reinterpret_cast<const int32_t*>(p.pos)[b];
    *slot = 0;
    if (s < 0 || s >= p.max_batch) { if (report) raise_status(p.status, FPKV_STATUS_BAD_SLOT); return 0; }
    if (at < 0 || at / 128 >= p.n_pages) { if (report) raise_status(p.status, FPKV_STATUS_BAD_POS); return 0; }
    *slot = (int)s;
    return (int)at + 1;
}
// A group as the kernels use it: rows inside the batch and pages inside the table, or nothing.
__device__ __forceinline__ int4 group_at(const RowParams& p, int g) {
    int4 d = p.groups[g];
    if (d.x < 0 || d.y <= 0 || d.x >= p.B || d.y > p.B - d.x || d.z <= 0) d.y = d.z = 0;
    d.z = min(d.z, p.n_pages);
    return d;
}
__device__ __forceinline__ int tiles_of(const RowParams& p, const int4& d) { return (d.y + p.rows_per_tile - 1) / p.rows_per_tile; }
// Group of a row, -1 for none.
__device__ __forceinline__ int group_of_row(const RowParams& p, int b, int4* d) {
    const int g = p.n_groups > 0 ? p.row_group[b] : -1;
    if (g < 0 || g >= p.n_groups) return -1;
    *d = group_at(p, g);
    return (d->y > 0 && b >= d->x && b < d->x + d->y) ? g : -1;
}

// Whether a slot maps pages at all: padding (slot 0) and erased slots do not.  Such a row of a group -- a request that has ended
// since the groups were made -- is as good as in none, and the pages are read through another row's table.
__device__ __forceinline__ bool slot_maps_pages(const RowParams& p, long long slot) {
    if (slot <= 0 || slot >= p.max_batch) return false;
    const long long page = p.page_table[slot * p.n_pages];
    return page >= 0 && page < p.n_pages;
}
// Slot of the first of `rows` batch rows from b0 on that maps pages, 0 if none does.  One warp.
__device__ __forceinline__ int mapping_slot(const RowParams& p, int b0, int rows, int lane) {
    for (int r0 = 0; r0 < rows; r0 += 32) {
        const long long slot = r0 + lane < rows ? p.batch_idx[b0 + r0 + lane] : 0;
        const uint32_t maps = __ballot_sync(0xffffffffu, slot_maps_pages(p, slot));
        if (maps) return (int)__shfl_sync(0xffffffffu, slot, __ffs(maps) - 1);
    }
    return 0;
}

// ---- the schedule: key tiles of all segments in a row -- group by group, head by head, query tile by query tile -- in equal
// shares.  flat_before[g], mt_before[g]: key tiles (over all segments) and query tiles before group g; mt_before[n_groups + 1]:
// the longest segment's key tiles.  The workspace has room for max_tiles query tiles, all that groups without common rows can
// have; groups are device data, so what does not fit that is left out, and said in the status. --------------------
// A share is what the fullest one has to hold, so that as few as possible are used: a share more is a partial more, and the
// fullest one sets the time.  Nor is the longest segment cut into more than kMaxPieces, because the merge goes through a row's
// partials one after the other.  Whole call, 8 query heads over one stored head of 128, bf16, at most 64 pieces against no bound:
// ten groups of up to 3 rows and 29 440 shared keys 72 instead of 133 us, three groups of up to 2 rows and 16 384 keys 37 instead
// of 143, one group of 4 rows and 32 768 keys 35 instead of 45.  At most 40 in the own part: 90 us for the first (a warp's
// share then sets the time), 96 and 128: 88 and 94.  A batch whose even share is larger already is cut as before.
constexpr int kMaxPieces = 64;
__device__ __forceinline__ long long share_size(long long total, int sharers, int longest) {
    return max(max((total + sharers - 1) / sharers, (long long)(longest + kMaxPieces - 1) / kMaxPieces), 1ll);
}
__device__ __forceinline__ void prefix_schedule(const RowParams& p, int max_tiles, long long* flat_before, int* mt_before, int lane) {      // one warp
    long long flat = 0;
    int mt = 0, longest = 0;
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        const int g = g0 + lane;
        const int4 d = g < p.n_groups ? group_at(p, g) : make_int4(0, 0, 0, 0);
        const int t = tiles_of(p, d);
        longest = max(longest, d.z);
        long long f = (long long)t * p.H * d.z;
        int m = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long yf = __shfl_up_sync(0xffffffffu, f, o);
            const int ym = __shfl_up_sync(0xffffffffu, m, o);
            if (lane >= o) { f += yf; m += ym; }
        }
        const int fit = __popc(__ballot_sync(0xffffffffu, mt + m <= max_tiles));     // a leading run of the lanes
        if (fit < 32) {
            const long long last_f = __shfl_sync(0xffffffffu, f, max(fit - 1, 0));
            const int last_m = __shfl_sync(0xffffffffu, m, max(fit - 1, 0));
            if (lane >= fit) { f = fit > 0 ? last_f : 0; m = fit > 0 ? last_m : 0; }
            if (lane == 0) raise_status(p.status, FPKV_STATUS_BAD_SLOT);
        }
        if (g < p.n_groups) { flat_before[g + 1] = flat + f; mt_before[g + 1] = mt + m; }
        flat += __shfl_sync(0xffffffffu, f, 31);
        mt += __shfl_sync(0xffffffffu, m, 31);
    }
    longest = (int)__reduce_max_sync(0xffffffffu, (uint32_t)longest);
    if (lane == 0) { flat_before[0] = 0; mt_before[0] = 0; mt_before[p.n_groups + 1] = longest; }
}
struct Segment {
    int index;                                 // over all groups
    int b0, rows, h;                           // first batch row, query rows, stored head
    int pages, tile;                           // key tiles of the segment; the one at the position asked for
    int group_b0, group_rows;                  // the group's batch rows
};
__device__ __forceinline__ Segment segment_at(const RowParams& p, const long long* flat_before, const int* mt_before, long long pos) {
    int lo = 0, hi = p.n_groups;               // flat_before[lo] <= pos < flat_before[hi]
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (flat_before[mid] <= pos) lo = mid; else hi = mid; }
    const int4 d = group_at(p, lo);
    const int mt = mt_before[lo + 1] - mt_before[lo];
    const long long rel = pos - flat_before[lo];
    const int seg = (int)(rel / d.z), m = seg % mt;
    Segment s;
    s.tile = (int)(rel - (long long)seg * d.z);
    s.pages = d.z;
    s.h = seg / mt;
    s.index = mt_before[lo] * p.H + seg;
    s.b0 = d.x + m * p.rows_per_tile;
    s.rows = min(p.rows_per_tile, d.x + d.y - s.b0) * p.n_rep;
    s.group_b0 = d.x; s.group_rows = d.y;
    return s;
}

// Segment i of all, as the merge reads it.
__device__ __forceinline__ int4 segment_entry(const RowParams& p, const long long* flat_before, const int* mt_before, int i, int ctas) {
    int lo = 0, hi = p.n_groups;               // mt_before[lo] * H <= i < mt_before[hi] * H
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (mt_before[mid] * p.H <= i) lo = mid; else hi = mid; }
    const int4 d = group_at(p, lo);
    const int mt = mt_before[lo + 1] - mt_before[lo], in = i - mt_before[lo] * p.H, m = in % mt;
    const long long share = share_size(flat_before[p.n_groups], ctas, mt_before[p.n_groups + 1]), first = flat_before[lo] + (long long)in * d.z;
    const int c0 = (int)(first / share), b0 = d.x + m * p.rows_per_tile;
    return make_int4(b0, min(p.rows_per_tile, d.x + d.y - b0) * p.n_rep | (in / mt) << 8, c0 + i, (int)((first + d.z - 1) / share) - c0 + 1 | lo << 16);
}

}  // namespace fpkv
