// Decode attention of a batch whose rows share long prefixes (16-bit pools, page_size 128).
//
// With keys 0 .. s-1 the same for every row of a group, the softmax over a row's keys splits into the prefix part and
// the row's own part, each with its own maximum m, sum l and unnormalised result a (all in 32 bits):
//     M = max(m1, m2),  l = l1 2^(m1-M) + l2 2^(m2-M),  out = (a1 2^(m1-M) + a2 2^(m2-M)) / l
// (scores in base 2).  The prefix part of all rows of a group is one product over the prefix's keys, so they are read
// once a group instead of once a row.  Three launches:
//
//  * prefix part: shared_prefix_tc.cu.
//  * own part, below: the rows' own keys in blocks of 16, for every row and every 8 query heads of a stored head, one after
//    the other, in equal shares, one per WARP: a warp needs no other, so there is no barrier, and all have the same to do
//    however the lengths differ.  A block is
//        S^T = K Q^T   (16 keys x 8 heads),   O^T += V^T P^T   (dims x 8 heads)      in mma.sync.m16n8k16,
//    with P rounded to the 16-bit type of V, as there, and the sums of P in 32 bits before that.
//    K and V come by tensor copies (16 rows, 128-byte swizzle) into a ring of the warp's own, requested several blocks ahead
//    and across rows: with only what fits the registers in flight, 12 warps an SM reached 3.7 TB/s.  The order of the
//    contraction index and of the output's dims is free, so it is chosen such that every lane's 16-byte piece of a row is its
//    own operand and no access to the ring conflicts.  Bound by the bytes of the rows' own keys.
//  * merge: joins the partials of every (row, head), applies the sink gate, writes out and lse.
// The three are chained by programmatic dependent launch: the own part starts as soon as every CTA of the prefix part has
// (it needs nothing from it) and fills the SMs as they come free; it ends after the prefix part, so that the merge has only
// the own part to wait for.  Both parts write down for the merge which partials belong to whom.

#include "tc5.cuh"
#include "shared_prefix.cuh"

namespace fpkv {

namespace {

constexpr int kMaxRep = 16;                    // query heads of a stored head
constexpr int kHeads = 8;                      // of them, those of a CTA of the own part: the MMAs' columns
// One CTA an SM.  A block takes a warp about 1200 clocks from its arrival (products, maximum, exponentials, products, each
// waiting for the one before), so it takes many warps to keep up with memory: 12 with two blocks of 16 keys each did 256 rows
// of 1 to 512 own keys faster than 8 with three.
constexpr int kOwnWarps = 12;
constexpr int kRingBytes = 16 * 1024;          // of a warp
constexpr int kBlock = 16, kPageBlocks = kPage / kBlock;
constexpr int kMaxRows = 1024;                 // batch rows of a launch of the own part

struct OwnParams {
    RowParams rows;
    const void* q;
    // partials [slot][8 heads] (m, l) and [slot][8 heads][D]; slot = worker number + segment number, segments counted row by
    // row, stored head by stored head, 8 query heads by 8 query heads
    float2* ml;
    float* acc;
    int4* entries;                             // [rows][segments] for the merge: {first slot, partials, group + 1, 0}
    long long q_stride_b, q_stride_h;
    int row0, n_rows, head_blocks;             // the launch's rows; blocks of kHeads query heads of a stored head
    int rows_per_plane;
    float scale_log2;
};

struct MergeParams {
    const int4* segments;                      // of the prefix part
    const int4* entries;                       // of the own part
    const float2* pre_ml; const float* pre_acc;
    const float2* own_ml; const float* own_acc;
    size_t own_slots;                          // partials of one launch of the own part
    int B, Hq, n_rep, head_blocks, n_segments; // n_segments: upper bound, of the prefix part
    void* out;
    float* lse;
    Epilogue epi;
};

template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint4 ld16(const char* p) { return *reinterpret_cast<const uint4*>(p); }

// The transpose of an 8 x 8 block of 16-bit numbers held two a lane.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

template <typename T, int D>
__global__ void __launch_bounds__(kOwnWarps * 32, 1)
own_part_kernel(const __grid_constant__ CUtensorMap map, const OwnParams prm)
{
    constexpr int NH = D / 64;                 // 64-column groups of a row
    constexpr int kHalf = kBlock * 128, kTile = NH * kHalf;  // a block's K (or V): column groups of 16 rows of 128 bytes
    constexpr int kStages = kRingBytes / (2 * kTile);
    const RowParams& rp = prm.rows;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    extern __shared__ uint8_t smem_raw[];
    __shared__ long long s_before[kMaxRows + 1];
    __shared__ int s_slot[kMaxRows], s_first[kMaxRows], s_keys[kMaxRows];    // slot, first own page, visible keys of each row
    __shared__ short s_group[kMaxRows];        // its group + 1, 0 for none
    __shared__ uint64_t s_bars[kOwnWarps][kStages];
    __shared__ int s_abort, s_longest;         // s_longest: blocks of the longest segment
    asm volatile("griddepcontrol.launch_dependents;");       // the merge may take its seats
    const uint32_t ring = ((s32(smem_raw) + 1023u) & ~1023u) + warp * kRingBytes, bars = s32(&s_bars[warp][0]);
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
        s_abort = 0;
    }
    if (lane < kStages) bar_init(bars + 8 * lane, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

    // ---- the schedule -----------------------------------------------------------------
    const int n_segs = rp.H * prm.head_blocks;               // of a row
    for (int i = threadIdx.x; i < prm.n_rows; i += kOwnWarps * 32) {
        const int b = prm.row0 + i;
        int slot; int4 d;
        const int keys = row_keys(rp, b, &slot, blockIdx.x == 0);
        int group = group_of_row(rp, b, &d);
        if (group >= 0 && !slot_maps_pages(rp, slot)) group = -1;
        const int first = group >= 0 ? d.z : 0;
        s_slot[i] = slot; s_first[i] = first; s_keys[i] = keys; s_group[i] = (short)(group + 1);
        s_before[i + 1] = (long long)max(0, (keys + kBlock - 1) / kBlock - first * kPageBlocks) * n_segs;
    }
    __syncthreads();
    if (warp == 0) {
        long long carry = 0;
        int longest = 0;
        for (int i0 = 0; i0 < prm.n_rows; i0 += 32) {
            const int i = i0 + lane;
            long long v = i < prm.n_rows ? s_before[i + 1] : 0;
            longest = max(longest, (int)(v / n_segs));
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += y; }
            if (i < prm.n_rows) s_before[i + 1] = v + carry;
            carry += __shfl_sync(0xffffffffu, v, 31);
        }
        longest = (int)__reduce_max_sync(0xffffffffu, (uint32_t)longest);
        if (lane == 0) { s_before[0] = 0; s_longest = longest; }
    }
    __syncthreads();
    const long long total = s_before[prm.n_rows];
    const int me = blockIdx.x * kOwnWarps + warp;
    const long long share = share_size(total, gridDim.x * kOwnWarps, s_longest), end = min(total, (me + 1) * share);
    long long pos = min(end, me * share);
    // the merge's table
    for (int i = blockIdx.x * kOwnWarps * 32 + threadIdx.x; i < prm.n_rows * n_segs; i += gridDim.x * kOwnWarps * 32) {
        const int r = i / n_segs, seg = i - r * n_segs;
        const long long blocks = s_before[r + 1] - s_before[r];
        int4 e = make_int4(0, 0, s_group[r], 0);
        if (blocks > 0) {
            const long long nb = blocks / n_segs, first = s_before[r] + nb * seg;
            const int w0 = (int)(first / share);
            e.x = w0 + i; e.y = (int)((first + nb - 1) / share) - w0 + 1;
        }
        prm.entries[i] = e;
    }

    // A piece: blocks [blk0, blk0 + n) of a segment.
    struct Piece { int row, first, keys, seg, blk0, n, h; };
    auto piece_at = [&](long long at) -> Piece {
        int lo = 0, hi = prm.n_rows;                         // s_before[lo] <= at < s_before[hi]
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_before[mid] <= at) lo = mid; else hi = mid; }
        Piece p;
        p.row = lo; p.first = s_first[lo]; p.keys = s_keys[lo];
        const int nb = (p.keys + kBlock - 1) / kBlock - p.first * kPageBlocks;
        const unsigned rel = (unsigned)(at - s_before[lo]);  // blocks of one row
        p.seg = (int)(rel / (unsigned)nb); p.blk0 = (int)(rel - (unsigned)p.seg * nb);
        p.n = (int)min((long long)(nb - p.blk0), end - at);
        p.h = p.seg / prm.head_blocks;
        return p;
    };
    // ---- requests run ahead of the work, across pieces -------------------------------------
    // Pages of a piece are looked up 32 at a time, one a lane; the table entries of the first 32 of the piece after next are on
    // their way while the present one is requested.
    auto page_of = [&](const Piece& p, int w) -> long long {
        const int page = p.first + p.blk0 / kPageBlocks + w * 32 + lane;
        return page * kPage < p.keys ? rp.page_table[(long long)s_slot[p.row] * rp.n_pages + page] : -1;
    };
    Piece ahead, next;                                       // the piece that is being requested, the one after it
    long long next_pos = pos, next_page = -1;                // end of `next`; this lane's table entry of it
    auto advance = [&]() {
        if (next_pos >= end) { next.n = 0; return; }
        next = piece_at(next_pos);
        next_pos += next.n;
        next_page = page_of(next, 0);
    };
    advance();
    int ahead_t = 0, window = 0, pool_rows = -1;             // pool rows of 32 pages of `ahead`; -1 = not visible
    ahead.n = 0;
    uint32_t requested = 0, visible = 0;                     // blocks requested; of the stages' blocks, those on visible pages
    auto request = [&]() {
        bool lookup = false;
        long long pg = -1;
        if (ahead_t == ahead.n) {
            if (next.n == 0) return;
            ahead = next; pg = next_page; ahead_t = 0; window = 0;
            lookup = true;
            advance();
            // the queries will be wanted soon
            if (lane < min(kHeads, rp.n_rep) * NH) {
                const int r0 = (ahead.seg % prm.head_blocks) * kHeads + lane / NH;
                if (r0 < rp.n_rep)
                    asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const T*>(prm.q) + (prm.row0 + ahead.row) * prm.q_stride_b +
                                                                   (ahead.h * rp.n_rep + r0) * prm.q_stride_h + lane % NH * 64));
            }
        }
        const int at_blk = ahead.blk0 + ahead_t, p = at_blk / kPageBlocks, w = (p - ahead.blk0 / kPageBlocks) / 32;
        if (w != window) { window = w; pg = page_of(ahead, w); lookup = true; }
        if (lookup) {
            pool_rows = -1;
            if (pg >= rp.n_pages) raise_status(rp.status, FPKV_STATUS_BAD_PAGE);
            else if (pg >= 0 && rp.p2l[(long long)s_slot[ahead.row] * rp.n_pages + pg] >= 0) pool_rows = (int)pg * kPage;
        }
        const int row0 = __shfl_sync(0xffffffffu, pool_rows, (p - ahead.blk0 / kPageBlocks) % 32);
        const uint32_t st = requested % kStages;
        visible = row0 >= 0 ? visible | (1u << st) : visible & ~(1u << st);
        if (lane == 0) {
            const uint32_t bar = bars + 8 * st, dst = ring + st * (2 * kTile);
            if (row0 >= 0) {
                const int row = ahead.h * prm.rows_per_plane + row0 + at_blk % kPageBlocks * kBlock;
                bar_expect_tx(bar, 2 * kTile);
                tma_3d(dst, &map, 0, row, 0, bar);
                tma_3d(dst + kTile, &map, 0, row + rp.H * prm.rows_per_plane, 0, bar);
            } else bar_arrive(bar);
        }
        ++requested; ++ahead_t;
    };
    const uint32_t n_blocks = (uint32_t)(end - pos);
    for (int i = 0; i < kStages; ++i) request();
    uint32_t done = 0;
    bool alive = true;
    while (pos < end && alive) {
        const Piece pc = piece_at(pos);
        pos += pc.n;
        const int r0 = (pc.seg % prm.head_blocks) * kHeads, heads = min(kHeads, rp.n_rep - r0);
        // queries: head g, dims a * 64 + c * 16 + e * 8 .. + 7
        uint4 qa[NH][2];
        const T* q = reinterpret_cast<const T*>(prm.q) + (prm.row0 + pc.row) * prm.q_stride_b + (pc.h * rp.n_rep + r0 + g) * prm.q_stride_h;
#pragma unroll
        for (int a = 0; a < NH; ++a)
#pragma unroll
            for (int e = 0; e < 2; ++e) qa[a][e] = g < heads ? ld16(reinterpret_cast<const char*>(q + a * 64 + c * 16 + e * 8)) : make_uint4(0, 0, 0, 0);
        float acc[NH][4][4];                   // O^T: rows dims a * 64 + g * 8 + 2 e (+ 1), columns heads 2 c and 2 c + 1
#pragma unroll
        for (int a = 0; a < NH; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[a][e][k] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // heads 2 c and 2 c + 1; l this lane's keys alone

        for (int t = 0; t < pc.n; ++t, ++done) {
            const uint32_t st = done % kStages;
            if (!bar_wait(bars + 8 * st, (done / kStages) & 1u, &s_abort)) { alive = false; break; }
            if (visible >> st & 1u) {
                const int key0 = pc.first * kPage + (pc.blk0 + t) * kBlock;
                const uint32_t ks = ring + st * (2 * kTile), vs = ks + kTile;
                // keys g and g + 8: 16-byte pieces 2 c and 2 c + 1 of their rows (row & 7 = g); two chains of products
                float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int a = 0; a < NH; ++a)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t at = ks + a * kHalf + g * 128 + (((2 * c + e) ^ g) << 4);
                        const uint4 k0 = lds16(at), k1 = lds16(at + 8 * 128);
                        const uint32_t a0[4] = {k0.x, k1.x, k0.y, k1.y}, a1[4] = {k0.z, k1.z, k0.w, k1.w};
                        mma16816<T>(s, a0, qa[a][e].x, qa[a][e].y);
                        mma16816<T>(s2, a1, qa[a][e].z, qa[a][e].w);
                    }
                uint4 v[4][NH];                // keys 2c, 2c + 1, 2c + 8, 2c + 9: piece g
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int a = 0; a < NH; ++a) {
                        const int r = 2 * c + (k & 1) + (k >> 1) * 8;
                        v[k][a] = lds16(vs + a * kHalf + r * 128 + ((g ^ (r & 7)) << 4));
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += s2[e];   // S^T: keys g (0, 1) and g + 8 (2, 3), heads 2 c and 2 c + 1
                // keys past the row's end: no weight, and (never appended, perhaps) no value either
                if (key0 + kBlock > pc.keys) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (key0 + g + (e >> 1) * 8 >= pc.keys) s[e] = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (key0 + 2 * c + (k & 1) + (k >> 1) * 8 >= pc.keys)
#pragma unroll
                            for (int a = 0; a < NH; ++a) v[k][a] = make_uint4(0, 0, 0, 0);
                }
                float mx[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(s[r], s[2 + r]);           // the scale is positive: the maximum commutes with it
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 4));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 8));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 16)) * prm.scale_log2;
                }
                if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float mn = fmaxf(m[r], mx[r]), alpha = m[r] == -INFINITY ? 0.f : exp2f(m[r] - mn);
                        m[r] = mn;
                        l[r] *= alpha;
#pragma unroll
                        for (int a = 0; a < NH; ++a)
#pragma unroll
                            for (int e = 0; e < 4; ++e) { acc[a][e][r] *= alpha; acc[a][e][2 + r] *= alpha; }
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = e & 1;
                    s[e] = m[r] == -INFINITY ? 0.f : exp2f(s[e] * prm.scale_log2 - m[r]);
                    l[r] += s[e];
                }
                const uint32_t p0 = transposed(pack_pair<T>(s[0], s[1])), p1 = transposed(pack_pair<T>(s[2], s[3]));
#pragma unroll
                for (int a = 0; a < NH; ++a) {
                    const uint32_t* x0 = &v[0][a].x; const uint32_t* x1 = &v[1][a].x;
                    const uint32_t* x2 = &v[2][a].x; const uint32_t* x3 = &v[3][a].x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t vt[4] = {__byte_perm(x0[e], x1[e], 0x5410u), __byte_perm(x0[e], x1[e], 0x7632u),
                                                __byte_perm(x2[e], x3[e], 0x5410u), __byte_perm(x2[e], x3[e], 0x7632u)};
                        mma16816<T>(acc[a][e], vt, p0, p1);
                    }
                }
            }
            __syncwarp();                      // all lanes have read the stage
            if (requested < n_blocks) request();
        }
        if (!alive) break;
        // ---- the piece's partial --------------------------------------------------------
        const size_t slot = (size_t)me + (size_t)pc.row * n_segs + pc.seg;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
            const int head = 2 * c + r;
            if (head >= heads) continue;
            if (g == 0) prm.ml[slot * kHeads + head] = make_float2(m[r], l[r]);
            float4* dst = reinterpret_cast<float4*>(prm.acc + (slot * kHeads + head) * D + g * 8);
#pragma unroll
            for (int a = 0; a < NH; ++a)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    dst[a * 16 + e] = make_float4(acc[a][2 * e][r], acc[a][2 * e][2 + r], acc[a][2 * e + 1][r], acc[a][2 * e + 1][2 + r]);
        }
    }
    if (!alive) {                              // a copy did not come: say so, and wait (bounded) for those in flight
        if (lane == 0) { raise_status(rp.status, FPKV_STATUS_TIMEOUT); *reinterpret_cast<volatile int*>(&s_abort) = 1; }
        for (; done < requested; ++done)
            for (uint32_t k = 0; k < kSpin && !bar_try(bars + 8 * (done % kStages), (done / kStages) & 1u); ++k) {}
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");       // not done before the prefix part is
}

// Block: 32 (row, head) pairs, one a lane, and 64 columns: four column groups x two halves of the partials, a warp each.  The
// pairs are a quarter of a query tile of the prefix part, whose partials lie side by side; behind those blocks come some for
// the rows that are in no group.  The weights of all partials are worked out first, in parallel, so that the loads of the sums
// do not wait for one another.
constexpr int kMergePieces = 32;

template <typename T, int D>
__global__ void __launch_bounds__(256, 2)
shared_merge_kernel(const MergeParams prm)
{
    constexpr int kColBlocks = D / 64;
    __shared__ float2 s_ml[kMergePieces][32];
    __shared__ float s_half[4][17][32];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, half = warp / 4;
    const int col4 = (blockIdx.x % kColBlocks) * 16 + warp % 4 * 4, block = blockIdx.x / kColBlocks;
    const int tile_blocks = prm.n_segments * (kPrefixTileRows / 32);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int b = -1, hq = 0, n_pre = 0, slot = 0, trow = 0, group = 0;
    if (block < tile_blocks) {
        const int4 sg = prm.segments[block / (kPrefixTileRows / 32)];
        const int rows = sg.y & 255;
        trow = block % (kPrefixTileRows / 32) * 32 + lane;
        if (trow < rows) { b = sg.x + trow / prm.n_rep; hq = (sg.y >> 8) * prm.n_rep + trow % prm.n_rep; }
        slot = sg.z; n_pre = sg.w & 0xffff; group = (sg.w >> 16) + 1;
    } else {
        const int i = (block - tile_blocks) * 32 + lane;
        if (i < prm.B * prm.Hq) { b = i / prm.Hq; hq = i % prm.Hq; }
    }
    // the row's partials of the own part: first one (times 8, plus the head) and number
    size_t own = 0;
    int n_own = 0;
    if (b >= 0) {
        const int rep = hq % prm.n_rep, seg = hq / prm.n_rep * prm.head_blocks + rep / kHeads, n_segs = prm.Hq / prm.n_rep * prm.head_blocks;
        const int4 e = prm.entries[(size_t)b * n_segs + seg];
        n_own = e.y;
        own = ((size_t)(b / kMaxRows) * prm.own_slots + e.x) * kHeads + rep % kHeads;
        if (e.z != group) b = -1;              // a row of the tile that does not name the group, or here a row that is in one
    }
    if (__ballot_sync(0xffffffffu, b >= 0) == 0) return;     // the same for all warps
    if (b < 0) n_own = 0;
    const int n = n_pre + (int)__reduce_max_sync(0xffffffffu, (uint32_t)n_own);
    float M = -INFINITY, L = 0.f, a[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] = 0.f;
    for (int p0 = 0; p0 < n; p0 += kMergePieces) {
        const int here = min(kMergePieces, n - p0);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kMergePieces / 8; ++r) {
            const int p = warp + 8 * r, i = p0 + p;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (p < here && b >= 0) {
                if (i < n_pre) ml = prm.pre_ml[(size_t)(slot + i) * kPrefixTileRows + trow];
                else if (i - n_pre < n_own) ml = prm.own_ml[own + (size_t)(i - n_pre) * kHeads];
            }
            s_ml[p][lane] = ml;
        }
        __syncthreads();
        float mn = M;
        for (int p = 0; p < here; ++p) mn = fmaxf(mn, s_ml[p][lane].x);
        const float alpha = M == -INFINITY ? 0.f : exp2f(M - mn);
        M = mn;
        L *= alpha;
#pragma unroll
        for (int k = 0; k < 16; ++k) a[k] *= alpha;
#pragma unroll 4
        for (int p = half; p < here; p += 2) {
            const float2 ml = s_ml[p][lane];
            const int i = p0 + p;
            const float4* src = i < n_pre ? reinterpret_cast<const float4*>(prm.pre_acc) + ((size_t)(slot + i) * (D / 4) + col4) * kPrefixTileRows + trow
                                          : reinterpret_cast<const float4*>(prm.own_acc) + (own + (size_t)(i - n_pre) * kHeads) * (D / 4) + col4;
            const size_t step = i < n_pre ? kPrefixTileRows : 1;
            const bool some = ml.y != 0.f;                   // nothing visible: no sums were written
            const float w = some ? exp2f(ml.x - M) : 0.f;
            L += ml.y * w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 x = some ? src[k * step] : make_float4(0.f, 0.f, 0.f, 0.f);
                a[4 * k] += w * x.x; a[4 * k + 1] += w * x.y; a[4 * k + 2] += w * x.z; a[4 * k + 3] += w * x.w;
            }
        }
    }
    if (half == 1) {
#pragma unroll
        for (int k = 0; k < 16; ++k) s_half[warp - 4][k][lane] = a[k];
        s_half[warp - 4][16][lane] = L;
    }
    __syncthreads();
    if (half == 1 || b < 0) return;
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] += s_half[warp][k][lane];
    L += s_half[warp][16][lane];
    const size_t row = (size_t)b * prm.Hq + hq;
    const float lse = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    const float gate = sink_gate(prm.epi, hq, lse), inv = L == 0.f ? 0.f : 1.f / L;
    __align__(16) T o[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = gated_out<T>(a[k] * inv, gate, prm.epi.sinks != nullptr);
    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(prm.out) + row * D + col4 * 4);
    dst[0] = reinterpret_cast<const uint4*>(o)[0];
    dst[1] = reinterpret_cast<const uint4*>(o)[1];
    if (col4 == 0) prm.lse[row] = lse;
}

struct Plan { int n_rep, rows_per_tile, tiles, head_blocks, workers, chunks; size_t slots, own_slots, pre_ml, pre_acc, own_ml, own_acc, entries, segments, bytes; };
Plan plan_of(const PoolView& pv, int B, int Hq, int n_groups)
{
    Plan p;
    p.n_rep = Hq / pv.H;
    p.rows_per_tile = kPrefixTileRows / p.n_rep;
    // each group's tiles: its rows over the rows of a tile, rounded up
    p.tiles = n_groups > 0 ? (int)((B + (long long)(n_groups < B ? n_groups : B) * (p.rows_per_tile - 1)) / p.rows_per_tile) : 0;
    p.head_blocks = (p.n_rep + kHeads - 1) / kHeads;
    p.workers = prefix_ctas() * kOwnWarps;
    p.chunks = (B + kMaxRows - 1) / kMaxRows;
    // slots are worker (or CTA) number + segment number
    p.slots = p.tiles > 0 ? (size_t)p.tiles * pv.H + prefix_ctas() : 0;
    p.own_slots = (size_t)(B < kMaxRows ? B : kMaxRows) * pv.H * p.head_blocks + p.workers;
    auto place = [at = (size_t)0](size_t n) mutable { const size_t was = at; at += (n + 255) / 256 * 256; return was; };
    p.pre_ml = place(p.slots * kPrefixTileRows * sizeof(float2));
    p.pre_acc = place(p.slots * kPrefixTileRows * pv.D * sizeof(float));
    p.own_ml = place(p.chunks * p.own_slots * kHeads * sizeof(float2));
    p.own_acc = place(p.chunks * p.own_slots * kHeads * pv.D * sizeof(float));
    p.entries = place((size_t)B * pv.H * p.head_blocks * sizeof(int4));
    p.segments = place((size_t)p.tiles * pv.H * sizeof(int4));
    p.bytes = place(0);
    return p;
}

}  // namespace

bool decode_shared_supported(const PoolView& pv, int Hq)
{
    return (pv.dtype == FPKV_BF16 || pv.dtype == FPKV_F16) && pv.split_hq == 0 && pv.P == kPage && Hq / pv.H <= kMaxRep && prefix_supported(pv);
}

size_t decode_shared_workspace_bytes(const PoolView& pv, int B, int Hq, int n_groups) { return plan_of(pv, B, Hq, n_groups).bytes; }

int launch_decode_shared(const PoolView& pv, int layer, void* out, float* lse, const void* q, long long qsb, long long qsh,
                         const int64_t* batch_idx, const void* pos, int pos_type, int B, int Hq, const int32_t* groups,
                         int n_groups, const int32_t* row_group, float sm_scale, void* workspace, const Epilogue& epi,
                         int32_t* status, cudaStream_t stream)
{
    const Plan pl = plan_of(pv, B, Hq, n_groups);
    char* ws = static_cast<char*>(workspace);
    RowParams rows;
    rows.page_table = pv.page_table; rows.p2l = pv.p2l; rows.batch_idx = batch_idx; rows.pos = pos;
    rows.groups = reinterpret_cast<const int4*>(groups); rows.row_group = row_group; rows.status = status;
    rows.B = B; rows.Hq = Hq; rows.H = pv.H; rows.n_rep = pl.n_rep; rows.n_groups = n_groups; rows.n_pages = pv.n_pages;
    rows.max_batch = pv.max_batch; rows.pos_is_64 = pos_type == FPKV_I64; rows.rows_per_tile = pl.rows_per_tile;
    if (n_groups > 0) {
        PrefixParams pre;
        pre.rows = rows; pre.ml = reinterpret_cast<float2*>(ws + pl.pre_ml); pre.acc = reinterpret_cast<float*>(ws + pl.pre_acc);
        pre.segments = reinterpret_cast<int4*>(ws + pl.segments); pre.max_segments = pl.tiles * pv.H;
        pre.rows_per_plane = 0; pre.q_box_rows = 0; pre.scale_log2 = sm_scale * kLog2e;
        const int rc = launch_prefix(pv, layer, q, qsb, qsh, pre, stream);
        if (rc) return rc;
    }
    OwnParams own;
    own.rows = rows; own.q = q; own.rows_per_plane = pv.n_pages * pv.P;
    own.q_stride_b = qsb; own.q_stride_h = qsh; own.head_blocks = pl.head_blocks; own.scale_log2 = sm_scale * kLog2e;
    MergeParams mrg;
    mrg.segments = reinterpret_cast<int4*>(ws + pl.segments); mrg.entries = reinterpret_cast<int4*>(ws + pl.entries);
    mrg.pre_ml = reinterpret_cast<float2*>(ws + pl.pre_ml); mrg.pre_acc = reinterpret_cast<float*>(ws + pl.pre_acc);
    mrg.own_ml = reinterpret_cast<float2*>(ws + pl.own_ml); mrg.own_acc = reinterpret_cast<float*>(ws + pl.own_acc);
    mrg.own_slots = pl.own_slots; mrg.B = B; mrg.Hq = Hq; mrg.n_rep = pl.n_rep; mrg.head_blocks = pl.head_blocks;
    mrg.n_segments = pl.tiles * pv.H;
    mrg.out = out; mrg.lse = lse; mrg.epi = epi;
    CUtensorMap map;
    if (!encode_rows(&map, pv, layer, kBlock)) return FPKV_ELAUNCH;
    constexpr int kOwnSmem = 1024 + kOwnWarps * kRingBytes;
    auto launch = [&](auto kern, int grid, int threads, int smem, bool chained, const auto&... args) {
        if (smem > 0 && launch_code(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return false;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr; cfg.numAttrs = chained ? 1 : 0;
        return launch_code(cudaLaunchKernelEx(&cfg, kern, args...)) == FPKV_OK;
    };
    auto run = [&](auto part, auto merge) {
        // (launches of further rows wait for the one before: each ends after the prefix part, and so after all of its own kind)
        for (int k = 0; k < pl.chunks; ++k) {
            own.row0 = k * kMaxRows; own.n_rows = B - own.row0 < kMaxRows ? B - own.row0 : kMaxRows;
            own.ml = reinterpret_cast<float2*>(ws + pl.own_ml) + k * pl.own_slots * kHeads;
            own.acc = reinterpret_cast<float*>(ws + pl.own_acc) + k * pl.own_slots * kHeads * pv.D;
            own.entries = reinterpret_cast<int4*>(ws + pl.entries) + (size_t)own.row0 * pv.H * pl.head_blocks;
            if (!launch(part, prefix_ctas(), kOwnWarps * 32, kOwnSmem, n_groups > 0 && k == 0, map, own)) return FPKV_ELAUNCH;
        }
        const int merge_grid = (pl.tiles * pv.H * (kPrefixTileRows / 32) + (B * Hq + 31) / 32) * (pv.D / 64);
        return launch(merge, merge_grid, 256, 0, true, mrg) ? FPKV_OK : FPKV_ELAUNCH;
    };
    if (pv.dtype == FPKV_BF16)
        return pv.D == 128 ? run(own_part_kernel<__nv_bfloat16, 128>, shared_merge_kernel<__nv_bfloat16, 128>)
                           : run(own_part_kernel<__nv_bfloat16, 64>, shared_merge_kernel<__nv_bfloat16, 64>);
    return pv.D == 128 ? run(own_part_kernel<__half, 128>, shared_merge_kernel<__half, 128>)
                       : run(own_part_kernel<__half, 64>, shared_merge_kernel<__half, 64>);
}

}  // namespace fpkv
