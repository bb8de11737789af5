// Decode attention of a batch whose rows share long prefixes (16-bit pools, page_size 128).
//
// With keys 0 .. s-1 the same for every row of a group, the softmax over a row's keys splits into the prefix part and
// the row's own part, each with its own maximum m, sum l and unnormalised result a (all in 32 bits):
//     M = max(m1, m2),  l = l1 2^(m1-M) + l2 2^(m2-M),  out = (a1 2^(m1-M) + a2 2^(m2-M)) / l
// (scores in base 2).  The prefix part of all rows of a group is one product over the prefix's keys, so they are read
// once a group instead of once a row.  Three launches:
//
//  * prefix part: shared_prefix_tc.cu.
//  * own part, below: a CTA takes up to 8 query heads of one stored head of one batch row and a share of the row's keys
//    behind the prefix.  Its warps walk blocks of 16 keys with mma.sync.m16n8k16,
//        S^T = K Q^T   (16 keys x 8 heads),   O^T += V^T P^T   (dims x 8 heads)
//    and K and V go from memory straight into the registers of the MMAs: the order of the contraction index and of the
//    output's dims is free, so it is chosen such that every lane's 16-byte piece of a row is its own operand.  No shared
//    memory and no barrier in the loop; 16 warps an SM keep 128 KB of loads in flight.  Bound by the bytes of the rows' own
//    keys.
//  * merge: joins the partials of every (row, head), applies the sink gate, writes out and lse.
// The three are chained by programmatic dependent launch: the own part starts as soon as every CTA of the prefix part has
// (it needs nothing from it) and fills the SMs as they come free; it ends after the prefix part, so that the merge, whose
// set-up overlaps both, has only the own part to wait for.

#include "shared_prefix.cuh"

namespace fpkv {

namespace {

constexpr int kPage = 128;
constexpr int kMaxRep = 16;                    // query heads of a stored head
constexpr int kHeads = 8;                      // of them, those of a CTA of the own part: the MMAs' columns
constexpr int kPartWarps = 4;
constexpr int kListTiles = 64;                 // pages resolved at a time

struct OwnParams {
    RowParams rows;
    const char* k;                             // K plane of stored head 0
    const char* v;
    size_t plane_bytes;
    const void* q;
    float2* ml;                                // partials [B][Hq][splits] (m, l)
    float* acc;                                // [B][Hq][splits][D]
    long long q_stride_b, q_stride_h;
    int splits, head_blocks;                   // shares of a row's keys; blocks of kHeads query heads of a stored head
    float scale_log2;
};

struct MergeParams {
    RowParams rows;
    const float2* pre_ml; const float* pre_acc;
    const float2* own_ml; const float* own_acc;
    int splits, ctas, tiles;                   // of the own part; of the prefix part; upper bound of its query tiles
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

template <typename T, int D>
__global__ void __launch_bounds__(kPartWarps * 32, 4)
own_part_kernel(const OwnParams prm)
{
    constexpr int NI = D / 32, NH = D / 64;    // 16-byte pieces of a K row per lane; 64-column groups of a V row
    const RowParams& rp = prm.rows;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    __shared__ int s_row[kListTiles];          // pool row of each resolved page, -1 = not visible
    __shared__ float s_m[kPartWarps][kHeads], s_l[kPartWarps][kHeads];
    __shared__ __align__(16) float s_acc[kPartWarps][kHeads][D + 4];
    asm volatile("griddepcontrol.launch_dependents;");       // the merge may take its seats

    int id = blockIdx.x;
    const int split = id % prm.splits; id /= prm.splits;
    const int r0 = (id % prm.head_blocks) * kHeads; id /= prm.head_blocks;
    const int h = id % rp.H, b0 = id / rp.H;
    const int heads = min(kHeads, rp.n_rep - r0);
    int slot0; int4 d;
    const int keys = row_keys(rp, b0, &slot0, h == 0 && split == 0 && r0 == 0 && threadIdx.x == 0);
    const int first_page = group_of_row(rp, b0, &d) >= 0 ? d.z : 0, end_page = (keys + kPage - 1) / kPage;
    const int n_pg = max(0, end_page - first_page);
    const int pg0 = first_page + (int)((long long)n_pg * split / prm.splits), pg1 = first_page + (int)((long long)n_pg * (split + 1) / prm.splits);

    // queries: head g, dims i * 32 + c * 8 .. + 7
    uint4 qa[NI];
    const T* q = reinterpret_cast<const T*>(prm.q) + b0 * prm.q_stride_b + (h * rp.n_rep + r0 + g) * prm.q_stride_h;
#pragma unroll
    for (int i = 0; i < NI; ++i) qa[i] = g < heads ? ld16(reinterpret_cast<const char*>(q + i * 32 + c * 8)) : make_uint4(0, 0, 0, 0);
    float acc[NH][4][4];                       // O^T: rows dims a * 64 + g * 8 + 2 e (+ 1), columns heads 2 c and 2 c + 1
#pragma unroll
    for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[a][e][k] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // heads 2 c and 2 c + 1; l this lane's keys alone
    const char* kp = prm.k + (size_t)h * prm.plane_bytes;
    const char* vp = prm.v + (size_t)h * prm.plane_bytes;

    for (int p0 = pg0; p0 < pg1; p0 += kListTiles) {
        __syncthreads();
        for (int j = threadIdx.x; j < min(kListTiles, pg1 - p0); j += kPartWarps * 32) {
            const long long pg = rp.page_table[(long long)slot0 * rp.n_pages + p0 + j];
            int row = -1;
            if (pg >= rp.n_pages) raise_status(rp.status, FPKV_STATUS_BAD_PAGE);
            else if (pg >= 0 && rp.p2l[(long long)slot0 * rp.n_pages + pg] >= 0) row = (int)pg * kPage;
            s_row[j] = row;
        }
        __syncthreads();
        const int blocks = min(kListTiles, pg1 - p0) * (kPage / 16);
        for (int k16 = warp; k16 < blocks; k16 += kPartWarps) {
            const int row0 = s_row[k16 / (kPage / 16)];
            const int key0 = p0 * kPage + k16 * 16;
            if (row0 < 0 || key0 >= keys) continue;
            const size_t at = (size_t)(row0 + (k16 % (kPage / 16)) * 16);
            uint4 kk[2][NI], vv[4][NH];
#pragma unroll
            for (int j = 0; j < 2; ++j)        // keys g and g + 8 of the block
#pragma unroll
                for (int i = 0; i < NI; ++i) kk[j][i] = ld16(kp + ((at + j * 8 + g) * D + i * 32 + c * 8) * 2);
#pragma unroll
            for (int k = 0; k < 4; ++k)        // keys 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
                for (int a = 0; a < NH; ++a) vv[k][a] = ld16(vp + ((at + 2 * c + (k & 1) + (k >> 1) * 8) * D + a * 64 + g * 8) * 2);
            float s[4] = {0.f, 0.f, 0.f, 0.f}; // S^T: keys g (0, 1) and g + 8 (2, 3), heads 2 c and 2 c + 1
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const uint32_t a0[4] = {kk[0][i].x, kk[1][i].x, kk[0][i].y, kk[1][i].y}, a1[4] = {kk[0][i].z, kk[1][i].z, kk[0][i].w, kk[1][i].w};
                mma16816<T>(s, a0, qa[i].x, qa[i].y);
                mma16816<T>(s, a1, qa[i].z, qa[i].w);
            }
            // keys past the row's end: no weight, and (never appended, perhaps) no value either
            float mx[2];
            if (key0 + 16 > keys) {
#pragma unroll
                for (int e = 0; e < 4; ++e) if (key0 + g + (e >> 1) * 8 >= keys) s[e] = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (key0 + 2 * c + (k & 1) + (k >> 1) * 8 >= keys)
#pragma unroll
                        for (int a = 0; a < NH; ++a) vv[k][a] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(s[r], s[2 + r]);                             // the scale is positive: the maximum commutes with it
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
            const uint32_t b0_ = transposed(pack_pair<T>(s[0], s[1])), b1_ = transposed(pack_pair<T>(s[2], s[3]));
#pragma unroll
            for (int a = 0; a < NH; ++a) {
                const uint32_t* x0 = &vv[0][a].x; const uint32_t* x1 = &vv[1][a].x;
                const uint32_t* x2 = &vv[2][a].x; const uint32_t* x3 = &vv[3][a].x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t at_[4] = {__byte_perm(x0[e], x1[e], 0x5410u), __byte_perm(x0[e], x1[e], 0x7632u),
                                             __byte_perm(x2[e], x3[e], 0x5410u), __byte_perm(x2[e], x3[e], 0x7632u)};
                    mma16816<T>(acc[a][e], at_, b0_, b1_);
                }
            }
        }
    }
    // ---- join the warps, write the partial ------------------------------------------
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
        if (g == 0) { s_m[warp][2 * c + r] = m[r]; s_l[warp][2 * c + r] = l[r]; }
    }
#pragma unroll
    for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) s_acc[warp][2 * c + (k & 1)][a * 64 + g * 8 + 2 * e + (k >> 1)] = acc[a][e][k];
    __syncthreads();
    for (int i = threadIdx.x; i < heads * (D / 4); i += kPartWarps * 32) {
        const int r = i / (D / 4), col = i % (D / 4) * 4;
        const size_t part = ((size_t)b0 * rp.Hq + h * rp.n_rep + r0 + r) * prm.splits + split;
        float M = -INFINITY;
        for (int w = 0; w < kPartWarps; ++w) M = fmaxf(M, s_m[w][r]);
        float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < kPartWarps; ++w) {
            if (s_m[w][r] == -INFINITY) continue;
            const float f = exp2f(s_m[w][r] - M);
            const float4 v = *reinterpret_cast<const float4*>(&s_acc[w][r][col]);
            L += s_l[w][r] * f;
            o[0] += v.x * f; o[1] += v.y * f; o[2] += v.z * f; o[3] += v.w * f;
        }
        *reinterpret_cast<float4*>(prm.acc + part * D + col) = make_float4(o[0], o[1], o[2], o[3]);
        if (col == 0) prm.ml[part] = make_float2(M, L);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");       // not done before the prefix part is
}

// Block: 32 (row, head) pairs, one a lane, and 32 columns, eight a warp.  The pairs are a quarter of a query tile of the
// prefix part, whose partials lie side by side; behind those blocks come some for the rows that are in no group.  The
// weights of all partials are worked out first, in parallel, so that the loads of the sums do not wait for one another.
constexpr int kMergePieces = 32;

template <typename T, int D>
__global__ void __launch_bounds__(128)
shared_merge_kernel(const MergeParams prm)
{
    constexpr int kColBlocks = D / 32;
    const RowParams& rp = prm.rows;
    __shared__ long long flat_before[FPKV_MAX_GROUPS + 1];
    __shared__ int mt_before[FPKV_MAX_GROUPS + 1];
    __shared__ float2 s_ml[kMergePieces][32];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int col4 = (blockIdx.x % kColBlocks) * 8 + warp * 2, block = blockIdx.x / kColBlocks;
    const int tile_blocks = prm.tiles * rp.H * (kPrefixTileRows / 32);
    int b = -1, hq = 0, c0 = 0, n_pre = 0, index = 0, trow = 0;
    if (block < tile_blocks) {
        if (warp == 0) prefix_schedule(rp, flat_before, mt_before, lane);
        __syncthreads();
        const int quarter = block % (kPrefixTileRows / 32), seg0 = block / (kPrefixTileRows / 32);
        if (seg0 >= mt_before[rp.n_groups] * rp.H) return;
        int lo = 0, hi = rp.n_groups;          // the group whose segments (query tiles times stored heads) hold this one
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (mt_before[mid] * rp.H <= seg0) lo = mid; else hi = mid; }
        const int4 d = group_at(rp, lo);
        const long long total = flat_before[rp.n_groups], first = flat_before[lo] + (long long)(seg0 - mt_before[lo] * rp.H) * d.z;
        const Segment sg = segment_at(rp, flat_before, mt_before, first);
        trow = quarter * 32 + lane;
        if (quarter * 32 >= sg.rows) return;
        const int ctas = sharers(total, prm.ctas);
        c0 = share_of(total, first, ctas);
        n_pre = share_of(total, first + d.z - 1, ctas) - c0 + 1;
        index = sg.index;
        hq = sg.h * rp.n_rep + trow % rp.n_rep;
        int4 mine;
        // (a row of the tile that does not name the group has all its keys in its own part)
        if (trow < sg.rows && group_of_row(rp, sg.b0 + trow / rp.n_rep, &mine) == lo) b = sg.b0 + trow / rp.n_rep;
    } else {
        const int i = (block - tile_blocks) * 32 + lane;
        int4 mine;
        if (i < rp.B * rp.Hq && group_of_row(rp, i / rp.Hq, &mine) < 0) { b = i / rp.Hq; hq = i % rp.Hq; }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (__ballot_sync(0xffffffffu, b >= 0) == 0) return;     // the same for all warps
    const size_t row = (size_t)max(b, 0) * rp.Hq + hq, own = row * prm.splits;
    const int n = n_pre + prm.splits;
    float M = -INFINITY, L = 0.f, a[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = 0.f;
    for (int p0 = 0; p0 < n; p0 += kMergePieces) {
        const int here = min(kMergePieces, n - p0);
        __syncthreads();
#pragma unroll 8
        for (int p = warp; p < here; p += 4) {
            const int i = p0 + p;
            s_ml[p][lane] = b < 0 ? make_float2(-INFINITY, 0.f)
                                  : i < n_pre ? prm.pre_ml[(size_t)(c0 + i + index) * kPrefixTileRows + trow] : prm.own_ml[own + i - n_pre];
        }
        __syncthreads();
        float mn = M;
        for (int p = 0; p < here; ++p) mn = fmaxf(mn, s_ml[p][lane].x);
        const float alpha = M == -INFINITY ? 0.f : exp2f(M - mn);
        M = mn;
        L *= alpha;
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] *= alpha;
#pragma unroll 8
        for (int p = 0; p < here; ++p) {
            const float2 ml = s_ml[p][lane];
            const int i = p0 + p;
            const float4* src = i < n_pre ? reinterpret_cast<const float4*>(prm.pre_acc) + ((size_t)(c0 + i + index) * (D / 4) + col4) * kPrefixTileRows + trow
                                          : reinterpret_cast<const float4*>(prm.own_acc) + (own + i - n_pre) * (D / 4) + col4;
            const size_t step = i < n_pre ? kPrefixTileRows : 1;
            const bool some = ml.y != 0.f;                   // nothing visible: no sums were written
            const float4 x = some ? src[0] : make_float4(0.f, 0.f, 0.f, 0.f), y = some ? src[step] : make_float4(0.f, 0.f, 0.f, 0.f);
            const float w = some ? exp2f(ml.x - M) : 0.f;
            L += ml.y * w;
            a[0] += w * x.x; a[1] += w * x.y; a[2] += w * x.z; a[3] += w * x.w;
            a[4] += w * y.x; a[5] += w * y.y; a[6] += w * y.z; a[7] += w * y.w;
        }
    }
    if (b < 0) return;
    const float lse = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    const float gate = sink_gate(prm.epi, hq, lse), inv = L == 0.f ? 0.f : 1.f / L;
    __align__(16) T o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = gated_out<T>(a[k] * inv, gate, prm.epi.sinks != nullptr);
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(prm.out) + row * D + col4 * 4) = *reinterpret_cast<const uint4*>(o);
    if (col4 == 0) prm.lse[row] = lse;
}

struct Plan { int n_rep, rows_per_tile, tiles, splits, head_blocks; size_t slots, pre_ml, pre_acc, own_ml, own_acc, bytes; };
Plan plan_of(const PoolView& pv, int B, int Hq, int n_groups)
{
    Plan p;
    p.n_rep = Hq / pv.H;
    p.rows_per_tile = kPrefixTileRows / p.n_rep;
    // a group leaves at most one tile that is not full
    p.tiles = n_groups > 0 ? B / p.rows_per_tile + (n_groups < B ? n_groups : B) : 0;
    p.head_blocks = (p.n_rep + kHeads - 1) / kHeads;
    // Own part: four CTAs an SM when there are few rows.
    p.splits = 4 * 148 / (B * pv.H > 0 ? B * pv.H * p.head_blocks : 1);
    p.splits = p.splits < 1 ? 1 : p.splits > 32 ? 32 : p.splits;
    p.slots = p.tiles > 0 ? (size_t)p.tiles * pv.H + prefix_ctas() : 0;
    auto place = [at = (size_t)0](size_t n) mutable { const size_t was = at; at += (n + 255) / 256 * 256; return was; };
    p.pre_ml = place(p.slots * kPrefixTileRows * sizeof(float2));
    p.pre_acc = place(p.slots * kPrefixTileRows * pv.D * sizeof(float));
    p.own_ml = place((size_t)B * Hq * p.splits * sizeof(float2));
    p.own_acc = place((size_t)B * Hq * p.splits * pv.D * sizeof(float));
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
        pre.rows_per_plane = 0; pre.q_box_rows = 0; pre.scale_log2 = sm_scale * kLog2e;
        const int rc = launch_prefix(pv, layer, q, qsb, qsh, pre, stream);
        if (rc) return rc;
    }
    OwnParams own;
    own.rows = rows; own.k = pv.plane(layer, 0, 0); own.v = pv.plane(layer, 1, 0); own.plane_bytes = pv.plane_bytes(); own.q = q;
    own.ml = reinterpret_cast<float2*>(ws + pl.own_ml); own.acc = reinterpret_cast<float*>(ws + pl.own_acc);
    own.q_stride_b = qsb; own.q_stride_h = qsh; own.splits = pl.splits; own.head_blocks = pl.head_blocks; own.scale_log2 = sm_scale * kLog2e;
    MergeParams mrg;
    mrg.rows = rows; mrg.pre_ml = reinterpret_cast<float2*>(ws + pl.pre_ml); mrg.pre_acc = reinterpret_cast<float*>(ws + pl.pre_acc);
    mrg.own_ml = own.ml; mrg.own_acc = own.acc; mrg.splits = pl.splits; mrg.ctas = prefix_ctas(); mrg.tiles = pl.tiles;
    mrg.out = out; mrg.lse = lse; mrg.epi = epi;
    auto launch = [&](auto kern, int grid, bool chained, const auto& args) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3(128); cfg.stream = stream;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr; cfg.numAttrs = chained ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, kern, args) == cudaSuccess;
    };
    static_assert(kPartWarps * 32 == 128, "both kernels run blocks of 128 threads");
    auto run = [&](auto part, auto merge) {
        const int merge_grid = (pl.tiles * pv.H * (kPrefixTileRows / 32) + (B * Hq + 31) / 32) * (pv.D / 32);
        return launch(part, B * pv.H * pl.head_blocks * pl.splits, n_groups > 0, own) && launch(merge, merge_grid, true, mrg) ? FPKV_OK : FPKV_ELAUNCH;
    };
    if (pv.dtype == FPKV_BF16)
        return pv.D == 128 ? run(own_part_kernel<__nv_bfloat16, 128>, shared_merge_kernel<__nv_bfloat16, 128>)
                           : run(own_part_kernel<__nv_bfloat16, 64>, shared_merge_kernel<__nv_bfloat16, 64>);
    return pv.D == 128 ? run(own_part_kernel<__half, 128>, shared_merge_kernel<__half, 128>)
                       : run(own_part_kernel<__half, 64>, shared_merge_kernel<__half, 64>);
}

}  // namespace fpkv
