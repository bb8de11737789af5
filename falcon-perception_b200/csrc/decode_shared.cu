// Decode attention of a batch whose rows share long prefixes (16-bit pools, page_size 128).
//
// With keys 0 .. s-1 the same for every row of a group, the softmax over a row's keys splits into the prefix part and
// the row's own part, each with its own maximum m, sum l and unnormalised result a (all in 32 bits):
//     M = max(m1, m2),  l = l1 2^(m1-M) + l2 2^(m2-M),  out = (a1 2^(m1-M) + a2 2^(m2-M)) / l
// (scores in base 2).  The prefix part of all rows of a group is one product over the prefix's keys, so they are read
// once a group instead of once a row.  Three launches:
//
//  * prefix part: shared_prefix_tc.cu.
//  * own part, below: a CTA takes the query heads of one stored head of one batch row (up to 16, the M rows of
//    mma.sync.m16n8k16) and a share of the row's keys behind the prefix.  Its warps walk blocks of 16 keys; K and V go
//    from memory straight into the registers of the MMAs: the order of the contraction index and of the output columns is
//    free, so it is chosen such that every lane's 16-byte piece of a row is its own operand.  No shared memory, no barrier
//    in the loop.  Bound by the bytes of the rows' own keys.
//  * merge: joins the partials of every (row, head), applies the sink gate, writes out and lse.

#include "shared_prefix.cuh"

namespace fpkv {

namespace {

constexpr int kPage = 128;
constexpr int kMaxRep = 16;                    // query heads of a stored head: rows of the own part's MMAs
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
    int splits;
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

template <typename T, int D>
__global__ void __launch_bounds__(kPartWarps * 32)
own_part_kernel(const OwnParams prm)
{
    constexpr int NI = D / 32, NH = D / 64;    // 16-byte pieces of a K row per lane; 64-column groups of a V row
    const RowParams& rp = prm.rows;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    __shared__ int s_row[kListTiles];          // pool row of each resolved page, -1 = not visible
    __shared__ float s_m[kPartWarps][kMaxRep], s_l[kPartWarps][kMaxRep];
    __shared__ float s_acc[kPartWarps][kMaxRep][D + 4];

    const int split = blockIdx.x % prm.splits, h = (blockIdx.x / prm.splits) % rp.H, b0 = blockIdx.x / (prm.splits * rp.H);
    const int rows = rp.n_rep;
    int slot0; int4 d;
    const int hi_keys = row_keys(rp, b0, &slot0, h == 0 && split == 0 && threadIdx.x == 0);
    const int first_page = group_of_row(rp, b0, &d) >= 0 ? d.z : 0, end_page = (hi_keys + kPage - 1) / kPage;
    const int n_pg = max(0, end_page - first_page);
    const int pg0 = first_page + (int)((long long)n_pg * split / prm.splits), pg1 = first_page + (int)((long long)n_pg * (split + 1) / prm.splits);
    const int keys[2] = {hi_keys, hi_keys};

    // queries: rows g and g + 8 of the MMAs, dims i * 32 + c * 8 .. + 7
    uint4 qa[NI], qb[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        qa[i] = qb[i] = make_uint4(0, 0, 0, 0);
        const T* q = reinterpret_cast<const T*>(prm.q);
        if (g < rows) qa[i] = ld16(reinterpret_cast<const char*>(q + b0 * prm.q_stride_b + (h * rows + g) * prm.q_stride_h + i * 32 + c * 8));
        if (g + 8 < rows) qb[i] = ld16(reinterpret_cast<const char*>(q + b0 * prm.q_stride_b + (h * rows + g + 8) * prm.q_stride_h + i * 32 + c * 8));
    }
    float acc[NH][8][4];
#pragma unroll
    for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[a][e][k] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
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
            if (row0 < 0 || key0 >= hi_keys) continue;
            const size_t at = (size_t)(row0 + (k16 % (kPage / 16)) * 16);
            uint4 kk[2][NI], vv[4][NH];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < NI; ++i) kk[j][i] = ld16(kp + ((at + j * 8 + g) * D + i * 32 + c * 8) * 2);
#pragma unroll
            for (int k = 0; k < 4; ++k)        // keys 2c, 2c + 1, 2c + 8, 2c + 9 of the block
#pragma unroll
                for (int a = 0; a < NH; ++a) vv[k][a] = ld16(vp + ((at + 2 * c + (k & 1) + (k >> 1) * 8) * D + a * 64 + g * 8) * 2);
            float s[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const uint32_t a0[4] = {qa[i].x, qb[i].x, qa[i].y, qb[i].y}, a1[4] = {qa[i].z, qb[i].z, qa[i].w, qb[i].w};
                    mma16816<T>(s[j], a0, kk[j][i].x, kk[j][i].y);
                    mma16816<T>(s[j], a1, kk[j][i].z, kk[j][i].w);
                }
            }
            // keys past a row's end: no weight, and (never appended, perhaps) no value either
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = e >> 1, key = key0 + j * 8 + 2 * c + (e & 1);
                    s[j][e] = key < keys[r] ? s[j][e] * prm.scale_log2 : -INFINITY;
                    mx[r] = fmaxf(mx[r], s[j][e]);
                }
            if (key0 + 16 > hi_keys) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (key0 + 2 * c + (k & 1) + (k >> 1) * 8 >= hi_keys)
#pragma unroll
                        for (int a = 0; a < NH; ++a) vv[k][a] = make_uint4(0, 0, 0, 0);
            }
            float alpha[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const float mn = fmaxf(m[r], mx[r]);
                alpha[r] = m[r] == -INFINITY ? 0.f : exp2f(m[r] - mn);
                m[r] = mn;
                l[r] *= alpha[r];
            }
#pragma unroll
            for (int a = 0; a < NH; ++a)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    acc[a][e][0] *= alpha[0]; acc[a][e][1] *= alpha[0];
                    acc[a][e][2] *= alpha[1]; acc[a][e][3] *= alpha[1];
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = e >> 1;
                    s[j][e] = m[r] == -INFINITY ? 0.f : exp2f(s[j][e] - m[r]);
                    l[r] += s[j][e];
                }
            const uint32_t p[4] = {pack_pair<T>(s[0][0], s[0][1]), pack_pair<T>(s[0][2], s[0][3]),
                                   pack_pair<T>(s[1][0], s[1][1]), pack_pair<T>(s[1][2], s[1][3])};
#pragma unroll
            for (int a = 0; a < NH; ++a) {
                const uint32_t* x0 = &vv[0][a].x; const uint32_t* x1 = &vv[1][a].x;
                const uint32_t* x2 = &vv[2][a].x; const uint32_t* x3 = &vv[3][a].x;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
                    mma16816<T>(acc[a][e], p, __byte_perm(x0[e >> 1], x1[e >> 1], sel), __byte_perm(x2[e >> 1], x3[e >> 1], sel));
                }
            }
        }
    }
    // ---- join the warps, write the partial ------------------------------------------
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (c == 0) { s_m[warp][g + 8 * r] = m[r]; s_l[warp][g + 8 * r] = l[r]; }
    }
#pragma unroll
    for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) s_acc[warp][g + 8 * (k >> 1)][a * 64 + (2 * c + (k & 1)) * 8 + e] = acc[a][e][k];
    __syncthreads();
    for (int i = threadIdx.x; i < rows * D; i += kPartWarps * 32) {
        const int r = i / D, col = i % D;
        const size_t part = ((size_t)b0 * rp.Hq + h * rows + r) * prm.splits + split;
        float M = -INFINITY;
        for (int w = 0; w < kPartWarps; ++w) M = fmaxf(M, s_m[w][r]);
        float L = 0.f, o = 0.f;
        for (int w = 0; w < kPartWarps; ++w)
            if (s_m[w][r] != -INFINITY) { const float f = exp2f(s_m[w][r] - M); L += s_l[w][r] * f; o += s_acc[w][r][col] * f; }
        prm.acc[part * D + col] = o;
        if (col == 0) prm.ml[part] = make_float2(M, L);
    }
}

// Columns [4 * col4, +4 * N) of one (row, head): the weighted sum of its partials.
template <int N> struct Sum {
    float a[4 * N], L, M;
    __device__ __forceinline__ void add(float w, const float4* src, size_t step) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float4 v = src[k * step];
            a[4 * k] += w * v.x; a[4 * k + 1] += w * v.y; a[4 * k + 2] += w * v.z; a[4 * k + 3] += w * v.w;
        }
    }
};

// Block: 32 query rows of a query tile (one stored head), a row a lane, the columns dealt out to the warps; behind those one
// block for each batch row that is in no group.
template <typename T, int D>
__global__ void __launch_bounds__(128)
shared_merge_kernel(const MergeParams prm)
{
    constexpr int N = D / 16;                  // column groups of four a warp (a block has four warps)
    const RowParams& rp = prm.rows;
    __shared__ long long flat_before[FPKV_MAX_GROUPS + 1];
    __shared__ int mt_before[FPKV_MAX_GROUPS + 1];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int tile_blocks = prm.tiles * rp.H * (kPrefixTileRows / 32);
    int b, hq, c0 = 0, c1 = -1, index = 0, trow = 0;
    if ((int)blockIdx.x < tile_blocks) {
        if (warp == 0) prefix_schedule(rp, flat_before, mt_before, lane);
        __syncthreads();
        const int quarter = blockIdx.x % (kPrefixTileRows / 32), seg0 = blockIdx.x / (kPrefixTileRows / 32);
        if (seg0 >= mt_before[rp.n_groups] * rp.H) return;
        int lo = 0, hi = rp.n_groups;          // the group whose segments (query tiles times stored heads) hold this one
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (mt_before[mid] * rp.H <= seg0) lo = mid; else hi = mid; }
        const int4 d = group_at(rp, lo);
        const Segment sg = segment_at(rp, flat_before, mt_before, flat_before[lo] + (long long)(seg0 - mt_before[lo] * rp.H) * d.z);
        trow = quarter * 32 + lane;
        if (quarter * 32 >= sg.rows) return;
        const long long total = flat_before[rp.n_groups], first = flat_before[lo] + (long long)(seg0 - mt_before[lo] * rp.H) * d.z;
        const int ctas = sharers(total, prm.ctas);
        c0 = share_of(total, first, ctas); c1 = share_of(total, first + d.z - 1, ctas);
        index = sg.index;
        b = sg.b0 + trow / rp.n_rep; hq = sg.h * rp.n_rep + trow % rp.n_rep;
        int4 mine;
        // a row of the tile that does not name the group has all its keys in its own part
        if (trow >= sg.rows) b = -1;
        else if (group_of_row(rp, b, &mine) != lo) b = -1;
    } else {
        const int i = (blockIdx.x - tile_blocks) * 32 + lane;
        b = i / rp.Hq; hq = i % rp.Hq;
        int4 mine;
        if (b >= rp.B || group_of_row(rp, b, &mine) >= 0) b = -1;
    }
    if (b < 0) return;
    const size_t row = (size_t)b * rp.Hq + hq, own = row * prm.splits;
    Sum<N> s;
    s.M = -INFINITY; s.L = 0.f;
#pragma unroll
    for (int k = 0; k < 4 * N; ++k) s.a[k] = 0.f;
    for (int c = c0; c <= c1; ++c) s.M = fmaxf(s.M, prm.pre_ml[(size_t)(c + index) * kPrefixTileRows + trow].x);
    for (int k = 0; k < prm.splits; ++k) s.M = fmaxf(s.M, prm.own_ml[own + k].x);
    for (int c = c0; c <= c1; ++c) {
        const float2 ml = prm.pre_ml[(size_t)(c + index) * kPrefixTileRows + trow];
        if (ml.y == 0.f) continue;             // nothing visible: no sums were written
        const float w = exp2f(ml.x - s.M);
        s.L += ml.y * w;
        s.add(w, reinterpret_cast<const float4*>(prm.pre_acc) + ((size_t)(c + index) * (D / 4) + warp * N) * kPrefixTileRows + trow, kPrefixTileRows);
    }
    for (int k = 0; k < prm.splits; ++k) {
        const float2 ml = prm.own_ml[own + k];
        if (ml.y == 0.f) continue;
        const float w = exp2f(ml.x - s.M);
        s.L += ml.y * w;
        s.add(w, reinterpret_cast<const float4*>(prm.own_acc) + (own + k) * (D / 4) + warp * N, 1);
    }
    const float lse = s.L == 0.f ? -INFINITY : (s.M + log2f(s.L)) * kLn2;
    const float gate = sink_gate(prm.epi, hq, lse), inv = s.L == 0.f ? 0.f : 1.f / s.L;
    T o[4 * N];
#pragma unroll
    for (int k = 0; k < 4 * N; ++k) o[k] = gated_out<T>(s.a[k] * inv, gate, prm.epi.sinks != nullptr);
    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(prm.out) + row * D + warp * 4 * N);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) dst[k] = reinterpret_cast<const uint4*>(o)[k];
    if (warp == 0) prm.lse[row] = lse;
}

struct Plan { int n_rep, rows_per_tile, tiles, splits; size_t slots, pre_ml, pre_acc, own_ml, own_acc, bytes; };
Plan plan_of(const PoolView& pv, int B, int Hq, int n_groups)
{
    Plan p;
    p.n_rep = Hq / pv.H;
    p.rows_per_tile = kPrefixTileRows / p.n_rep;
    // a group leaves at most one tile that is not full
    p.tiles = n_groups > 0 ? B / p.rows_per_tile + (n_groups < B ? n_groups : B) : 0;
    // Own part: four CTAs an SM when there are few rows.
    p.splits = 4 * 148 / (B * pv.H > 0 ? B * pv.H : 1);
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
    own.q_stride_b = qsb; own.q_stride_h = qsh; own.splits = pl.splits; own.scale_log2 = sm_scale * kLog2e;
    MergeParams mrg;
    mrg.rows = rows; mrg.pre_ml = reinterpret_cast<float2*>(ws + pl.pre_ml); mrg.pre_acc = reinterpret_cast<float*>(ws + pl.pre_acc);
    mrg.own_ml = own.ml; mrg.own_acc = own.acc; mrg.splits = pl.splits; mrg.ctas = prefix_ctas(); mrg.tiles = pl.tiles;
    mrg.out = out; mrg.lse = lse; mrg.epi = epi;
    auto run = [&](auto part, auto merge) {
        part<<<B * pv.H * pl.splits, kPartWarps * 32, 0, stream>>>(own);
        if (cudaGetLastError() != cudaSuccess) return FPKV_ELAUNCH;
        merge<<<pl.tiles * pv.H * (kPrefixTileRows / 32) + (B * Hq + 31) / 32, 128, 0, stream>>>(mrg);
        return cudaGetLastError() == cudaSuccess ? FPKV_OK : FPKV_ELAUNCH;
    };
    if (pv.dtype == FPKV_BF16)
        return pv.D == 128 ? run(own_part_kernel<__nv_bfloat16, 128>, shared_merge_kernel<__nv_bfloat16, 128>)
                           : run(own_part_kernel<__nv_bfloat16, 64>, shared_merge_kernel<__nv_bfloat16, 64>);
    return pv.D == 128 ? run(own_part_kernel<__half, 128>, shared_merge_kernel<__half, 128>)
                       : run(own_part_kernel<__half, 64>, shared_merge_kernel<__half, 64>);
}

}  // namespace fpkv
