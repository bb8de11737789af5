// Decode attention of a batch whose rows share long prefixes (16-bit pools, page_size 128).
//
// With keys 0 .. s-1 the same for every row of a group, the softmax over a row's keys splits into the prefix part and
// the row's own part, each with its own maximum m, sum l and unnormalised result a (all in 32 bits):
//     M = max(m1, m2),  l = l1 2^(m1-M) + l2 2^(m2-M),  out = (a1 2^(m1-M) + a2 2^(m2-M)) / l
// (scores in base 2).  The prefix part of all rows of a group is one pass over the prefix's keys, so they are read
// once a group instead of once a row.
//
//  * partial kernel: a CTA takes a tile of up to 16 query rows of one stored head -- the GQA group of one batch row over
//    that row's own keys, or the GQA groups of several rows over their common prefix -- and a share of the keys.  Its
//    warps walk blocks of 16 keys; K and V go from memory straight into the registers of mma.sync.m16n8k16: the order of
//    the contraction index and of the output columns is free, so it is chosen such that every lane's 16-byte piece of a
//    row is its own operand.  No shared memory, no barrier in the loop.
//  * merge kernel: joins the partials of every (row, head), applies the sink gate, writes out and lse.

#include "common.cuh"

namespace fpkv {

namespace {

constexpr int kPage = 128;
constexpr int kTileRows = 16;                  // query rows of a partial
constexpr int kPartWarps = 4;
constexpr int kListTiles = 64;                 // pages resolved at a time

struct SharedParams {
    const char* k;                             // K plane of stored head 0
    const char* v;
    size_t plane_bytes;
    const int64_t* page_table;
    const int64_t* p2l;
    const int64_t* batch_idx;
    const void* pos;
    const void* q;
    const int4* groups;                        // {first row, rows, shared pages, 0}
    const int* row_group;
    void* out;
    float* lse;
    float* ws;                                 // partials [part][16 rows][D + 2]: m, l, a[D]
    int32_t* status;
    long long q_stride_b, q_stride_h;
    int B, Hq, H, n_rep, rows_per_tile, n_groups, n_pages, max_batch, pos_is_64;
    int prefix_tiles, prefix_splits, own_splits;        // grid: prefix_tiles * H * prefix_splits, then B * H * own_splits
    float scale_log2;
    Epilogue epi;
};

__device__ __forceinline__ long long pos_of(const SharedParams& p, int b) {
    return p.pos_is_64 ? reinterpret_cast<const int64_t*>(p.pos)[b] : (long long)reinterpret_cast<const int32_t*>(p.pos)[b];
}
// Slot and visible keys of a row; a slot or position out of range gives no keys.
__device__ __forceinline__ int row_keys(const SharedParams& p, int b, int* slot, bool report) {
    const long long s = p.batch_idx[b], at = pos_of(p, b);
    *slot = 0;
    if (s < 0 || s >= p.max_batch) { if (report) raise_status(p.status, FPKV_STATUS_BAD_SLOT); return 0; }
    if (at < 0 || at / kPage >= p.n_pages) { if (report) raise_status(p.status, FPKV_STATUS_BAD_POS); return 0; }
    *slot = (int)s;
    return (int)at + 1;
}
// A group as the kernels use it: rows and pages inside the batch and the table, or nothing.
__device__ __forceinline__ int4 group_at(const SharedParams& p, int g) {
    int4 d = p.groups[g];
    if (d.x < 0 || d.y <= 0 || d.x >= p.B || d.y > p.B - d.x || d.z <= 0) d.y = d.z = 0;
    d.z = min(d.z, p.n_pages);
    return d;
}
__device__ __forceinline__ int tiles_of(const SharedParams& p, const int4& d) { return (d.y + p.rows_per_tile - 1) / p.rows_per_tile; }
// Group of a row (or -1) and, when asked for, the row's tile number over all groups.
__device__ __forceinline__ int group_of_row(const SharedParams& p, int b, int4* d) {
    const int g = p.n_groups > 0 ? p.row_group[b] : -1;
    if (g < 0 || g >= p.n_groups) return -1;
    *d = group_at(p, g);
    return (d->y > 0 && b >= d->x && b < d->x + d->y) ? g : -1;
}

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
shared_partial_kernel(const SharedParams prm)
{
    constexpr int NI = D / 32, NH = D / 64;    // 16-byte pieces of a K row per lane; 64-column groups of a V row
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    __shared__ int s_row[kListTiles];          // pool row of each resolved page, -1 = not visible
    __shared__ float s_m[kPartWarps][kTileRows], s_l[kPartWarps][kTileRows];
    __shared__ float s_acc[kPartWarps][kTileRows][D + 4];

    // ---- which tile, which keys ---------------------------------------------------
    const int n_prefix = prm.prefix_tiles * prm.H * prm.prefix_splits;
    const int id = blockIdx.x;
    int h, b0, nb, split, splits, first_page, end_page;
    if (id < n_prefix) {
        split = id % prm.prefix_splits; splits = prm.prefix_splits;
        h = (id / prm.prefix_splits) % prm.H;
        int t = id / (prm.prefix_splits * prm.H);
        int gr = 0; int4 d = make_int4(0, 0, 0, 0);
        for (; gr < prm.n_groups; ++gr) {      // tile t of all groups' tiles
            d = group_at(prm, gr);
            const int n = tiles_of(prm, d);
            if (t < n) break;
            t -= n;
        }
        if (gr == prm.n_groups) return;
        b0 = d.x + t * prm.rows_per_tile;
        nb = min(prm.rows_per_tile, d.x + d.y - b0);
        first_page = 0; end_page = d.z;
    } else {
        const int k = id - n_prefix;
        split = k % prm.own_splits; splits = prm.own_splits;
        h = (k / prm.own_splits) % prm.H;
        b0 = k / (prm.own_splits * prm.H); nb = 1;
        int4 d;
        first_page = group_of_row(prm, b0, &d) >= 0 ? d.z : 0;
        end_page = prm.n_pages;
    }
    // the rows of this tile: lane's rows g and g + 8
    int keys[2], hi_keys = 0, slot0 = 0;
    for (int r = 0; r < nb; ++r) {
        int s; const int n = row_keys(prm, b0 + r, &s, h == 0 && split == 0 && threadIdx.x == 0 && id >= n_prefix);
        if (r == 0) slot0 = s;
        hi_keys = max(hi_keys, n);
    }
    const int rows = nb * prm.n_rep;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = g + 8 * r;
        int s;
        keys[r] = row < rows ? row_keys(prm, b0 + row / prm.n_rep, &s, false) : 0;
    }
    {   // the prefix is read through the first row's slot; a first row out of range leaves the group to no one
        long long s = prm.batch_idx[b0];
        slot0 = (s >= 0 && s < prm.max_batch) ? (int)s : 0;
    }
    end_page = min(end_page, (hi_keys + kPage - 1) / kPage);
    const int n_pg = max(0, end_page - first_page);
    const int pg0 = first_page + (int)((long long)n_pg * split / splits), pg1 = first_page + (int)((long long)n_pg * (split + 1) / splits);
    const int lim = id < n_prefix ? end_page * kPage : 0x7fffffff;      // keys past the shared pages are the own part's
    keys[0] = min(keys[0], lim); keys[1] = min(keys[1], lim);

    // ---- queries: row g and row g + 8, dims i * 32 + c * 8 .. + 7 --------------------------
    uint4 qa[NI], qb[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        qa[i] = qb[i] = make_uint4(0, 0, 0, 0);
        const T* q = reinterpret_cast<const T*>(prm.q);
        if (g < rows) qa[i] = ld16(reinterpret_cast<const char*>(q + (b0 + g / prm.n_rep) * prm.q_stride_b + (h * prm.n_rep + g % prm.n_rep) * prm.q_stride_h + i * 32 + c * 8));
        if (g + 8 < rows) qb[i] = ld16(reinterpret_cast<const char*>(q + (b0 + (g + 8) / prm.n_rep) * prm.q_stride_b + (h * prm.n_rep + (g + 8) % prm.n_rep) * prm.q_stride_h + i * 32 + c * 8));
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
            const long long pg = prm.page_table[(long long)slot0 * prm.n_pages + p0 + j];
            int row = -1;
            if (pg >= prm.n_pages) raise_status(prm.status, FPKV_STATUS_BAD_PAGE);
            else if (pg >= 0 && prm.p2l[(long long)slot0 * prm.n_pages + pg] >= 0) row = (int)pg * kPage;
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
    float* dst = prm.ws + (size_t)id * kTileRows * (D + 2);
    for (int i = threadIdx.x; i < rows * D; i += kPartWarps * 32) {
        const int r = i / D, d = i % D;
        float M = -INFINITY;
        for (int w = 0; w < kPartWarps; ++w) M = fmaxf(M, s_m[w][r]);
        float L = 0.f, o = 0.f;
        for (int w = 0; w < kPartWarps; ++w)
            if (s_m[w][r] != -INFINITY) { const float f = exp2f(s_m[w][r] - M); L += s_l[w][r] * f; o += s_acc[w][r][d] * f; }
        dst[r * (D + 2) + 2 + d] = o;
        if (d == 0) { dst[r * (D + 2)] = M; dst[r * (D + 2) + 1] = L; }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(D)
shared_merge_kernel(const SharedParams prm)
{
    const int b = blockIdx.x / prm.Hq, hq = blockIdx.x % prm.Hq, h = hq / prm.n_rep, rep = hq % prm.n_rep, d = threadIdx.x;
    const int n_prefix = prm.prefix_tiles * prm.H * prm.prefix_splits;
    const float* own = prm.ws + ((size_t)n_prefix + ((size_t)b * prm.H + h) * prm.own_splits) * kTileRows * (D + 2) + (size_t)rep * (D + 2);
    const float* pre = nullptr;
    int4 gd;
    const int g = group_of_row(prm, b, &gd);
    if (g >= 0) {
        int t = 0;
        for (int i = 0; i < g; ++i) { const int4 o = group_at(prm, i); t += tiles_of(prm, o); }
        const int in = b - gd.x;
        t += in / prm.rows_per_tile;
        pre = prm.ws + ((size_t)t * prm.H + h) * prm.prefix_splits * kTileRows * (D + 2) +
              (size_t)((in % prm.rows_per_tile) * prm.n_rep + rep) * (D + 2);
    }
    const size_t step = (size_t)kTileRows * (D + 2);
    float M = -INFINITY;
    for (int s = 0; s < prm.own_splits; ++s) M = fmaxf(M, own[s * step]);
    if (pre != nullptr) for (int s = 0; s < prm.prefix_splits; ++s) M = fmaxf(M, pre[s * step]);
    float L = 0.f, o = 0.f;
    auto add = [&](const float* x) {
        if (x[0] == -INFINITY) return;
        const float w = exp2f(x[0] - M);
        L += x[1] * w; o += x[2 + d] * w;
    };
    for (int s = 0; s < prm.own_splits; ++s) add(own + s * step);
    if (pre != nullptr) for (int s = 0; s < prm.prefix_splits; ++s) add(pre + s * step);
    const float lse = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    reinterpret_cast<T*>(prm.out)[(size_t)blockIdx.x * D + d] =
        gated_out<T>(L == 0.f ? 0.f : o / L, sink_gate(prm.epi, hq, lse), prm.epi.sinks != nullptr);
    if (d == 0) prm.lse[blockIdx.x] = lse;
}

struct Plan { int rows_per_tile, prefix_tiles, prefix_splits, own_splits; size_t parts; };
Plan plan_of(const PoolView& pv, int B, int Hq, int n_groups)
{
    Plan p;
    const int n_rep = Hq / pv.H;
    p.rows_per_tile = kTileRows / n_rep;
    p.prefix_tiles = n_groups > 0 ? B / p.rows_per_tile + (n_groups < B ? n_groups : B) : 0;
    auto splits = [](int tiles) { const int s = tiles > 0 ? 4 * 148 / tiles : 1; return s < 1 ? 1 : s > 32 ? 32 : s; };
    p.prefix_splits = splits(p.prefix_tiles * pv.H);
    p.own_splits = splits(B * pv.H);
    p.parts = (size_t)p.prefix_tiles * pv.H * p.prefix_splits + (size_t)B * pv.H * p.own_splits;
    return p;
}

}  // namespace

bool decode_shared_supported(const PoolView& pv, int Hq)
{
    return (pv.dtype == FPKV_BF16 || pv.dtype == FPKV_F16) && pv.split_hq == 0 && pv.P == kPage && Hq / pv.H <= kTileRows;
}

size_t decode_shared_workspace_bytes(const PoolView& pv, int B, int Hq, int n_groups)
{
    return plan_of(pv, B, Hq, n_groups).parts * kTileRows * (pv.D + 2) * sizeof(float);
}

int launch_decode_shared(const PoolView& pv, int layer, void* out, float* lse, const void* q, long long qsb, long long qsh,
                         const int64_t* batch_idx, const void* pos, int pos_type, int B, int Hq, const int32_t* groups,
                         int n_groups, const int32_t* row_group, float sm_scale, void* workspace, const Epilogue& epi,
                         int32_t* status, cudaStream_t stream)
{
    const Plan pl = plan_of(pv, B, Hq, n_groups);
    SharedParams prm;
    prm.k = pv.plane(layer, 0, 0); prm.v = pv.plane(layer, 1, 0); prm.plane_bytes = pv.plane_bytes();
    prm.page_table = pv.page_table; prm.p2l = pv.p2l; prm.batch_idx = batch_idx; prm.pos = pos; prm.q = q;
    prm.groups = reinterpret_cast<const int4*>(groups); prm.row_group = row_group;
    prm.out = out; prm.lse = lse; prm.ws = static_cast<float*>(workspace); prm.status = status;
    prm.q_stride_b = qsb; prm.q_stride_h = qsh;
    prm.B = B; prm.Hq = Hq; prm.H = pv.H; prm.n_rep = Hq / pv.H; prm.rows_per_tile = pl.rows_per_tile;
    prm.n_groups = n_groups; prm.n_pages = pv.n_pages; prm.max_batch = pv.max_batch; prm.pos_is_64 = pos_type == FPKV_I64;
    prm.prefix_tiles = pl.prefix_tiles; prm.prefix_splits = pl.prefix_splits; prm.own_splits = pl.own_splits;
    prm.scale_log2 = sm_scale * kLog2e; prm.epi = epi;
    auto run = [&](auto part, auto merge) {
        part<<<(unsigned)pl.parts, kPartWarps * 32, 0, stream>>>(prm);
        if (cudaGetLastError() != cudaSuccess) return FPKV_ELAUNCH;
        merge<<<B * Hq, pv.D, 0, stream>>>(prm);
        return cudaGetLastError() == cudaSuccess ? FPKV_OK : FPKV_ELAUNCH;
    };
    if (pv.dtype == FPKV_BF16)
        return pv.D == 128 ? run(shared_partial_kernel<__nv_bfloat16, 128>, shared_merge_kernel<__nv_bfloat16, 128>)
                           : run(shared_partial_kernel<__nv_bfloat16, 64>, shared_merge_kernel<__nv_bfloat16, 64>);
    return pv.D == 128 ? run(shared_partial_kernel<__half, 128>, shared_merge_kernel<__half, 128>)
                       : run(shared_partial_kernel<__half, 64>, shared_merge_kernel<__half, 64>);
}

}  // namespace fpkv
