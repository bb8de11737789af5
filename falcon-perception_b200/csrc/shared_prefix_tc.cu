// Attention of many query rows over one shared prefix (tcgen05.mma, accumulators in tensor memory), 16-bit pools,
// page_size 128, head_dim 128 or 64.  The prefix part of fpkv_decode_attn_shared; what a row sees of its own is
// decode_shared.cu's, which also joins the two.
//
// A query tile is 128 rows: the query heads of one stored head for 128 / n_rep rows of a group (tensor map over q, so the
// rows need no packing).  All of them see the same keys -- whole pages -- but for rows whose position lies inside the
// prefix.  "Segment" = query tile x stored head; "piece" = a run of key tiles of a segment.  The key tiles of all segments,
// one after the other, are cut into equal shares, one per CTA (persistent, one per SM): decode has few query tiles and long
// prefixes, so the keys are what is split.  A piece leaves (m, l) of its rows and the unnormalised result in 32 bits in the
// workspace, at slot (CTA number + segment number): both only grow along the cut, and one of them does at each piece.
//
// Inside a piece the key tiles are dealt out to two sides, even and odd: softmax group g (four warps, one thread a query
// row) and MMA issuer g work through tiles g, g + 2, ..., each side with its own score columns, reference maximum, row sum
// and accumulator; the two are joined in the epilogue, where each group writes half of the columns.  A tile is worked
// through in two halves of 64 keys with separate score columns,
//     S = Q K^T   128x64xD,   A = Q (shared), B = 64 rows of the K tile (shared)
//     O += P V    128xDx64,   A = P (tensor memory, over the first half of the S columns), B = 64 rows of the V tile
// with P rounded to 16 bits, the type the MMA takes it in (at most half a step each, as the decode and prefill kernels
// round it; the row sums are those of P before the rounding, in 32 bits), so that four chains
// S -> softmax -> P V -> next S are in flight.  Warp 8 issues the copies, warps 9 and 10 the MMAs, warp 11 prepares the
// next piece and, 64 key tiles ahead, the pool rows of its pages.
//
// Bound: with at most 128 query rows a segment by the bytes of K and V (a tile's MMAs take 1040 clocks, its exponentials
// 1024, its 64 KiB at the SM's share of memory 2800); with more by the MMAs and exponentials.
//
// Every wait is a bounded mbarrier wait; on expiry the CTA raises FPKV_STATUS_TIMEOUT, every role leaves its loops, the copies
// and MMAs in flight are drained (bounded), tensor memory is freed and the kernel returns.

#include <string.h>
#include <type_traits>
#include "tc5.cuh"
#include "shared_prefix.cuh"

namespace fpkv {
namespace {

constexpr int kStagesK = 2, kStagesV = 3;
constexpr int kSoftmaxWarps = 4;                       // per side
constexpr int kLoadWarp = 8, kMmaWarp = 9, kScoutWarp = 11;
constexpr int kThreads = 12 * 32;
constexpr int kChunk = 64;                             // key tiles resolved at a time
constexpr uint32_t kTmemCols = 512;                    // S/P side 0, S/P side 1, O side 0, O side 1: 128 columns each

struct PieceDesc {
    int valid;                  // 0: no more work for this CTA
    int b0, hkv;                // first batch row and stored head of the segment
    int n_tiles;                // key tiles of the piece that any row sees
    int key0;                   // first key of the piece
    int rows;                   // query rows of the tile
    int max_extent;             // visible keys from key0 on, largest among the rows
    int slot;                   // partial
    int extent[kTileM];         // visible keys of each row from key0 on
};
struct ChunkDesc {
    int page_row[kChunk];       // pool row of the K tile of each key tile (reserved page 0 when unmapped)
    unsigned char page_ok[kChunk];
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const PrefixParams prm)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_s = smem;                                   // 32 KiB
    uint8_t* k_s = q_s + kTileBytes;                       // kStagesK x 32 KiB
    uint8_t* v_s = k_s + kStagesK * kTileBytes;            // kStagesV x 32 KiB
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + kStagesV * kTileBytes);
    int* ints = reinterpret_cast<int*>(bars + 48);
    volatile int* abort_flag = ints;                       // [0] abort, [1] TMEM base
    int* tmem_slot = ints + 1;
    PieceDesc* desc = reinterpret_cast<PieceDesc*>(ints + 16);       // [2]
    ChunkDesc* chunks = reinterpret_cast<ChunkDesc*>(desc + 2);      // [2]
    float2* xch = reinterpret_cast<float2*>(chunks + 2);   // [2][2 groups][128 rows] (m, l)
    long long* flat_before = reinterpret_cast<long long*>(xch + 2 * 2 * kTileM);      // [n_groups + 1]
    int* mt_before = reinterpret_cast<int*>(flat_before + FPKV_MAX_GROUPS + 1);       // [n_groups + 2]

    uint32_t at = s32(bars);
    auto take = [&](int n) { const uint32_t b = at; at += 8 * n; return b; };
    const uint32_t desc_full0 = take(2), desc_empty0 = take(2), chunk_full0 = take(2), chunk_empty0 = take(2);
    const uint32_t q_full = take(1), q_empty = take(1);
    const uint32_t k_full0 = take(kStagesK), k_empty0 = take(kStagesK), v_full0 = take(kStagesV), v_empty0 = take(kStagesV);
    const uint32_t s_half0 = take(4), p_half0 = take(4);   // [side][half] scores of 64 keys are in tensor memory / P of 64 keys written
    const uint32_t pv_done0 = take(2);                     // [side] a half's P.V has completed (one phase per half)
    const uint32_t all_done0 = take(2), o_free0 = take(2); // [side] last P.V complete / O read by the epilogue
    const uint32_t drain0 = take(2), merge0 = take(1);     // give-up path / both groups have published (m, l)

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    constexpr int kTileBytesD = kTileM * D * 2;

    // ---- set-up: barriers, tensor memory, key tiles before each group -----------------
    if (warp == kLoadWarp && lane == 0) {                  // the maps themselves come from memory, too
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&q_map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kv_map)) : "memory");
    }
    if (tid == 0) {
        for (int b = 0; b < 2; ++b) {
            bar_init(desc_full0 + 8 * b, 1); bar_init(desc_empty0 + 8 * b, 3 + 2 * kSoftmaxWarps);
            bar_init(chunk_full0 + 8 * b, 1); bar_init(chunk_empty0 + 8 * b, 1 + 2 * kSoftmaxWarps);
            for (int hf = 0; hf < 2; ++hf) { bar_init(s_half0 + 16 * b + 8 * hf, 1); bar_init(p_half0 + 16 * b + 8 * hf, kSoftmaxWarps); }
            bar_init(pv_done0 + 8 * b, 1); bar_init(all_done0 + 8 * b, 1);
            bar_init(o_free0 + 8 * b, 2 * kSoftmaxWarps);  // both groups read both accumulators
            bar_init(drain0 + 8 * b, 1);
        }
        bar_init(q_full, 1); bar_init(q_empty, 2);
        bar_init(merge0, 2 * kSoftmaxWarps);
        for (int s = 0; s < kStagesK; ++s) { bar_init(k_full0 + 8 * s, 1); bar_init(k_empty0 + 8 * s, 1); }
        for (int s = 0; s < kStagesV; ++s) { bar_init(v_full0 + 8 * s, 1); bar_init(v_empty0 + 8 * s, 1); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == kScoutWarp) prefix_schedule(prm.rows, prm.max_segments / prm.rows.H, flat_before, mt_before, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;");     // the own part needs nothing from here
    if (warp < 2 * kSoftmaxWarps) {                        // the merge's table, while there are no scores yet
        const RowParams& rp = prm.rows;
        const int n_segments = mt_before[rp.n_groups] * rp.H;
        for (int i = blockIdx.x * 2 * kSoftmaxWarps * 32 + tid; i < prm.max_segments; i += gridDim.x * 2 * kSoftmaxWarps * 32)
            prm.segments[i] = i < n_segments ? segment_entry(rp, flat_before, mt_before, i, gridDim.x) : make_int4(0, 0, 0, 0);
    }
    const uint32_t tmem = (uint32_t)*tmem_slot;
    // S/P of side 0 [0,128), of side 1 [128,256), O of side 0 [256,384), of side 1 [384,512)
    bool alive = true;
    uint32_t k_requested = 0, v_requested = 0, q_requested = 0;      // copies requested so far by the producer thread

    if (warp == kScoutWarp) {
        // ============================== scout ===================================
        const RowParams& rp = prm.rows;
        const long long total = flat_before[rp.n_groups];
        const long long share = share_size(total, gridDim.x, mt_before[rp.n_groups + 1]), end = min(total, (blockIdx.x + 1) * share);
        long long pos = blockIdx.x * share;
        uint32_t it = 0, ch = 0;
        while (alive) {
            const uint32_t b = it & 1u;
            if (lane == 0) alive = bar_wait(desc_empty0 + 8 * b, ((it >> 1) & 1u) ^ 1u, abort_flag);
            alive = __shfl_sync(0xffffffffu, alive, 0);
            if (!alive) break;
            PieceDesc* d = desc + b;
            if (pos >= end) {
                if (lane == 0) { d->valid = 0; bar_arrive(desc_full0 + 8 * b); }
                break;
            }
            const Segment sg = segment_at(rp, flat_before, mt_before, pos);
            const int here = (int)min((long long)(sg.pages - sg.tile), end - pos);
            const int key0 = sg.tile * kPage;
            int ex[4], emax = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = lane + 32 * r;
                int slot = 0;
                int n = row < sg.rows ? row_keys(rp, sg.b0 + row / rp.n_rep, &slot, false) : 0;
                if (!slot_maps_pages(rp, slot)) n = 0;
                ex[r] = max(0, min(n, sg.pages * kPage) - key0);
                d->extent[row] = ex[r];
                emax = max(emax, ex[r]);
            }
            emax = (int)__reduce_max_sync(0xffffffffu, (uint32_t)emax);
            const int n_tiles = min(here, (emax + kTileN - 1) / kTileN);
            if (lane == 0) {
                d->valid = 1; d->b0 = sg.b0; d->hkv = sg.h; d->n_tiles = n_tiles; d->key0 = key0; d->rows = sg.rows;
                d->max_extent = emax; d->slot = blockIdx.x + sg.index;
            }
            __syncwarp();
            if (lane == 0) bar_arrive(desc_full0 + 8 * b);
            ++it;
            // pool rows of its key tiles
            const long long trow = (long long)mapping_slot(rp, sg.group_b0, sg.group_rows, lane) * rp.n_pages;
            for (int j0 = 0; j0 < n_tiles && alive; j0 += kChunk, ++ch) {
                const uint32_t cb = ch & 1u;
                long long pg[2];
                bool ok[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int j = j0 + lane + 32 * r;
                    pg[r] = j < n_tiles ? rp.page_table[trow + sg.tile + j] : -1;
                    ok[r] = pg[r] >= 0 && pg[r] < rp.n_pages;
                    if (pg[r] >= rp.n_pages) raise_status(rp.status, FPKV_STATUS_BAD_PAGE);
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) if (ok[r]) ok[r] = rp.p2l[trow + pg[r]] >= 0;
                if (lane == 0) alive = bar_wait(chunk_empty0 + 8 * cb, ((ch >> 1) & 1u) ^ 1u, abort_flag);
                alive = __shfl_sync(0xffffffffu, alive, 0);
                if (!alive) break;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    chunks[cb].page_row[lane + 32 * r] = sg.h * prm.rows_per_plane + (ok[r] ? (int)pg[r] : 0) * kPage;
                    chunks[cb].page_ok[lane + 32 * r] = ok[r];
                }
                __syncwarp();
                if (lane == 0) bar_arrive(chunk_full0 + 8 * cb);
            }
            pos += here;
        }
    } else if (warp == kLoadWarp) {
        // ============================== TMA producer ========================
        if (lane == 0) {
            uint32_t gk = 0, wit = 0, ch = 0;              // key tiles requested, pieces with work, chunks taken
            for (uint32_t it = 0; alive; ++it) {
                const uint32_t b = it & 1u;
                if (!bar_wait(desc_full0 + 8 * b, (it >> 1) & 1u, abort_flag)) { alive = false; break; }
                const PieceDesc* d = desc + b;
                if (!d->valid) break;
                const int n = d->n_tiles;
                if (n > 0) {
                    if (!bar_wait(q_empty, (wit & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                    // the tile's rows x n_rep heads, 64 elements wide, one box per 64-element column group; rows of q past
                    // the batch read as zeros, rows of the box past the tile's are another group's and go unused
                    bar_expect_tx(q_full, prm.q_box_rows * D * 2);
                    for (int hf = 0; hf < D / 64; ++hf)
                        tma_3d(s32(q_s + hf * kHalfBytes), &q_map, hf * 64, d->hkv * prm.rows.n_rep, d->b0, q_full);
                    q_requested = wit + 1;
                    // The K ring and the V ring advance independently; a chunk of pool rows is given back when both are past it.
                    int jk = 0, jv = 0, have = 0, past = 0;      // tiles of K and V requested, resolved, in chunks given back
                    const uint32_t ch0 = ch;
                    uint32_t idle = 0;
                    while ((jk < n || jv < n) && alive) {
                        bool progress = false;
                        if (jk == have && have < n) {
                            const uint32_t c = ch0 + have / kChunk;
                            if (bar_try(chunk_full0 + 8 * (c & 1u), (c >> 1) & 1u)) {
                                have = min(n, have + kChunk);
                                progress = true;
                            }
                        }
                        if (jk < have) {
                            const uint32_t g = gk + jk, st = g % kStagesK;
                            if (bar_try(k_empty0 + 8 * st, ((g / kStagesK) & 1u) ^ 1u)) {
                                bar_expect_tx(k_full0 + 8 * st, kTileBytesD);
                                tma_3d(s32(k_s + st * kTileBytes), &kv_map, 0, chunks[(ch0 + jk / kChunk) & 1u].page_row[jk % kChunk], 0, k_full0 + 8 * st);
                                k_requested = g + 1; ++jk; progress = true;
                            }
                        }
                        if (jv < have) {
                            const uint32_t g = gk + jv, st = g % kStagesV;
                            if (bar_try(v_empty0 + 8 * st, ((g / kStagesV) & 1u) ^ 1u)) {
                                bar_expect_tx(v_full0 + 8 * st, kTileBytesD);
                                tma_3d(s32(v_s + st * kTileBytes), &kv_map, 0,
                                       chunks[(ch0 + jv / kChunk) & 1u].page_row[jv % kChunk] + prm.rows.H * prm.rows_per_plane, 0, v_full0 + 8 * st);
                                v_requested = g + 1; ++jv; progress = true;
                            }
                        }
                        while (past < n && min(jk, jv) >= min(past + kChunk, n)) {
                            bar_arrive(chunk_empty0 + 8 * (ch & 1u));
                            past += kChunk; ++ch;
                        }
                        if (progress) idle = 0;
                        else if (++idle > kSpin || ((idle & 255u) == 255u && *abort_flag)) alive = false;
                    }
                    gk += n;
                    ++wit;
                }
                if (alive) bar_arrive(desc_empty0 + 8 * b);
            }
        }
    } else if (warp >= kMmaWarp && warp < kMmaWarp + 2) {
        // ============================== MMA issuers =========================
        const int g = warp - kMmaWarp;
        if (lane == 0) {
            const bool is_bf16 = std::is_same<T, __nv_bfloat16>::value;
            const uint32_t idesc_qk = umma_idesc(is_bf16, false, 64);
            const uint32_t idesc_pv = umma_idesc(is_bf16, true, D);
            const uint32_t desc_hi = (uint32_t)(umma_desc(0, 0, 1024) >> 32);
            const uint32_t q_lo = (s32(q_s) & 0x3FFFF) >> 4, k_lo = (s32(k_s) & 0x3FFFF) >> 4;
            const uint32_t v_lo0 = ((s32(v_s) & 0x3FFFF) >> 4) | (uint32_t)umma_desc(0, kHalfBytes, 1024);
            const uint32_t t_s = tmem + g * kTileN, t_o = tmem + 256 + g * kTileN;
            const uint32_t s_lo = s_half0 + 16 * g, s_hi = s_lo + 8, p_lo = p_half0 + 16 * g, p_hi = p_lo + 8;
            const uint32_t pv_done = pv_done0 + 8 * g;
            uint32_t gk = 0, th = 0, wit = 0, wg = 0;      // key tiles of all pieces, this side's tiles, pieces with work, with work for this side
            for (uint32_t it = 0; alive; ++it) {
                const uint32_t b = it & 1u;
                if (!bar_wait(desc_full0 + 8 * b, (it >> 1) & 1u, abort_flag)) { alive = false; break; }
                const PieceDesc* d = desc + b;
                if (!d->valid) break;
                const int n = d->n_tiles;
                if (n > g) {
                    const uint32_t c0 = gk + g, st0 = c0 % kStagesK;
                    alive = bar_wait(q_full, wit & 1u, abort_flag) && bar_wait(k_full0 + 8 * st0, (c0 / kStagesK) & 1u, abort_flag);
                    if (!alive) break;
                    tc_fence_after();
                    issue_qk_half<0, D>(t_s, q_lo, k_lo + st0 * (kTileBytes >> 4), desc_hi, idesc_qk, s_lo);
                    issue_qk_half<1, D>(t_s + 64, q_lo, k_lo + st0 * (kTileBytes >> 4), desc_hi, idesc_qk, s_hi);
                    umma_commit(k_empty0 + 8 * st0);
                    if (g + 2 >= n) umma_commit(q_empty);  // that was this side's only Q.K^T of the piece
                    for (int j = g; j < n; j += 2) {
                        const uint32_t cur = gk + j, nxt = cur + 2;
                        const uint32_t sv = cur % kStagesV, sn = nxt % kStagesK;
                        const bool more = j + 2 < n;
                        if (!bar_wait(v_full0 + 8 * sv, (cur / kStagesV) & 1u, abort_flag)) { alive = false; break; }
                        // O of the previous piece must have been read before the first P.V overwrites it
                        if (j == g && !bar_wait(o_free0 + 8 * g, (wg & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                        if (!bar_wait(p_lo, th & 1u, abort_flag)) { alive = false; break; }
                        tc_fence_after();
                        const uint32_t v_lo = v_lo0 + sv * (kTileBytes >> 4);
                        issue_pv_half<0>(t_o, t_s, v_lo, desc_hi, idesc_pv, j > g);
                        umma_commit(pv_done);
                        if (more && !bar_wait(k_full0 + 8 * sn, (nxt / kStagesK) & 1u, abort_flag)) { alive = false; break; }
                        if (more) issue_qk_half<0, D>(t_s, q_lo, k_lo + sn * (kTileBytes >> 4), desc_hi, idesc_qk, s_lo);
                        if (!bar_wait(p_hi, th & 1u, abort_flag)) { alive = false; break; }
                        tc_fence_after();
                        issue_pv_half<1>(t_o, t_s + 64, v_lo, desc_hi, idesc_pv, 1u);
                        umma_commit(pv_done);
                        umma_commit(v_empty0 + 8 * sv);
                        ++th;
                        if (more) {
                            issue_qk_half<1, D>(t_s + 64, q_lo, k_lo + sn * (kTileBytes >> 4), desc_hi, idesc_qk, s_hi);
                            umma_commit(k_empty0 + 8 * sn);
                            if (j + 4 >= n) umma_commit(q_empty);        // this side's last Q.K^T of the piece
                        }
                    }
                    if (!alive) break;
                    umma_commit(all_done0 + 8 * g);
                    ++wg;
                } else if (n > 0) {
                    // One key tile: nothing for this side, only its share of the hand-back -- of this piece's queries, so not
                    // before they are there: two pieces' shares would pass for both sides' of one.
                    if (!bar_wait(q_full, wit & 1u, abort_flag)) { alive = false; break; }
                    bar_arrive(q_empty);
                }
                if (n > 0) { gk += n; ++wit; }
                bar_arrive(desc_empty0 + 8 * b);
            }
            if (!alive) {                                  // wait (bounded) for the MMAs already in the pipe
                umma_commit(drain0 + 8 * g);
                for (uint32_t k = 0; k < kSpin && !bar_try(drain0 + 8 * g, 0); ++k) {}
            }
        }
    } else if (warp < 2 * kSoftmaxWarps) {
        // ============================== softmax groups ======================
        const int grp = warp / kSoftmaxWarps, quarter = warp % kSoftmaxWarps;
        const int row = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t ts = tmem + grp * kTileN + lane_base;
        const uint32_t to = tmem + 256 + grp * kTileN + lane_base;
        const uint32_t pv_done = pv_done0 + 8 * grp;
        uint32_t gk = 0, th = 0, wit = 0, wg = 0, ch = 0;
        for (uint32_t it = 0; alive; ++it) {
            const uint32_t b = it & 1u;
            if (!bar_wait(desc_full0 + 8 * b, (it >> 1) & 1u, abort_flag)) { alive = false; break; }
            const PieceDesc* d = desc + b;
            if (!d->valid) break;
            const int n = d->n_tiles, max_extent = d->max_extent, my_extent = d->extent[row];
            float m_ref = -INFINITY, l = 0.f;
            uint32_t sv[2][32], pk[32];
            // tiles below `wfull` are fully visible to every row of this warp that has any (the others' results go unused)
            const int wfull = (int)__reduce_min_sync(0xffffffffu, row < d->rows ? (uint32_t)(my_extent / kTileN) : 0x7fffffffu);
            for (int j0 = 0; j0 < n && alive; j0 += kChunk, ++ch) {
                if (!bar_wait(chunk_full0 + 8 * (ch & 1u), (ch >> 1) & 1u, abort_flag)) { alive = false; break; }
                const ChunkDesc* cd = chunks + (ch & 1u);
                const int j1 = min(n, j0 + kChunk);
                for (int j = j0 + ((j0 + grp) & 1); j < j1 && alive; j += 2) {
                    const bool page_ok = cd->page_ok[j - j0] != 0;
                    // Value rows past the last key that any row of this tile sees (or all of an unmapped page's stand-in) may
                    // hold anything, and 0 x NaN would poison O: clear them in shared memory ahead of the tile's P.V.
                    const int tile_rows = page_ok ? min(kTileN, max_extent - j * kTileN) : 0;
                    if (tile_rows < kTileN) {
                        const uint32_t cur = gk + j, st = cur % kStagesV;
                        if (!bar_wait(v_full0 + 8 * st, (cur / kStagesV) & 1u, abort_flag)) { alive = false; break; }
                        for (int i = row; i < (kTileN - tile_rows) * (D / 8); i += kSoftmaxWarps * 32) {
                            const int r = tile_rows + i / (D / 8), c = i % (D / 8);
                            *reinterpret_cast<uint4*>(v_s + st * kTileBytes + (c >> 3) * kHalfBytes + r * 128 + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    const bool full = j < wfull && page_ok;
                    const int valid_row = full ? kTileN : (page_ok ? min(kTileN, my_extent - j * kTileN) : 0);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const uint32_t unit = 2 * th + hf;
                        const int valid_cols = valid_row - 64 * hf;
                        if (!bar_wait(s_half0 + 16 * grp + 8 * hf, th & 1u, abort_flag)) { alive = false; break; }
                        tc_fence_after();
                        tmem_ld32_nowait(ts + 64 * hf, sv[0]);
                        tmem_ld32_nowait(ts + 64 * hf + 32, sv[1]);
                        tmem_wait_ld();
                        // The reference maximum is raised only when a score lies more than 2^8 above it (the probabilities stay
                        // below 256), so that O in tensor memory is rarely rescaled; O is stable once all P.V so far are done.
                        const float mx = (full ? max64<true>(sv, 64) : max64<false>(sv, valid_cols)) * prm.scale_log2;   // scale > 0
                        const bool raise = mx > m_ref + kRescaleThreshold || (m_ref == -INFINITY && mx > -INFINITY);
                        if (__any_sync(0xffffffffu, raise)) {
                            const float m_new = raise ? mx : m_ref;
                            const float alpha = (m_ref == -INFINITY) ? 0.f : exp2f(m_ref - m_new);
                            if (j > grp || hf > 0) {
                                if (!bar_wait(pv_done, (unit - 1) & 1u, abort_flag)) { alive = false; break; }
                                tc_fence_after();
#pragma unroll 1
                                for (int c4 = 0; c4 < D / 32; ++c4) {
                                    tmem_ld32(to + c4 * 32, pk);
#pragma unroll
                                    for (int c = 0; c < 32; ++c) pk[c] = __float_as_uint(__uint_as_float(pk[c]) * alpha);
                                    tmem_st32(to + c4 * 32, pk);
                                }
                            }
                            l *= alpha;
                            m_ref = m_new;
                        }
                        const float neg_m = (m_ref == -INFINITY) ? 0.f : -m_ref;
                        F2 rs[2] = {F2{0.f, 0.f}, F2{0.f, 0.f}};
                        if (full) probabilities64<T, true>(sv, pk, rs, prm.scale_log2, neg_m, 64);
                        else probabilities64<T, false>(sv, pk, rs, prm.scale_log2, neg_m, valid_cols);
                        tmem_st32_nowait(ts + 64 * hf, pk);
                        l += (rs[0].x + rs[0].y) + (rs[1].x + rs[1].y);
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(p_half0 + 16 * grp + 8 * hf);
                    }
                    ++th;
                }
                __syncwarp();
                if (lane == 0 && alive) bar_arrive(chunk_empty0 + 8 * (ch & 1u));
            }
            if (!alive) break;
            gk += n;
            // ---- epilogue: both sides' accumulators to the common maximum, half of the columns each ----
            const bool own_tiles = n > grp, oth_tiles = n > (grp ^ 1);
            if (own_tiles) {
                if (!bar_wait(all_done0 + 8 * grp, wg & 1u, abort_flag)) { alive = false; break; }
                tc_fence_after();
                ++wg;
            }
            float w_own = 1.f, w_oth = 0.f;
            if (n > 0) {
                float2* told = xch + (wit & 1u) * (2 * kTileM);
                told[grp * kTileM + row] = make_float2(m_ref, l);
                __syncwarp();
                if (lane == 0) bar_arrive(merge0);
                if (!bar_wait(merge0, wit & 1u, abort_flag)) { alive = false; break; }
                tc_fence_after();
                const float2 oth = told[(grp ^ 1) * kTileM + row];
                const float m = fmaxf(m_ref, oth.x);
                w_own = (m_ref == -INFINITY) ? 0.f : exp2f(m_ref - m);
                w_oth = (oth.x == -INFINITY) ? 0.f : exp2f(oth.x - m);
                l = l * w_own + oth.y * w_oth;
                m_ref = m;
                ++wit;
            }
            if (grp == 0) prm.ml[(size_t)d->slot * kTileM + row] = make_float2(l == 0.f ? -INFINITY : m_ref, l);
            if (n > 0) {
                // partial: [D/4 column groups][128 rows] of four columns, so that a warp's rows lie side by side
                float4* dst = reinterpret_cast<float4*>(prm.acc) + (size_t)d->slot * (D / 4) * kTileM + row;
                constexpr int kCols = D / 2;
                const uint32_t to_oth = tmem + 256 + (grp ^ 1) * kTileN + lane_base;
#pragma unroll 1
                for (int c2 = 0; c2 < kCols / 32; ++c2) {
                    const int col0 = grp * kCols + c2 * 32;
                    if (own_tiles) tmem_ld32_nowait(to + col0, sv[0]);
                    if (oth_tiles) tmem_ld32_nowait(to_oth + col0, sv[1]);
                    tmem_wait_ld();
                    if (c2 == kCols / 32 - 1) {            // read: the next piece's P.V may overwrite them
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0 && own_tiles) bar_arrive(o_free0 + 8 * grp);
                        if (lane == 0 && oth_tiles) bar_arrive(o_free0 + 8 * (grp ^ 1));
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)        // an accumulator without a tile of this piece holds whatever was there
                            v[e] = (own_tiles ? __uint_as_float(sv[0][c + e]) * w_own : 0.f) + (oth_tiles ? __uint_as_float(sv[1][c + e]) * w_oth : 0.f);
                        dst[(size_t)((col0 + c) / 4) * kTileM] = make_float4(v[0], v[1], v[2], v[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) bar_arrive(desc_empty0 + 8 * b);
        }
    }
    if (!alive && lane == 0) {
        if (!*abort_flag) raise_status(prm.rows.status, FPKV_STATUS_TIMEOUT);
        *abort_flag = 1;
    }
    // ---- teardown: everyone meets here, then the allocating warp frees TMEM ---
    tc_fence_before();
    __syncthreads();
    if (warp == kLoadWarp && lane == 0 && *abort_flag) {
        // copies still in flight target this CTA's shared memory: wait (bounded) for the last one into every buffer
        if (q_requested > 0) for (uint32_t k = 0; k < kSpin && !bar_try(q_full, (q_requested - 1) & 1u); ++k) {}
        for (uint32_t s = 0; s < (uint32_t)kStagesK; ++s)
            if (k_requested > s) {
                const uint32_t last = ((k_requested - 1 - s) / kStagesK) * kStagesK + s;
                for (uint32_t k = 0; k < kSpin && !bar_try(k_full0 + 8 * s, (last / kStagesK) & 1u); ++k) {}
            }
        for (uint32_t s = 0; s < (uint32_t)kStagesV; ++s)
            if (v_requested > s) {
                const uint32_t last = ((v_requested - 1 - s) / kStagesV) * kStagesV + s;
                for (uint32_t k = 0; k < kSpin && !bar_try(v_full0 + 8 * s, (last / kStagesV) & 1u); ++k) {}
            }
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

constexpr int kSmem = 1024 + (1 + kStagesK + kStagesV) * kTileBytes + 48 * 8 + 16 * 4 + 2 * (int)sizeof(PieceDesc) + 2 * (int)sizeof(ChunkDesc) +
                      2 * 2 * kTileM * 8 + (FPKV_MAX_GROUPS + 1) * 12 + 16;
static_assert(kSmem <= 227 * 1024, "shared memory");

}  // namespace

int prefix_ctas() { return sm_count(); }

bool prefix_supported(const PoolView& pv)
{
    // TMA coordinates are 32-bit token rows within one layer's K and V planes
    return (long long)2 * pv.H * pv.n_pages * pv.P < (1ll << 31);
}

bool encode_rows(CUtensorMap* map, const PoolView& pv, int layer, int rows)
{
    if (encoder() == nullptr) return false;
    const int halves = pv.D / 64;
    const cuuint64_t dims[3] = {64, (cuuint64_t)2 * pv.H * pv.n_pages * pv.P, (cuuint64_t)halves};
    const cuuint64_t strides[2] = {(cuuint64_t)halves * 128, 128};
    const cuuint32_t box[3] = {64, (cuuint32_t)rows, (cuuint32_t)halves};
    const cuuint32_t es[3] = {1, 1, 1};
    return encoder()(map, pv.dtype == FPKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, pv.plane(layer, 0, 0), dims,
                     strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_prefix(const PoolView& pv, int layer, const void* q, long long q_stride_b, long long q_stride_h, PrefixParams prm, cudaStream_t stream)
{
    if (encoder() == nullptr) return FPKV_EARCH;
    const CUtensorMapDataType dt = pv.dtype == FPKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap kv_map, q_map;
    if (!encode_rows(&kv_map, pv, layer, kPage)) return FPKV_ELAUNCH;
    {   // queries (head_dim, heads, rows): a box of 64 elements x n_rep heads x the rows of a tile is a block of 128-byte rows
        const RowParams& rp = prm.rows;
        prm.q_box_rows = rp.rows_per_tile * rp.n_rep;
        const cuuint64_t dims[3] = {(cuuint64_t)pv.D, (cuuint64_t)rp.Hq, (cuuint64_t)rp.B};
        const cuuint64_t strides[2] = {(cuuint64_t)q_stride_h * 2, (cuuint64_t)q_stride_b * 2};
        const cuuint32_t box[3] = {64, (cuuint32_t)rp.n_rep, (cuuint32_t)rp.rows_per_tile};
        const cuuint32_t es[3] = {1, 1, 1};
        if (encoder()(&q_map, dt, 3, const_cast<void*>(q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return FPKV_ELAUNCH;
    }
    prm.rows_per_plane = pv.n_pages * pv.P;
    auto launch = [&](auto kern) {
        if (const int rc = launch_code(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem))) return rc;
        kern<<<prefix_ctas(), kThreads, kSmem, stream>>>(q_map, kv_map, prm);
        return launch_code(cudaGetLastError());
    };
    if (pv.dtype == FPKV_BF16) return pv.D == 128 ? launch(shared_prefix_kernel<__nv_bfloat16, 128>) : launch(shared_prefix_kernel<__nv_bfloat16, 64>);
    return pv.D == 128 ? launch(shared_prefix_kernel<__half, 128>) : launch(shared_prefix_kernel<__half, 64>);
}

}  // namespace fpkv
