// Packed-row indices, block tables and slot maps of one step, from request lengths held on the device.
//
// One launch: every CTA scans the aligned lengths of all requests into shared memory (a few thousand
// entries at most; the repeated scan costs less than a second launch would), then the CTAs share out
// the packed tokens and the block-table entries.  A warp finds its first token's request by bisection in
// shared memory, its other tokens go on from there, and a token's page takes one table read.  Bound by
// instructions and the dependent reads of a token (slot, start, page) on long rows -- 512 requests, 790 K tokens:
// 18.5 us, issue slots 53 % busy, while the 25 MB stored stay in L2 and would take 4 us -- and by the launch plus
// three dependent memory reads (lengths, slot, page) on short ones.

#include "common.cuh"

namespace fpkv {

namespace {

constexpr int kStepThreads = 256;

struct StepParams {
    const int64_t* page_table;
    const int64_t* slots;
    const int32_t* starts;
    const int32_t* lens;
    const int64_t* tokens;
    int64_t n_tokens, pad_id;
    fpkv_step_out out;
    int32_t* status;
    int n_req, row_tokens, align, width, n_pages, max_batch, P;
};

// Sum of two saturating lengths: everything past 2^31 - 1 stays there (such rows are refused token by token anyway).
__device__ __forceinline__ int sat(long long v) { return v > 0x7fffffffll ? 0x7fffffff : (int)v; }

__global__ void __launch_bounds__(kStepThreads)
step_tables_kernel(const StepParams prm)
{
    extern __shared__ int s_scan[];
    const int N = prm.n_req;
    int* first = s_scan;                 // [N + 1] packed index of each request's first token
    int* cum = s_scan + N + 1;           // [N + 1] tokens before each request
    __shared__ long long w_al[kStepThreads / 32], w_ln[kStepThreads / 32];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

    long long base_al = 0, base_ln = 0;
    for (int r0 = 0; r0 < N; r0 += kStepThreads) {
        const int r = r0 + tid;
        long long n = 0;
        if (r < N) {
            const int len = prm.lens[r], st = prm.starts[r];
            if (len < 0 || st < 0) { if (blockIdx.x == 0) raise_status(prm.status, FPKV_STATUS_BAD_POS); }
            else n = len;
        }
        const unsigned runs = ((unsigned)n + (unsigned)prm.align - 1u) / (unsigned)prm.align;     // below 2^31 + 2^20
        const long long al = (long long)runs * prm.align;
        long long xa = al, xn = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long ya = __shfl_up_sync(0xffffffffu, xa, o), yn = __shfl_up_sync(0xffffffffu, xn, o);
            if (lane >= o) { xa += ya; xn += yn; }
        }
        if (lane == 31) { w_al[warp] = xa; w_ln[warp] = xn; }
        __syncthreads();
        long long pa = base_al, pn = base_ln;
        for (int w = 0; w < kStepThreads / 32; ++w) {
            if (w < warp) { pa += w_al[w]; pn += w_ln[w]; }
            base_al += w_al[w]; base_ln += w_ln[w];
        }
        if (r < N) {
            first[r] = sat(pa + xa - al); cum[r] = sat(pn + xn - n);
            // tokens past the row's end; a run's gap, or padding, may reach beyond it
            if (blockIdx.x == 0 && n > 0 && pa + xa - al + n > prm.row_tokens && prm.slots[r] != 0) raise_status(prm.status, FPKV_STATUS_BAD_POS);
        }
        __syncthreads();
    }
    if (tid == 0) { first[N] = sat(base_al); cum[N] = sat(base_ln); }
    __syncthreads();

    const int step = gridDim.x * kStepThreads, at = blockIdx.x * kStepThreads + tid;
    // ---- the packed row ------------------------------------------------------
    const int used = N > 0 ? first[N] : 0;
    for (int t = at; t < prm.row_tokens; t += step) {
        long long id = prm.pad_id, pos = 0, slot = 0, row = -1;
        if (t < used) {
            // the request of the warp's first token, by bisection (the same reads for all lanes), then on from there
            int lo = 0, hi = N;                                 // first[lo] <= t0 < first[hi]
            const int t0 = t - lane;
            while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (first[mid] <= t0) lo = mid; else hi = mid; }
            while (first[lo + 1] <= t) ++lo;
            const int i = t - first[lo];
            if (i < cum[lo + 1] - cum[lo]) {
                const long long s = prm.slots[lo];
                const unsigned p = (unsigned)prm.starts[lo] + (unsigned)i, page = p / (unsigned)prm.P;       // both below 2^31
                if (s < 0 || s >= prm.max_batch) raise_status(prm.status, FPKV_STATUS_BAD_SLOT);
                else if (s > 0) {
                    slot = s; pos = p;
                    if (page >= (unsigned)prm.n_pages) raise_status(prm.status, FPKV_STATUS_BAD_POS);
                    else {
                        const long long pg = prm.page_table[s * prm.n_pages + page];
                        if (pg >= 0 && pg < prm.n_pages) row = pg * prm.P + (p - page * (unsigned)prm.P);
                        else raise_status(prm.status, FPKV_STATUS_BAD_PAGE);
                    }
                    const long long k = (long long)cum[lo] + i;
                    if (prm.out.input_ids != nullptr) {
                        if (k < prm.n_tokens) id = prm.tokens[k];
                        else raise_status(prm.status, FPKV_STATUS_BAD_POS);
                    }
                }
            }
        }
        if (prm.out.input_ids != nullptr) prm.out.input_ids[t] = id;
        if (prm.out.input_pos != nullptr) prm.out.input_pos[t] = pos;
        if (prm.out.batch_idx != nullptr) prm.out.batch_idx[t] = slot;
        if (prm.out.pool_row != nullptr) prm.out.pool_row[t] = row;
    }
    // ---- block tables --------------------------------------------------------
    if (prm.out.block_table != nullptr) {
        const long long cells = (long long)N * prm.width;
        for (long long c = at; c < cells; c += step) {
            const unsigned r = cells < (1ll << 32) ? (unsigned)c / (unsigned)prm.width : (unsigned)(c / prm.width);
            const int j = (int)(c - (long long)r * prm.width);
            const long long s = prm.slots[r];
            const int len = prm.lens[r], st = prm.starts[r];
            int pg = -1;
            if (s > 0 && s < prm.max_batch && len >= 0 && st >= 0 && (long long)j * prm.P < (long long)st + len && j < prm.n_pages) {
                const long long v = prm.page_table[s * prm.n_pages + j];
                if (v >= 0 && v < prm.n_pages) pg = (int)v;
            }
            prm.out.block_table[c] = pg;
        }
    }
    // ---- per request ---------------------------------------------------------
    for (int r = at; r <= N; r += step) {
        if (prm.out.offsets != nullptr) prm.out.offsets[r] = first[r];
        if (r == N) break;
        const int n = cum[r + 1] - cum[r];
        if (prm.out.seq_lens != nullptr) prm.out.seq_lens[r] = (prm.lens[r] < 0 || prm.starts[r] < 0) ? 0 : sat((long long)prm.starts[r] + prm.lens[r]);
        if (prm.out.last != nullptr) prm.out.last[r] = (n > 0 && (long long)first[r] + n <= prm.row_tokens) ? first[r] + n - 1 : -1;
    }
}

}  // namespace

int launch_step_tables(const PoolView& pv, const int64_t* slots, const int32_t* starts, const int32_t* lens, int n_req,
                       int row_tokens, int align, int width, const int64_t* tokens, int64_t n_tokens, int64_t pad_id,
                       const fpkv_step_out& out, int32_t* status, cudaStream_t stream)
{
    StepParams prm;
    prm.page_table = pv.page_table; prm.slots = slots; prm.starts = starts; prm.lens = lens;
    prm.tokens = tokens; prm.n_tokens = n_tokens; prm.pad_id = pad_id; prm.out = out; prm.status = status;
    prm.n_req = n_req; prm.row_tokens = row_tokens; prm.align = align; prm.width = width;
    prm.n_pages = pv.n_pages; prm.max_batch = pv.max_batch; prm.P = pv.P;
    const long long items = (long long)row_tokens + (long long)n_req * width + n_req + 1;
    const long long want = (items + kStepThreads - 1) / kStepThreads;
    // Every CTA scans all lengths: four an SM (512 requests, 790 K tokens, caches cold: 18 us; two an SM 26, eight 21).
    const int grid = (int)(want < 4 * 148 ? want : 4 * 148);
    step_tables_kernel<<<grid, kStepThreads, 2 * (n_req + 1) * (int)sizeof(int), stream>>>(prm);
    return cudaGetLastError() == cudaSuccess ? FPKV_OK : FPKV_ELAUNCH;
}

}  // namespace fpkv
