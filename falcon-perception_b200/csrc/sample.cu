// Token sampling: temperature, top-k, top-p and min-p from one given uniform number a row.
//
// All filters keep a leading part of the row ordered by (value descending, index ascending).  That order is the order
// of one 64-bit number a entry -- the order-preserving integer image of the value above the inverted index -- so the
// kept set is everything at or above a threshold number, whatever mixture of filters made it.
//
// A row belongs to a cluster of 1 to 8 CTAs, each with a slice of the vocabulary in its shared memory: the logits are
// read from memory once.  Steps, with a cluster barrier behind each:
//   1. slices to shared memory (NaN becomes -inf, -0 becomes 0), largest and smallest value
//   2. top-k.  A small k: of every thread's largest value the k-th largest has k entries at or above it and hardly more;
//      those are collected and sorted, and the first CTA does the rest of the row on that list.  A large k: counts over 1024
//      even bins, then the entries of the bin of the k-th.
//   3. top-p: 32-bit sums of the weights over 16 wide bins, private to each thread (atomics of all entries on shared memory
//      took seven times as long), then counts over 1024 bins around the border; the entries around it are collected
//   4. weights exp((x - max) / T) in 64 bits and their sums over chunks of the slice; for top-p the collected entries are
//      sorted and added up behind the exact sum of all larger ones, and the guess of step 3 is checked by it
//   5. the slice, the chunk and then the entry in which the running sum passes u times the sum
// A value that more entries share than are collected is narrowed down to and its entries are counted off by index.
// Where a guess fails all the same, the threshold value is found by bisection, one sum over the slices a step.
//
// Sums are 64-bit and weights good to 1.5e-13: the token is the answer, and which one it is may hang on the last bits of a
// sum over the vocabulary (32-bit sums would draw another token in about one row of a hundred at 65536 flat entries).  The
// 64-bit pipe has half the lanes of the 32-bit one, so the exponential is the table-and-polynomial one below: 12 operations.
// No result depends on the order in which atomics arrive: counts are integers, collected entries are sorted.
//
// What bounds it: a few rows (1 x 65536 with top-p: 31 us) the chain of about ten barriers and lookups; many rows (512 x
// 131072 in 32 bits, 268 MB, 41 us of memory, 537 us) the instructions an entry takes, 139 with these settings -- about 15 to
// load and compare it, 25 for the wide bins, 10 for the counts, 50 for the 64-bit weight, and the searches -- which fill 52 % of
// the issue slots of 29 warps an SM; the rest is waiting at barriers (a fifth of the stalls) and for the slice.

#include "common.cuh"

namespace fpkv {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kWide = 16;                                // bins private to a thread; the last one is "behind"
constexpr int kFine = 1024;                              // counted bins
constexpr int kCand = kThreads;                          // entries collected and sorted at a time, over the cluster: one a thread
constexpr int kAround = 64;                              // entries collected on either side of the top-p border
constexpr int kMaxChunks = kThreads;                     // chunks of a slice, one thread each in the final search
constexpr int kMaxCluster = 8;
constexpr int kMaxSmem = 220 * 1024;
constexpr uint32_t kKeyNone = 0x007fffffu;               // image of -inf: never drawn

struct SampleParams {
    const void* logits;
    const float* uniform;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int64_t* token;
    float* logprob;
    long long row_stride;
    int vocab;
    int slice_vecs;                                      // 16-byte pieces of a row per CTA, a multiple of chunk_vecs
    int chunk_vecs;                                      // 16-byte pieces per chunk, a multiple of 32
};

// Integer image of a value that is neither NaN nor -0, and back: larger value, larger image.  Compared as integers,
// subnormal values keep their order.
__device__ __forceinline__ uint32_t key_of(uint32_t bits) { return bits ^ ((uint32_t)((int)bits >> 31) | 0x80000000u); }
__device__ __forceinline__ uint32_t bits_of(uint32_t key) { return (key & 0x80000000u) ? (key ^ 0x80000000u) : ~key; }
// The value in 64 bits, put together from its bits (the conversion unit is a quarter as wide as the 64-bit pipe).  Zero and
// subnormal values come out up to 2^-126 off, which is nothing next to any other value or temperature.
__device__ __forceinline__ double value_of(uint32_t u) {
    return __hiloint2double((int)((u & 0x80000000u) | (((u & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(u << 29));
}

// 16-byte pieces of a row.  `entry`: 32-bit value bits of entry e.  `clean`: NaN to -inf, -0 to 0.
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr uint32_t kMinusInf = 0xff800000u;
    static __device__ __forceinline__ uint32_t entry(const uint4& v, int e) { return (&v.x)[e]; }
    static __device__ __forceinline__ uint32_t clean(uint32_t u) {
        if ((u & 0x7fffffffu) > 0x7f800000u) return kMinusInf;
        return u == 0x80000000u ? 0u : u;
    }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr uint32_t kMinusInf = 0xff80u;
    static __device__ __forceinline__ uint32_t entry(const uint4& v, int e) {
        const uint32_t w = (&v.x)[e >> 1];
        return (e & 1) ? (w & 0xffff0000u) : (w << 16);
    }
    static __device__ __forceinline__ uint32_t clean1(uint32_t h) { return (h & 0x7fffu) > 0x7f80u ? kMinusInf : (h == 0x8000u ? 0u : h); }
    static __device__ __forceinline__ uint32_t clean(uint32_t u) { return clean1(u & 0xffffu) | (clean1(u >> 16) << 16); }
};
template <> struct Piece<__half> {
    static constexpr uint32_t kMinusInf = 0xfc00u;
    static __device__ __forceinline__ uint32_t entry(const uint4& v, int e) {
        const uint32_t w = (&v.x)[e >> 1];
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)((e & 1) ? (w >> 16) : (w & 0xffffu)))));
    }
    static __device__ __forceinline__ uint32_t clean1(uint32_t h) { return (h & 0x7fffu) > 0x7c00u ? kMinusInf : (h == 0x8000u ? 0u : h); }
    static __device__ __forceinline__ uint32_t clean(uint32_t u) { return clean1(u & 0xffffu) | (clean1(u >> 16) << 16); }
};

// ---- cluster ---------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same variable in the shared memory of CTA `rank` of the cluster.
template <typename V> __device__ __forceinline__ V peer(const V* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    V v;
    if constexpr (sizeof(V) == 8) {
        unsigned long long x;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(a) : "memory");
        memcpy(&v, &x, 8);
    } else {
        uint32_t x;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
        memcpy(&v, &x, 4);
    }
    return v;
}

struct __align__(16) Shared {
    union {
        float wide[kWide][kThreads];                     // step 3's private bins
        struct {
            unsigned long long list[kCand];              // this CTA's collected entries
            unsigned long long all[kCand];               // the cluster's, sorted
            uint32_t hist[kFine];                        // counts of the slice
        };
    };
    double exp_table[16];                                // 2^(i/16): one entry a pair of banks, no access of it conflicts
    double chunk_sum[kMaxChunks];
    unsigned long long chunk_extra[kMaxChunks];          // kept border entries of a chunk, in units of 2^-52
    double red_d[3 * kWarps];
    double pub_d[5];                                     // published to the peers: sums
    unsigned long long red_l[kWarps];
    unsigned long long pub_max;
    float wide_sum[kWide];                               // published: the CTA's sums over the wide bins
    uint32_t pub_low, pub_bound, pub_tops, pub_n, pub_ties;
    uint32_t red_u[kWarps], red_v[kWarps];
    uint32_t n_list;
    int at[16];
};

template <typename V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename V> __device__ __forceinline__ V warp_scan(V v) {          // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const V y = __shfl_up_sync(0xffffffffu, v, o); if ((threadIdx.x & 31) >= o) v += y; }
    return v;
}
// Sum over the CTA, the same bits in every thread.  Ends with every thread past its reads of `s`.
template <typename V> __device__ __forceinline__ V block_sum(V v, V* s) {
    v = warp_sum(v);
    if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
    __syncthreads();
    V t = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += s[w];
    __syncthreads();
    return t;
}
// Three sums at once.
__device__ __forceinline__ void block_sum3(double& a, double& b, double& c, double* s) {
    a = warp_sum(a); b = warp_sum(b); c = warp_sum(c);
    if (threadIdx.x % 32 == 0) { double* t = s + 3 * (threadIdx.x / 32); t[0] = a; t[1] = b; t[2] = c; }
    __syncthreads();
    a = b = c = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { a += s[3 * w]; b += s[3 * w + 1]; c += s[3 * w + 2]; }
    __syncthreads();
}
// Running sum over the CTA's threads, this thread's own included; *total gets the whole.  Ends as block_sum does.
template <typename V> __device__ __forceinline__ V block_scan(V v, V* s, V* total) {
    v = warp_scan(v);
    if (threadIdx.x % 32 == 31) s[threadIdx.x / 32] = v;
    __syncthreads();
    V t = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { if (w < (int)threadIdx.x / 32) v += s[w]; t += s[w]; }
    *total = t;
    __syncthreads();
    return v;
}

// Sorts the first n numbers of a (n <= kCand), largest first, and gives each thread the one at its place (0 past the n-th).
// Bitonic, one number a thread: exchanges inside a warp by shuffle, the others through `a`.
__device__ __forceinline__ unsigned long long sort_numbers(unsigned long long* a, int n) {
    const int i = threadIdx.x;
    int size = 32;
    while (size < n) size *= 2;
    unsigned long long x = i < n ? a[i] : 0ull;
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            unsigned long long y;
            if (j >= 32) {
                __syncthreads();
                a[i] = x;
                __syncthreads();
                y = a[i ^ j];
            } else {
                y = __shfl_xor_sync(0xffffffffu, x, j);
            }
            const bool first = (i & j) == 0, falling = (i & k) == 0;
            x = ((x > y) == (first == falling)) ? x : y;
        }
    __syncthreads();
    a[i] = x;
    __syncthreads();
    return x;
}

template <typename T, bool kStaged>
__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const SampleParams prm)
{
    using Pc = Piece<T>;
    constexpr int VE = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    uint4* slice = reinterpret_cast<uint4*>(smem + sizeof(Shared));
    const uint32_t C = cluster_size(), rank = cluster_rank();
    const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid / 32, lane = tid % 32, V = prm.vocab;
    // The row as 16-byte pieces of memory; the first and last may reach beyond it.
    const T* x = reinterpret_cast<const T*>(prm.logits) + (long long)row * prm.row_stride;
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));       // entries of the first piece before the row
    const int row_vecs = (off + V + VE - 1) / VE;
    const int v0 = (int)rank * prm.slice_vecs, nv = max(0, min(prm.slice_vecs, row_vecs - v0));
    const int i0 = v0 * VE - off;                        // index of the slice's first entry (may be negative: not of the row)
    auto from_memory = [&](int v) -> uint4 {
        const int i = i0 + v * VE;
        uint4 r;
        if (i >= 0 && i + VE <= V) r = __ldg(reinterpret_cast<const uint4*>(x + i));
        else {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    w[k] = i + k >= 0 && i + k < V ? reinterpret_cast<const uint32_t*>(x)[i + k] : Pc::kMinusInf;
                } else {
                    const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
                    const uint32_t lo = i + 2 * k >= 0 && i + 2 * k < V ? h[i + 2 * k] : Pc::kMinusInf;
                    const uint32_t hi = i + 2 * k + 1 >= 0 && i + 2 * k + 1 < V ? h[i + 2 * k + 1] : Pc::kMinusInf;
                    w[k] = lo | (hi << 16);
                }
            }
            r = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return make_uint4(Pc::clean(r.x), Pc::clean(r.y), Pc::clean(r.z), Pc::clean(r.w));
    };
    auto piece = [&](int v) -> uint4 { if constexpr (kStaged) return slice[v]; else return from_memory(v); };
    // f(bits, index) for every entry of the slice, -inf ones and those beyond the row (which read as -inf) included
    auto each = [&](auto f) {
        for (int v = tid; v < nv; v += kThreads) {
            const uint4 d = piece(v);
#pragma unroll
            for (int e = 0; e < VE; ++e) f(Pc::entry(d, e), i0 + v * VE + e);
        }
    };
    // one number a entry that orders the row
    auto number = [&](uint32_t key, int i) { return ((unsigned long long)key << 32) | (uint32_t)~i; };

    // ---- 1. the slice; its largest entry, its smallest value above -inf, the smallest of its threads' largest values, and how
    // many threads have one (the last slice is short, and masked ones read nothing else than -inf) ----
    const float temp = prm.temperature != nullptr ? prm.temperature[row] : 1.f;
    const float p_top = prm.top_p != nullptr ? prm.top_p[row] : 1.f;
    const int k_top = prm.top_k != nullptr ? prm.top_k[row] : 0;
    const float p_min = prm.min_p != nullptr ? prm.min_p[row] : 0.f;
    // A goal below zero would end the search in a slice, or chunk, without any kept entry.  NaN gives 0 too.
    const double u = fmax((double)prm.uniform[row], 0.0);
    unsigned long long best = 0;
    uint32_t low = 0xffffffffu, bound = 0xffffffffu;
    uint32_t top = 0;                                    // image of this thread's largest value
    {
        int at = 0;
        for (int v = tid; v < nv; v += kThreads) {
            const uint4 d = from_memory(v);
            if constexpr (kStaged) slice[v] = d;
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const uint32_t key = key_of(Pc::entry(d, e));
                if (key > top) { top = key; at = i0 + v * VE + e; }
                if (key > kKeyNone) low = min(low, key);
            }
        }
        if (top > kKeyNone) best = number(top, at);
        if (top > kKeyNone) bound = top;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
        best = y > best ? y : best;
    }
    low = __reduce_min_sync(0xffffffffu, low);
    bound = __reduce_min_sync(0xffffffffu, bound);
    uint32_t tops = __popc(__ballot_sync(0xffffffffu, top > kKeyNone));
    if (lane == 0) { sh.red_l[warp] = best; sh.red_u[warp] = low; sh.red_v[warp] = bound; sh.at[warp] = (int)tops; }
    if (tid < 16) sh.exp_table[tid] = exp2((double)tid * 0.0625);
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    // exchange between the CTAs: lane r reads from CTA r
    const uint32_t from = min((uint32_t)lane, C - 1);
    if (warp == 0) {
        best = sh.red_l[lane % kWarps]; low = sh.red_u[lane % kWarps]; bound = sh.red_v[lane % kWarps];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
            const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
            best = y > best ? y : best;
        }
        low = __reduce_min_sync(0xffffffffu, low);
        bound = __reduce_min_sync(0xffffffffu, bound);
        tops = __reduce_add_sync(0xffffffffu, lane < kWarps ? (uint32_t)sh.at[lane] : 0u);
        if (lane == 0) { sh.pub_max = best; sh.pub_low = low; sh.pub_bound = bound; sh.pub_tops = tops; }
    }
    cluster_sync();
    best = peer(&sh.pub_max, from);
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
        best = y > best ? y : best;
    }
    low = __reduce_min_sync(0xffffffffu, peer(&sh.pub_low, from));
    bound = __reduce_min_sync(0xffffffffu, peer(&sh.pub_bound, from));
    tops = __reduce_add_sync(0xffffffffu, lane < (int)C ? peer(&sh.pub_tops, from) : 0u);
    best = __shfl_sync(0xffffffffu, best, 0);
    const uint32_t kmax = (uint32_t)(best >> 32);
    if (best == 0 || !(temp > 0.f)) {                    // the same for the whole cluster
        if (rank == 0 && tid == 0) {
            prm.token[row] = best != 0 ? (long long)(uint32_t)~(uint32_t)best : -1;
            if (prm.logprob != nullptr) prm.logprob[row] = best != 0 ? 0.f : -INFINITY;
        }
        cluster_sync();                                  // nobody leaves while a peer may read its shared memory
        return;
    }

    // Weight of a value: 2^y with y = (x - max) log2(e) / T.  y = n + i / 16 + r with |r| <= 1/32; 2^r by its series up to r^5
    // (the next term is 1.5e-13 at most), 2^(i/16) from the table, 2^n into the exponent.  An infinite maximum leaves every
    // other value without weight.
    const bool endless = bits_of(kmax) == 0x7f800000u;
    const double xmax = value_of(bits_of(kmax)), slope = endless ? 1e300 : 1.4426950408889634074 / (double)temp;
    auto weight = [&](uint32_t bits) -> double {
        const double y = (value_of(bits) - xmax) * slope;
        const uint32_t hi = (uint32_t)__double2hiint(y);
        const double big = 422212465065984.0;            // 1.5 * 2^48: the sum's last place is 2^-4
        const double t = y + big;
        const int n = __double2loint(t);
        const double r = y - (t - big);
        double s = fma(r, 0.0013333558146428443, 0.0096181291076284772);       // ln(2)^k / k!
        s = fma(s, r, 0.0555041086648215800);
        s = fma(s, r, 0.2402265069591007123);
        s = fma(s, r, 0.6931471805599453094);
        s = fma(s, r, 1.0);
        const double w = s * sh.exp_table[n & 15];
        // no branch, so that several entries' chains overlap: 2^n in two factors, the second one below 1 for subnormal weights
        const int e = n >> 4, e1 = max(e, -1000);
        const double scaled = __hiloint2double(__double2hiint(w) + (e1 << 20), __double2loint(w)) * __hiloint2double((1023 + max(e - e1, -90)) << 20, 0);
        return hi >= 0xC0910000u ? 0.0 : scaled;         // y <= -1088, or no number at all
    };
    // Smallest image at which `holds` is true, which it stays for all larger ones; kmax + 1 if for none.  The lanes of each
    // warp probe 32 places at a time.
    // Looked for between near_lo and near_hi first.
    auto first_key = [&](auto holds, uint32_t near_lo, uint32_t near_hi) -> uint32_t {
        uint32_t lo = kKeyNone + 1u, hi = kmax + 1u;     // the answer is in [lo, hi]
        if (near_lo >= lo && near_hi < hi && near_lo < near_hi) {
            const uint32_t yes = __ballot_sync(0xffffffffu, holds(lane == 0 ? near_lo : near_hi));
            if ((yes & 3u) == 2u) { lo = near_lo + 1u; hi = near_hi; }
        }
        while (lo < hi) {
            const uint32_t step = (hi - lo) / 32u + 1u, at = lo + (uint32_t)lane * step;
            const uint32_t yes = __ballot_sync(0xffffffffu, at < hi ? holds(at) : true);
            const int f = yes ? __ffs(yes) - 1 : 32;     // the lanes below f say no
            hi = f < 32 ? min(hi, lo + (uint32_t)f * step) : hi;
            if (f > 0) lo += (uint32_t)(f - 1) * step + 1u;
        }
        return lo;
    };
    // smallest image that min_p keeps
    const double least = fmin((double)p_min, 1.0);
    const uint32_t k_least = p_min > 0.f ? first_key([&](uint32_t key) { return weight(bits_of(key)) >= least; }, 0u, 0u) : 0u;
    const unsigned long long n_least = (unsigned long long)k_least << 32;
    const bool by_k = k_top > 0 && k_top < V, by_p = p_top < 1.f;

    // ---- bins go by the distance from the maximum in 32 bits, which does not decrease as the value falls ------------
    const float fmx = __uint_as_float(bits_of(kmax)), fslope = (float)slope;
    // Cut off where one over it is still a normal number, for the bins divide by it.
    auto distance = [&](uint32_t bits) { return key_of(bits) == kmax ? 0.f : fminf(fmx - __uint_as_float(bits), 8e37f); };
    // Images around the value at a distance from the maximum, a few roundings to either side.
    auto near = [&](float d, bool above) {
        const float x_ = fmx - d, slack = 4e-7f * (fabsf(fmx) + d);
        return key_of(__float_as_uint(above ? x_ + slack : x_ - slack));
    };
    // Fine bins: the images in [k_first, k_last], even in the distance; -1 above them, kFine below.  With k_split, no bin holds
    // images on both sides of it: those below it start with bin split_bin.
    uint32_t k_first = 0, k_last = 0, k_split = 0;
    int split_bin = 0;
    float start = 0.f, per = 0.f;
    auto span = [&](uint32_t first, uint32_t last) {
        k_first = first; k_last = last; k_split = 0; split_bin = 0;
        start = distance(bits_of(last));
        per = (float)kFine * 0.999f / fmaxf(distance(bits_of(first)) - start, 1e-30f);
    };
    auto fine_of = [&](uint32_t key) -> int {
        if (key > k_last) return -1;
        if (key < k_first) return kFine;
        const int b = max(0, min((int)((distance(bits_of(key)) - start) * per), kFine - 1));
        return key < k_split ? max(b, split_bin) : b;
    };
    // Smallest image whose fine bin is at most b.
    auto edge = [&](int b) -> uint32_t {
        if (b < 0) return k_last + 1u;
        if (b >= kFine - 1) return b < kFine ? k_first : 0u;
        if (k_split != 0 && b == split_bin - 1) return k_split;
        const float d = start + (float)(b + 1) / per;
        return first_key([&](uint32_t key) { return fine_of(key) <= b; }, near(d, false), near(d, true));
    };
    auto collect = [&](unsigned long long n) {
        const uint32_t slot = atomicAdd(&sh.n_list, 1u);
        if (slot < (uint32_t)kCand) sh.list[slot] = n;
    };
    // All collected entries of the cluster into sh.all, sorted; returns how many (more than kCand: nothing copied).  *own is
    // the one at this thread's place.
    unsigned long long own_number = 0;
    auto gather = [&]() -> int {
        __syncthreads();
        if (tid == 0) sh.pub_n = sh.n_list;
        cluster_sync();
        const uint32_t m = lane < (int)C ? peer(&sh.pub_n, from) : 0u;
        const uint32_t n = __reduce_add_sync(0xffffffffu, min(m, (uint32_t)kCand + 1u));
        if (n > (uint32_t)kCand) return kCand + 1;
        const uint32_t before = warp_scan(m) - m;
        // this thread fetches the tid-th of them
        uint32_t src = 0, at = 0;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            const uint32_t b = __shfl_sync(0xffffffffu, before, r);
            if (r < (int)C && (uint32_t)tid >= b) { src = (uint32_t)r; at = (uint32_t)tid - b; }
        }
        unsigned long long x = 0;
        if ((uint32_t)tid < n) x = peer(&sh.list[at], src);
        __syncthreads();
        sh.all[tid] = x;
        own_number = sort_numbers(sh.all, (int)n);
        return (int)n;
    };
    // Counts over the fine bins, added up over the cluster: this thread's bins 2 tid and 2 tid + 1, and the running count
    // before them.  `add` counts this CTA's part into sh.hist.
    uint32_t c0 = 0, c1 = 0, c_before = 0;
    auto count = [&](auto add) {
        for (int i = tid; i < kFine; i += kThreads) sh.hist[i] = 0;
        __syncthreads();
        add();
        cluster_sync();
        unsigned long long y[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
            y[r] = r < (int)C ? peer(reinterpret_cast<const unsigned long long*>(sh.hist) + tid, r) : 0ull;
        c0 = c1 = 0;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) { c0 += (uint32_t)y[r]; c1 += (uint32_t)(y[r] >> 32); }
        uint32_t total;
        c_before = block_scan(c0 + c1, sh.red_u, &total) - c0 - c1;
    };
    // A sum over the cluster, in rank order: the same bits everywhere.
    auto over_cluster = [&](const double* published) {
        const double v = lane < (int)C ? peer(published, from) : 0.0;
        double t = 0;
        for (uint32_t r = 0; r < C; ++r) t += __shfl_sync(0xffffffffu, v, r);
        return t;
    };
    auto cluster_sum = [&](double part) -> double {
        part = block_sum(part, sh.red_d);
        cluster_sync();                                  // peers are past their reads of the last sum
        if (tid == 0) sh.pub_d[3] = part;
        cluster_sync();
        return over_cluster(&sh.pub_d[3]);
    };
    // Largest image at which `measure`, a sum over the entries at or above it, reaches the goal; *above is the sum over the
    // larger ones.  `lo` reaches it.
    auto bisect = [&](uint32_t lo, auto measure, double goal_, double* above) -> uint32_t {
        uint32_t hi = kmax;
        *above = 0;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            const double m = cluster_sum(measure(mid));
            if (m >= goal_) lo = mid; else { hi = mid - 1; *above = m; }
        }
        return lo;
    };
    const unsigned long long everything = (unsigned long long)(kKeyNone + 1u) << 32;      // every entry above -inf
    auto at_or_above = [&](uint32_t key, int i, unsigned long long thr) {
        return key > (uint32_t)(thr >> 32) || (key == (uint32_t)(thr >> 32) && number(key, i) >= thr);
    };
    auto count_entries = [&](unsigned long long thr) {   // the slice's, at or above thr, into sh.hist
        each([&](uint32_t bits, int i) {
            const uint32_t key = key_of(bits);
            if (key < k_first || key > k_last || !at_or_above(key, i, thr)) return;
            atomicAdd(&sh.hist[fine_of(key)], 1u);
        });
    };
    // Chunks of the slice, a warp each: `f(chunk, bits, index)` for every entry, then `done(chunk)`.
    const int n_chunks = (nv + prm.chunk_vecs - 1) / prm.chunk_vecs;
    auto each_chunk = [&](auto f, auto done) {
        for (int c = warp; c < n_chunks; c += kWarps) {
            const int end = min((c + 1) * prm.chunk_vecs, nv);
            for (int v = c * prm.chunk_vecs + lane; v < end; v += 32) {
                const uint4 d = piece(v);
#pragma unroll
                for (int e = 0; e < VE; ++e) f(Pc::entry(d, e), i0 + v * VE + e);
            }
            done(c);
        }
    };
    // The same, a piece at a time: f(chunk, piece, index of its first entry).
    auto each_piece = [&](auto f, auto done) {
        for (int c = warp; c < n_chunks; c += kWarps) {
            const int end = min((c + 1) * prm.chunk_vecs, nv);
            for (int v = c * prm.chunk_vecs + lane; v < end; v += 32) f(piece(v), i0 + v * VE);
            done(c);
        }
    };
    // Number of the n-th entry (from 1, in vocabulary order) among those whose image is `key`; n of them are there.
    auto nth_equal = [&](uint32_t key, uint32_t n) -> unsigned long long {
        uint32_t mine = 0;
        each_chunk([&](uint32_t bits, int) { mine += key_of(bits) == key; },
                   [&](int c) { mine = __reduce_add_sync(0xffffffffu, mine); if (lane == 0) sh.chunk_extra[c] = mine; mine = 0; });
        __syncthreads();
        const uint32_t own = tid < n_chunks ? (uint32_t)sh.chunk_extra[tid] : 0u;
        uint32_t total;
        uint32_t incl = block_scan(own, sh.red_u, &total);
        cluster_sync();
        if (tid == 0) sh.pub_ties = total;
        cluster_sync();
        const uint32_t m = lane < (int)C ? peer(&sh.pub_ties, from) : 0u;
        incl += __shfl_sync(0xffffffffu, warp_scan(m) - m, rank);
        if (tid == 0) sh.pub_max = 0;
        __syncthreads();
        if (own > 0 && incl - own < n && n <= incl) sh.at[7] = tid;
        const bool here = __syncthreads_or(own > 0 && incl - own < n && n <= incl) != 0;
        if (here) {
            if (tid == sh.at[7]) sh.at[6] = (int)(n - (incl - own));            // which of the chunk's, from 1
            __syncthreads();
            if (warp == 0) {
                int left = sh.at[6];
                const int c = sh.at[7], end = min((c + 1) * prm.chunk_vecs, nv);
                for (int vb = c * prm.chunk_vecs; vb < end && left > 0; vb += 32) {
                    const int v = vb + lane;
                    uint32_t eq = 0;
                    if (v < end) {
                        const uint4 d = piece(v);
#pragma unroll
                        for (int e = 0; e < VE; ++e) eq |= (uint32_t)(key_of(Pc::entry(d, e)) == key) << e;
                    }
                    const int have = __popc(eq), to = warp_scan(have);
                    if (to >= left && to - have < left) {
                        uint32_t rest = eq;
                        for (int k = 1; k < left - (to - have); ++k) rest &= rest - 1;
                        sh.pub_max = number(key, i0 + v * VE + __ffs(rest) - 1);
                    }
                    left -= __shfl_sync(0xffffffffu, to, 31);
                }
            }
        }
        cluster_sync();
        unsigned long long got = lane < (int)C ? peer(&sh.pub_max, from) : 0ull;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { const unsigned long long y = __shfl_xor_sync(0xffffffffu, got, o); got = y > got ? y : got; }
        return got;
    };
    // Smallest and largest image over the cluster.
    auto extremes = [&](uint32_t& lo, uint32_t& hi) {
        lo = __reduce_min_sync(0xffffffffu, lo); hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) { sh.red_u[warp] = lo; sh.red_v[warp] = hi; }
        __syncthreads();
        lo = __reduce_min_sync(0xffffffffu, sh.red_u[lane % kWarps]); hi = __reduce_max_sync(0xffffffffu, sh.red_v[lane % kWarps]);
        cluster_sync();
        if (tid == 0) { sh.pub_low = lo; sh.pub_bound = hi; }
        cluster_sync();
        lo = __reduce_min_sync(0xffffffffu, peer(&sh.pub_low, from)); hi = __reduce_max_sync(0xffffffffu, peer(&sh.pub_bound, from));
    };
    // Narrows the fine bins down to the images that the entries of bin b at or above thr have, and returns the one they share, or
    // 0 if they differ.  What is there is narrower than the bin by far where some entries lie far away -- masked by a large
    // finite value, say -- and all others in one bin.
    auto narrow = [&](int b, unsigned long long thr) -> uint32_t {
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](uint32_t bits, int i) {
            const uint32_t key = key_of(bits);
            if (key >= k_first && key <= k_last && at_or_above(key, i, thr) && fine_of(key) == b) { lo = min(lo, key); hi = max(hi, key); }
        });
        extremes(lo, hi);
        span(lo, hi);
        return lo == hi ? lo : 0u;
    };

    unsigned long long threshold = everything;
    int listed = -1;                                     // entries of sh.all if it holds everything that is kept
    // ---- 2. top-k ------------------------------------------------------------------
    if (by_k) {
        const uint32_t k = (uint32_t)k_top;
        // Every one of the `tops` threads has an entry at or above `bound`.
        const bool bounded = k <= tops;
        span(bounded ? bound : low, kmax);
        int j = -1; uint32_t in_j = 0, until_j = 0;
        // The bin of the k-th of what was counted, behind `before` others.
        auto find = [&](uint32_t before) {
            if (tid == 0) sh.at[0] = -1;
            __syncthreads();
            const uint32_t b0 = before + c_before;
            if (b0 < k && k <= b0 + c0) { sh.at[0] = 2 * tid; sh.at[1] = (int)b0; sh.at[2] = (int)c0; }
            else if (b0 + c0 < k && k <= b0 + c0 + c1) { sh.at[0] = 2 * tid + 1; sh.at[1] = (int)(b0 + c0); sh.at[2] = (int)c1; }
            __syncthreads();
            j = sh.at[0]; until_j = (uint32_t)sh.at[1]; in_j = (uint32_t)sh.at[2];
            __syncthreads();
        };
        bool all_kept = false, done = false;
        if (bounded && 4 * k <= 3 * kCand) {
            // The k-th largest of the threads' largest values has k entries at or above it, and hardly more: collect those.  A bin
            // of many values is narrowed down to them.
            uint32_t from_key = 0, before = 0;
            for (int turn = 0;; ++turn) {
                const bool counted = top >= k_first && top <= k_last;
                count([&] { if (counted) atomicAdd(&sh.hist[fine_of(top)], 1u); });
                find(before);
                if (j < 0) break;
                from_key = edge(j);
                if (in_j <= 64u || turn == 2) break;
                const bool here = counted && fine_of(top) == j;
                uint32_t lo = here ? top : 0xffffffffu, hi = here ? top : 0u;
                extremes(lo, hi);
                from_key = max(from_key, lo);
                if (lo == hi) break;
                before = until_j;
                span(lo, hi);
            }
            each([&](uint32_t bits, int i) { if (key_of(bits) >= from_key) collect(number(key_of(bits), i)); });
            done = gather() <= kCand && j >= 0;
            if (done) listed = (int)k;
            else {
                cluster_sync();                          // peers have read the number of entries
                if (tid == 0) sh.n_list = 0;
                __syncthreads();
                span(from_key, kmax);                    // which holds k entries
            }
        }
        if (!done) {
            uint32_t before = 0, one = 0;                // entries before the fine bins; the value that fills bin j
            for (int turn = 0;; ++turn) {
                count([&] { count_entries(everything); });
                find(before);
                if (j < 0) { all_kept = turn == 0; break; }              // fewer than k entries above -inf: no limit
                if (in_j <= (uint32_t)kCand) break;
                one = narrow(j, everything);
                before = until_j;
                if (one != 0 || turn == 3) break;
            }
            if (j >= 0 && in_j <= (uint32_t)kCand) {
                const uint32_t from_key = edge(j), to_key = edge(j - 1);
                each([&](uint32_t bits, int i) {
                    const uint32_t key = key_of(bits);
                    if (key >= from_key && key < to_key) collect(number(key, i));
                });
                gather();
                threshold = sh.all[k - until_j - 1];
            } else if (!all_kept) {
                if (one != 0) threshold = nth_equal(one, k - until_j);
                else {
                    double above;
                    const uint32_t key = bisect(kKeyNone + 1u, [&](uint32_t from_) {
                        double m = 0;
                        each([&](uint32_t bits, int) { m += key_of(bits) >= from_ ? 1.0 : 0.0; });
                        return m;
                    }, (double)k, &above);
                    threshold = nth_equal(key, k - (uint32_t)above);
                }
            }
        }
        cluster_sync();                                  // lists and counts have been read
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
    }
    if (listed >= 0) {
        // ---- everything kept is in the sorted list of every CTA: the first one finishes the row --------------------
        if (rank == 0) {
            double w = tid < listed ? weight(bits_of((uint32_t)(own_number >> 32))) : 0.0, total;
            const double before = block_scan(w, sh.red_d, &total) - w;
            const bool keep = tid < listed && (tid == 0 || !by_p || before < (double)p_top * total) && own_number >= n_least;
            const int kept = __syncthreads_count(keep);  // a leading run
            // in vocabulary order: the inverted index above the value's image
            sh.list[tid] = keep ? (own_number << 32) | (own_number >> 32) : 0ull;
            __syncthreads();
            const unsigned long long mine = sort_numbers(sh.list, kept);
            w = tid < kept ? weight(bits_of((uint32_t)mine)) : 0.0;
            const double to = block_scan(w, sh.red_d, &total), goal = u * total;
            if (tid == 0) { sh.at[0] = kCand; sh.at[1] = 0; }
            __syncthreads();
            if (w > 0) {
                if (to > goal) atomicMin(&sh.at[0], tid);
                atomicMax(&sh.at[1], tid);
            }
            __syncthreads();
            if (tid == (sh.at[0] < kCand ? sh.at[0] : sh.at[1])) {
                prm.token[row] = (long long)(uint32_t)~(uint32_t)(mine >> 32);
                if (prm.logprob != nullptr) prm.logprob[row] = (float)log(w / total);
            }
        }
        return;                                          // peers' shared memory was last read before the barrier above
    }

    // ---- 3. top-p: where the border lies -------------------------------------------------------
    int p_lo = kFine + 1, p_hi = kFine + 1;              // fine bins below p_lo are surely kept, those up to p_hi are collected
    uint32_t tie = 0;                                    // or: the one value on which the border lies
    bool lost = false;                                   // or: no guess
    if (by_p) {
        // Whatever weighs less than (1 - p) / (2 V) of the maximum cannot be kept: all of it together is less than the part
        // that is dropped.
        const float far = fminf(fminf(distance(bits_of(low)), temp * logf(2.f * (float)V / (1.f - p_top))), 1e37f);
        const float per_wide = (float)(kWide - 1) / fmaxf(far, 1e-30f);
        auto wide_of = [&](uint32_t key) { return (int)fminf(distance(bits_of(key)) * per_wide, (float)(kWide - 1)); };
#pragma unroll
        for (int b = 0; b < kWide; ++b) sh.wide[b][tid] = 0.f;
        each([&](uint32_t bits, int i) {
            if (!at_or_above(key_of(bits), i, threshold)) return;
            const float d = distance(bits);
            const float w = d > 0.f ? exp2f(-d * fslope) : 1.f;
            sh.wide[wide_of(key_of(bits))][tid] += w;
        });
        __syncthreads();
        {   // a warp a bin
            float t = 0.f;
            for (int i = lane; i < kThreads; i += 32) t += sh.wide[warp][i];
            t = warp_sum(t);
            if (lane == 0) sh.wide_sum[warp] = t;
        }
        cluster_sync();
        float mass = 0.f;                                // lane b: bin b
        if (lane < kWide) {
            float y[kMaxCluster];
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) y[r] = r < (int)C ? peer(&sh.wide_sum[lane], r) : 0.f;
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) mass += y[r];
        }
        if (lane == 0) mass = fmaxf(mass, 1.f);
        const float upto = warp_scan(mass), goal = fmaxf(p_top, 0.f) * __shfl_sync(0xffffffffu, upto, kWide - 1);
        const uint32_t past = __ballot_sync(0xffffffffu, lane < kWide && upto >= goal);
        const int wb = past ? __ffs(past) - 1 : kWide - 1;
        float mass_before = __shfl_sync(0xffffffffu, upto - mass, wb);       // weight of everything above it
        // fine bins over the images of that wide bin and half a bin on either side, where the border may be after all
        auto at_distance = [&](float d) {                // smallest image at most that far from the maximum
            return first_key([&](uint32_t key) { return distance(bits_of(key)) <= d; }, near(d, false), near(d, true));
        };
        const float width = 1.f / per_wide;
        const float from_d = (float)wb * width;          // where `mass_before` ends
        span(wb < kWide - 1 ? at_distance(((float)wb + 1.5f) * width) : low, wb > 0 ? at_distance(((float)wb - 0.5f) * width) - 1u : kmax);
        // The fine bins are cut where that wide bin starts.  A bin told by its middle to lie before or behind that place may be
        // a whole class of equal 16-bit values on the wrong side (32 to 79 of them in the rows seen, heavier than those at the
        // border), and the guess then misses: 11 rows in 3840 went to the bisection, and 10 batches of 60 (64 rows of 65536,
        // bf16) took 300 us instead of 64; none does with the cut.
        if (wb > 0) {
            const uint32_t at = first_key([&](uint32_t key) { return wide_of(key) < wb; }, near(from_d, false), near(from_d, true));
            const int b = at > k_last ? -1 : fine_of(at);
            if (b < kFine - 1) { split_bin = b + 1; k_split = b < 0 ? 0u : at; }
        }
        for (int turn = 0; turn < 4; ++turn) {
            count([&] { count_entries(threshold); });
            if (tid == 0) { sh.at[0] = sh.at[3] = kFine; sh.at[4] = sh.at[7] = sh.at[8] = sh.at[10] = -1; sh.at[6] = sh.at[9] = sh.at[11] = 0; }
            __syncthreads();
            const float d0 = start + ((float)(2 * tid) + 0.5f) / per, d1 = start + ((float)(2 * tid) + 1.5f) / per;
            const float m0 = c0 ? (float)c0 * exp2f(-d0 * fslope) : 0.f, m1 = c1 ? (float)c1 * exp2f(-d1 * fslope) : 0.f;
            float total;
            const float extra = block_sum((2 * tid < split_bin ? m0 : 0.f) + (2 * tid + 1 < split_bin ? m1 : 0.f), reinterpret_cast<float*>(sh.red_u));
            const float m_before = mass_before - extra + block_scan(m0 + m1, reinterpret_cast<float*>(sh.red_u), &total) - m0 - m1;
            // one atomic a warp: hundreds on one address take longer than all the rest of this
            const int here = c0 && m_before + m0 >= goal ? 2 * tid : c1 && m_before + m0 + m1 >= goal ? 2 * tid + 1 : kFine;
            const int first_here = __reduce_min_sync(0xffffffffu, here), last_here = __reduce_max_sync(0xffffffffu, c1 ? 2 * tid + 1 : c0 ? 2 * tid : -1);
            if (lane == 0 && first_here < kFine) atomicMin(&sh.at[0], first_here);
            if (lane == 0 && last_here >= 0) atomicMax(&sh.at[4], last_here);
            __syncthreads();
            // the border by this count; if the estimates do not reach it, the last bin with entries
            const int j = sh.at[0] < kFine ? sh.at[0] : sh.at[4];
            if (j < 0) { lost = true; break; }
            if (tid == j / 2) {
                const uint32_t b = (j & 1) ? c_before + c0 : c_before;
                sh.at[1] = (int)b; sh.at[2] = (int)((j & 1) ? c1 : c0);
                sh.at[5] = __float_as_int((j & 1) ? m_before + m0 : m_before);
                // which of its neighbours is nearer to the border
                sh.at[12] = goal - ((j & 1) ? m_before + m0 : m_before) > 0.5f * ((j & 1) ? m1 : m0);
            }
            __syncthreads();
            const int at_j = sh.at[1], in_j = sh.at[2];
            // bins that hold any of the entries up to kAround places from that bin
            const int first = at_j - kAround, last = at_j + in_j + kAround;
            const int a0 = (int)c_before, a1 = a0 + (int)c0, a2 = a1 + (int)c1;
            if (c0 && a1 > first && a0 < last) { atomicMin(&sh.at[3], 2 * tid); atomicMax(&sh.at[7], 2 * tid); atomicAdd(&sh.at[6], (int)c0); }
            if (c1 && a2 > first && a1 < last) { atomicMin(&sh.at[3], 2 * tid + 1); atomicMax(&sh.at[7], 2 * tid + 1); atomicAdd(&sh.at[6], (int)c1); }
            // the nearest bins with entries on either side
            if (c0 && a1 == at_j) { sh.at[8] = 2 * tid; sh.at[9] = (int)c0; }
            if (c1 && a2 == at_j) { sh.at[8] = 2 * tid + 1; sh.at[9] = (int)c1; }
            if (c0 && a0 == at_j + in_j) { sh.at[10] = 2 * tid; sh.at[11] = (int)c0; }
            if (c1 && a1 == at_j + in_j) { sh.at[10] = 2 * tid + 1; sh.at[11] = (int)c1; }
            __syncthreads();
            if (sh.at[6] <= kCand) { p_lo = sh.at[3]; p_hi = sh.at[7]; break; }
            if (in_j <= kCand) {                         // that bin and, if they fit, those of its nearer neighbour
                p_lo = p_hi = j;
                if (!sh.at[12] && sh.at[8] >= 0 && in_j + sh.at[9] <= kCand) p_lo = sh.at[8];
                if (sh.at[12] && sh.at[10] >= 0 && in_j + sh.at[11] <= kCand) p_hi = sh.at[10];
                break;
            }
            tie = narrow(j, threshold);
            lost = tie == 0 && turn == 3;
            if (tie != 0 || lost) break;
            mass_before = __int_as_float(sh.at[5]);
        }
    }

    // ---- 4. weights ---------------------------------------------------------------
    // chunk by chunk: the sums of what is surely kept stay per chunk, in the order of the vocabulary
    auto sum_chunks = [&](unsigned long long thr) {      // kept: at or above thr
        double kept = 0;
        each_piece([&](const uint4& d, int i) {
#pragma unroll
            for (int g = 0; g < VE; g += 4) {            // four chains of dependent 64-bit operations at a time
                double w[4];
                bool in[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) in[e] = at_or_above(key_of(Pc::entry(d, g + e)), i + g + e, thr);
                if (!(in[0] | in[1] | in[2] | in[3])) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) { const double y = weight(Pc::entry(d, g + e)); w[e] = in[e] ? y : 0.0; }
                kept += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }, [&](int c) {
            kept = warp_sum(kept);
            if (lane == 0) { sh.chunk_sum[c] = kept; sh.chunk_extra[c] = 0; }
            kept = 0;
        });
        __syncthreads();
    };
    if (!by_p) {
        threshold = threshold > n_least ? threshold : n_least;
        sum_chunks(threshold);
    } else {
        // images at or above k_sure are surely kept by top-p, those from k_coll are collected (or counted: the tie)
        const uint32_t k_sure = lost ? 0u : tie != 0 ? tie + 1u : edge(p_lo - 1);
        const uint32_t k_coll = lost ? 0u : tie != 0 ? tie : edge(p_hi);
        const uint32_t k_chunk = max(k_sure, k_least);   // what counts for the chunks
        const bool split = k_least > k_sure;             // entries that top-p surely keeps and min_p does not
        double m_all = 0, m_mid = 0, m_ties = 0, kept = 0;
        each_piece([&](const uint4& d, int i) {
#pragma unroll
            for (int g = 0; g < VE; g += 4) {
                double w[4];
                uint32_t key[4];
                bool in[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    key[e] = key_of(Pc::entry(d, g + e));
                    in[e] = at_or_above(key[e], i + g + e, threshold);
                }
                if (!(in[0] | in[1] | in[2] | in[3])) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) { const double y = weight(Pc::entry(d, g + e)); w[e] = in[e] ? y : 0.0; }
                m_all += (w[0] + w[1]) + (w[2] + w[3]);
                if (split) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (key[e] >= k_sure) m_mid += w[e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (key[e] < k_sure && key[e] >= k_coll && in[e]) {
                        if (tie != 0) m_ties += 1.0; else collect(number(key[e], i + g + e));
                    }
                    w[e] = key[e] >= k_chunk ? w[e] : 0.0;
                }
                kept += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }, [&](int c) {
            kept = warp_sum(kept);
            if (lane == 0) { sh.chunk_sum[c] = kept; sh.chunk_extra[c] = 0; if (!split) m_mid += kept; }
            kept = 0;
        });
        block_sum3(m_all, m_mid, m_ties, sh.red_d);
        if (tid == 0) { sh.pub_d[0] = m_all; sh.pub_d[1] = m_mid; sh.pub_d[2] = m_ties; }
        const int n = gather();
        const double M = over_cluster(&sh.pub_d[0]), A = over_cluster(&sh.pub_d[1]);
        const double goal = (double)p_top * M;
        // entries of weight w from above on: as many as start below the goal, at least one
        auto taken = [&](double above, double w, double many) {
            double take = fmin(fmax(ceil((goal - above) / w), 1.0), many);
            while (take > 1.0 && above + (take - 1.0) * w >= goal) take -= 1.0;
            while (take < many && above + take * w < goal) take += 1.0;
            return (uint32_t)take;
        };
        bool right = false;                              // whether the border lies where it was guessed
        if (tie != 0) {
            const double many = over_cluster(&sh.pub_d[2]), w = weight(bits_of(tie));
            if (A < goal && A + many * w >= goal) {
                threshold = nth_equal(tie, taken(A, w, many));
                threshold = threshold > n_least ? threshold : n_least;
                sum_chunks(threshold);
                right = true;
            }
        } else if (n <= kCand && !lost) {
            // running sum over the sorted entries, behind the larger ones; the largest of all is kept whatever p is
            const double w = tid < n ? weight(bits_of((uint32_t)(own_number >> 32))) : 0.0;
            double total;
            const double before = A + (block_scan(w, sh.red_d, &total) - w);
            const int keep = __syncthreads_count(tid < n && (before < goal || own_number == best));      // a leading run
            // Right if the first one is kept, and the last one is not or all of these and the larger ones reach the goal.
            right = keep > 0 && (keep < n || A + total >= goal);
            if (right) {
                threshold = sh.all[keep - 1];
                threshold = threshold > n_least ? threshold : n_least;
                const int idx = (int)(uint32_t)~(uint32_t)own_number;
                if (tid < keep && own_number >= n_least && idx >= i0 && idx < i0 + nv * VE)
                    atomicAdd(&sh.chunk_extra[(idx - i0) / VE / prm.chunk_vecs], (unsigned long long)__double2ll_rn(w * 0x1p52));
                __syncthreads();
            }
        }
        if (!right) {
            double above;
            const uint32_t key = bisect((uint32_t)(threshold >> 32), [&](uint32_t from_) {
                double m = 0;
                each([&](uint32_t bits, int i) {
                    const uint32_t at = key_of(bits);
                    if (at >= from_ && at_or_above(at, i, threshold)) m += weight(bits);
                });
                return m;
            }, goal, &above);
            double many = 0;
            each([&](uint32_t bits, int i) { if (key_of(bits) == key && at_or_above(key, i, threshold)) many += 1.0; });
            many = cluster_sum(many);
            threshold = nth_equal(key, taken(above, weight(bits_of(key)), many));
            threshold = threshold > n_least ? threshold : n_least;
            sum_chunks(threshold);
        }
    }

    // ---- 5. the slice, the chunk, the entry ----------------------------------------------
    const double own = tid < n_chunks ? sh.chunk_sum[tid] + (double)(long long)sh.chunk_extra[tid] * 0x1p-52 : 0.0;
    double mine;
    const double incl = block_scan(own, sh.red_d, &mine);
    if (tid == 0) { sh.pub_d[4] = mine; sh.at[0] = kMaxChunks; sh.at[1] = -1; }
    cluster_sync();
    const double theirs = lane < (int)C ? peer(&sh.pub_d[4], from) : 0.0;
    double W = 0, pre = 0;
    for (uint32_t r = 0; r < C; ++r) { if (r == rank) pre = W; W += __shfl_sync(0xffffffffu, theirs, r); }
    const double goal = u * W;
    int owner = -1, last = 0;                            // the first slice that passes the goal; the last one with any mass
    {
        double run = 0;
        for (uint32_t r = 0; r < C; ++r) {
            const double m = __shfl_sync(0xffffffffu, theirs, r);
            if (m > 0) last = (int)r;
            run += m;
            if (owner < 0 && run > goal) owner = (int)r;
        }
        if (owner < 0) owner = last;                     // u at or past 1
    }
    if (owner == (int)rank) {
        // the first chunk that passes the goal, or the last one with any mass
        if (own > 0) {
            if (pre + incl > goal) atomicMin(&sh.at[0], tid);
            atomicMax(&sh.at[1], tid);
        }
        __syncthreads();
        const int c = sh.at[0] < kMaxChunks ? sh.at[0] : sh.at[1];
        if (tid == c) sh.red_d[0] = pre + incl - own;    // mass before the chunk
        __syncthreads();
        if (warp == 0) {
            double run = sh.red_d[0];
            int found = -1, fallback = -1;
            double w_found = 0, w_fallback = 0;
            const int end = min((c + 1) * prm.chunk_vecs, nv);
            for (int vb = c * prm.chunk_vecs; vb < end && found < 0; vb += 32) {
                const int v = vb + lane;
                double w[VE], sum = 0;
#pragma unroll
                for (int e = 0; e < VE; ++e) w[e] = 0.0;
                if (v < end) {
                    const uint4 d = piece(v);
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        const uint32_t bits = Pc::entry(d, e);
                        if (at_or_above(key_of(bits), i0 + v * VE + e, threshold)) w[e] = weight(bits);
                        sum += w[e];
                    }
                }
                const double to = warp_scan(sum);
                double at = run + (to - sum);
                int here = -1, some = -1; double wh = 0, ws = 0;
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    at += w[e];
                    if (w[e] > 0) { some = e; ws = w[e]; if (here < 0 && at > goal) { here = e; wh = w[e]; } }
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, here >= 0), any = __ballot_sync(0xffffffffu, some >= 0);
                if (hit) {
                    const int l = __ffs(hit) - 1;
                    found = i0 + (vb + l) * VE + __shfl_sync(0xffffffffu, here, l);
                    w_found = __shfl_sync(0xffffffffu, wh, l);
                } else if (any) {
                    const int l = 31 - __clz(any);
                    fallback = i0 + (vb + l) * VE + __shfl_sync(0xffffffffu, some, l);
                    w_fallback = __shfl_sync(0xffffffffu, ws, l);
                }
                run += __shfl_sync(0xffffffffu, to, 31);
            }
            // rounding may leave the last entry of the chunk a hair short of the goal
            if (found < 0) { found = fallback; w_found = w_fallback; }
            if (lane == 0) {
                prm.token[row] = found;
                if (prm.logprob != nullptr) prm.logprob[row] = (float)log(w_found / W);
            }
        }
    }
    cluster_sync();                                      // nobody leaves while a peer may read its shared memory
}

template <typename T>
int launch_typed(SampleParams prm, int rows, cudaStream_t stream)
{
    constexpr int VE = 16 / (int)sizeof(T);
    const int row_vecs = (prm.vocab + 2 * VE - 2) / VE;  // wherever the row starts within a piece
    // Few rows: split each until its slices are short (4096 entries) or two CTAs sit on every SM.  Many rows: only as far
    // as a slice has to be small for two CTAs to share an SM.
    int cluster = 1;
    while (cluster < kMaxCluster && (long long)prm.vocab > 4096ll * cluster && (long long)rows * cluster * 2 <= 2 * 148) cluster *= 2;
    const int half = 113 * 1024 - (int)sizeof(Shared), budget = kMaxSmem - (int)sizeof(Shared);
    auto shape = [&](int c) {
        prm.chunk_vecs = 32;
        while ((long long)prm.chunk_vecs * kMaxChunks * c < row_vecs) prm.chunk_vecs *= 2;
        const int per = (row_vecs + c - 1) / c;
        prm.slice_vecs = (per + prm.chunk_vecs - 1) / prm.chunk_vecs * prm.chunk_vecs;
    };
    shape(cluster);
    while (cluster < kMaxCluster && (long long)prm.slice_vecs * 16 > half) { cluster *= 2; shape(cluster); }
    const bool staged = (long long)prm.slice_vecs * 16 <= budget;
    const int bytes = (int)sizeof(Shared) + (staged ? prm.slice_vecs * 16 : 0);
    auto kern = staged ? sample_kernel<T, true> : sample_kernel<T, false>;
    // The same limit in every call: it belongs to the function, and another host thread may launch a larger row between a call's
    // setting of its own and its launch.
    if (const int rc = launch_code(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = bytes; cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    return launch_code(cudaLaunchKernelEx(&cfg, kern, prm));
}

}  // namespace

int launch_sample(const void* logits, int dtype, long long row_stride, int rows, int vocab, const float* uniform,
                  const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int64_t* token,
                  float* logprob, cudaStream_t stream)
{
    SampleParams prm{logits, uniform, temperature, top_k, top_p, min_p, token, logprob, row_stride, vocab, 0, 0};
    if (dtype == FPKV_F32) return launch_typed<float>(prm, rows, stream);
    if (dtype == FPKV_BF16) return launch_typed<__nv_bfloat16>(prm, rows, stream);
    return launch_typed<__half>(prm, rows, stream);
}

}  // namespace fpkv
