// Token sampling: temperature, top-k, top-p and min-p from one given uniform number a row.
//
// All filters keep a leading part of the row ordered by (value descending, index ascending), so the kept set is
// described by a threshold value and by how many of the entries equal to it are kept: "everything above t, and the
// first c entries equal to t".  t is found by bisection on the order-preserving integer image of the logits, with one
// count (top-k) or one sum of weights (top-p) over the row a step.  Weights are exp((x - max) / T) in 64 bits and so
// are all sums: the token is the answer, and which one it is may hang on the last bits of a sum over the vocabulary.
//
// One CTA a row.

#include "common.cuh"

namespace fpkv {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
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
};

// Integer image of a value: larger value, larger image; -0 and +0 have one image, NaN that of -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
    uint32_t u = __float_as_uint(x);                            // on the bits: arithmetic would flush subnormal values to zero
    if ((u & 0x7fffffffu) > 0x7f800000u) return kKeyNone;
    if (u == 0x80000000u) u = 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

template <typename V> __device__ __forceinline__ V block_sum(V v, V* s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
    __syncthreads();
    V t = 0;
    for (int w = 0; w < kWarps; ++w) t += s[w];
    return t;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_kernel(const SampleParams prm)
{
    __shared__ double s_d[kWarps];
    __shared__ int s_i[kWarps];
    __shared__ uint32_t s_k[kWarps];
    __shared__ int s_found, s_last;
    const int b = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32, V = prm.vocab;
    const T* x = reinterpret_cast<const T*>(prm.logits) + (long long)b * prm.row_stride;
    auto key_at = [&](int i) { return key_of(ElemTraits<T>::to_float(x[i])); };

    // ---- largest value and its first index -------------------------------------
    uint32_t kmax = 0; int imax = V;
    for (int i = tid; i < V; i += kThreads) { const uint32_t k = key_at(i); if (k > kmax) { kmax = k; imax = i; } }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint32_t k2 = __shfl_xor_sync(0xffffffffu, kmax, o);
        const int i2 = __shfl_xor_sync(0xffffffffu, imax, o);
        if (k2 > kmax || (k2 == kmax && i2 < imax)) { kmax = k2; imax = i2; }
    }
    if (lane == 0) { s_k[warp] = kmax; s_i[warp] = imax; }
    __syncthreads();
    for (int w = 0; w < kWarps; ++w)
        if (s_k[w] > kmax || (s_k[w] == kmax && s_i[w] < imax)) { kmax = s_k[w]; imax = s_i[w]; }
    const float temp = prm.temperature != nullptr ? prm.temperature[b] : 1.f;
    if (kmax <= kKeyNone || !(temp > 0.f)) {
        if (tid == 0) {
            const bool some = kmax > kKeyNone;
            prm.token[b] = some ? imax : -1;
            if (prm.logprob != nullptr) prm.logprob[b] = some ? 0.f : -INFINITY;
        }
        return;
    }
    const double xmax = (double)value_of(kmax), T64 = (double)temp;
    auto weight = [&](uint32_t key) -> double {
        if (key == kmax) return 1.0;                            // an infinite maximum too
        return key <= kKeyNone ? 0.0 : exp(((double)value_of(key) - xmax) / T64);
    };

    // ---- threshold -------------------------------------------------------------
    uint32_t t = kKeyNone;                                      // everything above t is kept ...
    int c = 0;                                                  // ... and the first c entries equal to t
    const int k = prm.top_k != nullptr ? prm.top_k[b] : 0;
    if (k > 0 && k < V) {
        uint32_t lo = kKeyNone, hi = kmax;                      // count(key >= lo) >= k where lo is above -inf
        int above = 0;
        while (lo < hi) {                                       // largest t with count(key >= t) >= k
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            int n = 0;
            for (int i = tid; i < V; i += kThreads) n += key_at(i) >= mid;
            n = block_sum(n, s_i);
            if (n >= k) lo = mid; else { hi = mid - 1; above = n; }
        }
        if (lo > kKeyNone) { t = lo; c = k - above; }
    }
    // sum of the kept weights at or above a key
    auto mass_from = [&](uint32_t from) {
        double m = 0;
        for (int i = tid; i < V; i += kThreads) { const uint32_t key = key_at(i); if (key >= from && key > t) m += weight(key); }
        m = block_sum(m, s_d);
        return (c > 0 && t >= from) ? m + c * weight(t) : m;
    };
    const float p = prm.top_p != nullptr ? prm.top_p[b] : 1.f;
    if (p < 1.f) {
        const double goal = (double)p * mass_from(kKeyNone + 1);
        uint32_t lo = c > 0 ? t : kKeyNone + 1, hi = kmax;
        double above = 0;
        while (lo < hi) {                                       // largest t' with mass(kept, key >= t') >= goal
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            const double m = mass_from(mid);
            if (m >= goal) lo = mid; else { hi = mid - 1; above = m; }
        }
        // entries equal to lo are taken while the mass before them is below the goal
        int n = 0;
        for (int i = tid; i < V; i += kThreads) n += key_at(i) == lo;
        n = block_sum(n, s_i);
        if (c > 0 && lo == t) n = c;
        const double w = weight(lo), need = (goal - above) / w;
        int take = need <= 1.0 ? 1 : (need >= (double)n ? n : (int)ceil(need));
        while (take > 1 && above + (take - 1) * w >= goal) --take;
        while (take < n && above + take * w < goal) ++take;
        t = lo; c = take;
    }
    const float mp = prm.min_p != nullptr ? prm.min_p[b] : 0.f;
    const double least = mp > 0.f ? (mp < 1.f ? (double)mp : 1.0) : 0.0;

    // ---- sum of the kept weights, then the first index past u of it ----------------
    double total = 0;
    if (tid == 0) { s_found = V; s_last = -1; }
    for (int pass = 0; pass < 2; ++pass) {
        const double goal = (double)prm.uniform[b] * total;
        double run = 0;                                         // mass before this tile
        int ties = 0;                                           // entries equal to t before this tile
        for (int i0 = 0; i0 < V; i0 += kThreads) {
            const int i = i0 + tid;
            const uint32_t key = i < V ? key_at(i) : 0;
            const bool tie = c > 0 && key == t;
            const uint32_t votes = __ballot_sync(0xffffffffu, tie);
            __syncthreads();
            if (lane == 0) s_i[warp] = __popc(votes);
            __syncthreads();
            int rank = ties + __popc(votes & ((1u << lane) - 1));          // this entry's rank among those equal to t
            for (int w = 0; w < kWarps; ++w) { if (w < warp) rank += s_i[w]; ties += s_i[w]; }
            const double wt = weight(key);
            const bool kept = (key > t || (tie && rank < c)) && key > kKeyNone && wt >= least;
            double sum = kept ? wt : 0.0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += y; }
            if (lane == 31) s_d[warp] = sum;
            __syncthreads();
            double before = run;
            for (int w = 0; w < kWarps; ++w) { if (w < warp) before += s_d[w]; run += s_d[w]; }
            if (pass == 1 && kept) {
                if (before + sum > goal) atomicMin(&s_found, i);
                if (wt > 0.0) atomicMax(&s_last, i);
            }
        }
        total = run;
    }
    __syncthreads();
    if (tid == 0) {
        const int tok = s_found < V ? s_found : s_last;         // uniform at or past 1: the last entry
        prm.token[b] = tok;
        if (prm.logprob != nullptr) prm.logprob[b] = (float)log(weight(key_at(tok)) / total);
    }
}

}  // namespace

int launch_sample(const void* logits, int dtype, long long row_stride, int rows, int vocab, const float* uniform,
                  const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int64_t* token,
                  float* logprob, cudaStream_t stream)
{
    SampleParams prm{logits, uniform, temperature, top_k, top_p, min_p, token, logprob, row_stride, vocab};
    if (dtype == FPKV_F32) sample_kernel<float><<<rows, kThreads, 0, stream>>>(prm);
    else if (dtype == FPKV_BF16) sample_kernel<__nv_bfloat16><<<rows, kThreads, 0, stream>>>(prm);
    else sample_kernel<__half><<<rows, kThreads, 0, stream>>>(prm);
    return cudaGetLastError() == cudaSuccess ? FPKV_OK : FPKV_ELAUNCH;
}

}  // namespace fpkv
