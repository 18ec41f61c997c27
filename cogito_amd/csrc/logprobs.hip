// logprobs.hip -- log probabilities of given tokens with their rank, the
// entropy and the top alternatives of rows of logits.
//
// With m = max x, d_j = x_j - m, z = sum exp(d_j): lse = m + log z,
// log p(x) = x - lse, H = log z - (sum d_j exp(d_j)) / z (a term with exp = 0
// adds nothing, so a masked token's -inf does not meet a 0).  Order of tokens:
// 64-bit keys, the value's bits mapped to unsigned order in the high word (-0
// as 0, NaN below -inf) and the complemented index in the low one, so every
// key is different and ties go to the lowest index.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "cgx_internal.h"

namespace {

inline hipStream_t stream() { return (hipStream_t)cgx_stream(); }

int launch_check(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        cgx_set_error("%s launch failed: %s", what, hipGetErrorString(e));
        return -1;
    }
    return 0;
}

constexpr int kThreads = 256, kWaves = kThreads / 64;

__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ unsigned long long key_of(float x, int i) {
    return (unsigned long long)order_of(x) << 32 | (uint32_t)~i;
}

template <typename T, typename F>
__device__ __forceinline__ T block_all(T v, T* sh, F f) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = f(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) v = f(v, sh[w]);
    return v;
}

// One block a row, one pass for the maximum, one for the sums and the rank,
// one per alternative.
__global__ __launch_bounds__(kThreads) void k_logprobs_row(const float* x, size_t ld, int V,
                                                           const int* tokens, int n_top,
                                                           float* logprob, int* rank,
                                                           float* entropy, int* top_tokens,
                                                           float* top_logprobs) {
    __shared__ unsigned long long s_u[kWaves];
    __shared__ double s_d[kWaves];
    __shared__ float s_f[kWaves];
    __shared__ int s_i[kWaves];
    const int r = blockIdx.x, tid = threadIdx.x;
    const float* row = x + (size_t)r * ld;
    const int tok = tokens ? tokens[r] : -1;
    const bool given = tok >= 0 && tok < V;
    const unsigned long long kt = given ? key_of(row[tok], tok) : 0;
    float m = -INFINITY;
    int nan = 0, before = 0;
    for (int i = tid; i < V; i += kThreads) {
        const float v = row[i];
        m = fmaxf(m, v);
        nan |= v != v;
        before += key_of(v, i) > kt;
    }
    m = block_all(m, s_f, [](float p, float q) { return fmaxf(p, q); });
    nan = block_all(nan, s_i, [](int p, int q) { return p | q; });
    before = block_all(before, s_i, [](int p, int q) { return p + q; });
    double z = 0.0, w = 0.0;
    for (int i = tid; i < V; i += kThreads) {
        const float d = row[i] - m, e = __expf(d);
        z += e;
        if (e > 0.0f) w += (double)(d * e);
    }
    z = block_all(z, s_d, [](double p, double q) { return p + q; });
    w = block_all(w, s_d, [](double p, double q) { return p + q; });
    const bool bad = nan || m == INFINITY || m == -INFINITY;
    const float logz = (float)log(z);
    auto lp = [&](float v) { return bad ? NAN : v - m - logz; };
    if (tid == 0) {
        if (logprob) logprob[r] = given ? lp(row[tok]) : -INFINITY;
        if (rank) rank[r] = given ? before : V;
        if (entropy) entropy[r] = bad ? NAN : (float)(log(z) - w / z);
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < n_top; k++) {
        unsigned long long best = 0;
        for (int i = tid; i < V; i += kThreads) {
            const unsigned long long u = key_of(row[i], i);
            if (u < last && u > best) best = u;
        }
        best = block_all(best, s_u, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
        last = best;
        if (tid == 0) {
            const int at = best ? (int)~(uint32_t)best : -1;
            top_tokens[(size_t)r * n_top + k] = at;
            top_logprobs[(size_t)r * n_top + k] = at < 0 ? -INFINITY : lp(row[at]);
        }
    }
}

}  // namespace

extern "C" size_t cgk_logprobs_ws(int rows, int V, int n_top) {
    (void)rows;
    (void)V;
    (void)n_top;
    return 0;
}

extern "C" int cgk_logprobs(const float* x, size_t ld, int rows, int V, const int* tokens,
                            int n_top, float* logprob, int* rank, float* entropy,
                            int* top_tokens, float* top_logprobs, void* ws) {
    (void)ws;
    hipLaunchKernelGGL(k_logprobs_row, dim3(rows), dim3(kThreads), 0, stream(), x, ld, V, tokens,
                       n_top, logprob, rank, entropy, top_tokens, top_logprobs);
    return launch_check("k_logprobs_row");
}
