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
constexpr int kMaxTop = 32;
constexpr int kWideBlocks = 1024;

// Two launches: k_logprobs_seg reads every logit once, a block a segment of a
// row held in registers (EPT values a thread), and leaves the segment's
// maximum, sums, count of tokens before the given one and its first n_top
// keys in order; k_logprobs_row joins a row's segments.  A row of one segment
// is done in the first.
//
// The first n_top of a segment: every wave finds the largest value T that at
// least n_top of the block's 256 lane maxima reach (a binary search over
// ballots), collects its values from T on (the block together little more than
// n_top: 22 for 20 of 8192), and the block ranks the few by counting.  Where
// ties make a wave's more than kCand, or nothing is above -inf, the wave takes
// its largest key n_top times instead.
//
// Bound by the logits' bytes: 301 rows of 128256 with 20 alternatives 37 us
// (4.1 TB/s); 5 rows of 32000 by latency, 6.6 us.  A threshold a wave took 4 us
// more, 64 values a thread 31 more.
constexpr int kCand = 128;                       // collected by a wave
constexpr int kRead = 8;                         // keys read at a time in ranking

__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return o == 0 ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

#define CGX_DPP_STEP(OP, CTRL, RMASK, IDENT)                                                   \
    v = OP(v, __builtin_bit_cast(decltype(v), __builtin_amdgcn_update_dpp(                     \
                  __builtin_bit_cast(int, (decltype(v))(IDENT)), __builtin_bit_cast(int, v), CTRL, RMASK, 0xF, false)))
#define CGX_DPP_ALL(OP, IDENT)         \
    CGX_DPP_STEP(OP, 0x111, 0xF, IDENT); \
    CGX_DPP_STEP(OP, 0x112, 0xF, IDENT); \
    CGX_DPP_STEP(OP, 0x114, 0xF, IDENT); \
    CGX_DPP_STEP(OP, 0x118, 0xF, IDENT); \
    CGX_DPP_STEP(OP, 0x142, 0xA, IDENT); \
    CGX_DPP_STEP(OP, 0x143, 0xC, IDENT)

__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ float last(float v) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
    CGX_DPP_ALL(fmaxf, -INFINITY);
    return last(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    CGX_DPP_ALL(add, 0.0f);
    return last(v);
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    CGX_DPP_ALL(umax, 0u);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

struct Args {
    const float* x;
    size_t ld;
    int V, nseg, len, n_top;                     // values a segment
    const int* tokens;
    float* logprob;
    int* rank;
    float* entropy;
    int* top_tokens;
    float* top_logprobs;
    float4* part;                                // [rows][nseg] maximum, sum, weighted sum, count
    unsigned long long* keys;                    // [rows][nseg][n_top]
};

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));   // rows start anywhere

// What a row's sums say; bad: a NaN or +inf, or nothing above -inf.
struct Row {
    double m, z, w;
    bool bad;
    float logz, mf;
};
__device__ __forceinline__ Row row_of(float m, double z, double w) {
    Row r;
    r.m = m;
    r.z = z;
    r.w = w;
    r.bad = !(z > 0.0) || m == INFINITY || m == -INFINITY;
    r.logz = (float)log(z);
    r.mf = m;
    return r;
}
__device__ __forceinline__ float lp_of(const Row& r, float v) { return r.bad ? NAN : v - r.mf - r.logz; }

// The given token's logit, `given` where it is one of the vocabulary.
__device__ __forceinline__ float given_logit(const Args& a, int r, bool& given, int& tok) {
    tok = a.tokens ? a.tokens[r] : -1;
    given = tok >= 0 && tok < a.V;
    return given ? a.x[(size_t)r * a.ld + tok] : 0.0f;
}
__device__ void write_row(const Args& a, int r, const Row& s, int before, bool given, float xt) {
    if (a.logprob) a.logprob[r] = given ? lp_of(s, xt) : -INFINITY;
    if (a.rank) a.rank[r] = given ? before : a.V;
    if (a.entropy) a.entropy[r] = s.bad ? NAN : (float)(log(s.z) - s.w / s.z);
}
__device__ __forceinline__ void write_top(const Args& a, int r, const Row& s, int k, unsigned long long key) {
    a.top_tokens[(size_t)r * a.n_top + k] = key ? (int)~(uint32_t)key : -1;
    a.top_logprobs[(size_t)r * a.n_top + k] = key ? lp_of(s, value_of((uint32_t)(key >> 32))) : -INFINITY;
}

template <int EPT>
__global__ __launch_bounds__(kThreads) void k_logprobs_seg(Args a) {
    // collected: bits of the value and the index; ranked: keys
    __shared__ __attribute__((aligned(16))) unsigned long long s_cand[kWaves][kCand], s_top[kMaxTop];
    __shared__ float s_m[kWaves], s_z[kWaves], s_w[kWaves];
    __shared__ int s_n[kWaves], s_before[kWaves];
    __shared__ uint32_t s_lane[kThreads];
    const int seg = blockIdx.x % a.nseg, r = blockIdx.x / a.nseg;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* row = a.x + (size_t)r * a.ld;
    const int begin = seg * a.len, size = min(a.V - begin, a.len), end = begin + size;
    int tok;
    bool given;
    const float xt = given_logit(a, r, given, tok);

    // value (j, c) of a thread is begin + 4 (256 j + tid) + c
    float v[EPT];
    if (size == EPT * kThreads) {
#pragma unroll
        for (int j = 0; j < EPT / 4; j++) {
            const f4 q = *(const f4*)(row + begin + 4 * (kThreads * j + tid));
#pragma unroll
            for (int c = 0; c < 4; c++) v[4 * j + c] = q[c];
        }
    } else {
#pragma unroll
        for (int j = 0; j < EPT / 4; j++) {
            const int i = begin + 4 * (kThreads * j + tid);
            f4 q = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (i + 4 <= end) {
                q = *(const f4*)(row + i);
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (i + c < end) q[c] = row[i + c];
            }
#pragma unroll
            for (int c = 0; c < 4; c++) v[4 * j + c] = q[c];
        }
    }

    // ---- maximum and sums of the wave
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < EPT; e++) m = fmaxf(m, v[e]);
    const float lane_max = m;
    m = wave_max(m);
    // values past the end are -inf and add nothing; a wave of nothing above
    // -inf has z = 0, a NaN or +inf makes z NaN
    const float mu = m == -INFINITY ? 0.0f : m;
    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f}, w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < EPT; e++) {
        const float d = v[e] - mu, x = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
        z[e & 3] += x;
        // below -200 the exponential is 0: the floor keeps -inf from meeting it
        w[e & 3] = fmaf(fmaxf(d, -200.0f), x, w[e & 3]);
    }
    const float zs = wave_sum((z[0] + z[1]) + (z[2] + z[3])), ws = wave_sum((w[0] + w[1]) + (w[2] + w[3]));

    // ---- tokens before the given one: larger, or equal and of a lower index;
    //      a NaN comes after every number
    int before = 0;
    if (a.rank && given && xt > -INFINITY && (end <= tok || begin > tok)) {
        // a segment on one side of the token (values past the end count as -inf)
        if (end <= tok) {
#pragma unroll
            for (int e = 0; e < EPT; e++) before += __popcll(__ballot(v[e] >= xt));
        } else {
#pragma unroll
            for (int e = 0; e < EPT; e++) before += __popcll(__ballot(v[e] > xt));
        }
    } else if (a.rank && given) {
        const bool nan = xt != xt;
#pragma unroll
        for (int e = 0; e < EPT; e++) {
            const int i = begin + 4 * (kThreads * (e / 4) + tid) + (e & 3);
            const bool ahead = nan ? i < end && (v[e] == v[e] || i < tok) : v[e] > xt || (v[e] == xt && i < min(tok, end));
            before += __popcll(__ballot(ahead));
        }
    }

    // ---- the wave's candidates
    const int n = a.n_top;
    if (n) {
        s_lane[tid] = order_of(lane_max);                    // of a lane's numbers: its maximum skips NaN
        __syncthreads();
        uint32_t q[kWaves], hi = 0;
#pragma unroll
        for (int x = 0; x < kWaves; x++) {
            q[x] = s_lane[64 * x + lane];
            hi = umax(hi, q[x]);
        }
        uint32_t lo = 0;                                     // lanes reaching lo: n at least; reaching hi: fewer
        hi = wave_umax(hi) + 1;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            int cnt = 0;
#pragma unroll
            for (int x = 0; x < kWaves; x++) cnt += __popcll(__ballot(q[x] >= mid));
            if (cnt >= n) lo = mid; else hi = mid;
            if (cnt == n) break;
        }
        const float T = value_of(lo > 0x007fffffu ? lo : 0x007fffffu);   // -inf at least
        int have = 0;
        if (T > -INFINITY) {
#pragma unroll
            for (int e = 0; e < EPT; e++) {
                const unsigned long long b = __ballot(v[e] >= T);
                if (b) {
                    const int at = have + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
                    if (v[e] >= T && at < kCand)
                        s_cand[wave][at] = (unsigned long long)__float_as_uint(v[e]) << 32 |
                                           (uint32_t)(begin + 4 * kThreads * (e / 4) + (e & 3) + 4 * tid);
                    have += __popcll(b);
                }
            }
            // a wave's own LDS words, in order: no barrier
            for (int c = lane; c < min(have, kCand); c += 64) {
                const unsigned long long q = s_cand[wave][c];
                s_cand[wave][c] = (unsigned long long)order_of(__uint_as_float((uint32_t)(q >> 32))) << 32 | (uint32_t)~(uint32_t)q;
            }
        }
        if (T == -INFINITY || have > kCand) {
            // the wave's largest keys one by one
            have = 0;
            unsigned long long bound = ~0ull;
            const int rounds = min(n, size);
            while (have < rounds) {
                unsigned long long best = 0;
#pragma unroll
                for (int e = 0; e < EPT; e++) {
                    const int i = begin + 4 * (kThreads * (e / 4) + tid) + (e & 3);
                    const unsigned long long k = (unsigned long long)order_of(v[e]) << 32 | (uint32_t)~i;
                    if (i < end && k < bound && k > best) best = k;
                }
                for (int o = 1; o < 64; o <<= 1) {
                    const unsigned long long k = __shfl_xor(best, o);
                    best = k > best ? k : best;
                }
                if (!best) break;                            // the wave has no more values
                if (lane == 0) s_cand[wave][have] = best;
                have++;
                bound = best;
            }
        }
        // the list's end up to whole reads of the ranking: keys below every other
        if (lane < kRead && have + lane < kCand) s_cand[wave][have + lane] = 0;
        if (lane == 0) s_n[wave] = have;
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_z[wave] = zs;
        s_w[wave] = ws;
        s_before[wave] = before;
    }
    if (tid < kMaxTop) s_top[tid] = 0;
    __syncthreads();
    if (n) {
        // a candidate's place is the number of larger keys, all keys different
        int cnt[kWaves];
#pragma unroll
        for (int x = 0; x < kWaves; x++) cnt[x] = s_n[x];
#pragma unroll 1
        for (int c = lane; c < cnt[wave]; c += 64) {
            const unsigned long long k = s_cand[wave][c];
            int place = 0;
#pragma unroll
            for (int x = 0; x < kWaves; x++)
#pragma unroll 1
                for (int y = 0; y < cnt[x]; y += kRead) {
                    unsigned long long q[kRead];
#pragma unroll
                    for (int i = 0; i < kRead; i++) q[i] = s_cand[x][y + i];
#pragma unroll
                    for (int i = 0; i < kRead; i++) place += q[i] > k;
                }
            if (place < n) s_top[place] = k;
        }
    }
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWaves; x++) M = fmaxf(M, s_m[x]);
    float Z = 0.0f, W = 0.0f;
    int all = 0;
#pragma unroll
    for (int x = 0; x < kWaves; x++) {
        const bool none = s_m[x] == -INFINITY && s_z[x] == 0.0f;
        const float d = none ? 0.0f : fmaxf(s_m[x] - M, -200.0f), f = none ? 0.0f : __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
        Z += f * s_z[x];
        W += f * (s_w[x] + d * s_z[x]);
        all += s_before[x];
    }
    if (n) __syncthreads();
    if (a.nseg == 1) {
        const Row s = row_of(M, Z, W);
        if (tid == 0) write_row(a, r, s, all, given, xt);
        if (tid < n) write_top(a, r, s, tid, s_top[tid]);
        return;
    }
    const size_t at = (size_t)r * a.nseg + seg;
    if (tid == 0) a.part[at] = make_float4(M, Z, W, __int_as_float(all));
    if (tid < n) a.keys[at * n + tid] = s_top[tid];
}

// One wave a row.  Sums: a lane takes every 64th segment.  Keys: a lane a
// segment's ordered list; the row's next is the largest head, the lowest lane
// of equal values (segments are in index order).  More than 64 segments come
// 63 at a time beside the list so far.  Bound by latency, n_top dependent steps
// among others: 7.5 us for 301 rows of 16 segments and 20 keys, 3.7 for 5.
__global__ __launch_bounds__(64) void k_logprobs_row(Args a) {
    __shared__ unsigned long long s_key[64][kMaxTop + 1];
    const int r = blockIdx.x, lane = threadIdx.x, n = a.n_top;
    const float4* part = a.part + (size_t)r * a.nseg;
    const unsigned long long* keys = a.keys + (size_t)r * a.nseg * n;
    // what the row needs from memory is asked for at once
    int tok;
    bool given;
    const float xt = given_logit(a, r, given, tok);
    const float4 p0 = lane < a.nseg ? part[lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    if (lane < a.nseg) {
#pragma unroll 8
        for (int k = 0; k < n; k++) s_key[lane][k] = keys[(size_t)lane * n + k];
    }
    float M = p0.x;
    for (int s = lane + 64; s < a.nseg; s += 64) M = fmaxf(M, part[s].x);
    M = wave_max(M);
    double Z = 0.0, W = 0.0;
    int before = 0;
    for (int s = lane; s < a.nseg; s += 64) {
        const float4 p = s < 64 ? p0 : part[s];
        const bool none = p.x == -INFINITY && p.y == 0.0f;
        const double d = none ? 0.0 : (double)p.x - (double)M, f = none ? 0.0 : exp(d);
        Z += f * p.y;
        W += f * (p.z + d * p.y);
        before += __float_as_int(p.w);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        Z += __shfl_xor(Z, o);
        W += __shfl_xor(W, o);
        before += __shfl_xor(before, o);
    }
    const Row s = row_of(M, Z, W);
    if (lane == 0) write_row(a, r, s, before, given, xt);
    if (!n) return;
    unsigned long long out = 0;                  // the row's key number `lane`
    for (int s0 = 0; s0 < a.nseg;) {
        const int first = s0 > 0, cnt = min(64 - first, a.nseg - s0);
        if (first) {
            __syncthreads();
            if (lane < n) s_key[0][lane] = out;
            if (lane < cnt)
                for (int k = 0; k < n; k++) s_key[1 + lane][k] = keys[(size_t)(s0 + lane) * n + k];
        }
        __syncthreads();
        // the list's next key is read while the one before it is compared
        int at = 1;
        const bool mine = lane < first + cnt;
        unsigned long long head = mine ? s_key[lane][0] : 0, next = mine && n > 1 ? s_key[lane][1] : 0;
        out = 0;
        for (int k = 0; k < n; k++) {
            const uint32_t hi = (uint32_t)(head >> 32);
            const uint32_t top = wave_umax(hi);
            // NaN keys have 0 in the high word, as an ended list has: those by their presence
            const unsigned long long b = __ballot(hi == top && head != 0);
            if (!b) break;
            const int win = __builtin_ctzll(b);
            const unsigned long long key = (unsigned long long)top << 32 |
                                           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)head, win);
            if (lane == k) out = key;
            if (lane == win) {
                head = next;
                at++;
                next = at < n ? s_key[lane][at] : 0;
            }
        }
        s0 += cnt;
    }
    if (lane < n) write_top(a, r, s, lane, out);
}

// Segments of 4096 values (16 a thread) while that gives few blocks, else of
// 8192: ranking a segment's candidates costs the same for both, but a few rows
// need the blocks (5 rows of 32000: 11.2 and 12.8 us; 301 of 128256: 53 and
// 43).  A row of 8192 or less is one segment, and needs no second launch (7.7
// us of two, 6.5 of one).
struct Shape {
    int nseg, len;
    bool wide;
};
Shape shape_of(int rows, int V) {
    Shape s;
    const long long wide = ((long long)V + 8191) / 8192;
    s.wide = wide * rows >= kWideBlocks || (V > 4096 && V <= 8192);
    s.len = s.wide ? 8192 : 4096;
    s.nseg = (int)(((long long)V + s.len - 1) / s.len);
    return s;
}

}  // namespace

// What a call with these sizes writes.
extern "C" size_t cgk_logprobs_need(int rows, int V, int n_top) {
    const Shape s = shape_of(rows, V);
    return s.nseg == 1 ? 0 : (size_t)rows * s.nseg * (sizeof(float4) + (size_t)n_top * 8);
}

// What no call of at most these sizes passes.  Segments of 4096 values are
// taken while those of 8192 number fewer than kWideBlocks, so they number at
// most 2 kWideBlocks - 2 of a call: the bound below holds for either length,
// and rises with rows and V where the segments' number itself falls.
extern "C" size_t cgk_logprobs_ws(int rows, int V, int n_top) {
    if (V <= 8192) return 0;
    const size_t narrow = (size_t)rows * (((size_t)V + 4095) / 4096), wide = (size_t)rows * (((size_t)V + 8191) / 8192);
    const size_t most = wide > 2 * kWideBlocks - 2 ? wide : 2 * kWideBlocks - 2;
    return (narrow < most ? narrow : most) * (sizeof(float4) + (size_t)n_top * 8);
}

extern "C" int cgk_logprobs(const float* x, size_t ld, int rows, int V, const int* tokens,
                            int n_top, float* logprob, int* rank, float* entropy,
                            int* top_tokens, float* top_logprobs, void* ws) {
    const Shape s = shape_of(rows, V);
    if ((long long)rows * s.nseg >= 1 << 24) {      // a launch has fewer than 2^32 threads
        cgx_set_error("cgx_token_logprobs_dev: too many rows for one call");
        return -1;
    }
    Args a;
    a.x = x;
    a.ld = ld;
    a.V = V;
    a.nseg = s.nseg;
    a.len = s.len;
    a.n_top = n_top;
    a.tokens = tokens;
    a.logprob = logprob;
    a.rank = rank;
    a.entropy = entropy;
    a.top_tokens = top_tokens;
    a.top_logprobs = top_logprobs;
    a.part = (float4*)ws;
    a.keys = (unsigned long long*)(a.part + (size_t)rows * s.nseg);
    const dim3 grid((unsigned)(rows * s.nseg));
    if (s.wide) hipLaunchKernelGGL(k_logprobs_seg<32>, grid, dim3(kThreads), 0, stream(), a);
    else hipLaunchKernelGGL(k_logprobs_seg<16>, grid, dim3(kThreads), 0, stream(), a);
    if (launch_check("k_logprobs_seg")) return -1;
    if (s.nseg == 1) return 0;
    hipLaunchKernelGGL(k_logprobs_row, dim3(rows), dim3(64), 0, stream(), a);
    return launch_check("k_logprobs_row");
}
