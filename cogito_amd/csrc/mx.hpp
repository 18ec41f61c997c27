// mx.hpp -- microscaled operands on the matrix cores: records of a 128-value
// chunk of the contraction, the cut of fp32 values into them, and the product
// kernel that the matmul, the vocabulary loss and its gradient share.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes per lane 32 consecutive values of one
// row (row lane % 16, values 32 (lane / 16) ..) in 4, 6 or 8 bits and the
// power of two of that block.  Error of one instruction against 64 bits over
// sum |a b|, measured: 2^-23.7 with 4- and 6-bit operands on both sides, 2^-12
// with an 8-bit one, so nothing here is held in 8 bits.  Rates, measured with
// operands in registers: 7.4-7.6 PFLOP/s 4 x 4 bits, 6.3 6 x 4, 6.8-7.1 6 x 6.
//
// Rows taken as they are (CGX_MX_FP32) are five 6-bit (E2M3) terms of the same
// block: each term rounds what the ones before left, 5 bits a term, so that a
// value is held to 2^-23 of the largest of its block.  With 6.3 / 5 = 1.26
// PFLOP/s of the product this beats two fp16 halves (0.70 at the rate measured for them),
// and the weight needs no decoding.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "cgx_internal.h"

namespace mx {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i2 __attribute__((ext_vector_type(2)));
typedef int i8 __attribute__((ext_vector_type(8)));
typedef unsigned u6 __attribute__((ext_vector_type(6)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef float f32 __attribute__((ext_vector_type(32)));

// operand formats of the instruction
constexpr int kE2M3 = 2, kE3M2 = 3, kE2M1 = 4;

// How rows enter a product: format, terms, and the bytes of a 16-row tile's
// chunk.  A 6-bit term is 16 bytes a lane (1 KiB) and behind them 8 (512 B).
template <int ACT>
struct Rows {
    static constexpr int fmt = ACT == CGX_MX_FP4 ? kE2M1 : kE2M3;
    static constexpr int terms = ACT == CGX_MX_FP32 ? 5 : 1;
    static constexpr int term = ACT == CGX_MX_FP4 ? 1024 : 1536;
    static constexpr int tile = terms * term;
    // smallest scale byte: the last term's power of two stays above 2^-127
    static constexpr int low = ACT == CGX_MX_FP32 ? 19 : 1;
};
// bytes of a chunk's record: tiles' codes, then 64 scale bytes a tile
template <int ACT>
constexpr int rows_record(int tiles) { return tiles * (Rows<ACT>::tile + 64); }
constexpr int kWTiles = 16;                        // 256 outputs a record
constexpr int kWRecord = kWTiles * (1024 + 64);    // the weight
constexpr int kTRecord = kWTiles * (1536 + 64);    // its transpose, E3M2

// exponent of term t below the block's
constexpr int term_shift(int t) { return t ? 5 * t - 2 : 0; }

__device__ __forceinline__ float pow2(int byte) { return __int_as_float(byte << 23); }

// 32 values of a block: scale byte (floor(log2 max) - 2, at least low; 255 for
// a NaN or an infinity) and codes.
__device__ __forceinline__ int block_byte(const float* v, int low) {
    int top = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const int b = __float_as_int(v[i]) & 0x7fffffff;
        top = b > top ? b : top;
    }
    top >>= 23;
    return top == 255 ? 255 : top - 2 > low ? top - 2 : low;
}

// 32 values (even ones in a, odd ones in b) over `scale` to 6 bits, to nearest
// even and saturating.  The instruction writes its result while it still reads
// its operands, which the compiler does not know: the empty statement keeps
// them in registers of their own until it is done.
template <int FMT>
__device__ __forceinline__ u6 to6(const f16& a, const f16& b, float scale) {
    u6 q = FMT == kE2M3 ? __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, scale)
                        : __builtin_amdgcn_cvt_scalef32_2xpk16_bf6_f32(a, b, scale);
    asm volatile("" : "+v"(q) : "v"(a), "v"(b), "v"(scale));
    return q;
}
// ... and back
__device__ __forceinline__ f32 from6(u6& q, float scale) {
    f32 w = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(q, scale);
    asm volatile("" : "+v"(w), "+v"(q) : "v"(scale));
    return w;
}

// One 6-bit term of v (rounded to nearest even at 2^e, saturating); v keeps
// the rest.
template <bool LAST>
__device__ __forceinline__ u6 cut6(float* v, float scale) {
    f16 a, b;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        a[i] = v[2 * i];
        b[i] = v[2 * i + 1];
    }
    u6 q = to6<kE2M3>(a, b, scale);
    if (!LAST) {
        const f32 w = from6(q, scale);
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] -= w[i];   // exact
    }
    return q;
}
__device__ __forceinline__ i4 cut4(const float* v, float scale) {
    i4 q;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        unsigned r = 0;
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[8 * w], v[8 * w + 1], scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[8 * w + 2], v[8 * w + 3], scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[8 * w + 4], v[8 * w + 5], scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[8 * w + 6], v[8 * w + 7], scale, 3);
        q[w] = (int)r;
    }
    return q;
}

// A lane's block as operands: q[t] for term t.
template <int ACT>
struct Cut {
    i8 q[Rows<ACT>::terms];
    int byte;
};
template <int ACT>
__device__ __forceinline__ Cut<ACT> cut(float* v) {
    Cut<ACT> c;
    c.byte = block_byte(v, Rows<ACT>::low);
    const float s = pow2(c.byte == 255 ? 127 : c.byte);
    if constexpr (ACT == CGX_MX_FP4) {
        const i4 q = cut4(v, s);
        c.q[0] = i8{q[0], q[1], q[2], q[3], 0, 0, 0, 0};
    } else {
#pragma unroll
        for (int t = 0; t < Rows<ACT>::terms; t++) {
            const float st = pow2((c.byte == 255 ? 127 : c.byte) - term_shift(t));
            const u6 q = t + 1 < Rows<ACT>::terms ? cut6<false>(v, st) : cut6<true>(v, st);
            c.q[t] = i8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], (int)q[4], (int)q[5], 0, 0};
        }
    }
    return c;
}
// ... into the record's tile (codes at `tile`, scales at `sc`)
template <int ACT>
__device__ __forceinline__ void put(uint8_t* tile, uint8_t* sc, int lane, const Cut<ACT>& c) {
#pragma unroll
    for (int t = 0; t < Rows<ACT>::terms; t++) {
        uint8_t* p = tile + t * Rows<ACT>::term;
        *(i4*)(p + lane * 16) = i4{c.q[t][0], c.q[t][1], c.q[t][2], c.q[t][3]};
        if constexpr (ACT != CGX_MX_FP4) *(i2*)(p + 1024 + lane * 8) = i2{c.q[t][4], c.q[t][5]};
    }
    sc[lane] = (uint8_t)c.byte;
}

template <int FMT>
__device__ __forceinline__ i8 operand(const uint8_t* p, int lane) {
    const i4 a = *(const i4*)(p + lane * 16);
    if constexpr (FMT == kE2M1) {
        return i8{a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    } else {
        const i2 b = *(const i2*)(p + 1024 + lane * 8);
        return i8{a[0], a[1], a[2], a[3], b[0], b[1], 0, 0};
    }
}

template <int FA, int FB>
__device__ __forceinline__ f4 mfma(i8 a, i8 b, f4 c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, FA, FB, 0, sa, 0, sb);
}

// One KiB (or its first n bytes) straight into LDS, 16 bytes a lane.
__device__ __forceinline__ void to_lds(const uint8_t* g, uint8_t* l, int lane, int n) {
    if (lane * 16 < n)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(g + lane * 16),
            (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// What a product's epilogue needs.
struct Gemm {
    const uint8_t* x;      // records of the rows [row block][chunk]
    const uint8_t* w;      // records of the weight [256 outputs][chunk]
    const int* list;       // weight chunk j takes the rows' chunk list[j] - list0 (NULL: j)
    int list0;
    int xk, wk;            // chunks of x and w
    int j0, j1;            // chunks of this launch
    int mbs, nbs, splits;  // blocks of rows, of outputs (from block nb0), of chunks
    int nb0;
    int M, N;              // rows and outputs that exist
    // store: y[split][m][n] (rows ld apart, splits `stride` apart)
    float* y;
    size_t ld, stride;
    int vec;               // y takes 16-byte stores
    // gradient: y (+)= row_scale[m] * sum, 0 in a row whose target is none of V
    const float* row_scale;
    const int* targets;
    int V, add;
    // loss: a block half's maximum and sum [m][2 nbs], the target's logit [m]
    float2* part;
    float* zt;
    // loss gradient: records of the rows' probabilities, lse
    const float* lse;
    uint8_t* p;
    int pk, pmt, pmbs;     // chunks of p, tiles of a record, row blocks
};

enum { kStore = 0, kGrad = 1, kStats = 2, kProbs = 3 };

// Probabilities of a lane's row in operand order.  Lane group g = lane / 16
// holds outputs 16 n + 4 g + r of its row (acc[n][r]); block b of 32 outputs is
// tiles 2 b and 2 b + 1.  Two swaps of lane halves and quarters transpose
// groups and blocks, after which group b holds its block's 32 values in order.
__device__ __forceinline__ void probs(float* v, const f4* acc, int col0, int N, int t, bool live,
                                      float lse) {
    unsigned q[2][4][4];                                        // [half][r][block]
#pragma unroll
    for (int n = 0; n < 8; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int c = col0 + 16 * n + r;
            float p = live && c < N ? expf(acc[n][r] - lse) : 0.0f;
            if (live && c == t) p = expm1f(acc[n][r] - lse);
            q[n & 1][r][n >> 1] = __float_as_uint(p);
        }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            unsigned* b = q[h][r];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const auto s = __builtin_amdgcn_permlane32_swap(b[k], b[k + 2], false, false);
                b[k] = s[0];
                b[k + 2] = s[1];
            }
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const auto s = __builtin_amdgcn_permlane16_swap(b[k], b[k + 1], false, false);
                b[k] = s[0];
                b[k + 1] = s[1];
            }
#pragma unroll
            for (int g = 0; g < 4; g++) v[16 * h + 4 * g + r] = __uint_as_float(b[g]);
        }
}

// Product of BM rows and 256 outputs a block: the weight's tile is the first
// operand, so that a lane holds four neighbouring outputs of one row.  A wave
// has BM / WM rows and 128 outputs.  Records of a chunk go into LDS without
// passing registers; two blocks a CU overlap one's loads with the other's
// matrix instructions.
template <int ACT, int WFMT, int BM, int WM, int EPI>
__global__ __launch_bounds__(128 * WM, WFMT == kE2M1 ? 2 : 1) void k_gemm(const Gemm a) {
    constexpr int MT = BM / 16, TM = MT / WM, TN = 8, NW = 2 * WM;
    using R = Rows<ACT>;
    constexpr int XR = rows_record<ACT>(MT), WT = WFMT == kE2M1 ? 1024 : 1536;
    constexpr int WR = kWTiles * (WT + 64), XU = (XR + 1023) / 1024, WU = (WR + 1023) / 1024;
    __shared__ __attribute__((aligned(16))) uint8_t lds[XR + WR];
    uint8_t *const lx = lds, *const lw = lds + XR;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    // each XCD (block b runs on XCD b % 8) takes a run of outputs with all their rows
    const int nblk = a.mbs * a.nbs, per = nblk / 8, b = blockIdx.x;
    const int sb = b < per * 8 ? (b % 8) * per + b / 8 : b;
    const int nb = sb / a.mbs, mb = sb - nb * a.mbs, nbw = a.nb0 + nb;
    const int z = blockIdx.y;
    const int j0 = a.j0 + (int)((long long)(a.j1 - a.j0) * z / a.splits);
    const int j1 = a.j0 + (int)((long long)(a.j1 - a.j0) * (z + 1) / a.splits);
    const uint8_t* xb = a.x + (size_t)mb * a.xk * XR;
    const uint8_t* wb = a.w + (size_t)nbw * a.wk * WR;
    f4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f4{0, 0, 0, 0};

    for (int j = j0; j < j1; j++) {
        const uint8_t* gx = xb + (size_t)(a.list ? a.list[j] - a.list0 : j) * XR;
        const uint8_t* gw = wb + (size_t)j * WR;
#pragma unroll
        for (int u = 0; u < XU; u += NW)
            if (u + wave < XU)
                to_lds(gx + (u + wave) * 1024, lx + (u + wave) * 1024, lane, XR - (u + wave) * 1024);
#pragma unroll
        for (int u = 0; u < WU; u += NW)
            if (u + wave < WU)
                to_lds(gw + (u + wave) * 1024, lw + (u + wave) * 1024, lane, WR - (u + wave) * 1024);
        __builtin_amdgcn_s_waitcnt(0x0f70);                   // vmcnt(0): the records are in LDS
        __syncthreads();
        i8 w[TN];
        int ws[TN];
#pragma unroll
        for (int n = 0; n < TN; n++) {
            w[n] = operand<WFMT>(lw + (wn * TN + n) * WT, lane);
            ws[n] = lw[kWTiles * WT + (wn * TN + n) * 64 + lane];
        }
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const uint8_t* t0 = lx + (wm * TM + i) * R::tile;
            const int xs = lx[MT * R::tile + (wm * TM + i) * 64 + lane];
#pragma unroll
            for (int t = 0; t < R::terms; t++) {
                const i8 x = operand<R::fmt>(t0 + t * R::term, lane);
#pragma unroll
                for (int n = 0; n < TN; n++)
                    acc[i][n] = mfma<WFMT, R::fmt>(w[n], x, acc[i][n], ws[n], xs - term_shift(t));
            }
        }
        __syncthreads();
    }

    const int col0 = nbw * 256 + wn * 128 + 4 * (lane >> 4);   // outputs col0 + 16 n + r
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = mb * BM + (wm * TM + i) * 16 + (lane & 15);
        if constexpr (EPI == kStore || EPI == kGrad) {
            if (m < a.M) {
                float* y = a.y + (size_t)z * a.stride + (size_t)m * a.ld;
                const float g = EPI == kGrad && a.row_scale ? a.row_scale[m] : 1.0f;
                const bool none = EPI == kGrad && (unsigned)a.targets[m] >= (unsigned)a.V;
#pragma unroll
                for (int n = 0; n < TN; n++) {
                    const int c = col0 + 16 * n;
                    f4 v = EPI == kGrad ? acc[i][n] * g : acc[i][n];
                    if (none) v = f4{0, 0, 0, 0};
                    if (a.vec && c + 3 < a.N) {
                        if (EPI == kGrad && a.add) v += *(const f4*)(y + c);
                        *(f4*)(y + c) = v;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (c + r < a.N)
                                y[c + r] = EPI == kGrad && a.add ? y[c + r] + v[r] : v[r];
                    }
                }
            }
        } else if constexpr (EPI == kStats) {
            const int t = m < a.M ? a.targets[m] : -1;
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int c = col0 + 16 * n + r;
                    if (c >= a.N) acc[i][n][r] = -INFINITY;
                    else if (c == t) a.zt[m] = acc[i][n][r];
                    top = fmaxf(top, acc[i][n][r]);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // nothing above -inf: the sum is 0, or NaN where a logit is
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) sum += expf(acc[i][n][r] - ref);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (m < a.M && lane < 16)
                a.part[(size_t)m * (2 * a.nbs) + 2 * nb + wn] = make_float2(top, sum);
        } else {
            // p = exp(z - lse) - [target]; rows past M and ignored ones are 0
            const int t = m < a.M ? a.targets[m] : -1;
            const bool live = t >= 0 && t < a.N;
            const float lse = live ? a.lse[m] : 0.0f;
            float v[32];
            probs(v, acc[i], col0, a.N, t, live, lse);
            const int mt = mb * MT + wm * TM + i;
            if (mt < a.pmt * a.pmbs) {
                using P = Rows<CGX_MX_FP32>;
                uint8_t* rec = a.p + ((size_t)(mt / a.pmt) * a.pk + 2 * nb + wn) *
                                         (size_t)(a.pmt * (P::tile + 64));
                const int at = mt % a.pmt;
                put<CGX_MX_FP32>(rec + at * P::tile, rec + a.pmt * P::tile + at * 64, lane,
                                 cut<CGX_MX_FP32>(v));
            }
        }
    }
}

}  // namespace mx
