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
// Rows that are not quantised (CGX_MX_FP32) are five 6-bit (E2M3) terms of the same
// block: each term rounds what the ones before left, 5 bits a term, so that a
// value is held to 2^-23 of the largest of its block (32/31 2^-24 by the terms' own
// steps), as fp32 holds that largest one.  The block's others are held to less than
// fp32 holds them, by their distance from it: an outlier channel a thousand times its
// neighbours leaves them 14 bits, which an output sees where the outlier's own weight
// is near 0 (elsewhere an fp32 sum would round as much).  With 6.3 / 5 = 1.26
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
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // rows start anywhere
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
// bytes of a chunk's record: tiles' codes, then 64 scale bytes a tile, up to
// whole KiB (what a wave copies to LDS at a time)
template <int ACT>
constexpr int rows_record(int tiles) { return (tiles * (Rows<ACT>::tile + 64) + 1023) & ~1023; }
constexpr int kWTiles = 16;                        // 256 outputs a record
constexpr int kWRecord = kWTiles * (1024 + 64);    // the weight
constexpr int kTRecord = kWTiles * (1536 + 64);    // its transpose, E3M2

// exponent of term t below the block's
constexpr int term_shift(int t) { return t ? 5 * t - 2 : 0; }

__device__ __forceinline__ float pow2(int byte) { return __int_as_float(byte << 23); }

// 32 values of a block, the first 16 in a.  The 6-bit conversion takes two
// vectors of 16 and interleaves them, so a block's codes hold value i at
// position 2 i and value 16 + i at 2 i + 1, in every record here, rows' and
// weights' alike: the order within a block does not change a product.
struct Block {
    f16 a, b;
};
__device__ __forceinline__ void set(Block& x, int i, float v) {
    if (i < 16) x.a[i] = v;
    else x.b[i - 16] = v;
}

// Scale byte: floor(log2 max) - 2, at least low; 255 for a NaN or an infinity.
__device__ __forceinline__ int block_byte(const Block& x, int low) {
    int top = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int p = __float_as_int(x.a[i]) & 0x7fffffff, q = __float_as_int(x.b[i]) & 0x7fffffff;
        top = max(top, max(p, q));
    }
    top >>= 23;
    return top == 255 ? 255 : top - 2 > low ? top - 2 : low;
}

// 32 values over `scale` to 6 bits, to nearest even and saturating, b's behind
// a's.  The instruction writes its result while it still reads
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

__device__ __forceinline__ i4 to4(const Block& x, float scale) {
    i4 q;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        unsigned r = 0;
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.a[4 * w], x.b[4 * w], scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.a[4 * w + 1], x.b[4 * w + 1], scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.a[4 * w + 2], x.b[4 * w + 2], scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.a[4 * w + 3], x.b[4 * w + 3], scale, 3);
        q[w] = (int)r;
    }
    return q;
}

// A lane's block as operands: f(t, codes) for each term t, the largest first;
// returns the scale byte.  x is left with what the last term rounded away.
template <int ACT, class F>
__device__ __forceinline__ int cut(Block& x, F f) {
    const int byte = block_byte(x, Rows<ACT>::low), e = byte == 255 ? 127 : byte;
    if constexpr (ACT == CGX_MX_FP4) {
        const i4 q = to4(x, pow2(e));
        f(0, i8{q[0], q[1], q[2], q[3], 0, 0, 0, 0});
    } else {
#pragma unroll
        for (int t = 0; t < Rows<ACT>::terms; t++) {
            const float scale = pow2(e - term_shift(t));
            u6 q = to6<kE2M3>(x.a, x.b, scale);
            if (t + 1 < Rows<ACT>::terms) {
                const f32 w = from6(q, scale);
#pragma unroll
                for (int i = 0; i < 16; i++) {       // exact
                    x.a[i] -= w[2 * i];
                    x.b[i] -= w[2 * i + 1];
                }
            }
            f(t, i8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], (int)q[4], (int)q[5], 0, 0});
        }
    }
    return byte;
}
// ... into the record's tile (codes at `tile`, scales at `sc`)
template <int ACT>
__device__ __forceinline__ void put(uint8_t* tile, uint8_t* sc, int lane, Block& x) {
    sc[lane] = (uint8_t)cut<ACT>(x, [&](int t, i8 q) {
        uint8_t* p = tile + t * Rows<ACT>::term;
        *(i4*)(p + lane * 16) = i4{q[0], q[1], q[2], q[3]};
        if constexpr (ACT != CGX_MX_FP4) *(i2*)(p + 1024 + lane * 8) = i2{q[4], q[5]};
    });
}

// The block from value k of a row on, 0 past the row's end.  whole: the lane's
// block lies within the row; the loads go to where the conversion reads, so that
// they stay in flight until then.  (Value by value in every lane, rows that end
// inside a block took 16.5 us for 12 x 2229 through 6144 outputs, now 9.1.)
__device__ __forceinline__ void load_block(Block& b, const float* x, int k, int cols, bool whole) {
    if (whole) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f4 v = *(const f4u*)(x + k + 4 * i), w = *(const f4u*)(x + k + 16 + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                b.a[4 * i + j] = v[j];
                b.b[4 * i + j] = w[j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const float v = x[min(k + i, cols - 1)];
            set(b, i, k + i < cols ? v : 0.0f);
        }
    }
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

typedef const __attribute__((address_space(1))) uint8_t* global_bytes;

// One KiB straight into LDS, 16 bytes a lane.
__device__ __forceinline__ void to_lds(const uint8_t* g, uint8_t* l, int lane) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(g + (unsigned)(lane * 16)),
        (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

typedef const __attribute__((address_space(4))) int* constant_ints;   // read by scalar loads

// s_waitcnt's operand that waits until n of a wave's loads are outstanding
constexpr int wait_loads(int n) { return 0x0f70 | (n & 15) | (n >> 4) << 14; }

// The block's waves meet, their reads of LDS done; the compiler moves none over it.
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);                       // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
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
    // gradient: y (+)= row_scale[m] * sum, 0 in a row whose target is none of V
    const float* row_scale;
    const int* targets;
    int V, add;
    // loss: a block half's part [m][2 nbs], the target's logit [m]
    float2* part;
    float* zt;
    // loss gradient: records of the rows' probabilities, lse
    const float* lse;
    uint8_t* p;
    int pk, pmt, pmbs;     // chunks of p, tiles of a record, row blocks
    int precord;
};

enum { kStore = 0, kGrad = 1, kStats = 2, kProbs = 3 };

// e^(z - z0), z0 not below z by much: the hardware's 2^x (an ulp) of the difference
// times log2(e).  Its two roundings cost 2^-24 |z - z0| of the result, which is the
// smaller the larger that is.  301 rows over 4096 x 128256 364 us, with expf 371; 1184
// quantised rows over 37 x 32000 28, 39.
__device__ __forceinline__ float exp_over(float z, float z0) {
    return __builtin_amdgcn_exp2f((z - z0) * 1.44269504f);
}
// Parts (top, sum) of a row's sum of e^z: where no logit is above -inf, the sum is
// taken over 0, and is 0, or NaN where a logit is.
__device__ __forceinline__ float over(float top) { return top == -INFINITY ? 0.0f : top; }

// Probabilities of a lane's row in operand order.  Lane group g = lane / 16
// holds outputs 16 n + 4 g + r of its row (acc[n][r]); block b of 32 outputs is
// tiles 2 b and 2 b + 1.  Two swaps of lane halves and quarters transpose
// groups and blocks, after which group b holds its block's 32 values in order.
__device__ __forceinline__ void probs(Block& v, const f4* acc, int col0, int N, int t, bool live,
                                      float lse) {
    unsigned q[2][4][4];                                        // [half][r][block]
#pragma unroll
    for (int n = 0; n < 8; n++) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int c = col0 + 16 * n + r;
            float p = live && c < N ? exp_over(acc[n][r], lse) : 0.0f;
            if (live && c == t) p = expm1f(acc[n][r] - lse);
            q[n & 1][r][n >> 1] = __float_as_uint(p);
        }
        __builtin_amdgcn_sched_barrier(0);                    // few registers beside the sums
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
            for (int g = 0; g < 4; g++) set(v, 16 * h + 4 * g + r, __uint_as_float(b[g]));
        }
}

// A row's part over a lane's logits v[n][r] (outputs col + 16 n + r) and those of
// the lanes that share the row, and its target's logit.
template <int TN>
__device__ __forceinline__ float2 stats(f4* v, int col, int N, int t, float* zt) {
    float top = -INFINITY, mine = 0.0f;
    if ((unsigned)t >= (unsigned)N) t = -1;
    const int at = t - col;                                   // 16 n + r where the target is here
#pragma unroll
    for (int n = 0; n < TN; n++) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            v[n][r] = 16 * n + r < N - col ? v[n][r] : -INFINITY;
            mine = at == 16 * n + r ? v[n][r] : mine;
            top = fmaxf(top, v[n][r]);
        }
        __builtin_amdgcn_sched_barrier(0);                    // few registers beside the logits
    }
    if (t >= 0 && at >= 0 && at < 16 * TN && (at & 15) < 4) *zt = mine;
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float ref = over(top);
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < TN; n++) {
#pragma unroll
        for (int r = 0; r < 4; r++) sum += exp_over(v[n][r], ref);
        __builtin_amdgcn_sched_barrier(0);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    return make_float2(top, sum);
}

// Product of 16 MT rows and 256 outputs a block of WM x 2 waves.  The weight's
// tile is the first operand, so that a lane holds four neighbouring outputs of
// one row.  Records go into LDS without passing registers, PER chunks of the
// contraction a step (more where a chunk is little work: one term).  The blocks
// of a CU overlap one's copies with another's matrix instructions; a launch of
// at most a block a CU (DEEP) copies the next chunk while it multiplies one,
// into a second array, so that the compiler sees that reads of the first need
// not wait for it.
template <int ACT, int WFMT, int MT, int WM, int PER, bool DEEP, int EPI>
__global__ __launch_bounds__(128 * WM, DEEP ? (WM + 1) / 2 : MT == 8 || WFMT == kE3M2 ? 2 : MT == 4 ? 3 : MT == 2 ? 4 : 2)
void k_gemm(const Gemm a) {
    constexpr int WN = 2, TM = MT / WM, TN = kWTiles / WN, NW = WM * WN;
    using R = Rows<ACT>;
    constexpr int XR = rows_record<ACT>(MT), WT = WFMT == kE2M1 ? 1024 : 1536;
    constexpr int WR = WFMT == kE2M1 ? kWRecord : kTRecord, XU = XR / 1024, U = XU + WR / 1024;
    constexpr int COPIES = (U + NW - 1) / NW;                 // of a wave a chunk
    static_assert(PER == 1 || !DEEP, "one chunk at a time");
    constexpr int kTurnRow = 256 + 16, kTurn = 16 * kTurnRow; // a wave's part in the epilogue
    constexpr int kChunks = PER * COPIES * NW * 1024, kParts = EPI == kStore || EPI == kGrad ? NW * kTurn : 0;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kChunks > kParts ? kChunks : kParts];
    __shared__ __attribute__((aligned(16))) uint8_t lds2[DEEP ? COPIES * NW * 1024 : 16];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
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

    // every wave issues the same number of copies; those past the record repeat its last KiB
    auto copy = [&](int j, uint8_t* l) {
        const uint8_t* gx = xb + (size_t)(a.list ? ((constant_ints)a.list)[j] - a.list0 : j) * XR;
        const uint8_t* gw = wb + (size_t)j * WR;
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
            const int u = i * NW + wave, v = i == COPIES - 1 ? min(u, U - 1) : u;
            to_lds(v < XU ? gx + v * 1024 : gw + (v - XU) * 1024, l + u * 1024, lane);
        }
    };
    auto multiply = [&](const uint8_t* lx) {
        const uint8_t* lw = lx + XR;
        __builtin_amdgcn_sched_barrier(0);
        i8 w[TN], x = operand<R::fmt>(lx + wm * TM * R::tile, lane);
        int ws[TN], xs[TM];
#pragma unroll
        for (int i = 0; i < TM; i++) xs[i] = lx[MT * R::tile + (wm * TM + i) * 64 + lane];
#pragma unroll
        for (int n = 0; n < TN; n++) {
            w[n] = operand<WFMT>(lw + (wn * TN + n) * WT, lane);
            ws[n] = lw[kWTiles * WT + (wn * TN + n) * 64 + lane];
        }
#pragma unroll
        for (int q = 0; q < TM * R::terms; q++) {
            const int i = q / R::terms, t = q % R::terms, p = q + 1;
            i8 next = x;                                      // read ahead of this one's instructions
            if (p < TM * R::terms)
                next = operand<R::fmt>(lx + (wm * TM + p / R::terms) * R::tile + p % R::terms * R::term, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < TN; n++)
                acc[i][n] = mfma<WFMT, R::fmt>(w[n], x, acc[i][n], ws[n], xs[i] - term_shift(t));
            x = next;
        }
    };
    if constexpr (DEEP) {
        copy(j0, lds);
        for (int j = j0; j < j1; j += 2) {
            copy(min(j + 1, j1 - 1), lds2);
            __builtin_amdgcn_s_waitcnt(wait_loads(COPIES));   // lds is there
            meet();
            multiply(lds);
            meet();
            if (j + 1 == j1) break;
            copy(min(j + 2, j1 - 1), lds);
            __builtin_amdgcn_s_waitcnt(wait_loads(COPIES));
            meet();
            multiply(lds2);
            meet();
        }
        __builtin_amdgcn_s_waitcnt(wait_loads(0));            // no copy is on its way any more
        meet();
    } else {
        for (int j = j0; j < j1; j += PER) {
#pragma unroll
            for (int s = 0; s < PER; s++)
                if (!s || j + s < j1) copy(j + s, lds + s * COPIES * NW * 1024);
            __builtin_amdgcn_s_waitcnt(wait_loads(0));
            __syncthreads();
#pragma unroll
            for (int s = 0; s < PER; s++)
                if (!s || j + s < j1) multiply(lds + s * COPIES * NW * 1024);
            __syncthreads();
        }
    }

    const int col0 = (nbw * kWTiles + wn * TN) * 16 + 4 * (lane >> 4);   // outputs col0 + 16 n + r
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = (mb * MT + wm * TM + i) * 16 + (lane & 15);
        if constexpr (EPI == kStore || EPI == kGrad) {
            // through the wave's part of LDS, so that a store writes 256 bytes of each of four
            // rows: 2039 rows of 4 bits through 4096 x 22016 150 us, 159 with 64 of sixteen
            uint8_t* own = lds + wave * kTurn;
#pragma unroll
            for (int h = 0; h < TN; h += 4) {
#pragma unroll
                for (int n = 0; n < 4; n++)
                    *(f4*)(own + (lane & 15) * kTurnRow + n * 64 + (lane >> 4) * 16) = acc[i][h + n];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const int c = (nbw * kWTiles + wn * TN + h) * 16 + 4 * (lane & 15);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int r = 4 * k + (lane >> 4), at = (mb * MT + wm * TM + i) * 16 + r;
                    f4 v = *(const f4*)(own + r * kTurnRow + (lane & 15) * 16);
                    if (at >= a.M) continue;
                    float* y = a.y + (size_t)z * a.stride + (size_t)at * a.ld + c;
                    if constexpr (EPI == kGrad) {
                        if (a.row_scale) v *= a.row_scale[at];
                        if ((unsigned)a.targets[at] >= (unsigned)a.V) v = f4{0, 0, 0, 0};
                    }
                    if (c + 3 < a.N) {
                        if (EPI == kGrad && a.add) v += *(const f4u*)y;
                        *(f4u*)y = v;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            if (c + q < a.N) y[q] = EPI == kGrad && a.add ? y[q] + v[q] : v[q];
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        } else if constexpr (EPI == kStats) {
            const int t = m < a.M ? a.targets[m] : -1;
            const float2 o = stats<TN>(acc[i], col0, a.N, t, a.zt + m);
            if (m < a.M && lane < 16) a.part[(size_t)m * (a.nbs * WN) + nb * WN + wn] = o;
        } else {
            // p = exp(z - lse) - [target]; rows past M and ignored ones are 0
            const int t = m < a.M ? a.targets[m] : -1;
            const bool live = t >= 0 && t < a.N;
            const float lse = live ? a.lse[m] : 0.0f;
            Block v;
            probs(v, acc[i], col0, a.N, t, live, lse);
            const int mt = mb * MT + wm * TM + i;
            if (mt < a.pmt * a.pmbs) {
                using P = Rows<CGX_MX_FP32>;
                uint8_t* rec = a.p + ((size_t)(mt / a.pmt) * a.pk + nb * WN + wn) * a.precord;
                const int at = mt % a.pmt;
                put<CGX_MX_FP32>(rec + at * P::tile, rec + a.pmt * P::tile + at * 64, lane, v);
            }
        }
    }
}

// Row blocks of mt tiles.  Launches of at most a block a CU take the DEEP form
// (40 rows through 4096 x 32000 in 250 blocks 39.6 -> 32.9 us; 61 x 768 over a
// contraction of 50304 in 255 blocks 17 us, 22 in 147 of the other form); one
// term in 128-row blocks takes two chunks a step (2039 rows of 4 bits through
// 4096 x 22016 130 -> 117 us).
template <int ACT, int WFMT, int EPI>
void gemm_launch(const Gemm& g, int mt, hipStream_t st) {
    const dim3 grid(g.mbs * g.nbs, g.splits);
    const bool deep = grid.x * grid.y <= 256;
#define CGX_MX_GEMM(MT, WM, PER, DEEP) \
    hipLaunchKernelGGL((k_gemm<ACT, WFMT, MT, WM, PER, DEEP, EPI>), grid, dim3(128 * WM), 0, st, g)
    if (mt == 1) {
        if (deep) CGX_MX_GEMM(1, 1, 1, true);
        else CGX_MX_GEMM(1, 1, 1, false);
        return;
    }
    if (mt == 2) {
        if (deep) CGX_MX_GEMM(2, 2, 1, true);
        else CGX_MX_GEMM(2, 2, 1, false);
        return;
    }
    if constexpr (WFMT == kE2M1)
        if (mt == 8) {
            CGX_MX_GEMM(8, 2, ACT == CGX_MX_FP32 ? 1 : 2, false);
            return;
        }
    if (deep) CGX_MX_GEMM(4, 4, 1, true);
    else CGX_MX_GEMM(4, 2, 1, false);
#undef CGX_MX_GEMM
}

// Splits of a contraction of kc chunks over which `blocks` blocks go: two blocks a
// CU, of at least four chunks each (a join costs what four or five chunks of a
// block do).
inline int gemm_splits(int blocks, int kc) {
    const int s = 512 / blocks, most = kc < 16 ? 1 : kc / 4;
    return s < 1 ? 1 : s < most ? s : most;
}

// Up to 16 rows: bound by the weight's bytes.  A block takes 16 T outputs at a
// time and its waves the chunks of the contraction in turn, operands of the
// weight going from memory to registers D chunks ahead.  The block cuts the
// rows once, a lane a block of 32 (cutting them in the lanes that multiply them
// would do M rows' work 16 / M times), into LDS without the rows that do not
// exist; where they do not fit, a segment of the chunks at a time.  The waves'
// sums meet in LDS.  At most a block a CU: where the outputs are more, a block
// keeps its rows and goes on with the next ones, whose first operands are on
// their way while it joins its waves' sums.
struct Gemv {
    const float* x;
    size_t ldx;
    const uint8_t* w;
    int M, K, N, kc;
    int tiles;             // of 16 outputs
    int seg;               // chunks cut at a time (gemv_seg)
    float* y;
    size_t ld;
    const int* targets;
    float2* part;          // [m][groups of T tiles]
    float* zt;
};
constexpr int kGemvWaves = 8, kGemvAhead = 2;
// bytes of a row's chunk in LDS
template <int ACT>
constexpr int gemv_chunk() { return 4 * (Rows<ACT>::terms * (ACT == CGX_MX_FP4 ? 16 : 24) + 1); }
constexpr int kGemvLds = 152 << 10;
constexpr int kGemvRound = kGemvAhead * kGemvWaves;    // chunks that the waves hold operands of
static_assert((kGemvRound + 1) * 16 * gemv_chunk<CGX_MX_FP32>() <= kGemvLds, "a segment fits");
// Chunks of a segment: all, or whole rounds.  An odd number of them is held.
template <int ACT>
int gemv_seg(int M, int kc) {
    const int fit = kGemvLds / (M * gemv_chunk<ACT>());
    return fit >= (kc | 1) ? kc : (fit - 1) / kGemvRound * kGemvRound;
}

template <int ACT, int T, int EPI>
__global__ __launch_bounds__(64 * kGemvWaves) void k_gemv(const Gemv a) {
    using R = Rows<ACT>;
    constexpr bool six = ACT != CGX_MX_FP4;
    constexpr int D = kGemvAhead, kRed = kGemvWaves * T * 1024;
    static_assert(kRed <= kGemvLds && T <= kGemvWaves, "the waves' sums fit");
    __shared__ __attribute__((aligned(16))) uint8_t lds[kGemvLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const unsigned l1 = lane, l16 = lane * 16;
    // in LDS: 16 bytes of a block [term][row][block], the 8 others, the scales; an odd
    // number of chunks a row, so that 16 rows' reads of one chunk spread over the banks
    const int ld = 4 * (a.seg | 1), n16 = R::terms * a.M * ld;
    uint8_t *const l8 = lds + n16 * 16, *const ls = l8 + (six ? n16 * 8 : 0);
    // the rows stay where the waves' sums fit behind them
    const int behind = (n16 * (six ? 24 : 16) + a.M * ld + 15) & ~15;
    const bool stay = a.seg == a.kc && behind + kRed <= kGemvLds;
    f4* red = (f4*)(lds + (stay ? behind : 0));
    i4 q[D][T];
    int s[D][T];
    auto fetch = [&](int group, int c, i4* q, int* s) {
        c = min(c, a.kc - 1);                                 // past the end: not used
#pragma unroll
        for (int t = 0; t < T; t++) {
            // tiles past the last repeat it
            const int tile = min(group * T + t, a.tiles - 1), at = tile & 15;
            global_bytes p = (global_bytes)a.w + ((size_t)(tile >> 4) * a.kc + c) * kWRecord;
            global_bytes codes = p + at * 1024, scale = p + kWTiles * 1024 + at * 64;
            // kept in scalar registers: with the lane's part added ahead of time the
            // addresses took 48 vector registers
            asm volatile("" : "+s"(codes), "+s"(scale));
            q[t] = *(const __attribute__((address_space(1))) i4*)(codes + l16);
            s[t] = scale[l1];
        }
    };
    // lanes past the last row repeat it: their products go nowhere
    const int row = min(r, a.M - 1), groups = (a.tiles + T - 1) / T;
    int group = blockIdx.x;
#pragma unroll
    for (int d = 0; d < D; d++) fetch(group, wave + d * kGemvWaves, q[d], s[d]);
    for (bool fresh = true;; fresh = !stay) {
        f4 acc[T];
#pragma unroll
        for (int t = 0; t < T; t++) acc[t] = f4{0, 0, 0, 0};
        for (int c0 = 0; c0 < a.kc; c0 += a.seg) {
            const int n = min(a.seg, a.kc - c0), blocks = 4 * n, total = a.M * blocks;
            if (c0) __syncthreads();                          // the last segment is multiplied
            if (fresh)
                for (int u0 = wave * 64; u0 < total; u0 += 64 * kGemvWaves) {
                    // lanes past the end repeat the last block
                    const int u = min(u0 + lane, total - 1), m = u / blocks, b = u - m * blocks;
                    Block x;
                    const int k = c0 * 128 + b * 32;
                    load_block(x, a.x + (size_t)m * a.ldx, k, a.K, k + 32 <= a.K);
                    const int top = cut<ACT>(x, [&](int t, i8 v) {
                        const int at = (t * a.M + m) * ld + b;
                        *(i4*)(lds + at * 16) = i4{v[0], v[1], v[2], v[3]};
                        if constexpr (six) *(i2*)(l8 + at * 8) = i2{v[4], v[5]};
                    });
                    ls[m * ld + b] = (uint8_t)top;
                }
            __syncthreads();
            for (int c = wave; c < n; c += kGemvRound)
#pragma unroll
                for (int d = 0; d < D; d++) {
                    const int e = c + d * kGemvWaves;
                    if (d && e >= n) break;
                    const int top = ls[row * ld + 4 * e + g];
#pragma unroll
                    for (int t = 0; t < R::terms; t++) {
                        const int at = (t * a.M + row) * ld + 4 * e + g;
                        const i4 u = *(const i4*)(lds + at * 16);
                        i8 x = {u[0], u[1], u[2], u[3], 0, 0, 0, 0};
                        if constexpr (six) {
                            const i2 v = *(const i2*)(l8 + at * 8);
                            x[4] = v[0];
                            x[5] = v[1];
                        }
#pragma unroll
                        for (int k = 0; k < T; k++)
                            acc[k] = mfma<kE2M1, R::fmt>(
                                i8{q[d][k][0], q[d][k][1], q[d][k][2], q[d][k][3], 0, 0, 0, 0}, x,
                                acc[k], s[d][k], top - term_shift(t));
                    }
                    if (c0 + e + kGemvRound < a.kc) fetch(group, c0 + e + kGemvRound, q[d], s[d]);
                }
        }
        const int next = group + (int)gridDim.x;
        if (next < groups)
#pragma unroll
            for (int d = 0; d < D; d++) fetch(next, wave + d * kGemvWaves, q[d], s[d]);
        if (!stay) __syncthreads();                           // the rows are multiplied
#pragma unroll
        for (int t = 0; t < T; t++) red[(wave * T + t) * 64 + lane] = acc[t];
        __syncthreads();
        auto sum = [&](int t) {
            f4 v = red[t * 64 + lane];
#pragma unroll
            for (int w = 1; w < kGemvWaves; w++) v += red[(w * T + t) * 64 + lane];
            return v;
        };
        const int col = group * T * 16 + 4 * g;
        if constexpr (EPI == kStore) {
            for (int t = wave; t < T; t += kGemvWaves) {
                const f4 v = sum(t);
                const int n = col + 16 * t;
                if (r >= a.M) continue;
                float* y = a.y + (size_t)r * a.ld + n;
                if (n + 3 < a.N) {
                    *(f4u*)y = v;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (n + k < a.N) y[k] = v[k];
                }
            }
        } else {
            // a wave a tile, then a lane a row
            const int t = r < a.M ? a.targets[r] : -1;
            f4 v = {0, 0, 0, 0};
            float2 o = {0, 0};
            if (wave < T) {
                v = sum(wave);
                o = stats<1>(&v, col + 16 * wave, a.N, t, a.zt + r);
            }
            __syncthreads();
            float2* tile = (float2*)red;
            if (wave < T && lane < 16) tile[wave * 16 + lane] = o;
            __syncthreads();
            if (wave == 0 && lane < 16 && r < a.M) {
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < T; k++) top = fmaxf(top, tile[k * 16 + lane].x);
                const float ref = over(top);
                float all = 0.0f;
#pragma unroll
                for (int k = 0; k < T; k++) {
                    const float2 p = tile[k * 16 + lane];
                    all += p.x == -INFINITY ? p.y : p.y * exp_over(p.x, ref);
                }
                a.part[(size_t)r * groups + group] = make_float2(top, all);
            }
        }
        if (next >= groups) return;
        group = next;
        __syncthreads();                                      // the sums are read
    }
}

// Whether rows take k_gemv.  Each of its blocks cuts all of them, which costs
// M K / 7100 us, against k_gemm's launch or two besides: 4096 outputs, K = 4096, ten
// rows 10.8 us, with k_gemm 11.8, twelve 11.5 and 11.8; K = 10208, three 12.3 and 13.7,
// eight 20.5 and 14.1.  From 256 blocks of 256 outputs on k_gemm fills the card
// with any rows: 128256 outputs with their loss, one row of K = 768 22.5 and 17.1, of
// 4096 55.3 and 56.5, ten 84.0 and 56.1 (50257: one of 768 13.8 and 13.6, of 4096 28.8
// and 33.9).
inline bool gemv_pays(int M, int K, int N) {
    return M <= 16 && M * (long long)K <= 48 << 10 && N <= 65536;
}

// Tiles a block: the fewest of 1, 2, 3, 4, 6 and 8 (each a kernel of its own for every
// kind of rows and epilogue: 5 and 7 are left out, for whose outputs 171 to 224 blocks
// of 6 or 8 tiles stand) that leave at most a block a CU, up to eight.  One
// block a CU and more tiles beat more blocks, each of which cuts the rows: one
// row through 4096 x 22016 10.3 us with 6 tiles (230 blocks), 13.2 with 3.
inline int gemv_tiles(int tiles) {
    for (int t : {1, 2, 3, 4, 6})
        if (tiles <= 256 * t) return t;
    return 8;
}
inline int gemv_groups(int tiles) { return (tiles + gemv_tiles(tiles) - 1) / gemv_tiles(tiles); }

template <int ACT, int EPI>
void gemv_launch(Gemv g, hipStream_t st) {
    g.seg = gemv_seg<ACT>(g.M, g.kc);
    const int groups = gemv_groups(g.tiles);
    const dim3 grid(groups < 256 ? groups : 256), block(64 * kGemvWaves);
    switch (gemv_tiles(g.tiles)) {
        case 1: hipLaunchKernelGGL((k_gemv<ACT, 1, EPI>), grid, block, 0, st, g); break;
        case 2: hipLaunchKernelGGL((k_gemv<ACT, 2, EPI>), grid, block, 0, st, g); break;
        case 3: hipLaunchKernelGGL((k_gemv<ACT, 3, EPI>), grid, block, 0, st, g); break;
        case 4: hipLaunchKernelGGL((k_gemv<ACT, 4, EPI>), grid, block, 0, st, g); break;
        case 6: hipLaunchKernelGGL((k_gemv<ACT, 6, EPI>), grid, block, 0, st, g); break;
        default: hipLaunchKernelGGL((k_gemv<ACT, 8, EPI>), grid, block, 0, st, g);
    }
}

}  // namespace mx
