// paged_attn.hip -- attention of ragged batches over the paged INT4 KV cache.
//
//   o_t = sum_j softmax_j(s_tj) v_j,  s_tj = (q_t . k_j) / sqrt(D)
// over the keys that row t sees (chain or tree mask), with one pass over the
// keys: running maximum m, running sum l and O, both held relative to m.
//
// Lengths, row offsets and tables are device words.  Every address formed from
// them is bounded here: a length by the table row, a page by the pool, a row
// by the row arrays.
//
// Head dimensions of 32 to 128 with scales per 32 dimensions or more run on
// the matrix cores (k_attn_paged); the rest takes k_attn_paged_row.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "cgx_internal.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

inline hipStream_t stream() { return (hipStream_t)cgx_stream(); }

int launch_check(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        cgx_set_error("%s launch failed: %s", what, hipGetErrorString(e));
        return -1;
    }
    return 0;
}

struct PagedArgs {
    const uint8_t* kp;           // this layer's pages
    const uint8_t* vp;
    const float* ks;
    const float* vs;
    int lp, num_pages, H, Hk, D, gs;
    int seqs, rows, table_ld;
    const int* table;
    const int* row_begin;
    const int* row_seq;
    const int* kv_len;
    const float* Q;
    const unsigned long long* anc;
    const int* tree_len;
    float scale;
    float* O;
    float* lse;
    // k_attn_paged: sequences of r_lo .. r_hi query rows times heads a KV
    // head, key chunks of at least c_min, about `target` units; partial
    // results of split tiles, this launch's from row part_row on, at most
    // max_parts tiles of them
    int r_lo, r_hi, c_min, target, max_parts;
    long long part_row, part_rows;
    float* part_o;               // [part_rows][D]
    float* part_ml;              // [part_rows][2]
    int4* info;                  // [rows][2] where k_paged_join finds a row's pieces: their number,
                                 // the sequence's first row of part_o (two words), the row's place
                                 // in the sequence; its tiles, rows a tile, 0, 0
};

__device__ __forceinline__ float code(unsigned n) { return (float)((int)(n << 28) >> 28); }

// A block a (row, head, piece of the keys), its waves take 64 keys a round in
// turn: scores with a key a lane (its row of K in 16-byte loads), then O with
// two dims a lane and byte, the keys' weights and pages from the lanes that
// have them, eight keys' loads together.  The waves' sums are joined in LDS,
// those of pieces by k_attn_paged_row_join.  Bound by the latency of a round
// (about 15 us at 256 dims: a key's 128 bytes are a lane's own, and a byte of V
// is a load): 5 rows of 8 heads of 256 at 4096 keys 34.5 us, 8 sequences of
// 1024 keys 22.9 (one wave a row without pieces: 1766 and 445).
constexpr int kRowWaves = 4, kVKeys = 8;

// the row's sequence and its place there; false: no sequence has it
__device__ __forceinline__ bool place_of(const PagedArgs& a, int t, int& b, int& n, int& i) {
    b = a.row_seq[t];
    if (b < 0 || b >= a.seqs) return false;
    const int r0 = a.row_begin[b];
    n = a.row_begin[b + 1] - r0;
    i = t - r0;
    return i >= 0 && i < n;
}

__global__ __launch_bounds__(64 * kRowWaves) void k_attn_paged_row(PagedArgs a) {
    constexpr int W = kRowWaves;
    __shared__ __attribute__((aligned(16))) float s_q[256];
    __shared__ float s_ml[W][2], s_o[W][256];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int b, n, i;
    if (!place_of(a, t, b, n, i)) return;
    const int D = a.D, half = D / 2, gs = a.gs, ng = D / gs, cb = D / 32;
    const int L = (int)min((long long)max(a.kv_len[b], 0), (long long)a.table_ld << a.lp);
    const int hk = h / (a.H / a.Hk);
    int base, end;                               // keys below base: seen; from base: bits
    unsigned long long bits = 0;
    if (a.anc) {
        base = L - min(max(a.tree_len ? a.tree_len[b] : n, 0), L);
        end = L;
        bits = a.anc[t];
    } else {
        end = min(L, max(0, L - n + i + 1));
        base = end;
    }
    const int S = gridDim.z, piece = ((end + S - 1) / S + 63) / 64 * 64, from = blockIdx.z * piece;
    end = min(end, from + piece);
    const float* q = a.Q + ((size_t)t * a.H + h) * D;
    for (int d = threadIdx.x; d < D; d += 64 * W) s_q[d] = q[d] * a.scale;
    __syncthreads();

    // the lane's dims d, d + 1 (and of D > 128, those 128 later) in a V block
    int voff[2], vg[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int d = min(2 * (lane + 64 * x), D - 2), nb = d / (D / 16);
        voff[x] = nb * 16 * cb + (d - nb * (D / 16)) / 2;
        vg[x] = d / gs;
    }
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = from + 64 * wave; k0 < end; k0 += 64 * W) {
        const int j = k0 + lane;
        bool see = j < end && (j < base || (j - base < 64 && ((bits >> (j - base)) & 1)));
        int page = -1;
        if (see) page = a.table[(size_t)b * a.table_ld + (j >> a.lp)];
        see = see && page >= 0 && page < a.num_pages;
        // the page's head: of 2^31 of them K alone would have 2^39 bytes
        const int ph = (see ? page : 0) * a.Hk + hk;
        const size_t pr = ((size_t)ph << a.lp) + (j & ((1 << a.lp) - 1));
        float s = -INFINITY;
        if (see) {
            const u32x4* kw = (const u32x4*)(a.kp + pr * half);
            const float* ks = a.ks + pr * ng;
            float sc = *ks;
            int left = gs;
            s = 0.0f;
            for (int w = 0; w < cb; w++) {
                const u32x4 x = kw[w];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const f32x4 q0 = *(const f32x4*)(s_q + 32 * w + 8 * c), q1 = *(const f32x4*)(s_q + 32 * w + 8 * c + 4);
                    float d[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const f32x4& qq = y < 2 ? q0 : q1;
                        d[y] = qq[2 * y & 3] * code(x[c] >> (8 * y)) + qq[(2 * y & 3) + 1] * code(x[c] >> (8 * y + 4));
                    }
                    if (gs % 8 == 0) {
                        s += ((d[0] + d[1]) + (d[2] + d[3])) * sc;
                        left -= 8;
                        if (!left && 32 * w + 8 * c + 8 < D) {
                            sc = *++ks;
                            left = gs;
                        }
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            s += d[y] * sc;
                            left -= 2;
                            if (!left && 32 * w + 8 * c + 2 * y + 2 < D) {
                                sc = *++ks;
                                left = gs;
                            }
                        }
                    }
                }
            }
        }
        float top = s;
        for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float mn = fmaxf(m, top);
        if (!__any(see)) continue;
        // a NaN score makes its weight, and so the row, NaN
        const float p = see ? __expf(s - mn) : 0.0f, f = m == mn ? 1.0f : __expf(m - mn);
        float sum = p;
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        l = l * f + sum;
        m = mn;
        for (int x = 0; x < 4; x++) o[x] *= f;
        // a key that is not seen has weight 0 and page 0: read, not added
        for (int kk = 0; kk < min(64, end - k0); kk += kVKeys) {
            uint32_t c[kVKeys][2];
            float v[kVKeys][2], w[kVKeys];
#pragma unroll
            for (int y = 0; y < kVKeys; y++) {
                w[y] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), kk + y));
                const size_t pk = (size_t)__builtin_amdgcn_readlane(ph, kk + y) << a.lp;
                const int ak = (k0 + kk + y) & ((1 << a.lp) - 1);
                const uint8_t* vp = a.vp + pk * half + (size_t)(ak >> 4) * (256 * cb) + (ak & 15) * cb;
                const float* vs = a.vs + (pk + ak) * ng;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    c[y][x] = vp[voff[x]];
                    v[y][x] = vs[vg[x]];
                }
            }
#pragma unroll
            for (int y = 0; y < kVKeys; y++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const float sv = w[y] == 0.0f ? 0.0f : w[y] * v[y][x];
                    o[2 * x] += sv * code(c[y][x] & 15);
                    o[2 * x + 1] += sv * code(c[y][x] >> 4);
                }
        }
    }
    if (lane == 0) {
        s_ml[wave][0] = m;
        s_ml[wave][1] = l;
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int d = 2 * (lane + 64 * x);
        if (d < D) *(f32x2*)&s_o[wave][d] = (f32x2){o[2 * x], o[2 * x + 1]};
    }
    __syncthreads();
    float M = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) M = fmaxf(M, s_ml[w][0]);
    float f[W];
#pragma unroll
    for (int w = 0; w < W; w++) {
        f[w] = s_ml[w][0] == M ? 1.0f : __expf(s_ml[w][0] - M);
        sum += f[w] * s_ml[w][1];
    }
    const size_t row = (size_t)t * a.H + h, pr = row * S + blockIdx.z;
    for (int d = threadIdx.x; d < D; d += 64 * W) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) v += f[w] * s_o[w][d];
        if (S > 1) a.part_o[pr * D + d] = v;
        else a.O[row * D + d] = sum != 0.0f ? v / sum : 0.0f;
    }
    if (threadIdx.x) return;
    if (S > 1) *(f32x2*)(a.part_ml + 2 * pr) = (f32x2){M, sum};
    else if (a.lse) a.lse[row] = sum != 0.0f ? M + logf(sum) : -INFINITY;
}

// Joins the S <= 64 pieces of a (row, head): one wave, four dims a lane.
__global__ __launch_bounds__(64) void k_attn_paged_row_join(PagedArgs a, int S) {
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, D = a.D;
    int b, n, i;
    if (!place_of(a, t, b, n, i)) return;
    const size_t row = (size_t)t * a.H + h, pr = row * S;
    const f32x2 ml = *(const f32x2*)(a.part_ml + 2 * (pr + min(lane, S - 1)));
    float M = ml.x;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
    const float w = ml.x == M ? 1.0f : __expf(ml.x - M);
    float l = lane < S ? w * ml.y : 0.0f;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
    const int d = min(4 * lane, D - 4);
    f32x4 o = (f32x4)(0.0f);
    for (int s = 0; s < S; s++) o += __shfl(w, s) * *(const f32x4*)(a.part_o + (pr + s) * D + d);
    if (4 * lane < D) *(f32x4*)(a.O + row * D + d) = l != 0.0f ? o / l : (f32x4)(0.0f);
    if (a.lse && lane == 0) a.lse[row] = l != 0.0f ? M + logf(l) : -INFINITY;
}

// ------------------------------------------------------- matrix-core kernel
//
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16.  The codes of K
// and V are exact fp16 integers.  Q (times scale log2 e) and the weights P v_s
// (v_s the key's V scale) are each two fp16 terms, hi + lo, of a value brought
// into [2^14, 2^15) by its row's power of two: 22 bits of it, and of values
// down to 2^-16 of the row's largest; products are exact, sums fp32.  The K
// scale multiplies the key's fp32 score.  A lane of group g (lane / 16) holds
// query row lane % 16 and the scores of keys 4g .. 4g + 3 of each half tile,
// which is the B operand of the second product, so P never moves.  Row state
// (m, l and the exponent e of the weights) is a lane's own; the maximum goes
// over the four lane groups with two lane-row swaps.
//
// The exponent follows the weights' largest of the tile, or what the sums so
// far still need (e minus the whole part of the maximum's rise): V scales may
// lie any distance apart.
//
// Bound, for one row a sequence, by the pages' bytes and the kernel's ends (64
// sequences of up to 4096 keys, 32/8 heads of 128: 51 us, the tiles 27 to 36 of
// them at 6 TB/s, search, first loads and operands 5, sums 3, join 6); for many
// rows by vector issue beside the products (509 rows after 2048 keys: 62 us, 9
// vector instructions a product: codes to fp16, softmax, hi + lo); for few rows
// by the chain of dependent steps (5 rows at 4096 keys: 17 us, tiles 5.5).
// Pieces of all items in even lengths (63 us instead of 54), the scores of the
// next tile beside the softmax (56 and 64 us), long pieces first (no change)
// and more than one round of blocks (57) were slower or no faster.
constexpr int kTile = 32;                        // keys of a wave's step

__device__ __forceinline__ float max_rows(float v) {     // over lanes l, l ^ 16, l ^ 32, l ^ 48
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// the same of the bits of values that are not negative
__device__ __forceinline__ uint32_t max_bits(float f) {
    const uint32_t v = __float_as_uint(f);
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t x = max(a[0], a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(b[0], b[1]);
}

__device__ __forceinline__ float sum_rows(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Masks in SGPRs and the fp16 exponent bits in VGPRs, made where the compiler
// does not see constants (VOP3 takes no literals here): a nibble's sign bit
// turned and its exponent set is then one instruction, else two or three.
struct Nib {
    uint32_t lo, hi, mag_lo, mag_hi;
};
__device__ __forceinline__ Nib nib_consts() {
    Nib k;
    asm volatile("s_mov_b32 %0, 0x000f000f" : "=s"(k.lo));
    asm volatile("s_mov_b32 %0, 0x00f000f0" : "=s"(k.hi));
    asm volatile("v_mov_b32 %0, 0x64086408" : "=v"(k.mag_lo));
    asm volatile("v_mov_b32 %0, 0x64806480" : "=v"(k.mag_hi));
    return k;
}

// Nibbles 0 and 4 (or 1 and 5) of a word of codes, exact: 0x6400 with a nibble
// is 1024 + n, or 1024 + 16 n; with its sign bit turned, 8 more than the code.
__device__ __forceinline__ uint32_t masked(uint32_t w, uint32_t mask, uint32_t mag) {
    return __builtin_amdgcn_bitop3_b32(w, mask, mag, 0x6A);      // (w & mask) ^ mag
}
__device__ __forceinline__ f16x2 low_nibbles(uint32_t w, const Nib& k) {
    const f16x2 m = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    return __builtin_bit_cast(f16x2, masked(w, k.lo, k.mag_lo)) + m;
}
__device__ __forceinline__ f16x2 high_nibbles(uint32_t w, const Nib& k) {
    const f16x2 s = {(_Float16)0.0625f, (_Float16)0.0625f}, m = {(_Float16)-72.0f, (_Float16)-72.0f};
    return __builtin_elementwise_fma(__builtin_bit_cast(f16x2, masked(w, k.hi, k.mag_hi)), s, m);
}

// Eight codes of a word: element p is nibble slot_of(p).
__device__ __forceinline__ int slot_of(int p) { return (p >> 1) + 4 * (p & 1); }
__device__ __forceinline__ f16x8 codes8(uint32_t w, const Nib& k) {
    const f16x2 a = low_nibbles(w, k), b = high_nibbles(w, k), c = low_nibbles(w >> 8, k),
                d = high_nibbles(w >> 8, k);
    f16x8 r;
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
    r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
    return r;
}

// x[p] * up as hi + lo, up a power of two: the product is exact, and so is
// what hi leaves of it.
__device__ __forceinline__ void split8(const float (&x)[8], float up, f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int p = 0; p < 8; p += 2) {
        const f32x2 v = {x[p] * up, x[p + 1] * up};
        const f16x2 h = __builtin_convertvector(v, f16x2);
        const f32x2 r = {fmaf(x[p], up, -(float)h[0]), fmaf(x[p + 1], up, -(float)h[1])};
        const f16x2 q = __builtin_convertvector(r, f16x2);
        hi[p] = h[0]; hi[p + 1] = h[1];
        lo[p] = q[0]; lo[p + 1] = q[1];
    }
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const u32x4 v = *(const u32x4*)p;
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N == 2) {
        const u32x2 v = *(const u32x2*)p;
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = ((const uint32_t*)p)[i];
    }
}

struct Unit {
    int b, hk, tile, split, nsplit, part, first, tiles, L, n, r0;
};

__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {      // inclusive scan over the wave
#define CGX_ROW(CTRL, RMASK) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, RMASK, 0xF, true)
    CGX_ROW(0x111, 0xF);
    CGX_ROW(0x112, 0xF);
    CGX_ROW(0x114, 0xF);
    CGX_ROW(0x118, 0xF);
    CGX_ROW(0x142, 0xA);
    CGX_ROW(0x143, 0xC);
#undef CGX_ROW
    return v;
}
__device__ __forceinline__ float dpp_total(float v) {          // the wave's sum, in every lane
#define CGX_ROW(CTRL, RMASK) \
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, RMASK, 0xF, true))
    CGX_ROW(0x111, 0xF);
    CGX_ROW(0x112, 0xF);
    CGX_ROW(0x114, 0xF);
    CGX_ROW(0x118, 0xF);
    CGX_ROW(0x142, 0xA);
    CGX_ROW(0x143, 0xC);
#undef CGX_ROW
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// The block's unit of work: sequences of r_lo .. r_hi rows in order, each with
// Hk * tiles * nsplit units.  The chunk length C follows from the keys of all
// of them, so that there are about `target` units whatever the lengths; a
// sequence is cut into round(len / C) even pieces.  Every wave finds this out
// for itself from the lengths, a lane taking B / 64 sequences: no LDS, no
// barrier, against a launch more and a wait for it.
//
// The counts are 32 bits: consistent lengths stay below the grid, and others
// may wrap, where a unit is only ever one that some sequence has.
__device__ __forceinline__ bool find_unit(const PagedArgs& a, int trows, Unit& u) {
    const int lane = threadIdx.x & 63, B = a.seqs, G = a.H / a.Hk;
    const long long most = (long long)a.table_ld << a.lp;
    struct Seq { int r0, n, L, tiles; };
    auto seq = [&](int b) {
        Seq s = {0, 0, 0, 0};
        if (b >= B) return s;
        const int r0 = a.row_begin[b], r1 = a.row_begin[b + 1], kv = a.kv_len[b];
        s.r0 = min(max(r0, 0), a.rows);
        s.n = max(0, min(r1, a.rows) - s.r0);
        s.L = (int)min((long long)max(kv, 0), most);
        const long long R = (long long)s.n * G;
        s.tiles = R >= a.r_lo && R <= a.r_hi ? (int)((R + trows - 1) / trows) : 0;
        return s;
    };
    const int per = (B + 63) >> 6, b0 = lane * per;
    const Seq s0 = seq(b0);
    // the work as a float: it only sets C, the same in every wave
    float work = (float)s0.tiles * (float)s0.L;
    for (int i = 1; i < per; i++) {
        const Seq s = seq(b0 + i);
        work += (float)s.tiles * (float)s.L;
    }
    work = dpp_total(work);
    const uint32_t cf = (uint32_t)fminf(work * (float)a.Hk / (float)a.target, 1.0e9f);
    const uint32_t C = (max(cf + 1, (uint32_t)a.c_min) + kTile - 1) / kTile * kTile;
    auto splits = [&](const Seq& s) { return max(1u, ((uint32_t)s.L + C / 2) / C); };
    const uint32_t ns0 = splits(s0), here0 = s0.tiles * a.Hk * ns0;
    uint32_t units = here0, parts = ns0 > 1 ? here0 : 0;
    for (int i = 1; i < per; i++) {
        const Seq s = seq(b0 + i);
        const uint32_t ns = splits(s), h = s.tiles * a.Hk * ns;
        units += h;
        parts += ns > 1 ? h : 0;
    }
    uint32_t pu = dpp_add(units) - units, pp = dpp_add(parts) - parts;
    const uint32_t me = blockIdx.x;
    const unsigned long long mine = __ballot(me >= pu && me - pu < units);
    if (!mine) return false;
    const int owner = __builtin_ctzll(mine);
    // the owner's first sequence of the unit, then its fields to every lane
    Seq s = s0;
    int b = b0;
    uint32_t ns = ns0, here = here0;
    if (lane == owner)
        while (me - pu >= here) {
            pu += here;
            if (ns > 1) pp += here;
            s = seq(++b);
            ns = splits(s);
            here = s.tiles * a.Hk * ns;
        }
    auto give = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
    u.b = give(b);
    u.L = give(s.L);
    u.n = give(s.n);
    u.r0 = give(s.r0);
    u.nsplit = give((int)ns);
    const uint32_t tiles = (uint32_t)give(s.tiles), x = me - (uint32_t)give((int)pu), y = x / a.Hk;
    const uint32_t first = min((uint32_t)give((int)pp), (uint32_t)a.max_parts);
    u.first = (int)first;
    u.tiles = (int)tiles;
    // KV heads fastest: with 8 of them a head's pieces share an XCD's L2
    u.hk = (int)(x - y * a.Hk);
    u.split = (int)(y / tiles);
    u.tile = (int)(y - (uint32_t)u.split * tiles);
    u.part = -1;
    if (u.nsplit > 1) {
        const unsigned long long at = first + ((unsigned long long)u.hk * tiles + u.tile) * u.nsplit + u.split;
        u.part = at < (unsigned)a.max_parts ? (int)at : -2;
    }
    return true;
}

// Barrier for LDS alone: loads from memory in flight stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// One unit.  NC = D / 32, NG scales a head row; the block's waves are RG groups
// of 16 RT query rows times KG that take the tiles of 32 keys in turn, their
// sums joined in LDS.
template <int NC, int NG, int RT, int RG, int KG, int WPS>
__global__ __launch_bounds__(64 * RG * KG, WPS) void k_attn_paged(PagedArgs a) {
    constexpr int D = 32 * NC, half = D / 2, TROWS = 16 * RT * RG;
    constexpr int GD = D / NG, TPG = GD / 16, NT = D / 16;   // dims, O tiles a group; O tiles
    constexpr int kQBytes = RG * RT * NC * 2 * 64 * (int)sizeof(f16x8);
    constexpr int kOBytes = KG / 2 * TROWS * (D + 4) * (int)sizeof(float);
    // the Q operands, and when the tiles are done, the waves' O
    __shared__ __attribute__((aligned(16))) unsigned char s_raw[kQBytes > kOBytes ? kQBytes : kOBytes];
    f16x8 (*s_q)[RT][NC][2][64] = (f16x8 (*)[RT][NC][2][64])s_raw;
    float (*s_o)[TROWS][D + 4] = (float (*)[TROWS][D + 4])s_raw;
    __shared__ float s_ml[KG][TROWS][2];
    Unit u;
    if (!find_unit(a, TROWS, u)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = wave % KG, rg = wave / KG;
    const int n = lane & 15, g = lane >> 4, G = a.H / a.Hk, R = u.n * G, L = u.L;
    const int row0 = u.tile * TROWS + rg * 16 * RT;
    const Nib nib = nib_consts();
    const int hk = u.hk, b = u.b, lp = a.lp, pmask = (1 << lp) - 1;

    // chain: keys up to base + i; tree: keys below base and those of the bits
    int base = L - u.n;
    if (a.anc && a.tree_len) base = L - min(max(a.tree_len[b], 0), L);
    if (a.anc) base = max(base, 0);
    // the lane's row of row tile rt, worked out again where it is needed: the
    // loop over the keys has no registers for it
    struct RowOf {
        bool ok;
        int i, j, t;                             // place in the sequence, head of the KV head, entry of
                                                 // the row arrays
        size_t q;                                // row of Q and O
    };
    auto row_of = [&](int rt) {
        int nn = n;
        asm volatile("" : "+v"(nn));
        const int r = row0 + 16 * rt + nn;
        RowOf x;
        x.ok = r < R;
        x.i = x.ok ? r / G : 0;
        x.j = x.ok ? r - x.i * G : 0;
        x.t = u.r0 + x.i;
        x.q = (size_t)x.t * a.H + hk * G + x.j;
        return x;
    };
    int end = 0;                                 // keys that any of the wave's rows may see
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int last = min(R - 1, row0 + 16 * rt + 15);
        if (row0 + 16 * rt < R) end = max(end, a.anc ? L : min(L, base + last / G + 1));
    }
    // the unit's piece of the keys, and what all of the wave's rows see of it
    const int piece = ((L + u.nsplit - 1) / u.nsplit + kTile - 1) / kTile * kTile;
    const int k_begin = u.split * piece;
    end = min(end, min(L, k_begin + piece));
    const int first_i = row0 < R ? row0 / G : 0;
    const int open_end = row0 < R ? min(L, a.anc ? base : base + first_i + 1) : 0;

    // ---- V^T operands: group y's O tile t has dims y GD + TPG n + t of lane
    //      n, that is bytes beta .. of block blk of the V page
    int voff[NG], beta[NG];
#pragma unroll
    for (int y = 0; y < NG; y++) {
        const int d0 = y * GD + n * TPG;
        voff[y] = (d0 / (2 * NC)) * (16 * NC) + 4 * g * NC;
        beta[y] = NG == 1 ? 0 : d0 % (2 * NC) / 2;
    }
    struct Tile {
        uint32_t k[2][NC], v[2][NG][NC];
        f32x4 ks[2][NG], vs[2][NG];
        int ok;                                  // bit h: half h's page is in the pool
    };
    // page numbers by scalar loads (nobody writes the table while this runs):
    // as vector loads each would wait for the tile in flight
    typedef const __attribute__((address_space(4))) int* scalar_ints;
    const scalar_ints tab = (scalar_ints)(uintptr_t)(a.table + (size_t)b * a.table_ld);
    struct Pages { int p[2]; };
    auto pages = [&](int kt) {
        Pages x;
#pragma unroll
        for (int h = 0; h < 2; h++) x.p[h] = kt + 16 * h < end ? tab[(kt + 16 * h) >> lp] : -1;
        return x;
    };
    auto load = [&](int kt, const Pages& pg, Tile& t) {
        t.ok = 0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool in = pg.p[h] >= 0 && pg.p[h] < a.num_pages;
            t.ok |= in << h;
            const size_t row = (((size_t)(in ? pg.p[h] : 0) * a.Hk + hk) << lp) + ((kt + 16 * h) & pmask);
            const uint8_t* kp = a.kp + row * half;
            if constexpr (NG == 1) {
                load_words<NC>(kp + (uint32_t)(n * half + 4 * NC * g), t.k[h]);
            } else {
#pragma unroll
                for (int c = 0; c < NC; c++) t.k[h][c] = *(const uint32_t*)(kp + (uint32_t)(n * half + 16 * c + 4 * g));
            }
            const float* sp = a.ks + row * NG;
#pragma unroll
            for (int y = 0; y < NG; y++) t.ks[h][y] = *(const f32x4*)(sp + (uint32_t)(4 * g * NG + 4 * y));
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool in = (t.ok >> h) & 1;
            const size_t row = (((size_t)(in ? pg.p[h] : 0) * a.Hk + hk) << lp) + ((kt + 16 * h) & pmask);
            const uint8_t* vp = a.vp + row * half;       // 16 positions of a head: 16 half bytes
#pragma unroll
            for (int y = 0; y < NG; y++) load_words<NC>(vp + (uint32_t)voff[y], t.v[h][y]);
            const float* sp = a.vs + row * NG;
#pragma unroll
            for (int y = 0; y < NG; y++) t.vs[h][y] = *(const f32x4*)(sp + (uint32_t)(4 * g * NG + 4 * y));
        }
    };

    // ---- Q^T operands: element p of chunk c is dim (NG == 1) g D/4 + 8 c +
    //      slot, (NG > 1) 32 c + 8 g + slot, so that a product never spans
    //      two scale groups.  Q's loads come first, then the first tile's, so
    //      that the operands are made while that is on its way.
    float qv[RT][NC][8];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const RowOf row = row_of(rt);
        const float* q = a.Q + row.q * D;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int x = 0; x < 8; x += 4) {
                const float4 t = *(const float4*)(q + (NG == 1 ? g * (D / 4) + 8 * c : 32 * c + 8 * g) + x);
                qv[rt][c][x] = row.ok ? t.x : 0.0f;
                qv[rt][c][x + 1] = row.ok ? t.y : 0.0f;
                qv[rt][c][x + 2] = row.ok ? t.z : 0.0f;
                qv[rt][c][x + 3] = row.ok ? t.w : 0.0f;
            }
    }
    constexpr int step = KG * kTile;
    int kt = k_begin + kg * kTile;
    Tile x;
    load(kt, pages(kt), x);
    Pages ahead = pages(kt + step);
    float qinv[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const float f = a.scale * 1.44269504088896340736f;
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                qv[rt][c][i] *= f;
                top = fmaxf(top, fabsf(qv[rt][c][i]));
            }
        top = max_rows(top);
        // 2^e <= top < 2^(e + 1); far exponents are cut where fp16's range covers them
        int e = (int)(__float_as_uint(top) >> 23) - 127;
        e = min(max(e, -100), 127);
        qinv[rt] = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
        const float up = __uint_as_float((uint32_t)(min(14 - e, 127) + 127) << 23);
        if (kg != rt % KG) continue;             // the group's rows: one writer
#pragma unroll
        for (int c = 0; c < NC; c++) {
            float v[8];
#pragma unroll
            for (int p = 0; p < 8; p++) v[p] = qv[rt][c][slot_of(p)];
            f16x8 hi, lo;
            split8(v, up, hi, lo);
            s_q[rg][rt][c][0][lane] = hi;
            s_q[rg][rt][c][1][lane] = lo;
        }
    }
    lds_barrier();

    float m[RT], l[RT];
    int ew[RT][NG];
    f32x4 o[RT][NT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int y = 0; y < NG; y++) ew[rt][y] = -100;
#pragma unroll
        for (int t = 0; t < NT; t++) o[rt][t] = (f32x4)(0.0f);
    }

    // OPEN: every key of the tile is seen by every row; NR: row tiles that hold
    // rows.  A wave that has 16 rows or fewer (a rest, or a sequence of few rows
    // beside ones of many) leaves the second one out: draft trees 27.8 us instead
    // of 28.9, 40 mixed batches 17.4 instead of 17.8.
    const bool two = R - row0 > 16;
    auto tile_of = [&](auto open, auto row_tiles, const Tile& td, int kt) {
        constexpr bool OPEN = decltype(open)::value;
        constexpr int NR = decltype(row_tiles)::value;
        int ql = lane;
        asm volatile("" : "+v"(ql));             // Q is read again each tile, not kept in registers
        f32x4 s[NR][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f32x4 acc[NR];
#pragma unroll
            for (int y = 0; y < NG; y++) {
#pragma unroll
                for (int rt = 0; rt < NR; rt++) acc[rt] = (f32x4)(0.0f);
#pragma unroll
                for (int c = y * NC / NG; c < (y + 1) * NC / NG; c++) {
                    const f16x8 kc = codes8(td.k[h][c], nib);
#pragma unroll
                    for (int rt = 0; rt < NR; rt++) {
                        acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, s_q[rg][rt][c][0][ql], acc[rt], 0, 0, 0);
                        acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, s_q[rg][rt][c][1][ql], acc[rt], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int rt = 0; rt < NR; rt++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        // scales of key x: [x * NG + y] of the four keys' scales
                        const float sc = td.ks[h][(x * NG + y) / 4][(x * NG + y) % 4];
                        s[rt][h][x] = y ? s[rt][h][x] + acc[rt][x] * sc : acc[rt][x] * sc;
                    }
            }
        }
        unsigned see[NR];
        float drop[NR], pr[NR][8];
        int whole[NR];
#pragma unroll
        for (int rt = 0; rt < NR; rt++) {
            see[rt] = 0xffu;
            if constexpr (!OPEN) {
                see[rt] = 0;
                const RowOf row = row_of(rt);
                const int lim = !row.ok ? -1 : a.anc ? base - 1 : base + row.i;     // last key seen without a bit
                const unsigned long long bits = a.anc && row.ok ? a.anc[row.t] : 0;
#pragma unroll
                for (int p = 0; p < 8; p++) {
                    const int key = kt + (p < 4 ? 4 * g + p : 12 + 4 * g + p), d = key - base;
                    const bool bit = key >= base && d < 64 && ((bits >> (d & 63)) & 1);
                    const bool yes = key < end && ((td.ok >> (p >> 2)) & 1) && (key <= lim || bit);
                    see[rt] |= (unsigned)yes << p;
                    s[rt][p >> 2][p & 3] = yes ? s[rt][p >> 2][p & 3] : -INFINITY;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int p = 0; p < 8; p++) top = fmaxf(top, s[rt][p >> 2][p & 3]);
            const float mn = fmaxf(m[rt], max_rows(top) * qinv[rt]);
            // a score that is NaN leaves m alone and makes l NaN; without any
            // score so far every weight is exp2(-inf) = 0
            const float mu = mn == -INFINITY ? 0.0f : mn;
            drop[rt] = m[rt] == mn ? 0.0f : mn - m[rt];
            m[rt] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int p = 0; p < 8; p++) {
                pr[rt][p] = __builtin_amdgcn_exp2f(fmaf(s[rt][p >> 2][p & 3], qinv[rt], -mu));
                sum += pr[rt][p];
            }
            l[rt] = l[rt] * __builtin_amdgcn_exp2f(-drop[rt]) + sum;
            whole[rt] = (int)fminf(drop[rt], 300.0f);
        }
#pragma unroll
        for (int y = 0; y < NG; y++) {
            f16x8 hi[NR], lo[NR];
#pragma unroll
            for (int rt = 0; rt < NR; rt++) {
                float w[8], big = 0.0f;
#pragma unroll
                for (int p = 0; p < 8; p++) {
                    const int e = (p & 3) * NG + y;
                    const float vs = td.vs[p >> 2][e / 4][e % 4];
                    // a hidden key's scale may be anything
                    w[p] = OPEN || ((see[rt] >> p) & 1) ? pr[rt][p] * vs : 0.0f;
                    big = fmaxf(big, fabsf(w[p]));
                }
                const int et = (int)(max_bits(big) >> 23) - 127;
                const int en = max(max(et, ew[rt][y] - whole[rt]), -100);
                const float f = __builtin_amdgcn_exp2f((float)(ew[rt][y] - en) - drop[rt]);
                ew[rt][y] = en;
                split8(w, __uint_as_float((uint32_t)(14 - en + 127) << 23), hi[rt], lo[rt]);
                if (__any(f != 1.0f)) {
#pragma unroll
                    for (int t = 0; t < TPG; t++) o[rt][y * TPG + t] *= f;
                }
            }
#pragma unroll
            for (int t = 0; t < TPG; t++) {
                const uint32_t at = (uint32_t)(beta[y] + t / 2) * 0x10001u;
                constexpr int b23 = NC == 4 ? 2 : NC == 1 ? 0 : 1;         // first word of keys 2, 3
                const uint32_t s01 = (0x0C000C00u | (NC << 16)) + at;
                const uint32_t s23 = (0x0C000C00u | ((3 * NC - 4 * b23) << 16) | (2 * NC - 4 * b23)) + at;
                f16x8 va;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t (&v)[NC] = td.v[h][y];
                    const uint32_t w01 = __builtin_amdgcn_perm(v[NC > 2 ? 1 : 0], v[0], s01);
                    const uint32_t w23 = __builtin_amdgcn_perm(v[NC > 2 ? b23 + 1 : b23], v[b23], s23);
                    const f16x2 x = t & 1 ? high_nibbles(w01, nib) : low_nibbles(w01, nib);
                    const f16x2 z = t & 1 ? high_nibbles(w23, nib) : low_nibbles(w23, nib);
                    va[4 * h] = x[0]; va[4 * h + 1] = x[1]; va[4 * h + 2] = z[0]; va[4 * h + 3] = z[1];
                }
#pragma unroll
                for (int rt = 0; rt < NR; rt++) {
                    o[rt][y * TPG + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, hi[rt], o[rt][y * TPG + t], 0, 0, 0);
                    o[rt][y * TPG + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, lo[rt], o[rt][y * TPG + t], 0, 0, 0);
                }
            }
        }
    };

    auto tile = [&](auto open, const Tile& td, int kt) {
        if constexpr (RT == 2) {
            if (!two) return tile_of(open, std::integral_constant<int, 1>(), td, kt);
        }
        tile_of(open, std::integral_constant<int, RT>(), td, kt);
    };

    // open tiles first, two in turn: one is loaded while the other is
    // multiplied (past the end page 0's first rows, which nobody looks at);
    // from the first tile on that is not open for all rows, one at a time
    //
    // A wave's priority falls as it nears its end: the waves of a SIMD else run
    // oldest first, and the last one ends alone, with nothing to overlap.
    const int open_to = min(open_end, end) - kTile;
    const int q2 = k_begin + (end - k_begin) / 2, q1 = (k_begin + q2) / 2, q3 = (q2 + end) / 2;
    auto pace = [&]() {
        if (kt >= q3) __builtin_amdgcn_s_setprio(0);
        else if (kt >= q2) __builtin_amdgcn_s_setprio(1);
        else if (kt >= q1) __builtin_amdgcn_s_setprio(2);
        else __builtin_amdgcn_s_setprio(3);
    };
    pace();
    if constexpr (NC * NG <= 4) {
        Tile y;
        for (;;) {
            if (kt > open_to || x.ok != 3) break;
            load(kt + step, ahead, y);
            ahead = pages(kt + 2 * step);
            tile(std::true_type(), x, kt);
            kt += step;
            pace();
            if (kt > open_to || y.ok != 3) {
                x = y;
                break;
            }
            load(kt + step, ahead, x);
            ahead = pages(kt + 2 * step);
            tile(std::true_type(), y, kt);
            kt += step;
            pace();
        }
    } else {
        // the words and scales of several groups leave no registers for a
        // second tile
        while (kt <= open_to && x.ok == 3) {
            tile(std::true_type(), x, kt);
            kt += step;
            pace();
            load(kt, ahead, x);
            ahead = pages(kt + step);
        }
    }
    while (kt < end) {
        tile(std::false_type(), x, kt);
        kt += step;
        load(kt, ahead, x);
        ahead = pages(kt + step);
    }
    __builtin_amdgcn_s_setprio(0);

    // ---- row sums, and O back to one scale relative to m
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        l[rt] = sum_rows(l[rt]);
#pragma unroll
        for (int y = 0; y < NG; y++) {
            const float dn = __uint_as_float((uint32_t)(ew[rt][y] - 14 + 127) << 23);
#pragma unroll
            for (int t = 0; t < TPG; t++) o[rt][y * TPG + t] *= dn;
        }
    }
    // element x of a group's O tiles is TPG neighbouring dims of lane group g
    auto dim = [&](int y, int x) { return y * GD + (4 * g + x) * TPG; };
    auto put = [&](float* to, const f32x4 (&v)[NT], float f) {
#pragma unroll
        for (int y = 0; y < NG; y++)
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int t = 0; t < TPG; t += 2)
                    *(f32x2*)(to + dim(y, x) + t) = (f32x2){v[y * TPG + t][x] * f, v[y * TPG + t + 1][x] * f};
    };

    // the key groups' maxima and sums, then O of the upper half of them onto
    // the lower until one is left
    const int lr = rg * 16 * RT + n;             // the row's place in the tile, plus 16 rt
    if (g == 0) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            s_ml[kg][lr + 16 * rt][0] = m[rt];
            s_ml[kg][lr + 16 * rt][1] = l[rt];
        }
    }
    lds_barrier();
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        float M = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < KG; w++) M = fmaxf(M, s_ml[w][lr + 16 * rt][0]);
#pragma unroll
        for (int w = 0; w < KG; w++) {
            const float mw = s_ml[w][lr + 16 * rt][0];
            sum += s_ml[w][lr + 16 * rt][1] * (mw == M ? 1.0f : __builtin_amdgcn_exp2f(mw - M));
        }
        const float f = m[rt] == M ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - M);
        m[rt] = M;
        l[rt] = sum;
#pragma unroll
        for (int t = 0; t < NT; t++) o[rt][t] *= f;
    }
#pragma unroll
    for (int from = KG / 2; from > 0; from >>= 1) {
        if (kg >= from && kg < 2 * from) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) put(&s_o[kg - from][lr + 16 * rt][0], o[rt], 1.0f);
        }
        lds_barrier();
        if (kg < from) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int y = 0; y < NG; y++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
#pragma unroll
                        for (int t = 0; t < TPG; t++)
                            o[rt][y * TPG + t][x] += s_o[kg][lr + 16 * rt][dim(y, x) + t];
        }
        if (from > 1) lds_barrier();
    }
    if (kg) return;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const RowOf row = row_of(rt);
        if (!row.ok) continue;
        if (a.part_rows && u.hk == 0 && u.split == 0 && g == 0) {
            // one of the row's lanes says where its pieces are
            if (row.j == 0) {
                const long long at = a.part_row + (long long)u.first * TROWS;
                a.info[2 * (size_t)row.t] = make_int4(u.nsplit, (int)at, (int)(at >> 32), row.i);
                a.info[2 * (size_t)row.t + 1] = make_int4(u.tiles, TROWS, 0, 0);
            }
        }
        if (u.part == -1) {
            const float inv = l[rt] != 0.0f ? 1.0f / l[rt] : 0.0f;
            put(a.O + row.q * D, o[rt], inv);
            if (a.lse && g == 0)
                a.lse[row.q] = l[rt] != 0.0f ? 0.69314718055994530942f * (m[rt] + log2f(l[rt])) : -INFINITY;
        } else if (u.part >= 0) {
            const size_t pr = (size_t)a.part_row + (size_t)u.part * TROWS + lr + 16 * rt;
            put(a.part_o + pr * D, o[rt], 1.0f);
            if (g == 0) {
                a.part_ml[2 * pr] = m[rt];
                a.part_ml[2 * pr + 1] = l[rt];
            }
        }
    }
}

// Joins the pieces of split rows: block = (row, every gridDim.y-th head), its
// waves take pieces in turn; m relative to the largest of the pieces, as in
// the block itself.  A row's place comes in one load, its pieces' sums and
// values together in the next.  Bound by those two and its launch: 3.6 us for 5
// rows of 32 heads, 6 to 8 for 64 and for 95 pieces of one row.
constexpr int kJoin = 4;                         // pieces a wave loads at a time
template <int W>
__global__ __launch_bounds__(64 * W) void k_paged_join(PagedArgs a) {
    __shared__ float s_o[W][128];
    const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int4 f = a.info[2 * (size_t)t], f2 = a.info[2 * (size_t)t + 1];
    const int b = a.row_seq[t], ns = f.x, tiles = f2.x, trows = f2.y, G = a.H / a.Hk, D = a.D;
    if (b < 0 || b >= a.seqs || ns < 2 || tiles < 1 || trows < 1) return;
    // a row that its sequence does not have, or of a sequence left out, holds
    // an earlier call's words
    const int r0 = min(max(a.row_begin[b], 0), a.rows), rn = min(a.row_begin[b + 1], a.rows) - r0;
    if (f.w != t - r0 || f.w < 0 || f.w >= rn || (long long)rn * G > a.r_hi) return;
    const long long base = (long long)(uint32_t)f.y | (long long)f.z << 32;
    const int d = min(2 * lane, D - 2);
    for (int h = blockIdx.y; h < a.H; h += gridDim.y) {
        const int hk = h / G;
        const uint32_t r = (uint32_t)f.w * G + (h - hk * G), tile = r / (uint32_t)trows;
        const long long p0 = base + (long long)(((uint32_t)hk * tiles + tile) * (uint32_t)ns) * trows + (r - tile * trows);
        if (base < 0 || tile >= (uint32_t)tiles || p0 + (long long)(ns - 1) * trows >= a.part_rows) return;
        float M = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int s0 = 0; s0 < ns; s0 += 64) {
            const f32x2 ml = *(const f32x2*)(a.part_ml + 2 * (p0 + (long long)min(s0 + lane, ns - 1) * trows));
            const int cnt = min(64, ns - s0);
            f32x2 v[kJoin];
            auto get = [&](int k0) {
#pragma unroll
                for (int x = 0; x < kJoin; x++)
                    v[x] = *(const f32x2*)(a.part_o + (p0 + (long long)(s0 + min(k0 + x, cnt - 1)) * trows) * D + d);
            };
            get(kJoin * wave);
            float top = ml.x;
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
            const float mn = fmaxf(M, top), g = M == mn ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
            M = mn;
            const float w = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
            l = l * g + (lane < cnt ? w * ml.y : 0.0f);
            o0 *= g;
            o1 *= g;
            for (int k0 = kJoin * wave; k0 < cnt; k0 += kJoin * W) {
                f32x2 now[kJoin];
#pragma unroll
                for (int x = 0; x < kJoin; x++) now[x] = v[x];
                if (k0 + kJoin * W < cnt) get(k0 + kJoin * W);
#pragma unroll
                for (int x = 0; x < kJoin; x++) {
                    const float wx = __shfl(w, min(k0 + x, cnt - 1));
                    if (k0 + x < cnt) {
                        o0 += wx * now[x].x;
                        o1 += wx * now[x].y;
                    }
                }
            }
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
        s_o[wave][d] = o0;
        s_o[wave][d + 1] = o1;
        __syncthreads();
        for (int e = threadIdx.x; e < D; e += 64 * W) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) v += s_o[w][e];
            a.O[((size_t)t * a.H + h) * D + e] = l != 0.0f ? v / l : 0.0f;
        }
        if (a.lse && threadIdx.x == 0)
            a.lse[(size_t)t * a.H + h] = l != 0.0f ? 0.69314718055994530942f * (M + log2f(l)) : -INFINITY;
        __syncthreads();
    }
}

int log2i(int x) {
    int l = 0;
    while ((1 << l) < x) l++;
    return l;
}

// How a call is cut: the split launch (few rows a KV head, keys over the
// waves) and the tile launch (more rows, rows over the waves).
struct Launch {
    int rt, r_lo, r_hi, c_min, target, max_parts;
    long long grid, part_row;
};
struct Plan {
    bool fast;
    int row_pieces;              // not fast: pieces of the keys
    Launch l[2];
    int n;
    long long part_rows;
    size_t info, part_o, total;
};

// Up to 32 rows times heads a KV head are one unit whose waves share the keys;
// with 16 the draft trees take 43 us instead of 28 and 5 rows of 4 heads each
// at 4096 keys 21 instead of 17.
constexpr int kSplitRows = 32;
// Blocks up to which k_attn_paged_row's keys are cut: 5 rows of 8 heads of 256
// at 4096 keys take 46 us with 512, 34.5 with 1024 and 2048, and 239 uncut.
constexpr int kRowBlocks = 1024;

// What the host knows of a step.
struct Sizes {
    bool fast;
    long long R, seqs, keys;     // rows times heads a KV head of one sequence, sequences, positions
    long long tiles;             // of 64 rows
    int row_keys;                // pieces that k_attn_paged_row's keys can be cut into
};
Sizes sizes_of(const cgx_kv_paged_int4* c, const cgx_paged_step* s, int H) {
    const int G = H / c->n_heads;
    const long long most = s->max_rows && s->max_rows < s->rows ? s->max_rows : s->rows;
    Sizes z;
    z.fast = c->head_dim <= 128 && c->group_size % 32 == 0;
    z.R = most * G;
    z.seqs = s->seqs < s->rows ? s->seqs : s->rows;
    z.keys = (long long)s->table_ld * c->page_size;
    z.tiles = ((long long)s->rows * G) / 64 + z.seqs;
    const long long n = (z.keys + 64 * kRowWaves - 1) / (64 * kRowWaves);
    z.row_keys = (int)(n > 64 ? 64 : n);
    return z;
}

// How finely the keys of a launch's tiles are cut, and the blocks and split
// tiles that follow.
struct Cut {
    int trows, c_min, target;
    long long grid(long long tiles, int heads, long long keys) const {
        // round(len / C) pieces: at most target units by length and one a tile
        const long long whole = tiles * heads, pieces = (keys + c_min / 2) / c_min, cut = whole * (pieces < 1 ? 1 : pieces);
        const long long g = whole + target + 8;      // 8: C is rounded in 32 bits
        return g > cut ? cut : g;
    }
    int parts(long long tiles, int heads, long long keys) const {
        if ((keys + c_min / 2) / c_min < 2) return 0;
        // a split tile has at least 1.5 C keys, so at most 4/3 target pieces in all
        const long long g = grid(tiles, heads, keys), most = target * 4 / 3 + 8;
        return (int)(g < most ? g : most);
    }
};
// Smallest chunks: a cut has to save more than the launch that joins its
// pieces (4-5 us).  Mean of 40 mixed batches: 128 and 256 keys 18.4 us, 384
// and 512 17.8, 384 and 768 18.2.  The units fill the card once (3, 2 and 1
// blocks a CU): with a third more 64 sequences take 57 us instead of 51.
constexpr Cut kCut16 = {16, 384, 768}, kCut32 = {32, 384, 448}, kCut64 = {64, 512, 256};

Plan plan_of(const cgx_kv_paged_int4* c, const cgx_paged_step* s, int H) {
    Plan p = {};
    const Sizes z = sizes_of(c, s, H);
    const int D = c->head_dim;
    p.fast = z.fast;
    if (!s->rows) return p;
    if (!p.fast) {
        const long long blocks = (long long)s->rows * H;
        const long long n = blocks < kRowBlocks ? kRowBlocks / blocks : 1;
        p.row_pieces = (int)(n < z.row_keys ? n : z.row_keys);
        if (p.row_pieces > 1) p.total = (size_t)blocks * p.row_pieces * (D + 2) * 4;
        return p;
    }
    auto add = [&](int rt, int lo, long long hi, long long tiles, const Cut& cut) {
        Launch& l = p.l[p.n++];
        l.rt = rt;
        l.r_lo = lo;
        l.r_hi = (int)(hi > 0x7fffffff ? 0x7fffffff : hi);
        l.c_min = cut.c_min;
        l.target = cut.target;
        l.grid = cut.grid(tiles, c->n_heads, z.keys);
        l.max_parts = cut.parts(tiles, c->n_heads, z.keys);
        l.part_row = p.part_rows;
        p.part_rows += (long long)l.max_parts * cut.trows;
    };
    // One sequence: one launch, whichever its bound on the rows asks for
    const bool tiles = z.R > kSplitRows, both = tiles && s->seqs > 1;
    if (!tiles || both)
        add(z.R > 16 ? 2 : 1, 1, z.R < kSplitRows ? z.R : kSplitRows, z.seqs, z.R > 16 ? kCut32 : kCut16);
    if (tiles) add(-2, both ? kSplitRows + 1 : 1, 0x7fffffff, z.tiles, kCut64);
    if (!p.part_rows) return p;
    p.info = 2 * (size_t)s->rows * sizeof(int4);
    p.part_o = (size_t)p.part_rows * D * 4;
    p.total = p.info + p.part_o + (size_t)p.part_rows * 2 * 4;
    return p;
}

template <int NC, int NG>
void launch_shape(const Launch& l, const PagedArgs& a) {
    // the words and scales of NC NG > 4 take the registers of a second row tile
    constexpr int RT = NC * NG > 4 ? 1 : 2, S = 2 / RT;
    const dim3 grid((unsigned)l.grid);
    if (l.rt == 1) hipLaunchKernelGGL((k_attn_paged<NC, NG, 1, 1, 4, (NC * NG > 4 ? 2 : 3)>), grid, dim3(256), 0, stream(), a);
    else if (l.rt == 2) hipLaunchKernelGGL((k_attn_paged<NC, NG, RT, S, 4 / S, 2>), grid, dim3(256), 0, stream(), a);
    else hipLaunchKernelGGL((k_attn_paged<NC, NG, RT, 2 * S, 4 / S, 2>), grid, dim3(512), 0, stream(), a);
}

void launch(const Launch& l, const PagedArgs& a) {
    const int nc = a.D / 32, ng = a.D / a.gs;
    switch (8 * nc + ng) {
        case 9: launch_shape<1, 1>(l, a); break;
        case 17: launch_shape<2, 1>(l, a); break;
        case 18: launch_shape<2, 2>(l, a); break;
        case 25: launch_shape<3, 1>(l, a); break;
        case 27: launch_shape<3, 3>(l, a); break;
        case 33: launch_shape<4, 1>(l, a); break;
        case 34: launch_shape<4, 2>(l, a); break;
        default: launch_shape<4, 4>(l, a); break;
    }
}

}  // namespace

// What this call writes.
extern "C" size_t cgk_paged_attention_need(const cgx_kv_paged_int4* c, const cgx_paged_step* s,
                                           int H) {
    return plan_of(c, s, H).total;
}

// What no call of at most these sequences, rows, positions and rows of one
// sequence passes: fewer rows may be cut into more pieces, or take launches
// that the step itself does not need.
extern "C" size_t cgk_paged_attention_ws(const cgx_kv_paged_int4* c, const cgx_paged_step* s,
                                         int H) {
    const Sizes z = sizes_of(c, s, H);
    const size_t word = (size_t)(c->head_dim + 2) * 4;           // a partial row
    if (!s->rows) return 0;
    if (!z.fast) {
        if (z.row_keys < 2 || 2 * H > kRowBlocks) return 0;
        const long long cut = (long long)s->rows * H * z.row_keys;
        return (size_t)(cut < kRowBlocks ? cut : kRowBlocks) * word;
    }
    auto rows_of = [&](const Cut& cut, long long tiles) { return (long long)cut.parts(tiles, c->n_heads, z.keys) * cut.trows; };
    const long long few = rows_of(kCut16, z.seqs), some = z.R > 16 ? rows_of(kCut32, z.seqs) : 0,
                    many = z.R > kSplitRows ? rows_of(kCut64, z.tiles) : 0;
    long long most = s->seqs > 1 ? some + many : some > many ? some : many;
    if (most < few) most = few;
    return most ? 2 * (size_t)s->rows * sizeof(int4) + (size_t)most * word : 0;
}

// whether the blocks stay within a launch's 2^32 threads
extern "C" int cgk_paged_attention_fits(const cgx_kv_paged_int4* c, const cgx_paged_step* s,
                                        int H) {
    const Plan p = plan_of(c, s, H);
    for (int i = 0; i < p.n; i++)
        if (p.l[i].grid >= 1 << 23) return 0;
    return 1;
}

extern "C" int cgk_paged_attention(const cgx_kv_paged_int4* c, int layer,
                                   const cgx_paged_step* s, const float* Q, int H,
                                   const unsigned long long* anc, const int* tree_len, float* O,
                                   float* lse, void* ws) {
    const size_t rows = (size_t)c->num_pages * c->page_size * c->n_heads;
    const size_t bytes = rows * (size_t)(c->head_dim / 2) * layer;
    const size_t groups = rows * (size_t)(c->head_dim / c->group_size) * layer;
    PagedArgs a = {};
    a.kp = c->k_pages + bytes;
    a.vp = c->v_pages + bytes;
    a.ks = c->k_scales + groups;
    a.vs = c->v_scales + groups;
    a.lp = log2i(c->page_size);
    a.num_pages = c->num_pages;
    a.H = H;
    a.Hk = c->n_heads;
    a.D = c->head_dim;
    a.gs = c->group_size;
    a.seqs = s->seqs;
    a.rows = s->rows;
    a.table_ld = s->table_ld;
    a.table = s->table;
    a.row_begin = s->row_begin;
    a.row_seq = s->row_seq;
    a.kv_len = s->kv_len;
    a.Q = Q;
    a.anc = anc;
    a.tree_len = tree_len;
    a.scale = 1.0f / sqrtf((float)c->head_dim);
    a.O = O;
    a.lse = lse;
    const Plan p = plan_of(c, s, H);
    if (!p.fast) {
        a.part_o = (float*)ws;
        a.part_ml = a.part_o + (size_t)s->rows * H * p.row_pieces * a.D;
        hipLaunchKernelGGL(k_attn_paged_row, dim3(s->rows, H, p.row_pieces), dim3(64 * kRowWaves), 0, stream(), a);
        if (launch_check("k_attn_paged_row")) return -1;
        if (p.row_pieces == 1) return 0;
        hipLaunchKernelGGL(k_attn_paged_row_join, dim3(s->rows, H), dim3(64), 0, stream(), a, p.row_pieces);
        return launch_check("k_attn_paged_row_join");
    }
    a.info = (int4*)ws;
    a.part_o = (float*)((char*)ws + p.info);
    a.part_ml = (float*)((char*)a.part_o + p.part_o);
    a.part_rows = p.part_rows;
    for (int i = 0; i < p.n; i++) {
        const Launch& l = p.l[i];
        a.r_lo = l.r_lo;
        a.r_hi = l.r_hi;
        a.c_min = l.c_min;
        a.target = l.target;
        a.max_parts = l.max_parts;
        a.part_row = l.part_row;
        launch(l, a);
        if (launch_check("k_attn_paged")) return -1;
    }
    if (!p.part_rows) return 0;
    // a block a head, or, of many rows, blocks that walk the heads.  Few blocks
    // have waves for the many pieces that a row may have, many blocks only take
    // each other's places with them: 2, 4 and 8 waves need for a row of 131071
    // keys 44.5, 41.4 and 39.8 us, for 64 rows of 32 heads 50.2, 51.6 and 52.6.
    const int ny = s->rows >= 2048 ? 1 : 2048 / s->rows, gy = ny < H ? ny : H;
    const dim3 grid(s->rows, gy);
    if ((long long)s->rows * gy < 512) hipLaunchKernelGGL(k_paged_join<8>, grid, dim3(512), 0, stream(), a);
    else hipLaunchKernelGGL(k_paged_join<2>, grid, dim3(128), 0, stream(), a);
    return launch_check("k_paged_join");
}
