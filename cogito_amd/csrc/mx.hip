// mx.hip -- microscaled blocks (32 values and a power of two): quantisation and
// read-back, the records of a 4-bit weight, and the product of rows with it.
#include "mx.hpp"

#include <algorithm>

namespace {

using namespace mx;

inline hipStream_t stream() { return (hipStream_t)cgx_stream(); }

int launch_check(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        cgx_set_error("%s launch failed: %s", what, hipGetErrorString(e));
        return -1;
    }
    return 0;
}

inline int up(long long a, int b) { return (int)((a + b - 1) / b); }

// ------------------------------------------------- quantise and read back
// Eight values of a row from k on, 0 past its end.
__device__ __forceinline__ void load8(float* v, const float* x, int k, int cols) {
    if (k + 8 <= cols) {
        const f4 a = *(const f4u*)(x + k), b = *(const f4u*)(x + k + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = k + i < cols ? x[k + i] : 0.0f;
    }
}

// A quad's lanes in another order
template <int ORDER>
__device__ __forceinline__ int quad(int v) {
    return __builtin_amdgcn_update_dpp(0, v, ORDER, 0xf, 0xf, false);
}

// Four lanes a block, eight values each; a wave takes 16 blocks of one row.
// The 6-bit conversion takes 32 values: a lane's eight go first and their six
// bytes are kept.  Bound by the bytes: 11008 rows of 4096 to 4 bits and back,
// 409 MB, 81 us (a copy of as many takes 71); four loads a wave in flight gained
// nothing, and one branch a wave around the row's end took 1.3 us more at rows of
// 1000.
template <int FMT>
__global__ __launch_bounds__(256) void k_quantize(const float* __restrict__ x, size_t ld, int rows,
                                                  int cols, int segs, uint8_t* __restrict__ codes,
                                                  uint8_t* __restrict__ scales) {
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int row = wave / segs, seg = wave - row * segs, blocks = (cols + 31) / 32;
    if (row >= rows) return;
    const int lane = threadIdx.x & 63, blk = seg * 16 + (lane >> 2), part = lane & 3;
    float v[8];
    load8(v, x + (size_t)row * ld, blk * 32 + part * 8, cols);
    int top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int b = __float_as_int(v[i]) & 0x7fffffff;
        top = b > top ? b : top;
    }
    top = max(top, quad<0xb1>(top));                          // lanes 1, 0, 3, 2
    top = max(top, quad<0x4e>(top)) >> 23;                    // lanes 2, 3, 0, 1
    const int byte = top == 255 ? 255 : top > 3 ? top - 2 : 1;
    if (blk >= blocks) return;
    const float s = pow2(byte == 255 ? 127 : byte);
    const size_t at = (size_t)row * blocks + blk;
    if (part == 0) scales[at] = (uint8_t)byte;
    if constexpr (FMT == CGX_MX_FP4) {
        unsigned r = 0;
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], s, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], s, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], s, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], s, 3);
        *(unsigned*)(codes + at * 16 + part * 4) = r;
    } else {
        f16 a = {}, b = {};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            a[i] = v[2 * i];
            b[i] = v[2 * i + 1];
        }
        const u6 q = to6<kE2M3>(a, b, s);
        uint16_t* p = (uint16_t*)(codes + at * 24 + part * 6);
        p[0] = (uint16_t)q[0];
        p[1] = (uint16_t)(q[0] >> 16);
        p[2] = (uint16_t)q[1];
    }
}

__device__ __forceinline__ float value4(int q) {
    const int e = (q >> 1) & 3;
    const float m = e ? __int_as_float(((e + 126) << 23) | (q & 1) << 22) : (q & 1) * 0.5f;
    return q & 8 ? -m : m;
}
__device__ __forceinline__ float value6(int q) {
    const int e = (q >> 3) & 3;
    const float m = e ? __int_as_float(((e + 126) << 23) | (q & 7) << 20) : (q & 7) * 0.125f;
    return q & 32 ? -m : m;
}

template <int FMT>
__global__ __launch_bounds__(256) void k_dequantize(const uint8_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, int rows,
                                                    int cols, int segs, float* __restrict__ y, size_t ld) {
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int row = wave / segs, seg = wave - row * segs, blocks = (cols + 31) / 32;
    const int lane = threadIdx.x & 63, blk = seg * 16 + (lane >> 2), part = lane & 3;
    if (row >= rows || blk >= blocks) return;
    const size_t at = (size_t)row * blocks + blk;
    const int byte = scales[at], k = blk * 32 + part * 8;
    float v[8];
    if constexpr (FMT == CGX_MX_FP4) {
        const unsigned r = *(const unsigned*)(codes + at * 16 + part * 4);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = value4((r >> (4 * i)) & 15);
    } else {
        const uint16_t* p = (const uint16_t*)(codes + at * 24 + part * 6);
        const unsigned long long r = p[0] | (unsigned long long)p[1] << 16 | (unsigned long long)p[2] << 32;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = value6((int)(r >> (6 * i)) & 63);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = byte == 255 ? NAN : ldexpf(v[i], byte - 127);
    float* o = y + (size_t)row * ld + k;
    if (k + 8 <= cols) {
        *(f4u*)o = f4{v[0], v[1], v[2], v[3]};
        *(f4u*)(o + 4) = f4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (k + i < cols) o[i] = v[i];
    }
}

// ------------------------------------------------------ weight records
// From rows of codes [N][blocks * 16] and scales [N][blocks]: a wave a tile
// (16 outputs) and chunk.  Outputs past N and blocks past K are 0.
__global__ __launch_bounds__(256) void k_weight(const uint8_t* __restrict__ codes,
                                                const uint8_t* __restrict__ scales, int N,
                                                int blocks, int kc, long long units,
                                                uint8_t* __restrict__ w) {
    const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= units) return;
    const int lane = threadIdx.x & 63, t = (int)(u % 16);
    const long long rec = u / 16;
    const int c = (int)(rec % kc), n = (int)(rec / kc) * 256 + t * 16 + (lane & 15);
    const int blk = c * 4 + (lane >> 4);
    i4 q = {0, 0, 0, 0}, o;
    int s = 127;
    if (n < N && blk < blocks) {
        const size_t at = (size_t)n * blocks + blk;
        q = *(const i4*)(codes + at * 16);
        s = scales[at];
    }
    // value i to position 2 i, value 16 + i to 2 i + 1
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned v = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int k = 4 * i + j;                          // values k and 16 + k
            v |= ((unsigned)q[k / 8] >> (4 * (k % 8)) & 15) << (8 * j);
            v |= ((unsigned)q[2 + k / 8] >> (4 * (k % 8)) & 15) << (8 * j + 4);
        }
        o[i] = (int)v;
    }
    uint8_t* p = w + (size_t)rec * kWRecord;
    *(i4*)(p + t * 1024 + lane * 16) = o;
    p[kWTiles * 1024 + t * 64 + lane] = (uint8_t)s;
}

// From a matrix [K][N], quantised along K: a thread an output and block.
__global__ __launch_bounds__(256) void k_weight_of(const float* __restrict__ x, int K, int N,
                                                   int kc, uint8_t* __restrict__ w) {
    const int n = blockIdx.x * 256 + threadIdx.x, blk = blockIdx.y, c = blk >> 2;
    Block v;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const int k = blk * 32 + i;
        set(v, i, n < N && k < K ? x[(size_t)k * N + n] : 0.0f);
    }
    uint8_t* p = w + ((size_t)blockIdx.x * kc + c) * kWRecord;
    const int t = threadIdx.x >> 4, lane = (blk & 3) * 16 + (threadIdx.x & 15);
    put<CGX_MX_FP4>(p + t * 1024, p + kWTiles * 1024 + t * 64, lane, v);
}

// ------------------------------------------------- transposed records
// For the gradient the contraction runs along the outputs, so a block is 32
// outputs of one input.  A weight's value is +-m 2^(s - 127), m in {.5 .. 6}, and s
// differs from output to output; E3M2 holds 4 m 2^-d for d = 0 .. 5 exactly.
// With top the block's largest s, layer p takes the outputs with top - s in
// 6 p .. 6 p + 5, under the scale 2^(top - 6 p - 2 - 127), so that the layers' sum
// is the weight exactly.  Layer 0 holds nearly every block; a chunk (128
// outputs) has further ones where a block of it has values there, each a chunk
// of the contraction of its own.  Layers between two that hold values are left out:
// with a row 1e-8 of the others in each chunk there are two, not the five down to it
// (1024 rows over 4096 x 32000, loss and gradient: 1163 us, with the empty ones 1869,
// without such rows 977; the copy 205 MB, 512, 102).
__device__ __forceinline__ int code_at(const uint8_t* w, int kc, int n, int k, int* s) {
    const uint8_t* p = w + ((size_t)(n >> 8) * kc + (k >> 7)) * kWRecord;
    const int t = (n >> 4) & 15, lane = ((k >> 5) & 3) * 16 + (n & 15), i = k & 31;
    *s = p[kWTiles * 1024 + t * 64 + lane];
    return p[t * 1024 + lane * 16 + (i & 15)] >> (4 * (i >> 4)) & 15;
}

// Layers of every chunk that hold a value, bit p for layer p (0 is taken to, in any
// chunk): a block a chunk and 128 inputs, a thread two blocks.  A block with a NaN
// has no values.
__global__ __launch_bounds__(256) void k_layers(const uint8_t* __restrict__ w, int N, int K,
                                                int kc, unsigned long long* __restrict__ layers) {
    const int c = blockIdx.x;
    unsigned long long held = 0;
    for (int u = threadIdx.x; u < 512; u += 256) {
        const int k = blockIdx.y * 128 + (u & 127), n0 = c * 128 + (u >> 7) * 32;
        if (k >= K) continue;
        int top = -1, low = 256, s;
        bool nan = false;
        for (int i = 0; i < 32 && n0 + i < N; i++) {
            const int q = code_at(w, kc, n0 + i, k, &s);
            nan |= s == 255;
            if (!(q & 7)) continue;
            top = s > top ? s : top;
            low = s < low ? s : low;
        }
        if (nan || top - low < 6) continue;                   // layer 0 alone
        for (int i = 0; i < 32 && n0 + i < N; i++)
            if (code_at(w, kc, n0 + i, k, &s) & 7) held |= 1ull << ((top - s) / 6);
    }
    if (held) atomicOr(&layers[c], held);
}

// A wave a tile (16 inputs) of a listed chunk and its layer.
__global__ __launch_bounds__(256) void k_transposed(const uint8_t* __restrict__ w, int N, int K,
                                                    int kc, const int* __restrict__ list,
                                                    const int* __restrict__ layers, int chunks,
                                                    uint8_t* __restrict__ out) {
    const int j = blockIdx.x, t = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int c = list[j], layer = layers[j];
    const int k = blockIdx.z * 256 + t * 16 + (lane & 15), n0 = c * 128 + (lane >> 4) * 32;
    int q[32], s[32], top = -1;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        q[i] = 0;
        s[i] = 0;
        if (k < K && n0 + i < N) q[i] = code_at(w, kc, n0 + i, k, &s[i]);
        if (s[i] == 255) nan = true;
        else if ((q[i] & 7) && s[i] > top) top = s[i];
    }
    int byte = top - 6 * layer - 2;
    byte = byte < 0 ? 0 : byte;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; i++)
        v[i] = !nan && (top - s[i]) / 6 == layer ? ldexpf(value4(q[i]), s[i] - byte) : 0.0f;
    Block x;
#pragma unroll
    for (int i = 0; i < 32; i++) set(x, i, v[i]);
    const u6 r = to6<kE3M2>(x.a, x.b, 1.0f);
    uint8_t* p = out + ((size_t)blockIdx.z * chunks + j) * kTRecord;
    *(i4*)(p + t * 1536 + lane * 16) = i4{(int)r[0], (int)r[1], (int)r[2], (int)r[3]};
    *(i2*)(p + t * 1536 + 1024 + lane * 8) = i2{(int)r[4], (int)r[5]};
    p[kWTiles * 1536 + t * 64 + lane] = (uint8_t)(nan ? 255 : top < 0 ? 127 : byte);
}

// ------------------------------------------------------- rows' records
// A wave a tile of 16 rows and a chunk, a lane a block.
template <int ACT>
__global__ __launch_bounds__(256) void k_rows(const float* __restrict__ x, size_t ld, int M, int K,
                                              int kc, int mt, long long units,
                                              uint8_t* __restrict__ out) {
    const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= units) return;
    const int lane = threadIdx.x & 63, tile = (int)(u / kc), c = (int)(u - (long long)tile * kc);
    // rows past the last repeat it: nothing of theirs is stored
    const int m = min(tile * 16 + (lane & 15), M - 1);
    Block v;
    const int k = c * 128 + (lane >> 4) * 32;
    load_block(v, x + (size_t)m * ld, k, K, k + 32 <= K);
    using R = Rows<ACT>;
    const int b = tile / mt, at = tile - b * mt;
    uint8_t* rec = out + ((size_t)b * kc + c) * (size_t)rows_record<ACT>(mt);
    put<ACT>(rec + at * R::tile, rec + mt * R::tile + at * 64, lane, v);
}

// Splits of a product: y[m][n] (+)= row_scale[m] * sum of part[s][m][n], 0 in a
// row whose target is none of V.  G lanes take the splits of four outputs in
// turn, four loads in flight, and their sums are added in order: 49 splits of
// 61 x 768 with one lane 6.3 us, with eight 4.7.
template <int G>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ part, int splits,
                                              size_t stride, int pld, int M, int N,
                                              float* __restrict__ y, size_t ld,
                                              const float* __restrict__ row_scale,
                                              const int* __restrict__ targets, int V, int add) {
    constexpr int Q = 256 / G;                                // fours of outputs
    __shared__ f4 sum[G][Q];
    const int q = threadIdx.x % Q, g = threadIdx.x / Q, m = blockIdx.y;
    const int n = 4 * (blockIdx.x * Q + q);
    f4 v = {0, 0, 0, 0};
    if (n < N) {
        const float* p = part + (size_t)m * pld + n;
        for (int s = g; s < splits; s += 4 * G) {
            f4 t[4];
#pragma unroll
            for (int i = 0; i < 4; i++) t[i] = *(const f4*)(p + (size_t)min(s + G * i, splits - 1) * stride);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (s + G * i < splits) v += t[i];
        }
    }
    if constexpr (G > 1) {
        sum[g][q] = v;
        __syncthreads();
        if (g) return;
#pragma unroll
        for (int i = 1; i < G; i++) v += sum[i][q];
    }
    if (n >= N) return;
    if (row_scale) v *= row_scale[m];
    if (targets && (unsigned)targets[m] >= (unsigned)V) v = f4{0, 0, 0, 0};
    float* o = y + (size_t)m * ld + n;
    if (n + 3 < N) {
        if (add) v += *(const f4u*)o;
        *(f4u*)o = v;
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (n + r < N) o[r] = add ? o[r] + v[r] : v[r];
    }
}

}  // namespace

// ------------------------------------------------------------ launchers
extern "C" int cgk_mx_quantize(const float* x, size_t ld, int rows, int cols, int format,
                               uint8_t* codes, uint8_t* scales) {
    const int segs = up(cols, 512);
    const dim3 grid(up((long long)rows * segs, 4));
    if (format == CGX_MX_FP4)
        hipLaunchKernelGGL((k_quantize<CGX_MX_FP4>), grid, dim3(256), 0, stream(), x, ld, rows, cols,
                           segs, codes, scales);
    else
        hipLaunchKernelGGL((k_quantize<CGX_MX_FP6>), grid, dim3(256), 0, stream(), x, ld, rows, cols,
                           segs, codes, scales);
    return launch_check("mx quantize");
}

extern "C" int cgk_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int cols,
                                 int format, float* y, size_t ld) {
    const int segs = up(cols, 512);
    const dim3 grid(up((long long)rows * segs, 4));
    if (format == CGX_MX_FP4)
        hipLaunchKernelGGL((k_dequantize<CGX_MX_FP4>), grid, dim3(256), 0, stream(), codes, scales,
                           rows, cols, segs, y, ld);
    else
        hipLaunchKernelGGL((k_dequantize<CGX_MX_FP6>), grid, dim3(256), 0, stream(), codes, scales,
                           rows, cols, segs, y, ld);
    return launch_check("mx dequantize");
}

extern "C" size_t cgk_mx_weight_bytes(int K, int N) {
    return (size_t)up(N, 256) * up(K, 128) * kWRecord;
}
extern "C" int cgk_mx_weight(const uint8_t* codes, const uint8_t* scales, int K, int N, uint8_t* w) {
    const int kc = up(K, 128);
    const long long units = (long long)up(N, 256) * kc * 16;
    hipLaunchKernelGGL(k_weight, dim3(up(units, 4)), dim3(256), 0, stream(), codes, scales, N,
                       up(K, 32), kc, units, w);
    return launch_check("mx weight");
}
extern "C" int cgk_mx_weight_of(const float* x, int K, int N, uint8_t* w) {
    const int kc = up(K, 128);
    hipLaunchKernelGGL(k_weight_of, dim3(up(N, 256), kc * 4), dim3(256), 0, stream(), x, K, N, kc, w);
    return launch_check("mx weight of a tensor");
}

// layers (device, 64 bits a chunk of 128 outputs, 0 before)
extern "C" int cgk_mx_layers(const uint8_t* w, int K, int N, uint64_t* layers) {
    hipLaunchKernelGGL(k_layers, dim3(up(N, 128), up(K, 128)), dim3(256), 0, stream(), w, N, K,
                       up(K, 128), (unsigned long long*)layers);
    return launch_check("mx layers");
}
extern "C" size_t cgk_mx_transposed_bytes(int K, int chunks) {
    return (size_t)up(K, 256) * chunks * kTRecord;
}
extern "C" int cgk_mx_transposed(const uint8_t* w, int K, int N, const int* list, const int* layers,
                                 int chunks, uint8_t* out) {
    hipLaunchKernelGGL(k_transposed, dim3(chunks, 4, up(K, 256)), dim3(256), 0, stream(), w, N, K,
                       up(K, 128), list, layers, chunks, out);
    return launch_check("mx transpose");
}

// Records of rows, mt tiles each, for the row blocks' whole height.
extern "C" int cgk_mx_rows(const float* x, size_t ld, int M, int K, int act, int mt, uint8_t* out) {
    const int kc = up(K, 128);
    const long long units = (long long)up(M, 16 * mt) * mt * kc;
    const dim3 grid(up(units, 4));
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, grid, dim3(256), 0, stream(), x, ld, M, K, kc, mt, units, out);
    };
    if (act == CGX_MX_FP4) go(k_rows<CGX_MX_FP4>);
    else if (act == CGX_MX_FP6) go(k_rows<CGX_MX_FP6>);
    else go(k_rows<CGX_MX_FP32>);
    return launch_check("mx rows");
}
extern "C" size_t cgk_mx_rows_bytes(int M, int K, int act, int mt) {
    const size_t rec = act == CGX_MX_FP4 ? rows_record<CGX_MX_FP4>(mt)
                       : act == CGX_MX_FP6 ? rows_record<CGX_MX_FP6>(mt) : rows_record<CGX_MX_FP32>(mt);
    return rec * up(M, 16 * mt) * up(K, 128);
}

extern "C" int cgk_mx_join(const float* part, int splits, size_t stride, int pld, int M, int N,
                           float* y, size_t ld, const float* row_scale, const int* targets,
                           int V, int add) {
    if (splits > 4)
        hipLaunchKernelGGL((k_join<8>), dim3(up(N, 128), M), dim3(256), 0, stream(), part, splits,
                           stride, pld, M, N, y, ld, row_scale, targets, V, add);
    else
        hipLaunchKernelGGL((k_join<1>), dim3(up(N, 1024), M), dim3(256), 0, stream(), part, splits,
                           stride, pld, M, N, y, ld, row_scale, targets, V, add);
    return launch_check("mx join");
}

namespace {

constexpr int kSlab = 4096;          // rows a launch: bounds the records' workspace

// How M rows go over a weight: tiles of a row block, blocks, and splits of K
// where there are fewer than two blocks a CU.
struct Plan {
    int mt, mbs, nbs, splits;
    size_t rows, part;               // bytes
};
Plan plan(const cgx_mx_weight* w, int M, int act) {
    Plan p = {};
    if (gemv_pays(M, w->K, w->N)) return p;
    p.mt = cgk_mx_tiles(M, w->N);
    p.mbs = up(M, 16 * p.mt);
    p.nbs = up(w->N, 256);
    p.splits = gemm_splits(p.mbs * p.nbs, up(w->K, 128));
    p.rows = (cgk_mx_rows_bytes(M, w->K, act, p.mt) + 255) & ~(size_t)255;
    p.part = p.splits > 1 ? (size_t)p.splits * M * ((w->N + 3) & ~3) * 4 : 0;
    return p;
}

template <int ACT>
void gemm(const Gemm& g, int mt) { gemm_launch<ACT, kE2M1, kStore>(g, mt, stream()); }
template <int ACT>
void gemv(const Gemv& g) {
    gemv_launch<ACT, kStore>(g, stream());
}

}  // namespace

// Tiles of a row block: 128 rows unless 64 leave a tenth fewer rows empty (fp32
// rows: 1024 through 4096 x 32000 304 us, with 64-row blocks 314, with 32-row ones 355;
// the loss of 301 over 4096 x 128256 374 us with 64, 438 with 128, 408 with 32), half
// where that leaves a CU without two blocks (200 through 4096 x 4096: 23 us with 32
// rows, 26 with 64, 31 with 128; 64: 14.9, 16.6 and 23.9; 61 through 768 x 50257: 16.2,
// 16.7 and 28.7, where one term prefers 64: 11.9 and 11.3).
extern "C" int cgk_mx_tiles(int M, int N) {
    if (M <= 16) return 1;
    int mt = 10 * up(M, 128) * 128 <= 11 * up(M, 64) * 64 ? 8 : 4;
    while (mt > 2 && (long long)up(M, 16 * mt) * up(N, 256) < 512) mt /= 2;
    return mt;
}

extern "C" size_t cgk_mx_matmul_need(const cgx_mx_weight* w, int M, int act) {
    size_t need = 0;
    if (M >= kSlab) {
        const Plan p = plan(w, kSlab, act);
        need = p.rows + p.part;
        M %= kSlab;
    }
    if (M) {
        const Plan p = plan(w, M, act);
        need = std::max(need, p.rows + p.part);
    }
    return need;
}
// ... of any call of at most M rows
extern "C" size_t cgk_mx_matmul_ws(const cgx_mx_weight* w, int M, int act) {
    const int top = std::min(M, kSlab);
    size_t need = top ? cgk_mx_matmul_need(w, top, act) : 0;
    for (int m = 16; m < top; m += 16) need = std::max(need, cgk_mx_matmul_need(w, m, act));
    return need;
}

extern "C" int cgk_mx_matmul(const float* x, size_t ldx, int M, const cgx_mx_weight* w, int act,
                             float* y, size_t ldy, void* ws) {
    for (int m0 = 0; m0 < M; m0 += kSlab) {
        const int m = std::min(kSlab, M - m0);
        const Plan p = plan(w, m, act);
        const float* xm = x + (size_t)m0 * ldx;
        float* ym = y + (size_t)m0 * ldy;
        if (gemv_pays(m, w->K, w->N)) {
            Gemv g = {};
            g.x = xm;
            g.ldx = ldx;
            g.w = w->codes;
            g.M = m;
            g.K = w->K;
            g.N = w->N;
            g.kc = up(w->K, 128);
            g.y = ym;
            g.ld = ldy;
            g.tiles = up(w->N, 16);
            if (act == CGX_MX_FP4) gemv<CGX_MX_FP4>(g);
            else if (act == CGX_MX_FP6) gemv<CGX_MX_FP6>(g);
            else gemv<CGX_MX_FP32>(g);
            if (launch_check("mx product of few rows")) return -1;
            continue;
        }
        uint8_t* rows = (uint8_t*)ws;
        if (cgk_mx_rows(xm, ldx, m, w->K, act, p.mt, rows)) return -1;
        const int kc = up(w->K, 128), pld = (w->N + 3) & ~3;
        Gemm g = {};
        g.x = rows;
        g.w = w->codes;
        g.xk = g.wk = g.j1 = kc;
        g.mbs = p.mbs;
        g.nbs = p.nbs;
        g.splits = p.splits;
        g.M = m;
        g.N = w->N;
        if (p.splits > 1) {
            g.y = (float*)(rows + p.rows);
            g.ld = pld;
            g.stride = (size_t)m * pld;
        } else {
            g.y = ym;
            g.ld = ldy;
        }
        if (act == CGX_MX_FP4) gemm<CGX_MX_FP4>(g, p.mt);
        else if (act == CGX_MX_FP6) gemm<CGX_MX_FP6>(g, p.mt);
        else gemm<CGX_MX_FP32>(g, p.mt);
        if (launch_check("mx product")) return -1;
        if (p.splits > 1 &&
            cgk_mx_join(g.y, p.splits, g.stride, pld, m, w->N, ym, ldy, nullptr, nullptr, 0, 0))
            return -1;
    }
    return 0;
}
