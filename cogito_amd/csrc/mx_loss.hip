// mx_loss.hip -- softmax cross entropy over the vocabulary of a microscaled
// lm_head, from hidden rows, and its gradient with respect to them.
//
// With z = x W: lse = log sum exp z, loss = lse - z[target].  The product's
// epilogue leaves a sum over the largest and the target's logit for each row and
// 128 outputs; a second launch joins a row's.
//
// Gradient: dx = g ((p - e_target) W^T), p = exp(z - lse).  Over pieces of the
// vocabulary: the product again, whose epilogue turns its logits into the
// 6-bit terms of p - e_target in the records that the next product reads, and
// that product with the transposed weight, added to dx piece by piece.
//
// Where the product has few blocks, its contraction is split: the parts of the
// logits, few then, go to the workspace, and a launch of its own adds them up and
// does what the epilogue does elsewhere.
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
inline size_t whole(size_t n) { return (n + 255) & ~(size_t)255; }

// Joins the parts of a row, a block a row: every part read once, its sum taken
// to the larger maximum, in double (a few a thread).
struct Sum {
    float top;
    double sum;
};
__device__ __forceinline__ Sum join(Sum a, Sum b) {
    const float top = fmaxf(a.top, b.top), ref = over(top);
    const float ea = a.top == -INFINITY ? 1.0f : exp_over(a.top, ref);
    const float eb = b.top == -INFINITY ? 1.0f : exp_over(b.top, ref);
    return {top, a.sum * ea + b.sum * eb};
}
__global__ __launch_bounds__(256) void k_loss(const float2* __restrict__ part, int parts,
                                              const float* __restrict__ zt,
                                              const int* __restrict__ targets, int V,
                                              float* __restrict__ loss, float* __restrict__ lse) {
    __shared__ Sum wave[4];
    const int m = blockIdx.x, lane = threadIdx.x & 63;
    const float2* p = part + (size_t)m * parts;
    Sum s = {-INFINITY, 0.0};
    for (int i = threadIdx.x; i < parts; i += 1024) {
        float2 q[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            q[j] = i + 256 * j < parts ? p[i + 256 * j] : make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; j++) s = join(s, Sum{q[j].x, q[j].y});
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) s = join(s, Sum{__shfl_xor(s.top, o), __shfl_xor(s.sum, o)});
    if (lane == 0) wave[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int w = 1; w < 4; w++) s = join(s, wave[w]);
    const double l = (double)over(s.top) + log(s.sum);
    const int t = targets[m];
    if (lse) lse[m] = (float)l;
    if (loss) loss[m] = t >= 0 && t < V ? (float)(l - (double)zt[m]) : 0.0f;
}

// Logits as the sum of their parts (four outputs from n on, n < N).
__device__ __forceinline__ f4 sum_of(const float* p, int splits, size_t stride, int n) {
    f4 v = {0, 0, 0, 0};
    for (int s = 0; s < splits; s += 4) {
        f4 t[4];
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = *(const f4*)(p + (size_t)min(s + i, splits - 1) * stride + n);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (s + i < splits) v += t[i];
    }
    return v;
}

// The epilogue's parts, a block 1024 outputs of a row.
__global__ __launch_bounds__(256) void k_stats(const float* __restrict__ z, int splits, size_t stride,
                                               int pld, int N, const int* __restrict__ targets,
                                               float2* __restrict__ part, float* __restrict__ zt) {
    __shared__ float2 wave[4];
    const int m = blockIdx.y, n = 4 * (blockIdx.x * 256 + threadIdx.x), lane = threadIdx.x & 63;
    f4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    float top = -INFINITY, sum = 0.0f;
    if (n < N) {
        v = sum_of(z + (size_t)m * pld, splits, stride, n);
        const int t = targets[m];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            v[r] = n + r < N ? v[r] : -INFINITY;
            if (n + r == t && t < N) zt[m] = v[r];
            top = fmaxf(top, v[r]);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float ref = over(top);
#pragma unroll
    for (int r = 0; r < 4; r++) sum += exp_over(v[r], ref);
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) wave[threadIdx.x >> 6] = make_float2(top, sum);
    __syncthreads();
    if (threadIdx.x >= 4) return;
    // four waves' parts, each a part of the row's
    part[((size_t)m * gridDim.x + blockIdx.x) * 4 + threadIdx.x] = wave[threadIdx.x];
}

// The epilogue's p - e_target as records of a piece from chunk c0 of the vocabulary
// on: a wave a tile of 16 rows and a chunk, a lane a block of 32 outputs.
__global__ __launch_bounds__(256) void k_probs(const float* __restrict__ z, int splits, size_t stride,
                                               int pld, int M, int N, const int* __restrict__ targets,
                                               const float* __restrict__ lse, int c0, int chunks,
                                               int mt, int units, uint8_t* __restrict__ out) {
    const int u = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= units) return;
    const int lane = threadIdx.x & 63, tile = u / chunks, c = u - tile * chunks;
    // rows past the last repeat it: nothing of theirs is stored
    const int m = min(tile * 16 + (lane & 15), M - 1), n0 = (c0 + c) * 128 + (lane >> 4) * 32;
    const int t = targets[m];
    const bool live = t >= 0 && t < N;
    const float l = live ? lse[m] : 0.0f;
    Block v;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int n = n0 + 4 * i;
        f4 q = {0, 0, 0, 0};
        if (live && n < N) q = sum_of(z + (size_t)m * pld, splits, stride, n);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float p = live && n + r < N ? exp_over(q[r], l) : 0.0f;
            if (live && n + r == t) p = expm1f(q[r] - l);
            set(v, 4 * i + r, p);
        }
    }
    using P = Rows<CGX_MX_FP32>;
    const int b = tile / mt, at = tile - b * mt;
    uint8_t* rec = out + ((size_t)b * chunks + c) * (size_t)rows_record<CGX_MX_FP32>(mt);
    put<CGX_MX_FP32>(rec + at * P::tile, rec + mt * P::tile + at * 64, lane, v);
}

constexpr int kSlab = 2048;                        // rows at a time
constexpr size_t kPiece = (size_t)128 << 20;       // bytes of a piece's probabilities

struct Plan {
    int mt, mbs, nbs;            // the product over the vocabulary
    int splits;                  // its contraction's
    size_t rows, part, zt, z;    // bytes (z: the parts of the logits)
    int parts;                   // of a row's sums
    int mt2, mbs2, kbs, piece;   // the second product; chunks of a piece
    size_t p, sum;
};
// Splits of a piece's chunks: a block a CU where few blocks would leave many
// parts to add, two otherwise (64 rows, K = 4096, 128 chunks: 19.7 us with 16
// splits, 20.5 with 32; 300 rows: 69 us with 3, 61 with 6).
int splits_of(const Plan& p, int chunks) {
    const int blocks = p.mbs2 * p.kbs;
    return std::max(1, std::min((blocks <= 64 ? 256 : 512) / blocks, chunks / 4));
}
Plan plan(const cgx_mx_weight* w, int M, int act, int grad) {
    Plan p = {};
    const int kc = up(w->K, 128), pld = (w->N + 3) & ~3;
    p.zt = grad ? 0 : whole((size_t)M * 4);
    if (!grad && gemv_pays(M, w->K, w->N)) {
        p.parts = gemv_groups(up(w->N, 16));
        p.part = whole((size_t)M * p.parts * sizeof(float2));
        return p;
    }
    p.mt = cgk_mx_tiles(M, w->N);
    p.mbs = up(M, 16 * p.mt);
    p.nbs = up(w->N, 256);
    p.parts = 2 * p.nbs;
    p.rows = whole(cgk_mx_rows_bytes(M, w->K, act, p.mt));
    // three splits or none, eight of one term: the logits' parts cost a launch and their
    // bytes (K = 4096, five terms: 30 rows and 32000 outputs, 125 blocks, 31 us in four and
    // 39 unsplit; 40 rows, 250 blocks, 41 in two, 39.  One: 30 rows and 500 outputs 15 us in
    // eight, 24; 32000 outputs 25 in four, 24)
    p.splits = gemm_splits(p.mbs * p.nbs, kc);
    if (p.splits < (act == CGX_MX_FP32 ? 3 : 8)) p.splits = 1;
    p.z = p.splits > 1 ? whole((size_t)p.splits * M * pld * 4) : 0;
    if (!grad) {
        if (p.splits > 1) p.parts = 4 * up(w->N, 1024);
        p.part = whole((size_t)M * p.parts * sizeof(float2));
        return p;
    }
    p.mt2 = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    p.mbs2 = up(M, 16 * p.mt2);
    p.kbs = up(w->K, 256);
    const size_t chunk = (size_t)p.mbs2 * rows_record<CGX_MX_FP32>(p.mt2);
    p.piece = 2 * (int)std::max<size_t>(1, std::min<size_t>(p.nbs, kPiece / (2 * chunk)));
    p.p = whole(chunk * p.piece);
    int most = 1;                // splits of any piece
    for (int c = 0; c < w->chunks128; c += p.piece) {
        const int e = std::min(c + p.piece, w->chunks128);
        most = std::max(most, splits_of(p, w->first[e] - w->first[c]));
    }
    p.sum = most > 1 ? (size_t)most * M * ((w->K + 3) & ~3) * 4 : 0;
    return p;
}
size_t bytes(const Plan& p) { return p.rows + p.part + p.zt + p.z + p.p + p.sum; }

template <int EPI>
int over_vocabulary(const Gemm& g, int mt, int act) {
    if (act == CGX_MX_FP4) gemm_launch<CGX_MX_FP4, kE2M1, EPI>(g, mt, stream());
    else if (act == CGX_MX_FP6) gemm_launch<CGX_MX_FP6, kE2M1, EPI>(g, mt, stream());
    else gemm_launch<CGX_MX_FP32, kE2M1, EPI>(g, mt, stream());
    return launch_check("mx loss");
}
template <int EPI>
int over_inputs(const Gemm& g, int mt) {
    gemm_launch<CGX_MX_FP32, kE3M2, EPI>(g, mt, stream());
    return launch_check("mx loss gradient");
}

// the product over the vocabulary from block nb0 on
Gemm logits(const cgx_mx_weight* w, const uint8_t* rows, const Plan& p, int M, const int* targets) {
    Gemm g = {};
    g.x = rows;
    g.w = w->codes;
    g.xk = g.wk = g.j1 = up(w->K, 128);
    g.mbs = p.mbs;
    g.nbs = p.nbs;
    g.splits = p.splits;
    g.M = M;
    g.N = w->N;
    g.targets = targets;
    return g;
}
// ... its parts where it is split
int split_logits(Gemm& g, int mt, int act, float* z) {
    g.y = z;
    g.ld = (g.N + 3) & ~3;
    g.stride = (size_t)g.M * g.ld;
    return over_vocabulary<kStore>(g, mt, act);
}

}  // namespace

extern "C" size_t cgk_mx_loss_need(const cgx_mx_weight* w, int M, int act, int grad) {
    size_t need = 0;
    if (M >= kSlab) {
        need = bytes(plan(w, kSlab, act, grad));
        M %= kSlab;
    }
    return M ? std::max(need, bytes(plan(w, M, act, grad))) : need;
}
// ... of any call of at most M rows
extern "C" size_t cgk_mx_loss_ws(const cgx_mx_weight* w, int M, int act, int grad) {
    const int top = std::min(M, kSlab);
    size_t need = top ? cgk_mx_loss_need(w, top, act, grad) : 0;
    for (int m = 16; m < top; m += 16) need = std::max(need, cgk_mx_loss_need(w, m, act, grad));
    return need;
}

extern "C" int cgk_mx_loss(const float* x, size_t ld, int M, const cgx_mx_weight* w, int act,
                           const int* targets, float* loss, float* lse, void* ws) {
    for (int m0 = 0; m0 < M; m0 += kSlab) {
        const int m = std::min(kSlab, M - m0);
        const Plan p = plan(w, m, act, 0);
        uint8_t* rows = (uint8_t*)ws;
        float2* part = (float2*)(rows + p.rows);
        float* zt = (float*)((uint8_t*)part + p.part);
        float* z = (float*)((uint8_t*)zt + p.zt);
        const float* xm = x + (size_t)m0 * ld;
        if (gemv_pays(m, w->K, w->N)) {
            Gemv g = {};
            g.x = xm;
            g.ldx = ld;
            g.w = w->codes;
            g.M = m;
            g.K = w->K;
            g.N = w->N;
            g.kc = up(w->K, 128);
            g.tiles = up(w->N, 16);
            g.targets = targets + m0;
            g.part = part;
            g.zt = zt;
            if (act == CGX_MX_FP4) gemv_launch<CGX_MX_FP4, kStats>(g, stream());
            else if (act == CGX_MX_FP6) gemv_launch<CGX_MX_FP6, kStats>(g, stream());
            else gemv_launch<CGX_MX_FP32, kStats>(g, stream());
            if (launch_check("mx loss of few rows")) return -1;
        } else {
            if (cgk_mx_rows(xm, ld, m, w->K, act, p.mt, rows)) return -1;
            Gemm g = logits(w, rows, p, m, targets + m0);
            if (p.splits > 1) {
                if (split_logits(g, p.mt, act, z)) return -1;
                hipLaunchKernelGGL(k_stats, dim3(p.parts / 4, m), dim3(256), 0, stream(), z, p.splits,
                                   g.stride, (int)g.ld, w->N, targets + m0, part, zt);
                if (launch_check("mx loss statistics")) return -1;
            } else {
                g.part = part;
                g.zt = zt;
                if (over_vocabulary<kStats>(g, p.mt, act)) return -1;
            }
        }
        hipLaunchKernelGGL(k_loss, dim3(m), dim3(256), 0, stream(), part, p.parts, zt,
                           targets + m0, w->N, loss ? loss + m0 : nullptr,
                           lse ? lse + m0 : nullptr);
        if (launch_check("mx loss join")) return -1;
    }
    return 0;
}

extern "C" int cgk_mx_loss_grad(const float* x, size_t ld, int M, const cgx_mx_weight* w, int act,
                                const int* targets, const float* lse, const float* dloss, float* dx,
                                size_t ldd, void* ws) {
    for (int m0 = 0; m0 < M; m0 += kSlab) {
        const int m = std::min(kSlab, M - m0);
        const Plan p = plan(w, m, act, 1);
        uint8_t *rows = (uint8_t*)ws, *probs = rows + p.rows;
        float *z = (float*)(probs + p.p), *sum = (float*)((uint8_t*)z + p.z);
        float* dm = dx + (size_t)m0 * ldd;
        const float* scale = dloss ? dloss + m0 : nullptr;
        if (cgk_mx_rows(x + (size_t)m0 * ld, ld, m, w->K, act, p.mt, rows)) return -1;
        for (int c = 0; c < w->chunks128; c += p.piece) {
            const int e = std::min(c + p.piece, w->chunks128);
            Gemm g = logits(w, rows, p, m, targets + m0);
            g.nb0 = c / 2;
            g.nbs = up(e - c, 2);
            if (p.splits > 1) {
                if (split_logits(g, p.mt, act, z)) return -1;
                const int units = p.mbs2 * p.mt2 * p.piece;
                hipLaunchKernelGGL(k_probs, dim3(up(units, 4)), dim3(256), 0, stream(), z, p.splits,
                                   g.stride, (int)g.ld, m, w->N, targets + m0, lse + m0, c, p.piece,
                                   p.mt2, units, probs);
                if (launch_check("mx loss probabilities")) return -1;
            } else {
                g.lse = lse + m0;
                g.p = probs;
                g.pk = p.piece;
                g.pmt = p.mt2;
                g.pmbs = p.mbs2;
                g.precord = rows_record<CGX_MX_FP32>(p.mt2);
                if (over_vocabulary<kProbs>(g, p.mt, act)) return -1;
            }
            Gemm t = {};
            t.x = probs;
            t.w = w->tcodes;
            t.list = w->list;
            t.list0 = c;
            t.xk = p.piece;
            t.wk = w->tchunks;
            t.j0 = w->first[c];
            t.j1 = w->first[e];
            t.mbs = p.mbs2;
            t.nbs = p.kbs;
            t.splits = splits_of(p, t.j1 - t.j0);
            t.M = m;
            t.N = w->K;
            const int pld = (w->K + 3) & ~3;
            if (t.splits > 1) {
                t.y = sum;
                t.ld = pld;
                t.stride = (size_t)m * pld;
                if (over_inputs<kStore>(t, p.mt2) ||
                    cgk_mx_join(sum, t.splits, t.stride, pld, m, w->K, dm, ldd, scale,
                                targets + m0, w->N, c > 0))
                    return -1;
            } else {
                t.y = dm;
                t.ld = ldd;
                t.row_scale = scale;
                t.targets = targets + m0;
                t.V = w->N;
                t.add = c > 0;
                if (over_inputs<kGrad>(t, p.mt2)) return -1;
            }
        }
    }
    return 0;
}
