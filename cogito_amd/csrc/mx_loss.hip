// mx_loss.hip -- softmax cross entropy over the vocabulary of a microscaled
// lm_head, from hidden rows, and its gradient with respect to them.  No logit
// is stored.
//
// With z = x W: lse = log sum exp z, loss = lse - z[target].  The product's
// epilogue leaves a maximum, a sum and the target's logit for each row and
// 128 outputs; a second launch joins a row's.
//
// Gradient: dx = g ((p - e_target) W^T), p = exp(z - lse).  Over pieces of the
// vocabulary: the product again, whose epilogue turns its logits into the
// 6-bit terms of p - e_target in the records that the next product reads, and
// that product with the transposed weight, added to dx piece by piece.
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
    // a part without a value above -inf holds 0, or NaN
    const float top = fmaxf(a.top, b.top), ref = top == -INFINITY ? 0.0f : top;
    const float ea = a.top == -INFINITY ? 1.0f : expf(a.top - ref);
    const float eb = b.top == -INFINITY ? 1.0f : expf(b.top - ref);
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
    const double l = (double)(s.top == -INFINITY ? 0.0f : s.top) + log(s.sum);
    const int t = targets[m];
    if (lse) lse[m] = (float)l;
    if (loss) loss[m] = t >= 0 && t < V ? (float)(l - (double)zt[m]) : 0.0f;
}

constexpr int kSlab = 2048;                        // rows at a time
constexpr size_t kPiece = (size_t)128 << 20;       // bytes of a piece's probabilities

struct Plan {
    int mt, mbs, nbs;            // the product over the vocabulary
    size_t rows, part, zt;       // bytes
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
    p.zt = grad ? 0 : whole((size_t)M * 4);
    if (!grad && gemv_pays(M, w->K)) {
        p.parts = gemv_groups(up(w->N, 16));
        p.part = whole((size_t)M * p.parts * sizeof(float2));
        return p;
    }
    p.mt = cgk_mx_tiles(M, w->N);
    p.mbs = up(M, 16 * p.mt);
    p.nbs = up(w->N, 256);
    p.parts = 2 * p.nbs;
    p.rows = whole(cgk_mx_rows_bytes(M, w->K, act, p.mt));
    if (!grad) {
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
size_t bytes(const Plan& p) { return p.rows + p.part + p.zt + p.p + p.sum; }

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
    g.splits = 1;
    g.M = M;
    g.N = w->N;
    g.targets = targets;
    return g;
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
        const float* xm = x + (size_t)m0 * ld;
        if (gemv_pays(m, w->K)) {
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
            g.part = part;
            g.zt = zt;
            if (over_vocabulary<kStats>(g, p.mt, act)) return -1;
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
        float* sum = (float*)(probs + p.p);
        float* dm = dx + (size_t)m0 * ldd;
        const float* scale = dloss ? dloss + m0 : nullptr;
        if (cgk_mx_rows(x + (size_t)m0 * ld, ld, m, w->K, act, p.mt, rows)) return -1;
        for (int c = 0; c < w->chunks128; c += p.piece) {
            const int e = std::min(c + p.piece, w->chunks128);
            Gemm g = logits(w, rows, p, m, targets + m0);
            g.nb0 = c / 2;
            g.nbs = up(e - c, 2);
            g.lse = lse + m0;
            g.p = probs;
            g.pk = p.piece;
            g.pmt = p.mt2;
            g.pmbs = p.mbs2;
            g.precord = rows_record<CGX_MX_FP32>(p.mt2);
            if (over_vocabulary<kProbs>(g, p.mt, act)) return -1;
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
