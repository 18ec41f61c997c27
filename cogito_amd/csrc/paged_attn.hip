// paged_attn.hip -- attention of ragged batches over the paged INT4 KV cache.
//
//   o_t = sum_j softmax_j(s_tj) v_j,  s_tj = (q_t . k_j) / sqrt(D)
// over the keys that row t sees (chain or tree mask), with one pass over the
// keys: running maximum m, running sum l and O, both held relative to m.
//
// Lengths, row offsets and tables are device words.  Every address formed from
// them is bounded here: a length by the table row, a page by the pool.
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
};

__device__ __forceinline__ float code(unsigned n) { return (float)((int)(n << 28) >> 28); }

// One wave a (row, head), 64 keys a round: scores with a key a lane, then the
// O update with two dims a lane and byte.
__global__ __launch_bounds__(64) void k_attn_paged_row(PagedArgs a) {
    __shared__ float s_q[256];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int b = a.row_seq[t];
    if (b < 0 || b >= a.seqs) return;
    const int r0 = a.row_begin[b], n = a.row_begin[b + 1] - r0, i = t - r0;
    if (i < 0 || i >= n) return;
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
    const float* q = a.Q + ((size_t)t * a.H + h) * D;
    for (int d = lane; d < D; d += 64) s_q[d] = q[d] * a.scale;
    __syncthreads();

    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < end; k0 += 64) {
        const int j = k0 + lane;
        bool see = j < end && (j < base || (j - base < 64 && ((bits >> (j - base)) & 1)));
        int page = -1;
        if (see) page = a.table[(size_t)b * a.table_ld + (j >> a.lp)];
        see = see && page >= 0 && page < a.num_pages;
        const size_t ph = (size_t)(see ? page : 0) * a.Hk + hk;
        const int at = j & ((1 << a.lp) - 1);
        const size_t pr = (ph << a.lp) + at;
        float s = -INFINITY;
        if (see) {
            s = 0.0f;
            for (int g = 0; g < ng; g++) {
                float dot = 0.0f;
                for (int d = g * gs; d < (g + 1) * gs; d += 2) {
                    const unsigned c = a.kp[pr * half + d / 2];
                    dot += s_q[d] * code(c & 15) + s_q[d + 1] * code(c >> 4);
                }
                s += dot * a.ks[pr * ng + g];
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
        const int nk = min(64, end - k0);
        for (int kk = 0; kk < nk; kk++) {
            const float w = __shfl(p, kk);
            const size_t pk = (size_t)__shfl((long long)ph, kk);
            if (w == 0.0f) continue;
            const int ak = (k0 + kk) & ((1 << a.lp) - 1);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int d = 2 * (lane + 64 * x);
                if (d >= D) break;
                const int nb = d / (D / 16);
                const unsigned c = a.vp[(pk << a.lp) * half +
                                        ((size_t)(ak >> 4) * 16 + nb) * (16 * cb) +
                                        (size_t)(ak & 15) * cb + (d - nb * (D / 16)) / 2];
                const float sv = w * a.vs[((pk << a.lp) + ak) * ng + d / gs];
                o[2 * x] += sv * code(c & 15);
                o[2 * x + 1] += sv * code(c >> 4);
            }
        }
    }
    float* out = a.O + ((size_t)t * a.H + h) * D;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int d = 2 * (lane + 64 * x);
        if (d >= D) break;
        out[d] = l != 0.0f ? o[2 * x] / l : 0.0f;
        out[d + 1] = l != 0.0f ? o[2 * x + 1] / l : 0.0f;
    }
    if (a.lse && lane == 0) a.lse[(size_t)t * a.H + h] = l != 0.0f ? m + logf(l) : -INFINITY;
}

int log2i(int x) {
    int l = 0;
    while ((1 << l) < x) l++;
    return l;
}

}  // namespace

extern "C" size_t cgk_paged_attention_ws(const cgx_kv_paged_int4* c, const cgx_paged_step* s,
                                         int H) {
    (void)c;
    (void)s;
    (void)H;
    return 0;
}

extern "C" int cgk_paged_attention(const cgx_kv_paged_int4* c, int layer,
                                   const cgx_paged_step* s, const float* Q, int H,
                                   const unsigned long long* anc, const int* tree_len, float* O,
                                   float* lse, void* ws) {
    (void)ws;
    const size_t rows = (size_t)c->num_pages * c->page_size * c->n_heads;
    const size_t bytes = rows * (size_t)(c->head_dim / 2) * layer;
    const size_t groups = rows * (size_t)(c->head_dim / c->group_size) * layer;
    PagedArgs a;
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
    hipLaunchKernelGGL(k_attn_paged_row, dim3(s->rows, H), dim3(64), 0, stream(), a);
    return launch_check("k_attn_paged_row");
}
