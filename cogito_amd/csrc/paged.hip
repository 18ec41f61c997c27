// paged.hip -- the paged INT4 KV cache's tables, append and read-back.
//
//   k_paged_plan    block tables, slots and row offsets of a step from the
//                   sequences' lengths, pages given back and taken on a stack
//   k_paged_append  RoPE of a step's q and k rows (cg_apply_rope's operations,
//                   src/attention/flash_attn.c:335-360) and the INT4 append of
//                   k and v (src/quantize/int4.c:155-231) into their slots
//   k_paged_gather  values of given slots
//
// Built without implicit contraction: x0 c - x1 s rounds each product on its
// own, so that a key's codes are those the contiguous cache gets.
#include <hip/hip_runtime.h>

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

// ------------------------------------------------------------------ tables
//
// With P positions a page, held_b = ceil(old_b / P), need_b = ceil((keep_b +
// new_b) / P), give_b = max(0, held_b - need_b), take_b = max(0, need_b -
// held_b): three exclusive prefix sums over the batch (rows, take, give) give
// every output word by itself.  The stack is read as if all pages given back
// lay on it first (position count + g: the g-th of them, table_old[c][need_c +
// g - before_c]); the k-th page taken is position count + G - 1 - k.
//
// Every block scans the whole batch (4096 sequences: 16 per thread) and keeps
// the three prefix sums in LDS, then all blocks share the rows, the table
// entries and the returned pages.  No block waits for another and nothing is
// read that another block writes, which one launch needs; the scan costs each
// block less than a second launch would.
constexpr int kPlanThreads = 256;

struct PlanArgs {
    cgx_paged_step s;
    int lp, num_pages;           // page_size = 1 << lp
    int* free_pages;
    const int* free_count;
    int* free_left;
};

__device__ __forceinline__ long long wave_scan(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// the last b with pre[b] <= x: the b of item x, x < pre[B]
__device__ __forceinline__ int find(const int* pre, int B, int x) {
    int lo = 0, hi = B;          // pre[lo] <= x < pre[hi]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (pre[m] <= x) lo = m; else hi = m;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PlanArgs a) {
    extern __shared__ int s_pre[];
    __shared__ long long s_sum[3][kPlanThreads / 64];
    __shared__ int s_bad;
    const cgx_paged_step& s = a.s;
    const int B = s.seqs, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* begin = s_pre;
    int* take = begin + B + 1;
    int* give = take + B + 1;
    const int P1 = (1 << a.lp) - 1;
    if (tid == 0) s_bad = 0;
    __syncthreads();

    // lengths of sequence b; a bad one counts as empty and refuses the step
    struct Len { int old, keep, add, held, need, bad; };
    auto lens = [&](int b) {
        Len l;
        l.bad = 0;
        l.old = s.kv_old[b];
        l.keep = s.kv_keep ? s.kv_keep[b] : l.old;
        l.add = s.rows_new[b];
        if (l.keep < 0 || l.keep > l.old || l.add < 0) l.bad = 1;
        const long long most = (long long)s.table_ld << a.lp;
        if (!l.bad && (l.old > most || (long long)l.keep + l.add > most)) l.bad = 2;
        if (!l.bad && (l.add > s.rows || (s.max_rows && l.add > s.max_rows))) l.bad = 4;
        if (l.bad) l.old = l.keep = l.add = 0;
        l.held = (l.old >> a.lp) + ((l.old & P1) != 0);
        const int kv = l.keep + l.add;
        l.need = (kv >> a.lp) + ((kv & P1) != 0);
        return l;
    };

    const int per = (B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
    long long v[3] = {0, 0, 0};
    int bad = 0;
    for (int b = b0; b < b1; b++) {
        const Len l = lens(b);
        bad |= l.bad;
        v[0] += l.add;
        v[1] += max(0, l.need - l.held);
        v[2] += max(0, l.held - l.need);
    }
    long long pre[3], tot[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        const long long inc = wave_scan(v[k], lane);
        if (lane == 63) s_sum[k][wave] = inc;
        pre[k] = inc - v[k];
    }
    if (bad) atomicOr(&s_bad, bad);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; k++) {
        tot[k] = 0;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 64; w++) {
            if (w < wave) pre[k] += s_sum[k][w];
            tot[k] += s_sum[k][w];
        }
    }
    const int count = *a.free_count;
    bad = s_bad;
    if (tot[0] > s.rows) bad |= 4;
    if (count < 0 || count > a.num_pages || count + tot[2] > a.num_pages) bad |= 16;
    else if (tot[1] > count + tot[2]) bad |= 8;
    if (bad) tot[0] = tot[1] = tot[2] = 0;
    for (int b = b0; b < b1; b++) {
        begin[b] = bad ? 0 : (int)pre[0];
        take[b] = bad ? 0 : (int)pre[1];
        give[b] = bad ? 0 : (int)pre[2];
        const Len l = lens(b);
        pre[0] += l.add;
        pre[1] += max(0, l.need - l.held);
        pre[2] += max(0, l.held - l.need);
        if (blockIdx.x == 0) {
            s.row_begin[b] = begin[b];
            s.kv_len[b] = bad ? s.kv_old[b] : l.keep + l.add;
        }
    }
    const int T = (int)tot[0], K = (int)tot[1], G = (int)tot[2];
    if (tid == 0) {
        begin[B] = T;
        take[B] = K;
        give[B] = G;
        if (blockIdx.x == 0) {
            s.row_begin[B] = T;
            *a.free_left = count + G - K;
            s.status[0] = bad;
            s.status[1] = T;
            s.status[2] = K;
            s.status[3] = G;
        }
    }
    __syncthreads();

    const int* told = s.table_old ? s.table_old : s.table;
    const bool in_place = told == s.table;
    const size_t ld = (size_t)s.table_ld;
    auto returned = [&](int g) {                 // the g-th page given back
        const int c = find(give, B, g);
        return told[c * ld + lens(c).need + (g - give[c])];
    };
    auto taken = [&](int k) {
        const int at = count + G - 1 - k;
        return at >= count ? returned(at - count) : a.free_pages[at];
    };

    const int stride = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + tid;
    for (int t = first; t < s.rows; t += stride) {
        int seq = -1, pos = -1, slot = -1;
        if (t < T) {
            seq = find(begin, B, t);
            const Len l = lens(seq);
            pos = l.keep + (t - begin[seq]);
            const int j = pos >> a.lp;
            const int page = j < l.held ? told[seq * ld + j] : taken(take[seq] + j - l.held);
            if (page >= 0 && page < a.num_pages) slot = (page << a.lp) + (pos & P1);
        }
        s.row_seq[t] = seq;
        s.row_pos[t] = pos;
        s.row_slot[t] = slot;
    }
    for (int g = first; g < G; g += stride)
        if (count + g < count + G - K) a.free_pages[count + g] = returned(g);
    if (in_place) {
        for (int k = first; k < K; k += stride) {
            const int b = find(take, B, k);
            s.table[b * ld + lens(b).held + (k - take[b])] = taken(k);
        }
        return;
    }
    // another table: held entries copied, new ones taken, -1 after
    const size_t n = (size_t)B * ld;
    for (size_t e = first; e < n; e += stride) {
        const int b = (int)(e / ld), j = (int)(e - b * ld);
        const Len l = lens(b);
        // a refused step copies the table as it is
        if (bad || j < min(l.held, l.need)) s.table[e] = told[e];
        else s.table[e] = j < l.need ? taken(take[b] + j - l.held) : -1;
    }
}

// ------------------------------------------------------------------ append
//
// Block = (row, chunk of at most 8 KV heads and their share of the query
// heads).  A thread rotates four neighbouring pairs (d, d + D/2) from 16-byte
// loads; q goes straight out, k and v into LDS, where 16 lanes a group find
// its absmax and pack its bytes.  Bound by its bytes: (H + 2 Hk) D in, H D
// out a row, the packed row is a sixteenth of that.
constexpr int kAppThreads = 256, kAppHeads = 8;

struct AppendArgs {
    uint8_t* kp;
    uint8_t* vp;
    float* ks;
    float* vs;
    int lp, Hk, D, gs, num_slots;
    const int* row_slot;
    const int* row_pos;
    const float* qkv;
    int ldq, H, q_per;
    const float2* rope;
    int rope_rows;
    float* q_out;
};

// byte of dims d, d + 1 (d even) of position `at` of a page's head, V layout
__device__ __forceinline__ size_t v_byte(int D, int at, int d) {
    const int c = D / 16, n = d / c;             // block of c dims
    return ((size_t)(at >> 4) * 16 + n) * (16 * (D / 32)) + (size_t)(at & 15) * (D / 32) +
           (d - n * c) / 2;
}

__global__ __launch_bounds__(kAppThreads) void k_paged_append(AppendArgs a) {
    __shared__ __attribute__((aligned(16))) float s_kv[2 * kAppHeads * 256];
    const int row = blockIdx.x, tid = threadIdx.x;
    const int slot = a.row_slot[row];
    if (slot < 0 || slot >= a.num_slots) return;
    const int pos = a.rope ? a.row_pos[row] : 0;
    if (a.rope && (pos < 0 || pos >= a.rope_rows)) return;
    const int D = a.D, half = D / 2, per = D / 8;    // items of four pairs a head
    const int h0 = blockIdx.y * kAppHeads, nh = min(kAppHeads, a.Hk - h0);
    const int q0 = blockIdx.y * a.q_per, nq = a.q_out ? max(0, min(a.q_per, a.H - q0)) : 0;
    const float* x = a.qkv + (size_t)row * a.ldq;
    const float2* cs = a.rope ? a.rope + (size_t)pos * half : nullptr;
    for (int e = tid; e < (nq + 2 * nh) * per; e += kAppThreads) {
        const int u = e / per, i = 4 * (e - u * per);
        // u: nq query heads, nh keys, nh values
        const int kind = u < nq ? 0 : u < nq + nh ? 1 : 2;
        const int head = kind == 0 ? q0 + u : kind == 1 ? a.H + h0 + u - nq
                                            : a.H + a.Hk + h0 + u - nq - nh;
        const float4 lo = *(const float4*)(x + (size_t)head * D + i);
        const float4 hi = *(const float4*)(x + (size_t)head * D + i + half);
        const float l[4] = {lo.x, lo.y, lo.z, lo.w}, g[4] = {hi.x, hi.y, hi.z, hi.w};
        float p[4], q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            p[j] = l[j];
            q[j] = g[j];
        }
        if (cs && kind != 2) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 t = cs[i + j];
                p[j] = __fsub_rn(__fmul_rn(l[j], t.x), __fmul_rn(g[j], t.y));
                q[j] = __fadd_rn(__fmul_rn(l[j], t.y), __fmul_rn(g[j], t.x));
            }
        }
        float* o = kind == 0 ? a.q_out + ((size_t)row * a.H + head) * D : s_kv + (u - nq) * D;
        *(float4*)(o + i) = make_float4(p[0], p[1], p[2], p[3]);
        *(float4*)(o + i + half) = make_float4(q[0], q[1], q[2], q[3]);
    }
    __syncthreads();
    const int sub = tid >> 4, l = tid & 15, gs = a.gs, ng = D / gs;
    const int page = slot >> a.lp, at = slot & ((1 << a.lp) - 1);
    for (int e = sub; e < 2 * nh * ng; e += kAppThreads / 16) {
        const int u = e / ng, g = e - u * ng;        // staged head, group
        const float* v = s_kv + u * D + g * gs;
        float m = 0.0f;
        for (int j = l; j < gs; j += 16) m = fmaxf(m, fabsf(v[j]));
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        float sc = __fdiv_rn(m, 7.0f);
        if (sc < 1e-8f) sc = 1.0f;
        const bool is_k = u < nh;
        const int hk = h0 + (is_k ? u : u - nh);
        const size_t ph = (size_t)page * a.Hk + hk;              // page's head
        const size_t pr = (ph << a.lp) + at;                     // its position
        if (l == 0) (is_k ? a.ks : a.vs)[pr * ng + g] = sc;
        for (int j = l; j < gs / 2; j += 16) {
            int c0 = (int)roundf(__fdiv_rn(v[2 * j], sc)), c1 = (int)roundf(__fdiv_rn(v[2 * j + 1], sc));
            c0 = c0 > 7 ? 7 : (c0 < -8 ? -8 : c0);
            c1 = c1 > 7 ? 7 : (c1 < -8 ? -8 : c1);
            const uint8_t byte = (uint8_t)((c0 & 0xF) | ((c1 & 0xF) << 4));
            const int d = g * gs + 2 * j;
            if (is_k) a.kp[pr * half + d / 2] = byte;
            else a.vp[(ph << a.lp) * half + v_byte(D, at, d)] = byte;
        }
    }
}

__device__ __forceinline__ float2 code_pair(uint8_t b) {
    const int lo = b & 15, hi = b >> 4;
    return make_float2((float)(lo >= 8 ? lo - 16 : lo), (float)(hi >= 8 ? hi - 16 : hi));
}

// One thread a byte of K and the byte of V of the same two dims.
__global__ __launch_bounds__(256) void k_paged_gather(const uint8_t* kp, const uint8_t* vp,
                                                      const float* ks, const float* vs, int lp,
                                                      int Hk, int D, int gs, int num_slots,
                                                      const int* slots, float* k, float* v) {
    const int i = blockIdx.x, slot = slots[i], half = D / 2, ng = D / gs;
    const bool ok = slot >= 0 && slot < num_slots;
    const int page = ok ? slot >> lp : 0, at = ok ? slot & ((1 << lp) - 1) : 0;
    for (int e = blockIdx.y * 256 + threadIdx.x; e < Hk * half; e += gridDim.y * 256) {
        const int h = e / half, d = 2 * (e - h * half);
        const size_t ph = (size_t)page * Hk + h, pr = (ph << lp) + at;
        float2 x = make_float2(0.0f, 0.0f), y = x;
        if (ok) {
            x = code_pair(kp[pr * half + d / 2]);
            y = code_pair(vp[(ph << lp) * half + v_byte(D, at, d)]);
            const float s = ks[pr * ng + d / gs], t = vs[pr * ng + d / gs];
            x.x *= s;
            x.y *= s;
            y.x *= t;
            y.y *= t;
        }
        const size_t o = ((size_t)i * Hk + h) * D + d;
        *(float2*)(k + o) = x;
        *(float2*)(v + o) = y;
    }
}

int log2i(int x) {
    int l = 0;
    while ((1 << l) < x) l++;
    return l;
}

}  // namespace

extern "C" int cgk_paged_plan(const cgx_paged_step* s, int page_size, int num_pages,
                              int* free_pages, const int* free_count, int* free_left) {
    PlanArgs a;
    a.s = *s;
    a.lp = log2i(page_size);
    a.num_pages = num_pages;
    a.free_pages = free_pages;
    a.free_count = free_count;
    a.free_left = free_left;
    const bool in_place = !s->table_old || s->table_old == s->table;
    const long long words = s->rows + (in_place ? 0ll : (long long)s->seqs * s->table_ld);
    long long blocks = (words + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
    blocks = blocks < 1 ? 1 : blocks > 256 ? 256 : blocks;
    hipLaunchKernelGGL(k_paged_plan, dim3((unsigned)blocks), dim3(kPlanThreads),
                       3 * (size_t)(s->seqs + 1) * sizeof(int), stream(), a);
    return launch_check("k_paged_plan");
}

extern "C" int cgk_paged_append(const cgx_kv_paged_int4* c, int layer, const cgx_paged_step* s,
                                const float* qkv, int ldq, int H, const float* rope,
                                int rope_rows, float* q_out) {
    const size_t rows = (size_t)c->num_pages * c->page_size * c->n_heads;
    const size_t bytes = rows * (size_t)(c->head_dim / 2) * layer;
    const size_t groups = rows * (size_t)(c->head_dim / c->group_size) * layer;
    const int ny = (c->n_heads + kAppHeads - 1) / kAppHeads;
    AppendArgs a;
    a.kp = c->k_pages + bytes;
    a.vp = c->v_pages + bytes;
    a.ks = c->k_scales + groups;
    a.vs = c->v_scales + groups;
    a.lp = log2i(c->page_size);
    a.Hk = c->n_heads;
    a.D = c->head_dim;
    a.gs = c->group_size;
    a.num_slots = c->num_pages * c->page_size;
    a.row_slot = s->row_slot;
    a.row_pos = s->row_pos;
    a.qkv = qkv;
    a.ldq = ldq;
    a.H = H;
    a.q_per = (H + ny - 1) / ny;
    a.rope = (const float2*)rope;
    a.rope_rows = rope_rows;
    a.q_out = q_out;
    hipLaunchKernelGGL(k_paged_append, dim3(s->rows, ny), dim3(kAppThreads), 0, stream(), a);
    return launch_check("k_paged_append");
}

extern "C" int cgk_paged_gather(const cgx_kv_paged_int4* c, int layer, const int* slots, int n,
                                float* k, float* v) {
    const size_t rows = (size_t)c->num_pages * c->page_size * c->n_heads;
    const size_t bytes = rows * (size_t)(c->head_dim / 2) * layer;
    const size_t groups = rows * (size_t)(c->head_dim / c->group_size) * layer;
    const int ny = (c->n_heads * (c->head_dim / 2) + 255) / 256;
    hipLaunchKernelGGL(k_paged_gather, dim3(n, ny > 64 ? 64 : ny), dim3(256), 0, stream(),
                       c->k_pages + bytes, c->v_pages + bytes, c->k_scales + groups,
                       c->v_scales + groups, log2i(c->page_size), c->n_heads, c->head_dim,
                       c->group_size, c->num_pages * c->page_size, slots, k, v);
    return launch_check("k_paged_gather");
}
