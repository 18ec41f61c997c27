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
// the three prefix sums in LDS; then a wave takes a part of a sequence: its
// rows, its table entries, its pages given back.  No block waits for another
// and nothing is read that another block writes, which one launch needs; the
// scan costs each block less than a second launch would.  Bound by latency:
// lengths, table and stack are three dependent loads.  64 sequences of up to 5
// rows take 4.4 us, 256 prompts of up to 381 rows 4.2, an empty launch 2.5.
constexpr int kPlanThreads = 256, kPlanWaves = kPlanThreads / 64;

struct PlanArgs {
    cgx_paged_step s;
    int lp, num_pages;           // page_size = 1 << lp
    int* free_pages;
    const int* free_count;
    int* free_left;
    int parts;                   // waves a sequence
};

// inclusive scan over the wave; a sum past 32 bits stays at the largest
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
#define CGX_ROW(CTRL, RMASK)                                                                     \
    v = __builtin_elementwise_add_sat(                                                           \
        v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, RMASK, 0xF, true))
    CGX_ROW(0x111, 0xF);
    CGX_ROW(0x112, 0xF);
    CGX_ROW(0x114, 0xF);
    CGX_ROW(0x118, 0xF);
    CGX_ROW(0x142, 0xA);
    CGX_ROW(0x143, 0xC);
#undef CGX_ROW
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
    __shared__ uint32_t s_sum[3][kPlanWaves];
    __shared__ int s_bad[kPlanWaves];
    const cgx_paged_step& s = a.s;
    const int B = s.seqs, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int* begin = s_pre;
    int* take = begin + B + 1;
    int* give = take + B + 1;
    const int P1 = (1 << a.lp) - 1;
    const long long most = (long long)s.table_ld << a.lp;

    // lengths of sequence b; a bad one counts as empty and refuses the step
    struct Len { int old, keep, add, held, need, bad; };
    auto lens = [&](int b) {
        Len l;
        l.bad = 0;
        l.old = s.kv_old[b];
        l.keep = s.kv_keep ? s.kv_keep[b] : l.old;
        l.add = s.rows_new[b];
        if (l.keep < 0 || l.keep > l.old || l.add < 0) l.bad = 1;
        else if (l.old > most || (long long)l.keep + l.add > most) l.bad = 2;
        else if (l.add > s.rows || (s.max_rows && l.add > s.max_rows)) l.bad = 4;
        if (l.bad) l.old = l.keep = l.add = 0;
        l.held = (l.old >> a.lp) + ((l.old & P1) != 0);
        const int kv = l.keep + l.add;
        l.need = (kv >> a.lp) + ((kv & P1) != 0);
        return l;
    };

    const int count = *a.free_count;
    const int per = (B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
    uint32_t v[3] = {0, 0, 0};
    int bad = 0;
    Len l0 = {};
    for (int b = b0; b < b1; b++) {
        const Len l = lens(b);
        if (b == b0) l0 = l;
        bad |= l.bad;
        v[0] = __builtin_elementwise_add_sat(v[0], (uint32_t)l.add);
        v[1] = __builtin_elementwise_add_sat(v[1], (uint32_t)max(0, l.need - l.held));
        v[2] = __builtin_elementwise_add_sat(v[2], (uint32_t)max(0, l.held - l.need));
    }
    uint32_t pre[3], tot[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        const uint32_t inc = wave_scan(v[k]);
        if (lane == 63) s_sum[k][wave] = inc;
        pre[k] = inc - v[k];
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {            // bits 1, 2, 4 of any lane
        const unsigned long long any = __ballot(bad & o);
        bad = any ? bad | o : bad & ~o;
    }
    if (lane == 0) s_bad[wave] = bad;
    __syncthreads();
    bad = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) bad |= s_bad[w];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        tot[k] = 0;
#pragma unroll
        for (int w = 0; w < kPlanWaves; w++) {
            if (w < wave) pre[k] = __builtin_elementwise_add_sat(pre[k], s_sum[k][w]);
            tot[k] = __builtin_elementwise_add_sat(tot[k], s_sum[k][w]);
        }
    }
    if (tot[0] > (uint32_t)s.rows) bad |= 4;
    if (count < 0 || count > a.num_pages || (unsigned long long)count + tot[2] > (uint32_t)a.num_pages) bad |= 16;
    else if (tot[1] > (unsigned long long)count + tot[2]) bad |= 8;
    if (bad) tot[0] = tot[1] = tot[2] = 0;
    for (int b = b0; b < b1; b++) {
        const Len l = b == b0 ? l0 : lens(b);
        begin[b] = bad ? 0 : (int)pre[0];
        take[b] = bad ? 0 : (int)pre[1];
        give[b] = bad ? 0 : (int)pre[2];
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

    const int first = blockIdx.x * kPlanThreads + tid, stride = gridDim.x * kPlanThreads;
    for (int t = T + first; t < s.rows; t += stride) s.row_seq[t] = s.row_pos[t] = s.row_slot[t] = -1;
    const int waves = gridDim.x * kPlanWaves;
    for (int w = blockIdx.x * kPlanWaves + wave; w < B * a.parts; w += waves) {
        const int b = w / a.parts, from = (w - b * a.parts) * 64 + lane, by = a.parts * 64;
        const Len l = lens(b);
        const int t0 = begin[b], k0 = take[b];
        const size_t row = b * ld;
        if (!bad)
            for (int i = from; i < l.add; i += by) {
                const int pos = l.keep + i, j = pos >> a.lp;
                const int page = j < l.held ? told[row + j] : taken(k0 + j - l.held);
                s.row_seq[t0 + i] = b;
                s.row_pos[t0 + i] = pos;
                s.row_slot[t0 + i] = page >= 0 && page < a.num_pages ? (page << a.lp) + (pos & P1) : -1;
            }
        if (in_place) {
            if (!bad)
                for (int j = l.held + from; j < l.need; j += by) s.table[row + j] = taken(k0 + j - l.held);
        } else {
            // another table: held entries copied, new ones taken, -1 after; a
            // refused step copies the table as it is
            const int same = bad ? s.table_ld : min(l.held, l.need);
            for (int j = from; j < s.table_ld; j += by)
                s.table[row + j] = j < same ? told[row + j] : j < l.need ? taken(k0 + j - l.held) : -1;
        }
        if (!bad)
            for (int j = l.need + from; j < l.held; j += by) {
                const int g = give[b] + (j - l.need);
                if (g < G - K) a.free_pages[count + g] = told[row + j];
            }
    }
}

// ------------------------------------------------------------------ append
//
// Block = 2048 values of one row: 256 items of four neighbouring pairs
// (d, d + D/2), two 16-byte loads each, a thread an item.  Blocks of query
// heads store them rotated; blocks of KV heads rotate K into LDS beside V,
// from where a thread packs eight neighbouring values of a head.  Row,
// slot and values are asked for together, then the rotary words.  Bound by
// latency for few rows (two dependent loads), then by bytes: (H + 2 Hk) D in,
// H D out a row, the packed row is a sixteenth of that.  5 rows of 32/8 heads
// of 128 take 4.0 us, 64 sequences of up to 5 rows 5.0, 2039 rows of 12/12
// heads of 64 11.9 (2.2 TB/s: a block has one round of loads, which nothing
// of its own overlaps).
constexpr int kAppThreads = 256;

struct AppendArgs {
    uint8_t* kp;
    uint8_t* vp;
    float* ks;
    float* vs;
    int lp, Hk, D, gs, num_slots;
    const int* row_slot;
    const int* row_pos;
    const float* qkv;
    int ldq, H;
    const float2* rope;
    int rope_rows;
    float* q_out;
    int rows;
    int q_heads, q_parts, q_rows;    // query heads of a block, blocks a row, rows a block
    int heads, kv_rows;              // KV heads of a block, rows a block
    // division of numbers below 256 by those of 256 or less: x m >> 16, m =
    // ceil(2^16 / d) (the excess of m adds less than 1/d); a division by a
    // variable is 25 instructions, and a thread has five of them
    uint32_t by_per, by_qheads, by_heads, by_gs, by_c;
};
__device__ __forceinline__ int quot(int x, uint32_t m) { return (int)((uint32_t)x * m >> 16); }

// byte of dims d, d + 1 (d even) of position `at` of a page's head, V layout
__device__ __forceinline__ size_t v_byte(int D, int at, int d, uint32_t by_c) {
    const int c = D / 16, n = quot(d, by_c);     // block of c dims
    return ((size_t)(at >> 4) * 16 + n) * (16 * (D / 32)) + (size_t)(at & 15) * (D / 32) +
           (d - n * c) / 2;
}

__device__ __forceinline__ uint32_t code_of(float v, float sc) {
    int c = (int)roundf(__fdiv_rn(v, sc));
    c = c > 7 ? 7 : (c < -8 ? -8 : c);
    return (uint32_t)c & 15u;
}

__global__ __launch_bounds__(kAppThreads) void k_paged_append(AppendArgs a) {
    __shared__ __attribute__((aligned(16))) float s_kv[8 * kAppThreads];
    __shared__ float s_max[kAppThreads];
    const int tid = threadIdx.x, D = a.D, half = D / 2, per = D / 8;   // items a head
    const bool is_q = (int)blockIdx.y < a.q_parts;
    // the item's row, its head among the row's H + 2 Hk and its first dim; K
    // and V of a block's heads lie side by side, w the head's place there
    const int w = quot(tid, a.by_per), i = 4 * (tid - w * per);
    int row, head, nh = 0;
    bool ok;
    if (is_q) {
        const int of = quot(w, a.by_qheads);
        row = blockIdx.x * a.q_rows + of;
        head = blockIdx.y * a.q_heads + w - of * a.q_heads;
        ok = of < a.q_rows && head < a.H;
    } else {
        const int h0 = (blockIdx.y - a.q_parts) * a.heads;
        nh = min(a.heads, a.Hk - h0);
        const int of = a.kv_rows == 1 ? w >= 2 * nh : quot(w, a.by_heads), u = w - of * 2 * nh;
        row = blockIdx.x * a.kv_rows + of;
        head = u < nh ? a.H + h0 + u : a.H + a.Hk + h0 + u - nh;
        ok = of < a.kv_rows;
    }
    ok = ok && row < a.rows;
    int slot = -1, pos = 0;
    float4 lo = make_float4(0.0f, 0.0f, 0.0f, 0.0f), hi = lo;
    if (ok) {
        const float* x = a.qkv + (size_t)row * a.ldq + (size_t)head * D + i;
        lo = *(const float4*)x;
        hi = *(const float4*)(x + half);
        slot = a.row_slot[row];
        if (a.rope) pos = a.row_pos[row];
    }
    ok = slot >= 0 && slot < a.num_slots && (!a.rope || (pos >= 0 && pos < a.rope_rows));
    if (ok) {
        const float l[4] = {lo.x, lo.y, lo.z, lo.w}, g[4] = {hi.x, hi.y, hi.z, hi.w};
        float p[4], q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            p[j] = l[j];
            q[j] = g[j];
        }
        if (a.rope && head < a.H + a.Hk) {
            const float4* cs = (const float4*)(a.rope + (size_t)pos * half + i);
            const float4 t0 = cs[0], t1 = cs[1];
            const float c[4] = {t0.x, t0.z, t1.x, t1.z}, s[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                p[j] = __fsub_rn(__fmul_rn(l[j], c[j]), __fmul_rn(g[j], s[j]));
                q[j] = __fadd_rn(__fmul_rn(l[j], s[j]), __fmul_rn(g[j], c[j]));
            }
        }
        float* o = is_q ? a.q_out + ((size_t)row * a.H + head) * D : s_kv + w * D;
        *(float4*)(o + i) = make_float4(p[0], p[1], p[2], p[3]);
        *(float4*)(o + i + half) = make_float4(q[0], q[1], q[2], q[3]);
    }
    if (is_q) return;
    __syncthreads();
    const int gs = a.gs, ng = D / gs, c = D / 16;
    // this thread's staged head is one of K, or of V
    const bool is_k = head < a.H + a.Hk;
    const int hk = head - a.H - (is_k ? 0 : a.Hk);
    const int page = slot >> a.lp, at = slot & ((1 << a.lp) - 1);
    if (gs % 8 == 0) {
        // a thread eight values of a head; its group's absmax from those of
        // the threads that share it
        const int d = 2 * i;
        float v[8], m = 0.0f;
        if (ok) {
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                const float4 f = *(const float4*)(s_kv + w * D + d + k);
                v[k] = f.x; v[k + 1] = f.y; v[k + 2] = f.z; v[k + 3] = f.w;
            }
#pragma unroll
            for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(v[k]));
            s_max[tid] = m;
        }
        __syncthreads();
        if (!ok) return;
        const int g = quot(d, a.by_gs), g0 = w * per + g * (gs / 8);
        for (int k = 0; k < gs / 8; k++) m = fmaxf(m, s_max[g0 + k]);
        float sc = __fdiv_rn(m, 7.0f);
        if (sc < 1e-8f) sc = 1.0f;
        const size_t ph = (size_t)page * a.Hk + hk;              // page's head
        const size_t pr = (ph << a.lp) + at;                     // its position
        if (d == g * gs) (is_k ? a.ks : a.vs)[pr * ng + g] = sc;
        uint32_t b = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) b |= code_of(v[k], sc) << (4 * k);
        uint8_t* vp = a.vp + (ph << a.lp) * half;
        if (is_k) {
            *(uint32_t*)(a.kp + pr * half + d / 2) = b;
        } else if (c % 8 == 0) {
            *(uint32_t*)(vp + v_byte(D, at, d, a.by_c)) = b;
        } else if (c % 4 == 0) {
            *(uint16_t*)(vp + v_byte(D, at, d, a.by_c)) = (uint16_t)b;
            *(uint16_t*)(vp + v_byte(D, at, d + 4, a.by_c)) = (uint16_t)(b >> 16);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) vp[v_byte(D, at, d + 2 * k, a.by_c)] = (uint8_t)(b >> (8 * k));
        }
        return;
    }
    // groups of any other even size: a thread walks the group of each
    // of its pairs
    if (!ok) return;
    const float* v = s_kv + w * D;
    const size_t ph = (size_t)page * a.Hk + hk, pr = (ph << a.lp) + at;
    for (int j = 2 * i; j < 2 * i + 8; j += 2) {
        const int g = j / gs;
        float m = 0.0f;
        for (int k = g * gs; k < (g + 1) * gs; k++) m = fmaxf(m, fabsf(v[k]));
        float sc = __fdiv_rn(m, 7.0f);
        if (sc < 1e-8f) sc = 1.0f;
        if (j == g * gs) (is_k ? a.ks : a.vs)[pr * ng + g] = sc;
        const uint8_t b = (uint8_t)(code_of(v[j], sc) | code_of(v[j + 1], sc) << 4);
        if (is_k) a.kp[pr * half + j / 2] = b;
        else a.vp[(ph << a.lp) * half + v_byte(D, at, j, a.by_c)] = b;
    }
}

__device__ __forceinline__ float2 code_pair(uint32_t b) {
    return make_float2((float)((int)(b << 28) >> 28), (float)((int)(b << 24) >> 28));
}

// Four dims of K and of V a thread: bound by latency (a slot, then its bytes
// and scales), 3.0 us for 5 rows, 6.0 for 2039 rows of 12 heads of 64.
__global__ __launch_bounds__(256) void k_paged_gather(const uint8_t* kp, const uint8_t* vp,
                                                      const float* ks, const float* vs, int lp,
                                                      int Hk, int D, int gs, int num_slots,
                                                      const int* slots, float* k, float* v,
                                                      uint32_t by_c, uint32_t by_gs) {
    const int i = blockIdx.x, slot = slots[i], half = D / 2, ng = D / gs, quads = D / 4;
    const bool ok = slot >= 0 && slot < num_slots;
    const int page = ok ? slot >> lp : 0, at = ok ? slot & ((1 << lp) - 1) : 0;
    for (int e = blockIdx.y * 256 + threadIdx.x; e < Hk * quads; e += gridDim.y * 256) {
        const int h = e / quads, d = 4 * (e - h * quads);
        const size_t ph = (size_t)page * Hk + h, pr = (ph << lp) + at;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
        if (ok) {
            const uint32_t kb = *(const uint16_t*)(kp + pr * half + d / 2);
            const uint8_t* vb = vp + (ph << lp) * half;
            const float2 k0 = code_pair(kb), k1 = code_pair(kb >> 8);
            const float2 v0 = code_pair(vb[v_byte(D, at, d, by_c)]), v1 = code_pair(vb[v_byte(D, at, d + 2, by_c)]);
            const int g0 = quot(d, by_gs), g1 = quot(d + 2, by_gs);    // groups hold an even number of dims
            const float s0 = ks[pr * ng + g0], s1 = ks[pr * ng + g1];
            const float t0 = vs[pr * ng + g0], t1 = vs[pr * ng + g1];
            x = make_float4(k0.x * s0, k0.y * s0, k1.x * s1, k1.y * s1);
            y = make_float4(v0.x * t0, v0.y * t0, v1.x * t1, v1.y * t1);
        }
        const size_t o = ((size_t)i * Hk + h) * D + d;
        *(float4*)(k + o) = x;
        *(float4*)(v + o) = y;
    }
}

uint32_t magic(int d) { return (65536u + d - 1) / d; }

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
    // waves enough for the sequences, or, of few, for their rows and entries
    a.parts = s->seqs >= 1024 ? 1 : 1024 / s->seqs;
    const long long each = s->rows > s->table_ld ? s->rows : s->table_ld;
    if (a.parts > (each + 63) / 64) a.parts = (int)((each + 63) / 64);
    int blocks = (s->seqs * a.parts + kPlanWaves - 1) / kPlanWaves;
    if (blocks > 256) blocks = 256;
    hipLaunchKernelGGL(k_paged_plan, dim3(blocks), dim3(kPlanThreads),
                       3 * (size_t)(s->seqs + 1) * sizeof(int), stream(), a);
    return launch_check("k_paged_plan");
}

extern "C" int cgk_paged_append(const cgx_kv_paged_int4* c, int layer, const cgx_paged_step* s,
                                const float* qkv, int ldq, int H, const float* rope,
                                int rope_rows, float* q_out) {
    const size_t rows = (size_t)c->num_pages * c->page_size * c->n_heads;
    const size_t bytes = rows * (size_t)(c->head_dim / 2) * layer;
    const size_t groups = rows * (size_t)(c->head_dim / c->group_size) * layer;
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
    a.rope = (const float2*)rope;
    a.rope_rows = rope_rows;
    a.q_out = q_out;
    const int per = c->head_dim / 8;             // items a head
    const int fit = kAppThreads / per;           // heads of a block
    a.rows = s->rows;
    a.q_heads = H < fit ? (H ? H : 1) : fit;
    a.q_parts = q_out ? (H + a.q_heads - 1) / a.q_heads : 0;
    a.q_rows = H > fit ? 1 : fit / a.q_heads;
    a.heads = c->n_heads < fit / 2 ? c->n_heads : fit / 2;
    const int kv_parts = (c->n_heads + a.heads - 1) / a.heads;
    a.kv_rows = kv_parts > 1 ? 1 : fit / (2 * a.heads);
    a.by_per = magic(per);
    a.by_qheads = magic(a.q_heads);
    a.by_heads = magic(2 * a.heads);
    a.by_gs = magic(c->group_size);
    a.by_c = magic(c->head_dim / 16);
    const int step = a.q_parts && a.q_rows < a.kv_rows ? a.q_rows : a.kv_rows;
    hipLaunchKernelGGL(k_paged_append, dim3((s->rows + step - 1) / step, a.q_parts + kv_parts),
                       dim3(kAppThreads), 0, stream(), a);
    return launch_check("k_paged_append");
}

extern "C" int cgk_paged_gather(const cgx_kv_paged_int4* c, int layer, const int* slots, int n,
                                float* k, float* v) {
    const size_t rows = (size_t)c->num_pages * c->page_size * c->n_heads;
    const size_t bytes = rows * (size_t)(c->head_dim / 2) * layer;
    const size_t groups = rows * (size_t)(c->head_dim / c->group_size) * layer;
    const int ny = (c->n_heads * (c->head_dim / 4) + 255) / 256;
    hipLaunchKernelGGL(k_paged_gather, dim3(n, ny > 64 ? 64 : ny), dim3(256), 0, stream(),
                       c->k_pages + bytes, c->v_pages + bytes, c->k_scales + groups,
                       c->v_scales + groups, log2i(c->page_size), c->n_heads, c->head_dim,
                       c->group_size, c->num_pages * c->page_size, slots, k, v,
                       magic(c->head_dim / 16), magic(c->group_size));
    return launch_check("k_paged_gather");
}
