/*
 * paged.c -- the paged INT4 KV cache, the steps of a serving loop over it and
 * token log probabilities: argument checks and the cache's memory (kernels:
 * paged.hip, paged_attn.hip, logprobs.hip).  No counterpart in the reference,
 * whose cache (src/quantize/int4.c:116-289) holds one sequence.
 *
 * Every call takes device pointers, enqueues its launches on the library
 * stream and returns; none allocates.  What device arrays hold (lengths,
 * tables, slots) cannot be checked here: the kernels bound every address they
 * form from it.
 */
#include <limits.h>
#include <stdlib.h>

#include "cg_mi355x.h"
#include "cgx_internal.h"

/* MAX_ROWS: a block of 512 threads a row stays within a launch's 2^32 threads;
 * MAX_KEYS: positions of a sequence plus a tile's stay within an int */
enum { MAX_SEQS = 4096, MAX_TOP = 32, MAX_ROWS = 1 << 23, MAX_KEYS = 1 << 30, MAX_VOCAB = 1 << 30 };

static int misaligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

static int check_shape(const char* who, int layers, int pages, int page, int heads, int D, int gs) {
    if (layers <= 0 || pages <= 0 || heads <= 0 || page < 16 || page > 4096 ||
        (page & (page - 1)) || D < 32 || D > 256 || D % 32 || gs < 2 || (gs & 1) || D % gs ||
        (long long)pages * page > INT_MAX) {
        cgx_set_error("%s: %d layers of %d pages of %d positions, %d heads of %d in groups of %d "
                      "(page_size a power of two 16..4096, head_dim a multiple of 32 up to 256, "
                      "group_size even and a divisor of head_dim, fewer than 2^31 positions)",
                      who, layers, pages, page, heads, D, gs);
        return -1;
    }
    /* byte offsets in 64 bits: a position's head has D / 2 bytes of codes, up to 2 D of scales */
    if ((double)pages * page * heads * layers * (2.0 * D) > (double)(1LL << 60)) {
        cgx_set_error("%s: %d layers of %d pages of %d positions, %d heads of %d are too large",
                      who, layers, pages, page, heads, D);
        return -1;
    }
    return 0;
}

static int check_cache(const char* who, const cgx_kv_paged_int4* c, int layer) {
    if (!c || !c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales) {
        cgx_set_error("%s: no cache", who);
        return -1;
    }
    if (check_shape(who, c->num_layers, c->num_pages, c->page_size, c->n_heads, c->head_dim,
                    c->group_size))
        return -1;
    if (layer < 0 || layer >= c->num_layers) {
        cgx_set_error("%s: layer %d of %d", who, layer, c->num_layers);
        return -1;
    }
    if (misaligned(c->k_pages, 16) || misaligned(c->v_pages, 16) || misaligned(c->k_scales, 16) ||
        misaligned(c->v_scales, 16)) {
        cgx_set_error("%s: the cache's arrays have to be 16-byte aligned", who);
        return -1;
    }
    return 0;
}

int cgx_check_spans(const char* who, const cgx_span* s, int n, int place) {
    for (int i = 0; i < n; i++)
        for (int j = 0; s[i].out && j < n; j++) {
            const uintptr_t a = (uintptr_t)s[i].p, b = (uintptr_t)s[j].p;
            if (i == j || !a || !b || !s[i].n || !s[j].n || (!i && j == place && a == b)) continue;
            if (a < b + s[j].n && b < a + s[i].n) {
                cgx_set_error("%s: an output or the workspace overlaps another argument", who);
                return -1;
            }
        }
    return 0;
}

/* The sizes of a step, and a table of which page_size positions an entry. */
static int check_step(const char* who, const cgx_paged_step* s, int page) {
    if (!s || s->seqs < 1 || s->seqs > MAX_SEQS || s->rows < 0 || s->rows >= MAX_ROWS ||
        s->max_rows < 0 || s->table_ld < 1 || (long long)s->table_ld * page > MAX_KEYS) {
        cgx_set_error("%s: a step of 1..%d sequences, 0..%d rows, max_rows >= 0 and table_ld >= 1 "
                      "(at most 2^30 positions) is required", who, MAX_SEQS, MAX_ROWS - 1);
        return -1;
    }
    return 0;
}

cgx_kv_paged_int4* cgx_kv_paged_int4_new(int num_layers, int num_pages, int page_size,
                                         int n_heads, int head_dim, int group_size) {
    if (check_shape("cgx_kv_paged_int4_new", num_layers, num_pages, page_size, n_heads, head_dim,
                    group_size))
        return NULL;
    if (cgx_ensure_init()) return NULL;
    cgx_kv_paged_int4* c = (cgx_kv_paged_int4*)calloc(1, sizeof(*c));
    if (!c) {
        cgx_set_error("cgx_kv_paged_int4_new: out of memory");
        return NULL;
    }
    c->num_layers = num_layers;
    c->num_pages = num_pages;
    c->page_size = page_size;
    c->n_heads = n_heads;
    c->head_dim = head_dim;
    c->group_size = group_size;
    const size_t rows = (size_t)num_layers * num_pages * page_size * n_heads;
    const size_t bytes = rows * (size_t)(head_dim / 2);
    const size_t groups = rows * (size_t)(head_dim / group_size) * 4;
    c->k_pages = (uint8_t*)cgx_malloc(bytes);
    c->v_pages = (uint8_t*)cgx_malloc(bytes);
    c->k_scales = (float*)cgx_malloc(groups);
    c->v_scales = (float*)cgx_malloc(groups);
    if (!c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales ||
        cgx_memset(c->k_pages, 0, bytes) || cgx_memset(c->v_pages, 0, bytes) ||
        cgx_memset(c->k_scales, 0, groups) || cgx_memset(c->v_scales, 0, groups)) {
        cgx_kv_paged_int4_free(c);
        return NULL;
    }
    return c;
}

void cgx_kv_paged_int4_free(cgx_kv_paged_int4* c) {
    if (!c) return;
    cgx_free(c->k_pages);
    cgx_free(c->v_pages);
    cgx_free(c->k_scales);
    cgx_free(c->v_scales);
    free(c);
}

static int overlap(const int* a, size_t na, const int* b, size_t nb) {
    return a && b && na && nb && (uintptr_t)a < (uintptr_t)(b + nb) &&
           (uintptr_t)b < (uintptr_t)(a + na);
}

int cgx_paged_plan_dev(const cgx_paged_step* s, int page_size, int num_pages, int* free_pages,
                       const int* free_count, int* free_left) {
    const char* who = "cgx_paged_plan_dev";
    if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1)) || num_pages < 1 ||
        (long long)num_pages * page_size > INT_MAX) {
        cgx_set_error("%s: %d pages of %d positions (a power of two 16..4096, fewer than 2^31 "
                      "positions)", who, num_pages, page_size);
        return -1;
    }
    if (check_step(who, s, page_size)) return -1;
    if (!s->kv_old || !s->rows_new || !s->table || !s->row_begin || !s->kv_len || !s->status ||
        (s->rows && (!s->row_seq || !s->row_pos || !s->row_slot)) || !free_pages || !free_count ||
        !free_left) {
        cgx_set_error("%s: kv_old, rows_new, table, row_begin, the row arrays, kv_len, status and "
                      "the stack of free pages are required", who);
        return -1;
    }
    /* every block reads the inputs while others write the outputs */
    const size_t B = (size_t)s->seqs, T = (size_t)s->rows, nt = B * (size_t)s->table_ld;
    struct { const int* p; size_t n; } in[] = {{s->kv_old, B}, {s->kv_keep, B}, {s->rows_new, B},
                                               {free_count, 1}, {s->table_old, nt}},
        out[] = {{s->table, nt}, {s->row_begin, B + 1}, {s->row_seq, T}, {s->row_pos, T},
                 {s->row_slot, T}, {s->kv_len, B}, {s->status, 4}, {free_left, 1},
                 {free_pages, (size_t)num_pages}};
    const int ni = sizeof(in) / sizeof(in[0]), no = sizeof(out) / sizeof(out[0]);
    for (int o = 0; o < no; o++) {
        for (int i = 0; i < ni; i++) {
            if (out[o].p == s->table && in[i].p == s->table_old && s->table == s->table_old) continue;
            if (overlap(in[i].p, in[i].n, out[o].p, out[o].n)) {
                cgx_set_error("%s: an output overlaps an input (only table_old may be table)", who);
                return -1;
            }
        }
        for (int i = 0; i < o; i++)
            if (overlap(out[i].p, out[i].n, out[o].p, out[o].n)) {
                cgx_set_error("%s: two outputs overlap", who);
                return -1;
            }
    }
    if (cgx_ensure_init()) return -1;
    return cgk_paged_plan(s, page_size, num_pages, free_pages, free_count, free_left);
}

int cgx_kv_paged_append_dev(cgx_kv_paged_int4* c, int layer, const cgx_paged_step* s,
                            const float* qkv, int ldq, int H, const float* rope, int rope_rows,
                            float* q_out) {
    const char* who = "cgx_kv_paged_append_dev";
    if (check_cache(who, c, layer) || check_step(who, s, c->page_size)) return -1;
    if (H < 0 || H > 65536 || c->n_heads > 65536 || !qkv ||
        ldq < (H + 2LL * c->n_heads) * c->head_dim || (rope && rope_rows < 1) ||
        (s->rows && (!s->row_slot || (rope && !s->row_pos)))) {
        cgx_set_error("%s: qkv rows of at least (H + 2 * %d) * %d values, row_slot, and with a "
                      "rotary table its rows and row_pos are required", who, c->n_heads,
                      c->head_dim);
        return -1;
    }
    if (misaligned(qkv, 16) || ldq % 4 || misaligned(q_out, 16) || misaligned(rope, 16)) {
        cgx_set_error("%s: qkv, rope and q_out have to be 16-byte aligned, ldq a multiple of 4",
                      who);
        return -1;
    }
    const size_t T = (size_t)s->rows, D = (size_t)c->head_dim;
    const cgx_span mem[] = {
        {q_out, T * H * D * 4, 1},
        {qkv, T ? ((T - 1) * ldq + (H + 2 * (size_t)c->n_heads) * D) * 4 : 0, 0},
        {rope, (size_t)(rope ? rope_rows : 0) * D * 4, 0},
        {s->row_slot, T * 4, 0},
        {rope ? s->row_pos : NULL, T * 4, 0}};
    /* one row may be rotated in its place: a thread's values are its own */
    if (cgx_check_spans(who, mem, 5, T == 1 ? 1 : -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!s->rows) return 0;
    return cgk_paged_append(c, layer, s, qkv, ldq, H, rope, rope_rows, q_out);
}

int cgx_kv_paged_gather_dev(const cgx_kv_paged_int4* c, int layer, const int* slots, int n,
                            float* k, float* v) {
    const char* who = "cgx_kv_paged_gather_dev";
    if (check_cache(who, c, layer)) return -1;
    if (n < 0 || n >= MAX_ROWS || !slots || !k || !v || misaligned(k, 16) || misaligned(v, 16)) {
        cgx_set_error("%s: 0..%d slots and 16-byte aligned outputs are required", who,
                      MAX_ROWS - 1);
        return -1;
    }
    const size_t bytes = (size_t)n * c->n_heads * c->head_dim * 4;
    const cgx_span mem[] = {{k, bytes, 1}, {v, bytes, 1}, {slots, (size_t)n * 4, 0}};
    if (cgx_check_spans(who, mem, 3, -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!n) return 0;
    return cgk_paged_gather(c, layer, slots, n, k, v);
}

static int check_heads(const char* who, const cgx_kv_paged_int4* c, const cgx_paged_step* s,
                       int H) {
    if (H < 1 || H > 65535 || H % c->n_heads) {
        cgx_set_error("%s: %d query heads over %d KV heads (a multiple is required)", who, H,
                      c->n_heads);
        return -1;
    }
    if ((long long)s->rows * H > INT_MAX || !cgk_paged_attention_fits(c, s, H)) {
        cgx_set_error("%s: %d rows of %d heads are too many for one call", who, s->rows, H);
        return -1;
    }
    return 0;
}

size_t cgx_attention_paged_ws(const cgx_kv_paged_int4* c, const cgx_paged_step* s, int H) {
    const char* who = "cgx_attention_paged_ws";
    if (!c || check_shape(who, c->num_layers, c->num_pages, c->page_size, c->n_heads, c->head_dim,
                          c->group_size) ||
        check_step(who, s, c->page_size) || check_heads(who, c, s, H))
        return 0;
    return cgk_paged_attention_ws(c, s, H);
}

int cgx_attention_paged_dev(const cgx_kv_paged_int4* c, int layer, const cgx_paged_step* s,
                            const float* Q, int H, const unsigned long long* anc,
                            const int* tree_len, float* O, float* lse, void* ws,
                            size_t ws_bytes) {
    const char* who = "cgx_attention_paged_dev";
    if (check_cache(who, c, layer) || check_step(who, s, c->page_size) || check_heads(who, c, s, H))
        return -1;
    if (!Q || !O || !s->table || !s->row_begin || !s->kv_len || (s->rows && !s->row_seq)) {
        cgx_set_error("%s: Q, O and the step's table, row_begin, row_seq and kv_len are required",
                      who);
        return -1;
    }
    if (tree_len && !anc) {
        cgx_set_error("%s: tree_len without ancestor bits", who);
        return -1;
    }
    if (anc && !tree_len && s->max_rows > 64 && s->rows > 64) {
        cgx_set_error("%s: ancestor bits of sequences of more than 64 rows (max_rows %d) need "
                      "tree_len", who, s->max_rows);
        return -1;
    }
    if (misaligned(Q, 16) || misaligned(O, 16) || misaligned(anc, 8)) {
        cgx_set_error("%s: Q and O have to be 16-byte aligned", who);
        return -1;
    }
    const size_t need = cgk_paged_attention_need(c, s, H);
    if (need && (!ws || misaligned(ws, 16) || ws_bytes < need)) {
        cgx_set_error("%s: a 16-byte aligned workspace of %zu bytes is required (%zu given)", who,
                      need, ws ? ws_bytes : (size_t)0);
        return -1;
    }
    const size_t T = (size_t)s->rows, B = (size_t)s->seqs;
    const cgx_span mem[] = {{O, T * H * c->head_dim * 4, 1},
                        {lse, T * H * 4, 1},
                        {ws, need, 1},
                        {Q, T * H * c->head_dim * 4, 0},
                        {s->table, B * s->table_ld * 4, 0},
                        {s->row_begin, (B + 1) * 4, 0},
                        {s->row_seq, T * 4, 0},
                        {s->kv_len, B * 4, 0},
                        {anc, T * 8, 0},
                        {tree_len, B * 4, 0}};
    /* O in the place of Q: a block writes the rows and heads that it has read */
    if (cgx_check_spans(who, mem, 10, 3)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!s->rows) return 0;
    return cgk_paged_attention(c, layer, s, Q, H, anc, tree_len, O, lse, ws);
}

size_t cgx_token_logprobs_ws(int rows, int V, int n_top) {
    if (rows < 0 || rows >= MAX_ROWS || V < 1 || V > MAX_VOCAB || n_top < 0 || n_top > MAX_TOP) {
        cgx_set_error("cgx_token_logprobs_ws: invalid argument");
        return 0;
    }
    return cgk_logprobs_ws(rows, V, n_top);
}

int cgx_token_logprobs_dev(const float* x, size_t ld, int rows, int V, const int* tokens,
                           int n_top, float* logprob, int* rank, float* entropy, int* top_tokens,
                           float* top_logprobs, void* ws, size_t ws_bytes) {
    const char* who = "cgx_token_logprobs_dev";
    if (!x || rows < 0 || rows >= MAX_ROWS || V < 1 || V > MAX_VOCAB || ld < (size_t)V ||
        n_top < 0 || n_top > MAX_TOP) {
        cgx_set_error("%s: rows of V >= 1 logits, ld >= V apart, and 0..%d alternatives are "
                      "required (fewer than 2^23 rows, V at most 2^30)", who, MAX_TOP);
        return -1;
    }
    if (!tokens && (logprob || rank)) {
        cgx_set_error("%s: log probabilities and ranks need the tokens", who);
        return -1;
    }
    if (n_top ? !top_tokens || !top_logprobs : top_tokens || top_logprobs) {
        cgx_set_error("%s: top_tokens and top_logprobs go with n_top > 0", who);
        return -1;
    }
    const size_t need = cgk_logprobs_need(rows, V, n_top);
    if (need && (!ws || misaligned(ws, 16) || ws_bytes < need)) {
        cgx_set_error("%s: a 16-byte aligned workspace of %zu bytes is required (%zu given)", who,
                      need, ws ? ws_bytes : (size_t)0);
        return -1;
    }
    const size_t T = (size_t)rows;
    const cgx_span mem[] = {{logprob, T * 4, 1},
                        {rank, T * 4, 1},
                        {entropy, T * 4, 1},
                        {top_tokens, T * n_top * 4, 1},
                        {top_logprobs, T * n_top * 4, 1},
                        {ws, need, 1},
                        {x, T ? ((T - 1) * ld + V) * 4 : 0, 0},
                        {tokens, T * 4, 0}};
    if (cgx_check_spans(who, mem, 8, -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!rows) return 0;
    return cgk_logprobs(x, ld, rows, V, tokens, n_top, logprob, rank, entropy, top_tokens,
                        top_logprobs, ws);
}
