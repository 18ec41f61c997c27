/*
 * mx.c -- microscaled 4-bit weights, the product with them and the loss over
 * a vocabulary of them: argument checks and the weights' memory (kernels:
 * mx.hip, mx_loss.hip).  No counterpart in the reference, whose 4-bit weights
 * (src/quantize/int4.c:10-114) are integers with fp32 scales.
 *
 * Every _dev call takes device pointers, enqueues its launches on the library
 * stream and returns; none allocates.
 */
#include <stdlib.h>

#include "cg_mi355x.h"
#include "cgx_internal.h"

/* MAX_ROWS as in paged.c; MAX_WAVES: a wave a row's 512 values, four a block of
 * 256 threads: 2^24 - 1 blocks, as a launch has fewer than 2^32 threads */
enum { MAX_ROWS = 1 << 23, MAX_K = 1 << 20, MAX_N = 1 << 24, MAX_WAVES = (1 << 26) - 4,
       MAX_COLS = 1 << 30 };

static int misaligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) != 0; }
static size_t blocks_of(int cols) { return ((size_t)cols + 31) / 32; }
/* bytes of rows that start ld floats apart */
static size_t row_bytes(int rows, size_t ld, int cols) {
    return rows ? ((size_t)(rows - 1) * ld + (size_t)cols) * 4 : 0;
}

static int check_format(const char* who, const float* x, size_t ld, int rows, int cols, int format,
                        const uint8_t* codes, const uint8_t* scales) {
    if (!x || !codes || !scales || rows < 0 || cols < 1 || cols > MAX_COLS ||
        ld < (size_t)cols ||
        ld >= (size_t)1 << 32 || (long long)rows * ((cols + 511LL) / 512) > MAX_WAVES ||
        (format != CGX_MX_FP4 && format != CGX_MX_FP6)) {
        cgx_set_error("%s: rows of cols >= 1 values, ld >= cols apart, to or from CGX_MX_FP4 or "
                      "CGX_MX_FP6 codes and scales are required (rows times ceil(cols / 512) "
                      "at most 2^26 - 4, cols at most 2^30, ld below 2^32)", who);
        return -1;
    }
    if (misaligned(codes, 16) || misaligned(x, 4)) {
        cgx_set_error("%s: codes have to be 16-byte aligned, values 4-byte", who);
        return -1;
    }
    return 0;
}

int cgx_mx_quantize_dev(const float* x, size_t ld, int rows, int cols, int format, uint8_t* codes,
                        uint8_t* scales) {
    const char* who = "cgx_mx_quantize_dev";
    if (check_format(who, x, ld, rows, cols, format, codes, scales)) return -1;
    const size_t n = (size_t)rows * blocks_of(cols);
    const cgx_span mem[] = {{codes, n * (format == CGX_MX_FP4 ? 16 : 24), 1},
                            {scales, n, 1},
                            {x, row_bytes(rows, ld, cols), 0}};
    if (cgx_check_spans(who, mem, 3, -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!rows) return 0;
    return cgk_mx_quantize(x, ld, rows, cols, format, codes, scales);
}

int cgx_mx_dequantize_dev(const uint8_t* codes, const uint8_t* scales, int rows, int cols,
                          int format, float* y, size_t ld) {
    const char* who = "cgx_mx_dequantize_dev";
    if (check_format(who, y, ld, rows, cols, format, codes, scales)) return -1;
    const size_t n = (size_t)rows * blocks_of(cols);
    const cgx_span mem[] = {{y, row_bytes(rows, ld, cols), 1},
                            {codes, n * (format == CGX_MX_FP4 ? 16 : 24), 0},
                            {scales, n, 0}};
    if (cgx_check_spans(who, mem, 3, -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!rows) return 0;
    return cgk_mx_dequantize(codes, scales, rows, cols, format, y, ld);
}

/* ------------------------------------------------------------- weights */
static cgx_mx_weight* weight(const char* who, int K, int N) {
    if (K < 1 || K > MAX_K || N < 1 || N > MAX_N || (long long)K * N > 1LL << 36) {
        cgx_set_error("%s: a weight of %d inputs and %d outputs (1..2^20, 1..2^24, together at "
                      "most 2^36)", who, K, N);
        return NULL;
    }
    if (cgx_ensure_init()) return NULL;
    if (cgx_is_capturing()) {
        cgx_set_error("%s: the library stream is being captured into a graph", who);
        return NULL;
    }
    cgx_mx_weight* w = (cgx_mx_weight*)calloc(1, sizeof(*w));
    if (!w) {
        cgx_set_error("%s: out of memory", who);
        return NULL;
    }
    w->K = K;
    w->N = N;
    w->chunks128 = (N + 127) / 128;
    w->codes = (uint8_t*)cgx_malloc(cgk_mx_weight_bytes(K, N));
    if (!w->codes) {
        cgx_mx_weight_free(w);
        return NULL;
    }
    return w;
}

/* The transposed copy: the layers of every chunk found on the device, the list of
 * chunks and layers made here.  Layer 0 is always there. */
static int transpose(const char* who, cgx_mx_weight* w) {
    const int n = w->chunks128;
    uint64_t* layers = (uint64_t*)malloc((size_t)n * sizeof(uint64_t));
    uint64_t* dev = (uint64_t*)cgx_malloc((size_t)n * sizeof(uint64_t));
    int rc = -1, *list = NULL;
    if (!layers) goto memory;
    if (!dev || cgx_memset(dev, 0, (size_t)n * sizeof(uint64_t)) ||
        cgk_mx_layers(w->codes, w->K, w->N, dev) ||
        cgx_memcpy_d2h(layers, dev, (size_t)n * sizeof(uint64_t)))
        goto done;
    w->first = (int*)malloc(((size_t)n + 1) * sizeof(int));
    if (!w->first) goto memory;
    w->first[0] = 0;
    for (int c = 0; c < n; c++) w->first[c + 1] = w->first[c] + __builtin_popcountll(layers[c] | 1);
    w->tchunks = w->first[n];
    list = (int*)malloc((size_t)w->tchunks * 2 * sizeof(int));
    if (!list) goto memory;
    for (int c = 0, j = 0; c < n; c++)
        for (uint64_t left = layers[c] | 1; left; left &= left - 1, j++) {
            list[j] = c;
            list[w->tchunks + j] = __builtin_ctzll(left);
        }
    w->list = (int*)cgx_malloc((size_t)w->tchunks * 2 * sizeof(int));
    w->tcodes = (uint8_t*)cgx_malloc(cgk_mx_transposed_bytes(w->K, w->tchunks));
    if (!w->list || !w->tcodes ||
        cgx_memcpy_h2d(w->list, list, (size_t)w->tchunks * 2 * sizeof(int)) ||
        cgk_mx_transposed(w->codes, w->K, w->N, w->list, w->list + w->tchunks, w->tchunks,
                          w->tcodes) ||
        cgx_synchronize())
        goto done;
    rc = 0;
    goto done;
memory:
    cgx_set_error("%s: out of memory", who);
done:
    free(layers);
    free(list);
    cgx_free(dev);
    return rc;
}

/* A device copy of host memory that the caller frees, or p itself. */
static const void* on_device(const void* p, size_t bytes, void** made) {
    *made = NULL;
    if (cgx_is_device_ptr(p)) return p;
    *made = cgx_malloc(bytes);
    return *made && !cgx_memcpy_h2d(*made, p, bytes) ? *made : NULL;
}

cgx_mx_weight* cgx_mx_weight_new(const uint8_t* codes, const uint8_t* scales, int K, int N,
                                 int grad) {
    const char* who = "cgx_mx_weight_new";
    if (!codes || !scales) {
        cgx_set_error("%s: codes and scales are required", who);
        return NULL;
    }
    cgx_mx_weight* w = weight(who, K, N);
    if (!w) return NULL;
    const size_t n = (size_t)N * blocks_of(K);
    void *c_made = NULL, *s_made = NULL;
    const uint8_t* c = (const uint8_t*)on_device(codes, n * 16, &c_made);
    const uint8_t* s = (const uint8_t*)on_device(scales, n, &s_made);
    int rc = -1;
    if (c && misaligned(c, 16))
        cgx_set_error("%s: device codes have to be 16-byte aligned", who);
    else if (c && s)
        rc = cgk_mx_weight(c, s, K, N, w->codes) || (grad && transpose(who, w)) ||
             cgx_synchronize();
    cgx_free(c_made);
    cgx_free(s_made);
    if (rc) {
        cgx_mx_weight_free(w);
        return NULL;
    }
    return w;
}

cgx_mx_weight* cgx_mx_weight_from_tensor(cg_tensor* t, int grad) {
    const char* who = "cgx_mx_weight_from_tensor";
    if (!t || !t->data || t->ndim != 2) {
        cgx_set_error("%s: a matrix [K, N] is required", who);
        return NULL;
    }
    cgx_mx_weight* w = weight(who, t->shape[0], t->shape[1]);
    if (!w) return NULL;
    void* made = NULL;
    const float* x = (const float*)on_device(t->data, (size_t)w->K * w->N * 4, &made);
    const int rc = !x || cgk_mx_weight_of(x, w->K, w->N, w->codes) ||
                   (grad && transpose(who, w)) || cgx_synchronize();
    cgx_free(made);
    if (rc) {
        cgx_mx_weight_free(w);
        return NULL;
    }
    return w;
}

void cgx_mx_weight_free(cgx_mx_weight* w) {
    if (!w) return;
    cgx_free(w->codes);
    cgx_free(w->tcodes);
    cgx_free(w->list);
    free(w->first);
    free(w);
}

/* ------------------------------------------------- product and loss */
static int check_rows(const char* who, const cgx_mx_weight* w, int rows, int act) {
    if (!w || rows < 0 || rows >= MAX_ROWS ||
        (act != CGX_MX_FP32 && act != CGX_MX_FP4 && act != CGX_MX_FP6)) {
        cgx_set_error("%s: a weight, 0..%d rows and CGX_MX_FP32, CGX_MX_FP4 or CGX_MX_FP6 are "
                      "required", who, MAX_ROWS - 1);
        return -1;
    }
    return 0;
}
static int check_ws(const char* who, const void* ws, size_t have, size_t need) {
    if (need && (!ws || misaligned(ws, 16) || have < need)) {
        cgx_set_error("%s: a 16-byte aligned workspace of %zu bytes is required (%zu given)", who,
                      need, ws ? have : (size_t)0);
        return -1;
    }
    return 0;
}
static int check_ld(const char* who, const float* x, size_t ld, int cols) {
    if (!x || misaligned(x, 4) || ld < (size_t)cols || ld >= (size_t)1 << 32) {
        cgx_set_error("%s: rows of %d floats, at least as far apart (fewer than 2^32), are required", who, cols);
        return -1;
    }
    return 0;
}

/* a loss's arrays of a value a row; optional ones are NULL */
static int check_arrays(const char* who, const int* targets, const float* a, const float* b) {
    if (misaligned(targets, 4) || misaligned(a, 4) || misaligned(b, 4)) {
        cgx_set_error("%s: targets and the values of a row have to be 4-byte aligned", who);
        return -1;
    }
    return 0;
}

size_t cgx_matmul_mx_ws(const cgx_mx_weight* w, int M, int act) {
    if (check_rows("cgx_matmul_mx_ws", w, M, act)) return 0;
    return cgk_mx_matmul_ws(w, M, act);
}

int cgx_matmul_mx_dev(const float* x, size_t ldx, int M, const cgx_mx_weight* w, int act, float* y,
                      size_t ldy, void* ws, size_t ws_bytes) {
    const char* who = "cgx_matmul_mx_dev";
    if (check_rows(who, w, M, act) || check_ld(who, x, ldx, w->K) || check_ld(who, y, ldy, w->N))
        return -1;
    const size_t need = cgk_mx_matmul_need(w, M, act);
    if (check_ws(who, ws, ws_bytes, need)) return -1;
    const cgx_span mem[] = {{y, row_bytes(M, ldy, w->N), 1},
                            {ws, need, 1},
                            {x, row_bytes(M, ldx, w->K), 0}};
    if (cgx_check_spans(who, mem, 3, -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!M) return 0;
    return cgk_mx_matmul(x, ldx, M, w, act, y, ldy, ws);
}

static int check_grad(const char* who, const cgx_mx_weight* w) {
    if (!w->tcodes) {
        cgx_set_error("%s: the weight was made without a gradient", who);
        return -1;
    }
    return 0;
}

size_t cgx_token_loss_mx_ws(const cgx_mx_weight* w, int rows, int act, int grad) {
    const char* who = "cgx_token_loss_mx_ws";
    if (check_rows(who, w, rows, act) || (grad && check_grad(who, w))) return 0;
    size_t n = cgk_mx_loss_ws(w, rows, act, 0);
    if (grad) {
        const size_t g = cgk_mx_loss_ws(w, rows, act, 1);
        n = g > n ? g : n;
    }
    return n;
}

int cgx_token_loss_mx_dev(const float* h, size_t ldh, int rows, const cgx_mx_weight* w, int act,
                          const int* targets, float* loss, float* lse, void* ws, size_t ws_bytes) {
    const char* who = "cgx_token_loss_mx_dev";
    if (check_rows(who, w, rows, act) || check_ld(who, h, ldh, w->K)) return -1;
    if (!targets || (!loss && !lse)) {
        cgx_set_error("%s: targets and loss or lse are required", who);
        return -1;
    }
    if (check_arrays(who, targets, loss, lse)) return -1;
    const size_t need = cgk_mx_loss_need(w, rows, act, 0), T = (size_t)rows;
    if (check_ws(who, ws, ws_bytes, need)) return -1;
    const cgx_span mem[] = {{loss, T * 4, 1},
                            {lse, T * 4, 1},
                            {ws, need, 1},
                            {h, row_bytes(rows, ldh, w->K), 0},
                            {targets, T * 4, 0}};
    if (cgx_check_spans(who, mem, 5, -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!rows) return 0;
    return cgk_mx_loss(h, ldh, rows, w, act, targets, loss, lse, ws);
}

int cgx_token_loss_mx_grad_dev(const float* h, size_t ldh, int rows, const cgx_mx_weight* w,
                               int act, const int* targets, const float* lse, const float* dloss,
                               float* dh, size_t ldd, void* ws, size_t ws_bytes) {
    const char* who = "cgx_token_loss_mx_grad_dev";
    if (check_rows(who, w, rows, act) || check_grad(who, w) || check_ld(who, h, ldh, w->K) ||
        check_ld(who, dh, ldd, w->K))
        return -1;
    if (!targets || !lse) {
        cgx_set_error("%s: targets and lse are required", who);
        return -1;
    }
    if (check_arrays(who, targets, lse, dloss)) return -1;
    const size_t need = cgk_mx_loss_need(w, rows, act, 1), T = (size_t)rows;
    if (check_ws(who, ws, ws_bytes, need)) return -1;
    const cgx_span mem[] = {{dh, row_bytes(rows, ldd, w->K), 1},
                            {ws, need, 1},
                            {h, row_bytes(rows, ldh, w->K), 0},
                            {targets, T * 4, 0},
                            {lse, T * 4, 0},
                            {dloss, T * 4, 0}};
    if (cgx_check_spans(who, mem, 6, -1)) return -1;
    if (cgx_ensure_init()) return -1;
    if (!rows) return 0;
    return cgk_mx_loss_grad(h, ldh, rows, w, act, targets, lse, dloss, dh, ldd, ws);
}
