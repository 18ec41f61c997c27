/*
 * mx_host.c -- drives the host side of the microscaled weights (host/mx.c: their
 * memory, and the list of chunks and layers of the transposed copy) under
 * AddressSanitizer and UndefinedBehaviorSanitizer, with the runtime and the launchers
 * replaced by host code: "device" memory is the heap, the layers that the device
 * would find are set by the test, and every allocation in turn fails once.  Exit
 * status 0 and no sanitizer report is a pass.  Test infrastructure only.
 */
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "cg_mi355x.h"
#include "cgx_internal.h"

/* ------------------------------------------------ the runtime's place */
static char g_err[1024];
static long g_live, g_calls, g_fail_at = -1;   /* device blocks held; calls that can fail */
static int g_fails, g_device;

static int fails_now(void) {
    if (g_calls++ != g_fail_at) return 0;
    cgx_set_error("made to fail");
    return 1;
}
void cgx_set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
}
int cgx_ensure_init(void) { return 0; }
int cgx_is_capturing(void) { return 0; }
int cgx_synchronize(void) { return 0; }
int cgx_is_device_ptr(const void* p) { return p && g_device; }
void* cgx_malloc(size_t b) {
    if (fails_now()) return NULL;
    g_live++;
    return aligned_alloc(16, (b + 15) / 16 * 16);
}
int cgx_free(void* p) {
    g_live -= p != NULL;
    free(p);
    return 0;
}
int cgx_memcpy_h2d(void* d, const void* s, size_t b) {
    if (fails_now()) return -1;
    memcpy(d, s, b);
    return 0;
}
int cgx_memcpy_d2h(void* d, const void* s, size_t b) { return cgx_memcpy_h2d(d, s, b); }
int cgx_memset(void* d, int v, size_t b) {
    if (fails_now()) return -1;
    memset(d, v, b);
    return 0;
}
int cgx_check_spans(const char* who, const cgx_span* s, int n, int place) { return 0; }

/* ---------------------------------------------- the launchers' places */
enum { RECORD = 16 * (1024 + 64), TRECORD = 16 * (1536 + 64) };
static const uint64_t* g_layers;   /* of the chunks, NULL: none beyond the first */
static int up(int a, int b) { return (a + b - 1) / b; }

size_t cgk_mx_weight_bytes(int K, int N) { return (size_t)up(N, 256) * up(K, 128) * RECORD; }
int cgk_mx_weight(const uint8_t* codes, const uint8_t* scales, int K, int N, uint8_t* w) {
    if (fails_now()) return -1;
    const size_t n = (size_t)N * up(K, 32);
    unsigned sum = 0;   /* reads what the kernel reads, writes what it writes */
    for (size_t i = 0; i < n * 16; i++) sum += codes[i];
    for (size_t i = 0; i < n; i++) sum += scales[i];
    memset(w, (int)(sum & 255), cgk_mx_weight_bytes(K, N));
    return 0;
}
int cgk_mx_weight_of(const float* x, int K, int N, uint8_t* w) {
    if (fails_now()) return -1;
    float sum = 0;
    for (size_t i = 0; i < (size_t)K * N; i++) sum += x[i];
    memset(w, sum > 0, cgk_mx_weight_bytes(K, N));
    return 0;
}
int cgk_mx_layers(const uint8_t* w, int K, int N, uint64_t* layers) {
    if (fails_now()) return -1;
    for (int c = 0; c < up(N, 128); c++) {
        g_fails += layers[c] != 0;   /* cleared before */
        if (g_layers) layers[c] |= g_layers[c];
    }
    return 0;
}
size_t cgk_mx_transposed_bytes(int K, int chunks) { return (size_t)up(K, 256) * chunks * TRECORD; }
int cgk_mx_transposed(const uint8_t* w, int K, int N, const int* list, const int* layers,
                      int chunks, uint8_t* out) {
    if (fails_now()) return -1;
    /* every layer that holds a value, and the first, once each and in order */
    int j = 0;
    for (int c = 0; c < up(N, 128); c++)
        for (int p = 0; p < 64; p++) {
            if (p && !(g_layers && g_layers[c] >> p & 1)) continue;
            g_fails += j >= chunks || list[j] != c || layers[j] != p;
            j++;
        }
    g_fails += j != chunks;
    memset(out, 1, cgk_mx_transposed_bytes(K, chunks));
    return 0;
}
int cgk_mx_quantize(const float* x, size_t ld, int rows, int cols, int format, uint8_t* codes,
                    uint8_t* scales) { return -1; }
int cgk_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int cols, int format,
                      float* y, size_t ld) { return -1; }
size_t cgk_mx_matmul_need(const cgx_mx_weight* w, int M, int act) { return 0; }
size_t cgk_mx_matmul_ws(const cgx_mx_weight* w, int M, int act) { return 0; }
int cgk_mx_matmul(const float* x, size_t ldx, int M, const cgx_mx_weight* w, int act, float* y,
                  size_t ldy, void* ws) { return -1; }
size_t cgk_mx_loss_need(const cgx_mx_weight* w, int M, int act, int grad) { return 0; }
size_t cgk_mx_loss_ws(const cgx_mx_weight* w, int M, int act, int grad) { return 0; }
int cgk_mx_loss(const float* x, size_t ld, int M, const cgx_mx_weight* w, int act,
                const int* targets, float* loss, float* lse, void* ws) { return -1; }
int cgk_mx_loss_grad(const float* x, size_t ld, int M, const cgx_mx_weight* w, int act,
                     const int* targets, const float* lse, const float* dloss, float* dx,
                     size_t ldd, void* ws) { return -1; }

/* ------------------------------------------------------------ checks */
static cgx_mx_weight* make(const uint8_t* codes, const uint8_t* scales, cg_tensor* t, int K, int N,
                           int grad) {
    return t ? cgx_mx_weight_from_tensor(t, grad) : cgx_mx_weight_new(codes, scales, K, N, grad);
}

static void weights(int K, int N, int grad, const uint64_t* layers) {
    const size_t n = (size_t)N * up(K, 32);
    uint8_t *codes = aligned_alloc(16, n * 16), *scales = malloc(n);
    float* x = calloc((size_t)K * N, sizeof(float));
    memset(codes, 0x21, n * 16);
    memset(scales, 127, n);
    cg_tensor t;
    memset(&t, 0, sizeof(t));
    t.data = x;
    t.ndim = 2;
    t.shape[0] = K;
    t.shape[1] = N;
    t.size = K * N;
    g_layers = layers;
    for (int tensor = 0; tensor < 2; tensor++)
        for (g_device = 0; g_device < 2; g_device++) {
            g_calls = 0;
            g_fail_at = -1;
            cgx_mx_weight* w = make(codes, scales, tensor ? &t : NULL, K, N, grad);
            const long calls = g_calls;
            g_fails += !w || g_live != (grad ? 3 : 1);
            if (w && grad) {
                g_fails += w->first[0] != 0 || w->first[w->chunks128] != w->tchunks;
                for (int c = 0; c < w->chunks128; c++)
                    g_fails += w->first[c + 1] - w->first[c] !=
                               (layers ? __builtin_popcountll(layers[c] | 1) : 1);
            }
            cgx_mx_weight_free(w);
            g_fails += g_live != 0;
            /* each call that can fail fails once: NULL, the error set, nothing kept */
            for (long i = 0; i < calls; i++) {
                g_calls = 0;
                g_fail_at = i;
                g_err[0] = 0;
                w = make(codes, scales, tensor ? &t : NULL, K, N, grad);
                g_fails += w != NULL || g_live != 0 || strcmp(g_err, "made to fail") != 0;
                cgx_mx_weight_free(w);
            }
        }
    free(codes);
    free(scales);
    free(x);
}

int main(void) {
    const uint64_t wide[] = {1, 0, 1ull | 1ull << 10, 1ull << 42 | 1ull << 41 | 2, 0x7ffffffffffull};
    const int sizes[][2] = {{1, 1}, {33, 128}, {130, 129}, {256, 600}};
    for (int i = 0; i < 4; i++)
        for (int grad = 0; grad < 2; grad++) {
            weights(sizes[i][0], sizes[i][1], grad, NULL);
            weights(sizes[i][0], sizes[i][1], grad, wide);
            weights(sizes[i][0], sizes[i][1], grad, wide + 5 - up(sizes[i][1], 128));
        }
    printf("mx host check: %s (%d failed checks)\n", g_fails ? "FAIL" : "ok", g_fails);
    return g_fails ? 1 : 0;
}
