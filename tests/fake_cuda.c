/* Stand-ins for the CUDA runtime calls and the kernel launchers behind ops_engine.c, so that its checks and the
 * arguments it hands on can be tested without a GPU: launches are counted, nothing runs. */
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include "../fomoe_b200/csrc/ops_launch.h"

static int device, devices = 2;
int fake_launches, fake_launch_device = -1, fake_fail;
int cudaGetDeviceCount(int *n) { *n = devices; return 0; }
int cudaGetDevice(int *d) { *d = device; return 0; }
int cudaSetDevice(int d) { device = d; return 0; }
int cudaDeviceGetAttribute(int *v, int attr, int d) { (void)d; *v = attr == 75 ? 10 : 148; return 0; } /* 75: compute capability, major */
int cudaHostAlloc(void **p, size_t n, unsigned f) { (void)f; *p = calloc(1, n); return 0; }
int cudaHostGetDevicePointer(void **d, void *h, unsigned f) { (void)f; *d = h; return 0; }
int cudaFreeHost(void *p) { free(p); return 0; }
int cudaGetLastError(void) { return 0; }
const char *cudaGetErrorString(int e) { (void)e; return "fake error"; }

static int launch(void) { fake_launches++; fake_launch_device = device; return fake_fail; }
int ops_rows_init(void) { return 0; }
int ops_f8_init(ops_device_t *d) { (void)d; return 0; }
int ops_launch_route(const ops_route_t *a, void *s) { (void)a; (void)s; return launch(); }
int ops_launch_norm(const fomoe_b200_norm_args_t *a, void *s) { (void)a; (void)s; return launch(); }
int ops_launch_f8_quantize(int rows, int cols, const void *x, int b, int64_t xs, uint8_t *q, int64_t qs, float *sc, int64_t ss, void *s) {
    (void)rows; (void)cols; (void)x; (void)b; (void)xs; (void)q; (void)qs; (void)sc; (void)ss; (void)s;
    return launch();
}
int ops_launch_f8_matmul(const fomoe_b200_f8_matmul_args_t *a, int *st, const ops_device_t *d, int *n, void *s) {
    (void)a; (void)st; (void)d; (void)s; *n += 1;
    return launch();
}
void ops_experts_layout(const fomoe_b200_f8_experts_args_t *a, ops_experts_ws_t *w) {
    memset(w, 0, sizeof(*w));
    w->bytes = 256 + (uint64_t)a->n_tokens * 1024;
}
int ops_launch_f8_experts(const fomoe_b200_f8_experts_args_t *a, uint8_t *ws, int *st, const ops_device_t *d, int *n, void *s) {
    (void)a; (void)ws; (void)st; (void)d; (void)s; *n += 1;
    return launch();
}
