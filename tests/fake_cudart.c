/* Stand-ins for the CUDA runtime under the launchers as they are built, so that what they launch, and what they make of
 * errors, can be tested without a GPU: launches are written down, nothing runs. */
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

typedef struct { unsigned x, y, z; } dim3_t;
typedef struct { /* cudaLaunchConfig_t */
    dim3_t grid, block;
    size_t smem;
    void *stream, *attrs;
    unsigned n_attrs;
} config_t;

#define MOST 64
static struct { const void *fun; const char *name; } known[256];
static int n_known;
int fake_launches, fake_fail_at = -1, fake_last; /* fake_fail_at: the launch that fails; fake_last: the pending last error */
const char *fake_name[MOST];
unsigned fake_grid[MOST][3];
static config_t pushed;

static int launch(const void *fun, dim3_t grid) {
    if (fake_launches == fake_fail_at) return fake_last = 701;
    if (fake_launches < MOST) {
        fake_name[fake_launches] = "?";
        for (int i = 0; i < n_known; i++)
            if (known[i].fun == fun) fake_name[fake_launches] = known[i].name;
        memcpy(fake_grid[fake_launches], &grid, sizeof(grid));
    }
    fake_launches++;
    return 0;
}

void **__cudaRegisterFatBinary(void *f) { static void *h; (void)f; return &h; }
void __cudaRegisterFatBinaryEnd(void **h) { (void)h; }
void __cudaUnregisterFatBinary(void **h) { (void)h; }
void __cudaRegisterFunction(void **h, const char *fun, char *dev, const char *name, int n, void *a, void *b, void *c, void *d, int *e) {
    (void)h; (void)dev; (void)n; (void)a; (void)b; (void)c; (void)d; (void)e;
    if (n_known < 256) known[n_known].fun = fun, known[n_known++].name = name;
}
unsigned __cudaPushCallConfiguration(dim3_t grid, dim3_t block, size_t smem, void *stream) {
    pushed = (config_t){grid, block, smem, stream, 0, 0};
    return 0;
}
int __cudaPopCallConfiguration(dim3_t *grid, dim3_t *block, size_t *smem, void **stream) {
    *grid = pushed.grid, *block = pushed.block, *smem = pushed.smem, *stream = pushed.stream;
    return 0;
}
int cudaLaunchKernel(const void *f, dim3_t grid, dim3_t block, void **args, size_t smem, void *stream) {
    (void)block; (void)args; (void)smem; (void)stream;
    return launch(f, grid);
}
int cudaLaunchKernelExC(const config_t *c, const void *f, void **args) { (void)args; return launch(f, c->grid); }

int cudaGetDeviceCount(int *n) { *n = 1; return 0; }
int cudaGetDevice(int *d) { *d = 0; return 0; }
int cudaSetDevice(int d) { (void)d; return 0; }
int cudaDeviceGetAttribute(int *v, int attr, int d) { (void)d; *v = attr == 75 ? 10 : 148; return 0; } /* 75: compute capability, major */
int cudaHostAlloc(void **p, size_t n, unsigned f) { (void)f; *p = calloc(1, n); return 0; }
int cudaHostGetDevicePointer(void **d, void *h, unsigned f) { (void)f; *d = h; return 0; }
int cudaFreeHost(void *p) { free(p); return 0; }
int cudaFuncGetAttributes(void *a, const void *f) { (void)a; (void)f; return 0; }
int cudaFuncSetAttribute(const void *f, int a, int v) { (void)f; (void)a; (void)v; return 0; }
int cudaOccupancyMaxActiveClusters(int *n, const void *f, const config_t *c) { (void)f; *n = 148 / (int)c->grid.x; return 0; }
int cudaGetLastError(void) { const int e = fake_last; fake_last = 0; return e; }
const char *cudaGetErrorString(int e) { (void)e; return "fake error"; }

static int encode(void) { return 0; }
int cudaGetDriverEntryPointByVersion(const char *name, void **fn, unsigned v, unsigned long long f, int *q) {
    (void)name; (void)v; (void)f;
    *fn = (void *)encode, *q = 0;
    return 0;
}
