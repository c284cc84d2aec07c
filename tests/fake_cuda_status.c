/* fake_cuda.c with host memory that is looked after: what the library frees is counted, and the launcher of the product
 * keeps the status words it was given, as a kernel that a graph holds does. */
#define cudaFreeHost plain_cudaFreeHost
#define ops_launch_f8_matmul plain_ops_launch_f8_matmul
#include "fake_cuda.c"
#undef cudaFreeHost
#undef ops_launch_f8_matmul
#include "../fomoe_b200/csrc/launch.h"

int fake_freed;
static int *kept;
int cudaFreeHost(void *p) { (void)p; fake_freed++; return 0; }
int ops_launch_f8_matmul(const fomoe_b200_f8_matmul_args_t *a, int *st, const ops_device_t *d, int *n, void *s) {
    kept = st;
    return plain_ops_launch_f8_matmul(a, st, d, n, s);
}
/* what the kept kernel does where something goes wrong */
void fake_goes_wrong(int what) {
#ifdef OPS_STATUS_WORD
    kept[OPS_STATUS_WORD(what)] = 1;
#else
    *kept = what;
#endif
}
