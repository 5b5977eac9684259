/* Stands in for the runtime calls that start a kernel, so that the host side of libispa_hip.so runs without a GPU: nothing is
 * launched, every launch is written down and judged by the limits of the hardware.  Loaded before the library. */
#include <stddef.h>
#include <stdio.h>

typedef struct {
    unsigned x, y, z;
} dim3;

enum { MAX_KERNELS = 4096, FREE_LDS = 65536, ALL_LDS = 163840 };
static struct {
    const void *kernel;
    int lds;
} allowed[MAX_KERNELS];
static int n_allowed, n_launches;
static char fault[256];

int recorder_launches(void) { return n_launches; }
const char *recorder_fault(void) { return fault; }
void recorder_clear(void) {
    n_launches = 0;
    fault[0] = 0;
}

/* <<<grid, block, lds, stream>>> hands its numbers over in these two. */
static dim3 next_grid, next_block;
static size_t next_lds;
static void *next_stream;
int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, void *stream) {
    next_grid = grid;
    next_block = block;
    next_lds = lds;
    next_stream = stream;
    return 0;
}
int __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, void **stream) {
    *grid = next_grid;
    *block = next_block;
    *lds = next_lds;
    *stream = next_stream;
    return 0;
}

int hipGetDevice(int *device) {
    *device = 0;
    return 0;
}

int hipGetLastError(void) { return 0; }

int hipFuncSetAttribute(const void *kernel, int attribute, int value) {
    int i = 0;
    if (attribute != 8) return 1;                         /* hipFuncAttributeMaxDynamicSharedMemorySize */
    while (i < n_allowed && allowed[i].kernel != kernel) ++i;
    if (i == MAX_KERNELS) return 1;
    if (i == n_allowed) ++n_allowed;
    allowed[i].kernel = kernel;
    allowed[i].lds = value;
    return 0;
}

int hipLaunchKernel(const void *kernel, dim3 grid, dim3 block, void **args, size_t lds, void *stream) {
    size_t limit = FREE_LDS;
    const unsigned long long blocks = (unsigned long long)grid.x * grid.y * grid.z;
    (void)args;
    (void)stream;
    ++n_launches;
    for (int i = 0; i < n_allowed; ++i)
        if (allowed[i].kernel == kernel && (size_t)allowed[i].lds > limit) limit = (size_t)allowed[i].lds;
    if (fault[0]) return 0;                               /* the first one is kept */
    if (blocks == 0)
        snprintf(fault, sizeof(fault), "an empty grid (%u,%u,%u)", grid.x, grid.y, grid.z);
    else if ((unsigned long long)grid.x * block.x >> 32 || grid.y > 65535 || grid.z > 65535)
        snprintf(fault, sizeof(fault), "a grid of (%u,%u,%u) x %u threads", grid.x, grid.y, grid.z, block.x);
    else if (lds > limit || lds > ALL_LDS)
        snprintf(fault, sizeof(fault), "%zu bytes of LDS where %zu are allowed", lds, limit);
    return 0;
}
