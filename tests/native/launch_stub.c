/* For tests of the library's launches without a GPU, preloaded into a process of its own: kernels are not run, their grids and workgroups along the
 * first axis are kept. */
#include <stddef.h>

typedef struct { unsigned x, y, z; } dim;

enum { MOST = 4096 };
int stub_launches = 0;
unsigned stub_grids[MOST], stub_groups[MOST];

static dim grid_now, group_now;
static size_t shared_now;
static void* stream_now;

unsigned __hipPushCallConfiguration(dim grid, dim group, size_t shared, void* stream) {
    grid_now = grid, group_now = group, shared_now = shared, stream_now = stream;
    return 0;
}
int __hipPopCallConfiguration(dim* grid, dim* group, size_t* shared, void** stream) {
    *grid = grid_now, *group = group_now, *shared = shared_now, *stream = stream_now;
    return 0;
}
int hipLaunchKernel(const void* kernel, dim grid, dim group, void** args, size_t shared, void* stream) {
    (void)kernel, (void)args, (void)shared, (void)stream;
    if (stub_launches < MOST) stub_grids[stub_launches] = grid.x, stub_groups[stub_launches] = group.x;
    ++stub_launches;
    return 0;
}
int hipGetLastError(void) { return 0; }
int hipPeekAtLastError(void) { return 0; }
