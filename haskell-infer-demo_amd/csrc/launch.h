/*
 * launch.h - What the library's kernel files share on the host: the launch with its measurement
 * hook, HIP statuses, the device's compute units and the checks of buffers.
 */
#ifndef W4A16_LAUNCH_H
#define W4A16_LAUNCH_H

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.h"

namespace w4a16 {

int hip_status(hipError_t e, const char *what);

/* Compute units of the current device (cached per device; 256 if the query fails). */
int device_cus();

/* Every device buffer of the compute entry points starts on a 16-byte boundary: the kernels
 * move 16 bytes a lane (buffer and direct-to-LDS loads). Allocator pointers always do. */
inline bool misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

/* Whether byte ranges [a, a + an) and [b, b + bn) share a byte. A kernel that reads one while
 * its other blocks write the other would race, so such pairs are refused. */
inline bool overlap(const void *a, size_t an, const void *b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return an && bn && x < y + bn && y < x + an;
}

/* Events that time one of the calling thread's next kernel launches (w4a16_time_next_launch): it
 * goes through hipExtLaunchKernel, whose events take the dispatch's own start and end times
 * (the times a kernel trace reports), and the pair is then forgotten. */
extern thread_local hipEvent_t t_next_launch_events[2];
extern thread_local int t_launches_to_skip;

template <typename... Params, typename... Args>
void launch_k(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, hipStream_t stream,
              Args... args) {
    hipEvent_t start = t_next_launch_events[0], stop = t_next_launch_events[1];
    if ((start || stop) && t_launches_to_skip > 0) {
        --t_launches_to_skip;
        start = stop = nullptr;
    }
    if (start || stop) {
        t_next_launch_events[0] = t_next_launch_events[1] = nullptr;
        hipExtLaunchKernelGGL(kernel, grid, block, (uint32_t)smem, stream, start, stop, 0u,
                              static_cast<Params>(args)...);
    } else {
        hipLaunchKernelGGL(kernel, grid, block, smem, stream, static_cast<Params>(args)...);
    }
}

} // namespace w4a16

#endif /* W4A16_LAUNCH_H */
