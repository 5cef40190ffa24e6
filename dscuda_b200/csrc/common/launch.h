// Kernel launches that may begin before the kernel in front of them on the stream has ended.
#pragma once

#include "cuda_common.h"

#include <cuda_runtime.h>

#include <cstddef>
#include <mutex>
#include <utility>

namespace dscuda {

// Programmatic dependent launch: the blocks of a grid may start when every block of the preceding grid has exited, so its
// launch latency, barrier set-up and tensor-memory allocation overlap the end of that grid (the flush of its writes).
// Every kernel launched this way calls sm100::grid_dependency_wait() before it touches memory that another kernel writes; that
// returns when the preceding grid has ended and its writes are visible.  The one thing read earlier is the kernel family's own
// status word.  Loads are plain, not ld.global.nc: that form wants memory that nothing writes while the kernel lives, and its
// life begins before the grid in front has ended.  No kernel lets its dependents go early
// (griddepcontrol.launch_dependents): blocks of the next grid that sit beside a running decode slowed it (8 ragged sequences,
// 128 heads: 35.3 us without, 41-44 us with), and nothing else gained.
// `cluster`: consecutive blocks (in x) that make a cluster; 1 for none.
template <class... Parameters, class... Arguments>
void launch_chained_clusters(void (*kernel)(Parameters...), dim3 grid, unsigned cluster, dim3 block, std::size_t shared_bytes, cudaStream_t stream,
                             Arguments&&... arguments) {
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = shared_bytes;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t result = cudaLaunchKernelEx(&config, kernel, std::forward<Arguments>(arguments)...);
    if (result != cudaSuccess) {
        (void)cudaGetLastError();       // reported here: the caller's next check must not find it again
    }
    CUDA_CHECK(result);
}

template <class... Parameters, class... Arguments>
void launch_chained(void (*kernel)(Parameters...), dim3 grid, dim3 block, std::size_t shared_bytes, cudaStream_t stream, Arguments&&... arguments) {
    launch_chained_clusters(kernel, grid, 1, block, shared_bytes, stream, std::forward<Arguments>(arguments)...);
}

// What is found out once for each device (the current one), by whichever host thread comes first; on devices behind the table each time.
template <class Value>
class PerDevice {
public:
    template <class Make>
    const Value& get(Make&& make) {
        int device = 0;
        CUDA_CHECK(cudaGetDevice(&device));
        if (device >= DEVICES) {
            thread_local Value value;
            return value = make();
        }
        std::call_once(made_[device], [&] { values_[device] = make(); });
        return values_[device];
    }

private:
    static constexpr int DEVICES = 16;
    std::once_flag made_[DEVICES];
    Value values_[DEVICES];
};

}  // namespace dscuda
