// Test-only: the choice of a cluster size for a loop, on given numbers of clusters that a device holds (no GPU), and what the device at hand holds of a small kernel.
#include "loop_parts.cuh"

#include "launch.h"

#include <exception>

namespace {
__global__ void nothing_kernel() {}
}  // namespace

// counts[n]: clusters of n CTAs, n = 0 .. 16
extern "C" int dscuda_test_loop_parts(long long ctas, long long tiles, double tile_us, const int* counts) {
    dscuda::ClusterCounts given;
    for (int n = 0; n <= dscuda::MOST_PARTS; ++n) {
        given.of[n] = counts[n];
    }
    return dscuda::loop_parts(ctas, tiles, tile_us, given);
}

// Fills counts[0 .. 16] for an empty kernel of so much shared memory; 1 where the runtime has an error left over.
extern "C" int dscuda_test_cluster_counts(int shared_bytes, int most, int* counts) {
    (void)cudaGetLastError();
    if (cudaFuncSetAttribute(nothing_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes) != cudaSuccess) {
        return 2;
    }
    const dscuda::ClusterCounts found = dscuda::cluster_counts(nothing_kernel, 128, static_cast<std::size_t>(shared_bytes), most);
    for (int n = 0; n <= dscuda::MOST_PARTS; ++n) {
        counts[n] = found.of[n];
    }
    return cudaPeekAtLastError() == cudaSuccess ? 0 : 1;
}

// 0: PerDevice asks once and hands out what it found
extern "C" int dscuda_test_per_device() {
    try {
        static dscuda::PerDevice<int> devices;
        int asked = 0;
        const int first = devices.get([&] { return 10 + ++asked; }), second = devices.get([&] { return 10 + ++asked; });
        return first == 11 && second == 11 && asked == 1 ? 0 : 1;
    } catch (const std::exception&) {
        return 2;
    }
}
