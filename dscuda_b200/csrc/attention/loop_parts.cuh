// Loops over tiles that are cut into parts where whole loops would leave SMs idle: the CTAs of a cluster take a part each, keep their fp32
// results in their own shared memory and read one another's (distributed shared memory) to add them in order.  No scratch in HBM, no
// second kernel.
#pragma once

#include "sm100_primitives.cuh"

#include <cuda_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace dscuda {

constexpr long long SMS = 148;
constexpr int MOST_PARTS = 16;

// Clusters of n CTAs of a kernel that a device holds at a time, of[n]; 0 for sizes that it cannot launch (a cluster stays inside one of the groups of 16 to
// 20 SMs that share a network, and these differ from one device or partition to another).  One cluster more waits for a whole wave: where 15 of 8 fit, 16 of them
// took 42 us and 15 of 7 take 27.
struct ClusterCounts {
    int of[MOST_PARTS + 1] = {0, static_cast<int>(SMS)};
};

// Asks the device, for sizes up to 8 (portable) and for 16 where `most` allows it.  Once for a device and kernel: the answers take a tenth of a millisecond.
template <class... Parameters>
ClusterCounts cluster_counts(void (*kernel)(Parameters...), unsigned threads, std::size_t shared_bytes, int most) {
    ClusterCounts counts;
    for (int parts = 2; parts <= most; parts += parts < 8 ? 1 : 8) {
        cudaLaunchAttribute attribute{};
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = static_cast<unsigned>(parts);
        attribute.val.clusterDim.y = 1;
        attribute.val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(static_cast<unsigned>(parts));
        config.blockDim = dim3(threads);
        config.dynamicSmemBytes = shared_bytes;
        config.attrs = &attribute;
        config.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&counts.of[parts], kernel, &config) != cudaSuccess) {
            (void)cudaGetLastError();
            counts.of[parts] = 0;
        }
    }
    return counts;
}

// What a cluster costs beside its loops in the gradients' kernels: launch, two cluster barriers, the reads.  (Backward of 4064 x 3 rows over 3 x 3821 ragged keys, 180
// whole loops for 148 SMs: 233 us whole, 144 in parts.)
constexpr double CLUSTER_US = 4.3;

// Parts that a loop of `tiles` tiles of `tile_us` microseconds is cut into when `ctas` whole loops would run: the cluster size of the shortest time, in as many waves
// as its clusters need.
inline int loop_parts(long long ctas, long long tiles, double tile_us, const ClusterCounts& counts) {
    int best = 1;
    double best_us = 0.0;
    for (int parts = 1; parts <= MOST_PARTS && parts <= tiles; ++parts) {
        if (counts.of[parts] == 0) {
            continue;
        }
        const long long waves = (ctas + counts.of[parts] - 1) / counts.of[parts];
        const double us = static_cast<double>(waves) * (static_cast<double>((tiles + parts - 1) / parts) * tile_us + (parts > 1 ? CLUSTER_US : 0.0));
        if (parts == 1 || us < best_us) {
            best = parts;
            best_us = us;
        }
    }
    return best;
}

// Where part `part` of `parts` begins in a loop of `count` tiles.  With fewer tiles than parts the last ones take one each and the first
// parts_without(count, parts) none.
__device__ __forceinline__ int part_begin(int count, int part, int parts) {
    return count < parts ? max(0, count - parts + part) : static_cast<int>(static_cast<long long>(count) * part / parts);
}

__device__ __forceinline__ int parts_without(int count, int parts) {
    return max(0, parts - count);
}

// A CTA's result of 128 rows x 128 fp32 columns in shared memory: 512 bytes to a row, 16-byte units swizzled so that neither a thread to a row
// (writing) nor a warp to a row (reading) meets bank conflicts.
constexpr int RESULT_BYTES = 128 * 512;

__device__ __forceinline__ uint32_t result_unit(int row, int unit) {
    return static_cast<uint32_t>(row * 512 + ((unit ^ (row & 7)) * 16));
}

__device__ __forceinline__ void result_store32(uint8_t* result, int row, int column, const uint32_t* values) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        *reinterpret_cast<uint4*>(result + result_unit(row, column / 4 + u)) = make_uint4(values[4 * u], values[4 * u + 1], values[4 * u + 2], values[4 * u + 3]);
    }
}

// 16 bytes of another CTA's shared memory (address from sm100::map_to_cta).
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// Rows of the results of `parts` CTAs added in order, by a whole warp, a lane to each 16-byte unit: rows first and first + step, as far as they are
// below `end`, times weight(k, part) for the k-th of them.  Parts below `skipped` have left nothing.  A read from another CTA takes most of a
// microsecond, so those of two rows and four parts are on the way at once.
constexpr int SUM_ROWS = 2;

template <class Weight>
__device__ __forceinline__ void cluster_sums(float4 (&sums)[SUM_ROWS], uint32_t result, int lane, int skipped, int parts, int first, int step, int end,
                                             Weight weight) {
    constexpr int AT_ONCE = 4;
#pragma unroll
    for (int k = 0; k < SUM_ROWS; ++k) {
        sums[k] = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
    }
#pragma unroll 1
    for (int base = skipped; base < parts; base += AT_ONCE) {
        float4 x[AT_ONCE][SUM_ROWS];
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const uint32_t from = sm100::map_to_cta(result, min(base + n, parts - 1));
#pragma unroll
            for (int k = 0; k < SUM_ROWS; ++k) {
                x[n][k] = base + n < parts && first + k * step < end ? cluster_load4(from + result_unit(first + k * step, lane)) : make_float4(0.0F, 0.0F, 0.0F, 0.0F);
            }
        }
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
#pragma unroll
            for (int k = 0; k < SUM_ROWS; ++k) {
                const float w = weight(k, min(base + n, parts - 1));
                sums[k] = make_float4(fmaf(w, x[n][k].x, sums[k].x), fmaf(w, x[n][k].y, sums[k].y), fmaf(w, x[n][k].z, sums[k].z), fmaf(w, x[n][k].w, sums[k].w));
            }
        }
    }
}

}  // namespace dscuda
