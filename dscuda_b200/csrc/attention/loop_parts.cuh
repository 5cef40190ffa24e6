// Loops over tiles that are cut into parts, a CTA each, where whole loops would leave SMs idle; the parts' fp32 results are joined in order by
// another kernel.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

namespace dscuda {

constexpr long long SMS = 148;

// Parts that a loop of `tiles` tiles is cut into when `ctas` whole loops would run: enough CTAs for every SM, parts of at least MIN_PART tiles, and no
// cut that saves less than the reduce kernel costs.
inline int loop_parts(long long ctas, long long tiles, int min_part) {
    const long long parts = std::min(SMS / std::max(ctas, 1LL), tiles / min_part);
    return parts >= 2 ? static_cast<int>(parts) : 1;
}

// The share of the loop over `count` tiles that part `part` of `parts` has; the last part's is never empty.
__device__ __forceinline__ int part_begin(int count, int part, int parts) {
    return static_cast<int>(static_cast<long long>(count) * part / parts);
}

// Partial sums: a warp's 32 rows of 32 fp32 columns through 4 KB of shared memory, so that a store instruction writes whole 128-byte lines.
template <class RowPointer>
__device__ __forceinline__ void store_f32_rows(uint8_t* slab, int lane, const uint32_t* values, RowPointer row_pointer) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        *reinterpret_cast<uint4*>(slab + lane * 128 + ((u ^ (lane & 7)) * 16)) = make_uint4(values[4 * u], values[4 * u + 1], values[4 * u + 2], values[4 * u + 3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = 4 * i + lane / 8;
        const uint4 v = *reinterpret_cast<const uint4*>(slab + row * 128 + (((lane % 8) ^ (row & 7)) * 16));
        float* dst = row_pointer(row);
        if (dst != nullptr) {
            reinterpret_cast<uint4*>(dst)[lane % 8] = v;
        }
    }
    __syncwarp();
}

}  // namespace dscuda
