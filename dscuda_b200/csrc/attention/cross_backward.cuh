// What the files of the cross attention's gradients share: sizes, parameters, output staging.
#pragma once

#include "sm100_primitives.cuh"

#include <cuda.h>
#include <cuda_bf16.h>

#include <cstdint>

namespace dscuda {
namespace cross {

using namespace sm100;

constexpr int HEAD = 128;
constexpr int BIG = 128;                    // rows of a resident tile (tensor-memory lanes)
constexpr int SUB = 64;                     // rows of a streamed query tile
constexpr int BIG_CHUNK = BIG * 128;        // 16 KB
constexpr int SUB_CHUNK = SUB * 128;        // 8 KB
constexpr int THREADS = 320;                // 8 softmax warps, the MMA warp, the load warp
constexpr int SOFTMAX_THREADS = 256;
constexpr int MMA_WARP = 8;
constexpr int LOAD_WARP = 9;
constexpr int TMEM_COLUMNS = 512;
constexpr float LOG2E = 1.4426950408889634F;

struct CrossBackwardParams {
    CUtensorMap q_sub, do_sub;          // group rows, box {64, group, tokens of a 64-row tile}
    CUtensorMap q_big, do_big, o_big;   // the same for 128-row tiles
    CUtensorMap k, v;                   // [B][Tk][Hkv * 128], boxes of 128 rows
    CUtensorMap dq;                     // like q_big
    CUtensorMap dk, dv;                 // like k
    float2* rows;                       // [B, Hkv, Tq, group]: lse * log2(e), delta
    const float* lse;                   // [B, Hq, Tq]
    const int* lengths;                 // null: Tk
    __nv_bfloat16 *dq_out, *dk_out, *dv_out;
    int query_parts, key_parts;         // CTAs (a cluster) that share a loop
    int tokens, keys, kv_heads, group;
    int sub_tokens, big_tokens;         // tokens of a query tile of each kind
    float scale, scale_log2;
    int batch, key_tiles;               // for the key kernel of short loops
};

__device__ __forceinline__ int length_of(const CrossBackwardParams& p, int entry) {
    return p.lengths == nullptr ? p.keys : min(max(p.lengths[entry], 0), p.keys);
}

// Output tiles leave through idle shared memory: thread r lays out its row of 32 columns in the 128-byte-swizzled chunk that a TMA store reads.
__device__ __forceinline__ void stage_bf16x32(uint8_t* chunk, int r, int half, const uint32_t* values, bool keep) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const uint32_t* x = values + 8 * u;
        const uint4 vec = keep ? make_uint4(pack_bf16x2(__uint_as_float(x[0]), __uint_as_float(x[1])), pack_bf16x2(__uint_as_float(x[2]), __uint_as_float(x[3])),
                                            pack_bf16x2(__uint_as_float(x[4]), __uint_as_float(x[5])), pack_bf16x2(__uint_as_float(x[6]), __uint_as_float(x[7])))
                               : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(chunk + r * 128 + (((half * 4 + u) ^ (r & 7)) * 16)) = vec;
    }
}

}  // namespace cross

// The key kernel for short loops (cross_backward_short.cu): whether it takes a call with that many items of 128 keys and row tiles, and its launch.
bool cross_key_short_takes(long long items, long long row_tiles);
void launch_cross_key_short(const cross::CrossBackwardParams& p, cudaStream_t stream);

// The same for the query kernel (cross_query_short.cu), items of 128 rows.
bool cross_query_short_takes(long long items, long long key_tiles);
void launch_cross_query_short(const cross::CrossBackwardParams& p, cudaStream_t stream);

}  // namespace dscuda
