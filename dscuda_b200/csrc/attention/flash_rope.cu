// Rotary position embedding with several position axes, for the heads of the grouped-query kernels (W = 128) and for 64 wide ones.
//
// Pair i of a head (elements i and i + W/2) belongs to one axis and is turned by angle = position[axis] * f_i:
//     out[i]       = x[i] * cos - x[i + W/2] * sin
//     out[i + W/2] = x[i] * sin + x[i + W/2] * cos
// (sin changes sign for `inverse`, which is the transpose and so the gradient).
//
// Angles.  position * f_i / (2 pi) is formed in double precision and reduced to the nearest whole turn there; sine and cosine are taken in double precision
// and rounded to fp32, the products and sums are separate fp32 operations, rounded once to bf16.  So a result has the bits that these steps have anywhere else, and
// codes made from it (the 8-bit cache) are the same; with fp32 sines one result in 2^15 rounded to its neighbour.  That costs nothing at 16384 rows of
// 32 + 8 heads (55.1 us) and 2 % where a row has 8 heads (16.3 us, with fp32 sines 16.0).
//
// Bound: HBM, every value is read and written once.  A warp takes a row: its lanes compute the row's W/2 sines and cosines once (two or
// one each) and exchange them through shared memory; then W/16 lanes cover a head, a lane with 16 bytes of either half, and the warp goes over
// the heads of queries and keys alike, four (eight) at a time with several loads in flight.  With few rows a row's heads are dealt out
// to several warps, each with the row's angles.
#include "flash_attention.h"
#include "cuda_common.h"
#include "attention_internal.h"
#include "sm100_primitives.cuh"
#include "../common/launch.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <stdexcept>

namespace dscuda {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_WARPS = ROPE_THREADS / 32;
constexpr int MAX_AXES = 4;
// Head groups whose loads are issued before the first store, in three CTAs to an SM: 16384 rows of 32 + 8 heads 55.6 us (93 % of the measured copy rate);
// without the bound on registers (two CTAs) 57.9, two groups in four CTAs 56.3, five groups in two 55.7.
constexpr int IN_FLIGHT = 4;

struct RopeParams {
    __nv_bfloat16* out[2];                  // queries, keys
    const __nv_bfloat16* in[2];
    long long out_stride[2], in_stride[2];
    const int* positions;                   // [axes, rows]
    long long rows;
    int query_heads;
    int heads;                              // queries and keys
    int parts;                              // warps that share a row
    int part_heads;                         // heads of each
    int section_end[MAX_AXES];              // pair index behind each section
    double exponent_step[MAX_AXES];         // log2(f) = -step * (pair - base)
    int exponent_base[MAX_AXES];
    float sign;                             // of the sine
};

__device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000U));
}

template <int WIDTH>
__global__ void __launch_bounds__(ROPE_THREADS, 3) flash_rope_kernel(const __grid_constant__ RopeParams p) {
    constexpr int PAIRS = WIDTH / 2;
    constexpr int LANES = PAIRS / 8;                    // lanes to a head
    constexpr int HEADS = 32 / LANES;                   // heads of one pass of the warp
    constexpr int OWN = PAIRS / 32;                     // pairs whose angle a lane computes
    __shared__ alignas(16) float2 turns[ROPE_WARPS][PAIRS];
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const int slot = lane % LANES;                      // pairs 8 slot .. 8 slot + 7
    double frequency[OWN];                              // turns per position
    int axis[OWN];
#pragma unroll
    for (int k = 0; k < OWN; ++k) {
        const int pair = lane + 32 * k;
        axis[k] = 0;
        while (pair >= p.section_end[axis[k]]) {
            ++axis[k];
        }
        frequency[k] = exp2(-p.exponent_step[axis[k]] * (pair - p.exponent_base[axis[k]])) * 0.15915494309189533577;
    }
    sm100::grid_dependency_wait();
    const long long items = p.rows * p.parts;
    for (long long item = static_cast<long long>(blockIdx.x) * ROPE_WARPS + warp; item < items; item += static_cast<long long>(gridDim.x) * ROPE_WARPS) {
        const long long row = p.parts == 1 ? item : item / p.parts;
        const int first = p.parts == 1 ? 0 : static_cast<int>(item - row * p.parts) * p.part_heads;
        const int last = min(p.heads, first + p.part_heads);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const double whole = p.positions[axis[k] * p.rows + row] * frequency[k];
            double s, c;
            sincospi(2.0 * (whole - rint(whole)), &s, &c);
            turns[warp][lane + 32 * k] = make_float2(static_cast<float>(c), static_cast<float>(s) * p.sign);
        }
        __syncwarp();
        float2 turn[8];
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            const float4 two = *reinterpret_cast<const float4*>(&turns[warp][slot * 8 + k]);
            turn[k] = make_float2(two.x, two.y);
            turn[k + 1] = make_float2(two.z, two.w);
        }
        for (int base = first + lane / LANES; base < last; base += HEADS * IN_FLIGHT) {
            uint4 lo[IN_FLIGHT], hi[IN_FLIGHT];
#pragma unroll
            for (int u = 0; u < IN_FLIGHT; ++u) {
                const int head = base + u * HEADS;
                if (head < last) {
                    const int side = head >= p.query_heads;
                    const uint4* src = reinterpret_cast<const uint4*>(p.in[side] + row * p.in_stride[side] + static_cast<long long>(head - side * p.query_heads) * WIDTH);
                    lo[u] = src[slot];
                    hi[u] = src[LANES + slot];
                }
            }
#pragma unroll
            for (int u = 0; u < IN_FLIGHT; ++u) {
                const int head = base + u * HEADS;
                if (head < last) {
                    const int side = head >= p.query_heads;
                    uint4* dst = reinterpret_cast<uint4*>(p.out[side] + row * p.out_stride[side] + static_cast<long long>(head - side * p.query_heads) * WIDTH);
                    uint4 out_lo, out_hi;
                    const uint32_t *a = reinterpret_cast<const uint32_t*>(&lo[u]), *b = reinterpret_cast<const uint32_t*>(&hi[u]);
                    uint32_t *x = reinterpret_cast<uint32_t*>(&out_lo), *y = reinterpret_cast<uint32_t*>(&out_hi);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 l = unpack(a[e]), h = unpack(b[e]), t0 = turn[2 * e], t1 = turn[2 * e + 1];
                        x[e] = sm100::pack_bf16x2(__fsub_rn(__fmul_rn(l.x, t0.x), __fmul_rn(h.x, t0.y)), __fsub_rn(__fmul_rn(l.y, t1.x), __fmul_rn(h.y, t1.y)));
                        y[e] = sm100::pack_bf16x2(__fadd_rn(__fmul_rn(l.x, t0.y), __fmul_rn(h.x, t0.x)), __fadd_rn(__fmul_rn(l.y, t1.y), __fmul_rn(h.y, t1.x)));
                    }
                    dst[slot] = out_lo;
                    dst[LANES + slot] = out_hi;
                }
            }
        }
    }
}

}  // namespace

void flash_rope_cuda(__nv_bfloat16* query_output, __nv_bfloat16* key_output, const __nv_bfloat16* query, const __nv_bfloat16* key,
                     const int* positions, long long rows, int query_heads, int key_heads, int head_size, long long query_output_stride,
                     long long key_output_stride, long long query_stride, long long key_stride, int axes, const int* sections, bool restart,
                     bool inverse, float theta, cudaStream_t stream) {
    if (head_size != 64 && head_size != 128) {
        throw std::invalid_argument("flash rope requires head_size 64 or 128");
    }
    if ((query == nullptr) != (query_output == nullptr) || (key == nullptr) != (key_output == nullptr) || (query == nullptr && key == nullptr)) {
        throw std::invalid_argument("null tensor pointer");
    }
    if (query == nullptr) {
        query_heads = 0;
    }
    if (key == nullptr) {
        key_heads = 0;
    }
    if (rows <= 0 || (query != nullptr && query_heads <= 0) || (key != nullptr && key_heads <= 0) || query_heads > 65535 || key_heads > 65535 ||
        !(theta > 1.0F) || !std::isfinite(theta)) {
        throw std::invalid_argument("flash rope requires positive rows and heads and theta > 1");
    }
    if (axes < 1 || axes > MAX_AXES || sections == nullptr) {
        throw std::invalid_argument("flash rope takes one to four position axes");
    }
    RopeParams p{};
    int pairs = 0;
    const double log2_theta = std::log2(static_cast<double>(theta));
    for (int a = 0; a < axes; ++a) {
        if (sections[a] <= 0 || sections[a] > head_size / 2) {
            throw std::invalid_argument("flash rope sections are positive and add up to head_size / 2");
        }
        p.exponent_base[a] = restart ? pairs : 0;
        p.exponent_step[a] = log2_theta / (restart ? sections[a] : head_size / 2);
        pairs += sections[a];
        p.section_end[a] = pairs;
    }
    if (pairs != head_size / 2) {
        throw std::invalid_argument("flash rope sections are positive and add up to head_size / 2");
    }
    if (query != nullptr) {
        internal::check_flash_pointers({query, query_output}, {positions});
    }
    if (key != nullptr) {
        internal::check_flash_pointers({key, key_output}, {positions});
    }
    const long long strides[4] = {query_output_stride, query_stride, key_output_stride, key_stride};
    for (int i = 0; i < 4; ++i) {
        const long long heads = i < 2 ? query_heads : key_heads;
        if (heads > 0 && (strides[i] % 8 != 0 || (rows > 1 && strides[i] < heads * head_size))) {
            throw std::invalid_argument("flash rope rows must not overlap and lie a multiple of 16 bytes apart");
        }
    }
    if ((query != nullptr && query == query_output && query_stride != query_output_stride && rows > 1) ||
        (key != nullptr && key == key_output && key_stride != key_output_stride && rows > 1)) {
        throw std::invalid_argument("flash rope in place needs the same distance between rows on both sides");
    }
    p.out[0] = query_output;
    p.out[1] = key_output;
    p.in[0] = query;
    p.in[1] = key;
    p.out_stride[0] = query_output_stride;
    p.out_stride[1] = key_output_stride;
    p.in_stride[0] = query_stride;
    p.in_stride[1] = key_stride;
    p.positions = positions;
    p.rows = rows;
    p.query_heads = query_heads;
    p.heads = query_heads + key_heads;
    p.sign = inverse ? -1.0F : 1.0F;
    // as many warps to a row as two CTAs to an SM hold, each with at least one pass of the kernel's loop
    const int pass = 32 / (head_size / 16);
    const int passes = (p.heads + pass - 1) / pass;
    constexpr long long WARPS = 148LL * 2 * ROPE_WARPS;
    const int parts = static_cast<int>(std::max(1LL, std::min<long long>(passes, WARPS / rows)));
    p.part_heads = (passes + parts - 1) / parts * pass;
    p.parts = (p.heads + p.part_heads - 1) / p.part_heads;
    const unsigned blocks = static_cast<unsigned>(std::min((rows * p.parts + ROPE_WARPS - 1) / ROPE_WARPS, 148LL * 8));
    launch_chained(head_size == 128 ? flash_rope_kernel<128> : flash_rope_kernel<64>, dim3(blocks), dim3(ROPE_THREADS), 0, stream, p);
}

}  // namespace dscuda
