// Appends keys and values to the paged 8-bit cache of the grouped-query decode: codes [blocks, Hkv, page, 128] (int8 or e4m3) with
// one fp32 scale for each page and head.
//
// A page's scale covers all values that the page holds.  For the new values x of a page and head
//     need  = max|x| * (1 / Q)           (Q = 127 or 448, 1 / Q as an fp32 constant; 0 if max|x| < 2^-100)
//     scale = max(old, need)             (old = 0 for a page that starts with a new token)
//     code  = round(x * (1 / scale))
// and where the scale grows, the page's older codes become round(code * (old * (1 / scale))).  Every step is a single fp32 operation,
// rounded to nearest, so the codes are the same on any machine.  Growing by the exact ratio instead of a power of two keeps the full range of the codes for
// the page's largest value; a code is rounded again only when a new maximum arrives (about ln(page) times for values in random order).
//
// Bound: HBM, 256 bytes read and 128 written per value row.  A block takes one page of one head of the keys or the values: its threads hold the
// new rows in registers between the maximum and the rounding.  Pages that get no rows cost a block that leaves at once.  A step of 64 sequences in the middle of their
// pages, 8 heads: 3.8 us where the scales stay, 7.1 where every page's grows.
#include "flash_attention.h"
#include "cuda_common.h"
#include "attention_internal.h"
#include "sm100_primitives.cuh"
#include "../common/launch.h"

#include <cuda_fp8.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>

namespace dscuda {
namespace {

constexpr int HEAD = 128;
constexpr int THREADS = 128;
constexpr int ROWS_PER_PASS = THREADS / 16;         // 16 lanes x 16 bytes of bf16 to a row
constexpr int HELD = 8;                             // passes whose rows stay in registers; larger pages read the rest again (from L2)
constexpr float SMALLEST = 7.888609052210118e-31F;  // 2^-100
constexpr uint32_t INFINITE = 0x7f80;               // bf16 magnitudes from here on are infinities and NaN

__device__ int flash_cache_status = 0;

struct AppendParams {
    uint8_t* cache[2];                  // keys, values
    float* scale[2];
    const __nv_bfloat16* rows[2];
    long long stride[2];                // elements between tokens
    const int* table;
    const int* starts;
    const int* counts;
    int tokens, kv_heads, page, pages, blocks;
};

__device__ __forceinline__ float low_bf16(uint32_t pair) {
    return __uint_as_float(pair << 16);
}

__device__ __forceinline__ float high_bf16(uint32_t pair) {
    return __uint_as_float(pair & 0xffff0000U);
}

// Four codes of finite values that lie in the type's range (up to the rounding of the product).
template <bool INT8>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (INT8) {
        // 1.5 * 2^23 + x rounds x half to even into the lowest bits
        constexpr float ROUND = 12582912.0F;
        const uint32_t low = __byte_perm(__float_as_uint(__fadd_rn(a, ROUND)), __float_as_uint(__fadd_rn(b, ROUND)), 0x0040);
        const uint32_t high = __byte_perm(__float_as_uint(__fadd_rn(c, ROUND)), __float_as_uint(__fadd_rn(d, ROUND)), 0x0040);
        return __byte_perm(low, high, 0x5410);
    } else {
        const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        return low | (high << 16);
    }
}

// One code of any value: NaN is 0, infinities the largest codes.
template <bool INT8>
__device__ __forceinline__ uint32_t encode_any(float x) {
    constexpr float LARGEST = INT8 ? 127.0F : 448.0F;
    const float inside = isnan(x) ? 0.0F : fminf(fmaxf(x, -LARGEST), LARGEST);
    return encode4<INT8>(inside, 0.0F, 0.0F, 0.0F) & 0xffU;
}

template <bool INT8>
__device__ __forceinline__ float decode(uint32_t code) {
    if constexpr (INT8) {
        return static_cast<float>(static_cast<int8_t>(code));
    } else {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3)));
    }
}

template <bool INT8>
__global__ void __launch_bounds__(THREADS) flash_cache_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr float LARGEST = INT8 ? 127.0F : 448.0F;
    __shared__ uint32_t warp_max[2][THREADS / 32];
    const int b = blockIdx.z;
    const int side = blockIdx.y % 2;                // keys, values
    const int head = blockIdx.y / 2;
    const int warp = threadIdx.x / 32;
    sm100::grid_dependency_wait();
    const long long start = p.starts != nullptr ? p.starts[b] : 0;
    const long long count = p.counts != nullptr ? min(max(p.counts[b], 0), p.tokens) : p.tokens;
    if (start < 0 && count > 0 && threadIdx.x == 0) {
        atomicExch(&flash_cache_status, sm100::STATUS_BAD_INDEX);       // its tokens in front of position 0 are left out
    }
    const long long logical = max(start, 0LL) / p.page + blockIdx.x;
    const long long begin = max(max(start, 0LL), logical * p.page), end = min(start + count, (logical + 1) * p.page);
    if (begin >= end) {
        return;
    }
    const int slot = static_cast<int>(begin - logical * p.page);        // of the first new row; the rows in front of it are older
    const int rows = static_cast<int>(end - begin);
    const __nv_bfloat16* source = p.rows[side] + (static_cast<long long>(b) * p.tokens + (begin - start)) * p.stride[side] + head * HEAD;
    const int part = threadIdx.x % 16;
    const int mine = threadIdx.x / 16;
    auto load = [&](int row) { return *reinterpret_cast<const uint4*>(source + row * p.stride[side] + part * 8); };
    uint4 held[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int row = k * ROWS_PER_PASS + mine;
        held[k] = row < rows ? load(row) : make_uint4(0, 0, 0, 0);
    }
    int physical = -1;
    if (logical < p.pages) {
        physical = p.table[static_cast<long long>(b) * p.pages + logical];
    }
    if (physical < 0 || physical >= p.blocks) {
        if (threadIdx.x == 0) {
            atomicExch(&flash_cache_status, sm100::STATUS_BAD_INDEX);
        }
        return;
    }
    const size_t head_page = static_cast<size_t>(physical) * p.kv_heads + head;
    uint8_t* page = p.cache[side] + head_page * p.page * HEAD;
    const float old = slot > 0 ? p.scale[side][head_page] : 0.0F;

    // the largest magnitude as bf16 bits, two at a time: their order is that of the integers, infinities and NaN on top
    auto block_max = [&](uint32_t pairs, int round) {
        const uint32_t top = __reduce_max_sync(0xffffffffU, max(pairs & 0xffffU, pairs >> 16));
        if (threadIdx.x % 32 == 0) {
            warp_max[round][warp] = top;
        }
        __syncthreads();
        uint32_t largest = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            largest = max(largest, warp_max[round][w]);
        }
        return largest;
    };
    uint32_t pairs = 0;
    auto measure = [&](const uint4& v) {
        pairs = __vmaxu2(pairs, v.x & 0x7fff7fffU);
        pairs = __vmaxu2(pairs, v.y & 0x7fff7fffU);
        pairs = __vmaxu2(pairs, v.z & 0x7fff7fffU);
        pairs = __vmaxu2(pairs, v.w & 0x7fff7fffU);
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        measure(held[k]);
    }
    for (int row = HELD * ROWS_PER_PASS + mine; row < rows; row += ROWS_PER_PASS) {
        measure(load(row));
    }
    uint32_t largest_bits = block_max(pairs, 0);
    const bool finite = largest_bits < INFINITE;
    if (!finite) {
        // again without the values that are not finite
        pairs = 0;
        for (int row = mine; row < rows; row += ROWS_PER_PASS) {
            const uint4 v = load(row);
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
            for (int e = 0; e < 4; ++e) {
                const uint32_t low = words[e] & 0x7fffU, high = (words[e] >> 16) & 0x7fffU;
                pairs = __vmaxu2(pairs, (low < INFINITE ? low : 0) | (high < INFINITE ? high << 16 : 0));
            }
        }
        largest_bits = block_max(pairs, 1);
    }
    const float largest = __uint_as_float(largest_bits << 16);
    const float need = largest < SMALLEST ? 0.0F : __fmul_rn(largest, 1.0F / LARGEST);
    const float scale = fmaxf(old, need);
    const float inverse = scale > 0.0F ? __fdiv_rn(1.0F, scale) : 0.0F;

    auto store = [&](int row, const uint4& v) {
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
        uint32_t codes[2];
        if (finite) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                codes[e] = encode4<INT8>(__fmul_rn(low_bf16(words[2 * e]), inverse), __fmul_rn(high_bf16(words[2 * e]), inverse),
                                         __fmul_rn(low_bf16(words[2 * e + 1]), inverse), __fmul_rn(high_bf16(words[2 * e + 1]), inverse));
            }
        } else {
            codes[0] = codes[1] = 0;
            for (int e = 0; e < 8; ++e) {
                const float x = e % 2 == 0 ? low_bf16(words[e / 2]) : high_bf16(words[e / 2]);
                codes[e / 4] |= encode_any<INT8>(__fmul_rn(x, inverse)) << (8 * (e % 4));
            }
        }
        *reinterpret_cast<uint2*>(page + static_cast<size_t>(slot + row) * HEAD + part * 8) = make_uint2(codes[0], codes[1]);
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int row = k * ROWS_PER_PASS + mine;
        if (row < rows) {
            store(row, held[k]);
        }
    }
    for (int row = HELD * ROWS_PER_PASS + mine; row < rows; row += ROWS_PER_PASS) {
        store(row, load(row));
    }
    if (slot > 0 && scale > old) {
        const float ratio = __fmul_rn(old, inverse);
        for (int unit = threadIdx.x; unit < slot * (HEAD / 16); unit += THREADS) {
            uint4* at = reinterpret_cast<uint4*>(page) + unit;
            const uint4 v = *at;
            uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = __fmul_rn(decode<INT8>((words[e] >> (8 * k)) & 0xffU), ratio);
                }
                words[e] = encode4<INT8>(x[0], x[1], x[2], x[3]);
            }
            *at = make_uint4(words[0], words[1], words[2], words[3]);
        }
    }
    if (threadIdx.x == 0) {
        p.scale[side][head_page] = scale;
    }
}

}  // namespace

namespace internal {

void check_flash_pointers(std::initializer_list<const void*> wide, std::initializer_list<const void*> narrow) {
    for (const void* pointer : wide) {
        if (pointer == nullptr) {
            throw std::invalid_argument("null tensor pointer");
        }
        if ((reinterpret_cast<std::uintptr_t>(pointer) & 15U) != 0) {
            throw std::invalid_argument("tensor pointers must be 16-byte aligned");
        }
    }
    for (const void* pointer : narrow) {
        if (pointer == nullptr) {
            throw std::invalid_argument("null tensor pointer");
        }
        if ((reinterpret_cast<std::uintptr_t>(pointer) & 3U) != 0) {
            throw std::invalid_argument("int32 and fp32 pointers must be 4-byte aligned");
        }
    }
}

void check_flash_cache_shape(int batch_size, int tokens, int key_value_heads, int head_size, int page_size, int pages_per_sequence,
                             int cache_blocks, FlashCacheType type) {
    if (head_size != HEAD) {
        throw std::invalid_argument("the flash cache requires head_size 128");
    }
    if (type != FlashCacheType::INT8 && type != FlashCacheType::E4M3) {
        throw std::invalid_argument("the flash cache holds int8 or e4m3 codes");
    }
    if (batch_size <= 0 || tokens <= 0 || key_value_heads <= 0 || pages_per_sequence <= 0 || cache_blocks <= 0) {
        throw std::invalid_argument("the flash cache requires positive batch, tokens, heads, pages and blocks");
    }
    if (page_size <= 0 || page_size % 16 != 0) {
        throw std::invalid_argument("the flash cache requires a page size that is a multiple of 16");
    }
    if (static_cast<long long>(page_size) * pages_per_sequence > (1LL << 30) ||
        static_cast<unsigned long long>(page_size) * key_value_heads > 0xffffffffULL / static_cast<unsigned>(cache_blocks)) {
        throw std::invalid_argument("the flash cache shape exceeds the supported index range");
    }
}

int flash_cache_device_status(bool reset) {
    int status = 0;
    CUDA_CHECK(cudaDeviceSynchronize());
    CUDA_CHECK(cudaMemcpyFromSymbol(&status, flash_cache_status, sizeof(int)));
    if (reset && status != 0) {
        const int zero = 0;
        CUDA_CHECK(cudaMemcpyToSymbol(flash_cache_status, &zero, sizeof(int)));
    }
    return status;
}

}  // namespace internal

void flash_cache_append_cuda(void* key_cache, void* value_cache, float* key_scale, float* value_scale, const __nv_bfloat16* key,
                             const __nv_bfloat16* value, const int* block_table, const int* start_positions, const int* token_counts, int batch_size,
                             int tokens, int key_value_heads, int head_size, long long key_stride, long long value_stride, int page_size,
                             int pages_per_sequence, int cache_blocks, FlashCacheType type, cudaStream_t stream) {
    internal::check_flash_cache_shape(batch_size, tokens, key_value_heads, head_size, page_size, pages_per_sequence, cache_blocks, type);
    if (batch_size > 65535 || key_value_heads > 32767) {
        throw std::invalid_argument("flash cache append shape exceeds the supported index range");
    }
    internal::check_flash_pointers({key_cache, value_cache, key, value}, {key_scale, value_scale, block_table});
    for (const int* pointer : {start_positions, token_counts}) {
        if (pointer != nullptr) {
            internal::check_flash_pointers({}, {pointer});
        }
    }
    for (const long long stride : {key_stride, value_stride}) {
        if (stride % 8 != 0 || (static_cast<long long>(batch_size) * tokens > 1 && stride < static_cast<long long>(key_value_heads) * HEAD)) {
            throw std::invalid_argument("flash cache append: tokens must not overlap and lie a multiple of 16 bytes apart");
        }
    }
    AppendParams p{};
    p.cache[0] = static_cast<uint8_t*>(key_cache);
    p.cache[1] = static_cast<uint8_t*>(value_cache);
    p.scale[0] = key_scale;
    p.scale[1] = value_scale;
    p.rows[0] = key;
    p.rows[1] = value;
    p.stride[0] = key_stride;
    p.stride[1] = value_stride;
    p.table = block_table;
    p.starts = start_positions;
    p.counts = token_counts;
    p.tokens = tokens;
    p.kv_heads = key_value_heads;
    p.page = page_size;
    p.pages = pages_per_sequence;
    p.blocks = cache_blocks;
    // T tokens touch at most ceil((T - 1) / page) + 1 pages, from any slot
    const int touched = (tokens + page_size - 2) / page_size + 1;
    launch_chained(type == FlashCacheType::INT8 ? flash_cache_append_kernel<true> : flash_cache_append_kernel<false>,
                   dim3(touched, 2 * key_value_heads, batch_size), dim3(THREADS), 0, stream, p);
}

}  // namespace dscuda
