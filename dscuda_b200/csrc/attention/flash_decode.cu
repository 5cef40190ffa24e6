// Grouped-query attention of a few query rows over many keys (D = 128), for single tokens and short drafts:
//
//   * over the paged 8-bit cache that flash_cache.cu writes: int8 or e4m3 codes [blocks, Hkv, page, 128] with one fp32 scale
//     for each page and head;
//   * over an encoder's states in bf16, [B, Tk, Hkv, 128], each entry with its own length.
//
// The rows of one key/value head are its group's heads times the new tokens (row = token * group + head), in blocks of 16 or 32,
// so a key is fetched once for all of them.  Per key x and row r: s = scale * ks * (q . x), online softmax, O += p * vs * v.
//
// Bound: HBM, 256 bytes per cached token and head (8 bits) against 4 * 128 FLOP per row.  With 16 rows that is 32 FLOP per byte,
// far below the tensor core's ratio, so the products run on mma.sync (m16n8k16, fp32 sums): 16 rows fit its tile, its operands
// come from registers where the codes are widened on the way, and at the copy rate it is a third busy.  tcgen05 would want
// 128 rows and the widened tile written back to shared memory.
//
// Operands.  Codes become f16 (exact for both types: int8 through 1024 + u - 1152, e4m3 by conversion) and so does Q, each row
// multiplied by a power of two that brings its largest element to 2^13..2^14; P is rounded to f16 (half a step is 2^-12 of it), relative to the largest
// value scale met so far and times 2^14, so that small weights of long rows keep their bits.  bf16 states are multiplied as they are, P
// rounded to bf16.  Sums, maxima and the softmax are fp32.
//
// The order of head columns inside a product is free as long as both factors agree, so a thread takes 16 consecutive bytes of a
// key (four k-steps of its fragment) instead of a gather, and of a value 16 consecutive bytes of four keys.  Rows in shared memory are
// swizzled by ((r & 7) >> 1) | ((r & 1) << 2) in 16-byte units, which makes both read patterns free of bank conflicts.
//
// Work split: tiles of 4 warps x 32 (16) keys of all (sequence, head, row block) items laid end to end and cut into equal ranges, one
// per CTA.  A warp streams its own keys through its own ring (cp.async, no barriers between warps); the four merge at the end of an
// item.  An item that one CTA sees whole is written at once, parts go to the workspace and flash_decode_combine_kernel joins
// them.  No atomics: results do not depend on the order in which CTAs run.
#include "flash_attention.h"
#include "cuda_common.h"
#include "attention_internal.h"
#include "sm100_primitives.cuh"
#include "../common/launch.h"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>

namespace dscuda {
namespace {

using sm100::exp2_approx;

constexpr int HEAD = 128;
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int STAGES = 3;
constexpr int CTAS = 2 * 148;               // two to an SM
constexpr float LOG2E = 1.4426950408889634F;
constexpr float LN2 = 0.6931471805599453F;
constexpr float WEIGHT_UNIT = 16384.0F;     // f16 weights are stored times this

enum Source { INT8 = 0, E4M3 = 1, BF16 = 2 };

__device__ int flash_decode_status = 0;

struct DecodeParams {
    const __nv_bfloat16* query;         // [B, T, Hq, 128]
    const uint8_t* keys;                // codes [blocks, Hkv, page, 128], or bf16 [B, Tk, Hkv, 128]
    const uint8_t* values;
    const float* key_scale;             // [blocks, Hkv]
    const float* value_scale;
    const int* table;                   // [B, pages]; null: dense bf16 states
    const int* lengths;                 // [B]; null: `keys_most` everywhere
    __nv_bfloat16* out;                 // [B, T, Hq, 128]
    float* lse;                         // [B, Hq, T]
    float* part_out;                    // [2 * CTAs][rows of a block][128], normalised
    float* part_lse;                    // [2 * CTAs][rows of a block], log2 domain
    int batch, tokens, heads, kv_heads, group;
    int page, pages, blocks;
    int keys_most;                      // pages * page, or Tk
    int row_blocks;
    int causal;                         // token t sees keys < length - tokens + 1 + t
    float scale;
};

template <int SOURCE, int MT>
struct Shape {
    static constexpr int KEYS = SOURCE == BF16 ? 16 : 32;          // of a warp's step
    static constexpr int TILE = WARPS * KEYS;
    static constexpr int ROW_BYTES = SOURCE == BF16 ? 256 : 128;
    static constexpr int OPERAND = KEYS * ROW_BYTES;               // 4 KB
    static constexpr int STAGE = 2 * OPERAND;
    static constexpr int RING = WARPS * STAGES * STAGE;            // 96 KB
    static constexpr int ROWS = 16 * MT;
    static constexpr int QUERY = MT > 1 ? MT * 8 * 512 : 0;        // fragments of Q, when registers do not hold them
    static constexpr int MERGE = WARPS * ROWS * HEAD * 4;          // in the ring's place, between items
    static_assert(MERGE <= RING, "merge buffer");
    static constexpr int BYTES = RING + QUERY;
};

struct Scales {
    float key[2], value[2];             // of the step's two groups of 16 keys
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
    // 16 bytes, or 16 zeros: keys behind the end of a sequence may hold anything
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

template <int SOURCE>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    if constexpr (SOURCE == BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t packed;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(packed) : "f"(hi), "f"(lo));
    return packed;
}

// Bytes 0, 1 and 2, 3 of a word of codes as pairs of f16.
template <int SOURCE>
__device__ __forceinline__ void widen(uint32_t word, uint32_t& lo, uint32_t& hi) {
    if constexpr (SOURCE == INT8) {
        // code + 128 as the low byte of 0x64xx is 1024 + code + 128
        const uint32_t offset = word ^ 0x80808080U;
        const __half2 bias = __half2half2(__ushort_as_half(0x6480));
        const uint32_t l = __byte_perm(offset, 0x64646464U, 0x4140), h = __byte_perm(offset, 0x64646464U, 0x4342);
        const __half2 dl = __hsub2(*reinterpret_cast<const __half2*>(&l), bias), dh = __hsub2(*reinterpret_cast<const __half2*>(&h), bias);
        lo = *reinterpret_cast<const uint32_t*>(&dl);
        hi = *reinterpret_cast<const uint32_t*>(&dh);
    } else {
        const __half2_raw dl = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(word & 0xffffU), __NV_E4M3);
        const __half2_raw dh = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(word >> 16), __NV_E4M3);
        lo = static_cast<uint32_t>(dl.x) | (static_cast<uint32_t>(dl.y) << 16);
        hi = static_cast<uint32_t>(dh.x) | (static_cast<uint32_t>(dh.y) << 16);
    }
}

__device__ __forceinline__ uint32_t swizzle(int row) {
    return static_cast<uint32_t>(((row & 7) >> 1) | ((row & 1) << 2));
}

// Sequences as runs of tiles: entry b has row_blocks * kv_heads items of tiles(b) tiles each.
__device__ __forceinline__ int length_of(const DecodeParams& p, int b) {
    const int length = p.lengths == nullptr ? p.keys_most : p.lengths[b];
    return min(max(length, 0), p.keys_most);
}

__device__ __forceinline__ long long tiles_of(const DecodeParams& p, int b, int tile) {
    return (static_cast<long long>(length_of(p, b)) + tile - 1) / tile;
}

// Sum of tiles(b) * items over [0, count) by the whole block; every thread gets it.
__device__ __forceinline__ long long sum_tiles(const DecodeParams& p, int count, int tile, long long* scratch) {
    long long sum = 0;
    for (int b = threadIdx.x; b < count; b += THREADS) {
        sum += tiles_of(p, b, tile);
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        sum += __shfl_xor_sync(0xffffffffU, sum, offset);
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) {
        scratch[threadIdx.x / 32] = sum;
    }
    __syncthreads();
    sum = 0;
    for (int w = 0; w < WARPS; ++w) {
        sum += scratch[w];
    }
    return sum * p.kv_heads * p.row_blocks;
}

__device__ __forceinline__ long long range_start(long long total, int ctas, int cta) {
    return total * cta / ctas;
}

// The address of a query or output row: row = token * group + head of the group.
__device__ __forceinline__ size_t row_offset(const DecodeParams& p, int b, int kv_head, int row) {
    const int token = row / p.group;
    return ((static_cast<size_t>(b) * p.tokens + token) * p.heads + kv_head * p.group + row % p.group) * HEAD;
}

__device__ __forceinline__ size_t lse_offset(const DecodeParams& p, int b, int kv_head, int row) {
    return (static_cast<size_t>(b) * p.heads + kv_head * p.group + row % p.group) * p.tokens + row / p.group;
}

template <int SOURCE, int MT>
__global__ void __launch_bounds__(THREADS, 2) flash_decode_kernel(const __grid_constant__ DecodeParams p) {
    using S = Shape<SOURCE, MT>;
    constexpr int KEYS = S::KEYS;
    constexpr int NT = KEYS / 8;                        // n-tiles of a step's scores
    constexpr int KU = KEYS / 16;                       // k-steps of P V
    constexpr int KSTEPS = HEAD / 16;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ long long scratch[WARPS];
    __shared__ Scales scales[WARPS][STAGES];
    __shared__ float merge_m[WARPS][S::ROWS], merge_l[WARPS][S::ROWS], merge_unit[WARPS];
    __shared__ long long found_first;
    __shared__ int found_entry;

    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const int g = lane / 4;                             // row of a fragment of A and C, column of one of B
    const int c = lane % 4;
    const uint32_t delta = static_cast<uint32_t>((g >> 1) | ((g & 1) << 2));        // which 16-byte unit of a value row this lane takes
    const uint32_t ring = warp * STAGES * S::STAGE;             // offset of the warp's ring
    const uint32_t smem_base = sm100::smem_u32(smem);
    auto lds128 = [&](uint32_t offset) { return *reinterpret_cast<const uint4*>(smem + offset); };

    sm100::grid_dependency_wait();
    const long long total = sum_tiles(p, p.batch, S::TILE, scratch);
    long long position = range_start(total, gridDim.x, blockIdx.x);
    const long long end = range_start(total, gridDim.x, blockIdx.x + 1);
    if (position >= end) {
        return;
    }
    // the entry that holds the first tile: blocks of THREADS entries, then inside the block
    const int items = p.kv_heads * p.row_blocks;
    long long entry_first = 0;
    int entry = 0;
    {
        long long before = 0;
        for (int base = 0; base < p.batch; base += THREADS) {
            const int b = base + threadIdx.x;
            const long long own = b < p.batch ? tiles_of(p, b, S::TILE) * items : 0;
            long long inclusive = own;
#pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const long long other = __shfl_up_sync(0xffffffffU, inclusive, offset);
                if (lane >= offset) {
                    inclusive += other;
                }
            }
            __syncthreads();
            if (lane == 31) {
                scratch[warp] = inclusive;
            }
            __syncthreads();
            long long sum = 0;
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) {
                    inclusive += scratch[w];
                }
                sum += scratch[w];
            }
            inclusive += before;
            if (position >= inclusive - own && position < inclusive) {
                found_entry = b;
                found_first = inclusive - own;
            }
            before += sum;
            __syncthreads();
            if (position < before) {
                break;
            }
        }
        entry = found_entry;
        entry_first = found_first;
    }

    bool first_segment = true;
    while (position < end) {
        const int length = length_of(p, entry);
        const long long entry_tiles = tiles_of(p, entry, S::TILE);
        if (position >= entry_first + entry_tiles * items) {
            entry_first += entry_tiles * items;
            ++entry;
            continue;
        }
        const long long item = (position - entry_first) / entry_tiles;
        const long long item_first = entry_first + item * entry_tiles;
        const int tile_begin = static_cast<int>(position - item_first);
        const int tile_end = static_cast<int>(min(entry_tiles, end - item_first));
        const int kv_head = static_cast<int>(item / p.row_blocks);
        const int row_base = static_cast<int>(item % p.row_blocks) * S::ROWS;
        const int rows = p.group * p.tokens;

        // ---- Q: fragments in the column order of the codes --------------------------------------------------
        uint4 qa[MT == 1 ? KSTEPS : 1];
        float factor[MT][2];            // scale * log2(e) * 2^-shift of the thread's two rows
        int limit[MT][2];               // keys that they see
        __syncthreads();                // the last item's merge buffer, and its fragments, have been read
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            uint32_t raw[2][KSTEPS * 2];
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                const int row = row_base + mt * 16 + g + side * 8;
                limit[mt][side] = row < rows ? (p.causal ? length - p.tokens + 1 + row / p.group : length) : 0;
                const uint4* src = reinterpret_cast<const uint4*>(p.query + (row < rows ? row_offset(p, entry, kv_head, row) : 0));
                // 8-bit: k-step 4 j + i holds columns 16 (c + 4 j) + 4 i .. + 3; bf16: k-step 2 j + i columns 8 (c + 4 j) + 4 i .. + 3
                constexpr int UNITS = 4;
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    const int unit = SOURCE == BF16 ? c + 4 * u : 2 * (c + 4 * (u / 2)) + u % 2;
                    const uint4 v = row < rows ? src[unit] : make_uint4(0, 0, 0, 0);
                    raw[side][4 * u] = v.x;
                    raw[side][4 * u + 1] = v.y;
                    raw[side][4 * u + 2] = v.z;
                    raw[side][4 * u + 3] = v.w;
                }
                factor[mt][side] = p.scale * LOG2E;
                if (SOURCE != BF16) {
                    float largest = 0.0F;
#pragma unroll
                    for (int e = 0; e < KSTEPS * 2; ++e) {
                        largest = fmaxf(largest, fmaxf(fabsf(__uint_as_float(raw[side][e] << 16)), fabsf(__uint_as_float(raw[side][e] & 0xffff0000U))));
                    }
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffU, largest, 1));
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffU, largest, 2));
                    const int exponent = static_cast<int>(__float_as_uint(largest) >> 23) - 127;
                    const int shift = largest > 0.0F && exponent < 128 ? min(13 - exponent, 120) : 0;
                    const float up = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
                    factor[mt][side] *= __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll
                    for (int e = 0; e < KSTEPS * 2; ++e) {
                        raw[side][e] = pack_f16x2(__uint_as_float(raw[side][e] << 16) * up, __uint_as_float(raw[side][e] & 0xffff0000U) * up);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
                const uint4 fragment = make_uint4(raw[0][2 * k], raw[1][2 * k], raw[0][2 * k + 1], raw[1][2 * k + 1]);
                if constexpr (MT == 1) {
                    qa[k] = fragment;
                } else if (warp == mt) {
                    *reinterpret_cast<uint4*>(smem + S::RING + ((mt * KSTEPS + k) * 32 + lane) * 16) = fragment;
                }
            }
        }
        if constexpr (MT > 1) {
            __syncthreads();
        }

        // ---- the warp's keys: steps of KEYS, one to a tile ------------------------------------------------
        const int first_key = tile_begin * S::TILE + warp * KEYS;
        const int steps = min(tile_end - tile_begin, max(0, (length - first_key + S::TILE - 1) / S::TILE));
        uint32_t place[2] = {0, 0};                     // lane l: where step (s / 32) * 32 + l finds its two groups of 16 keys
        float place_scale[4] = {1.0F, 1.0F, 1.0F, 1.0F};
        auto issue = [&](int s) {
            if (s < steps) {
                if (SOURCE != BF16 && s % 32 == 0) {
                    const int key = first_key + (s + lane) * S::TILE;
                    if (s + lane < steps) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int k = min(key + 16 * u, length - 1);
                            int page = p.table[static_cast<size_t>(entry) * p.pages + k / p.page];
                            if (page < 0 || page >= p.blocks) {
                                atomicExch(&flash_decode_status, sm100::STATUS_BAD_INDEX);
                                page = 0;
                            }
                            const uint32_t head_page = static_cast<uint32_t>(page) * p.kv_heads + kv_head;
                            place[u] = head_page * p.page + (k / 16 * 16) % p.page;
                            place_scale[u] = p.key_scale[head_page];
                            place_scale[2 + u] = p.value_scale[head_page];
                        }
                    }
                    __syncwarp();
                }
                const uint32_t dst = smem_base + ring + (s % STAGES) * S::STAGE;
                const int key0 = first_key + s * S::TILE;
                if constexpr (SOURCE != BF16) {
                    uint32_t at[2];
                    Scales meta;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        at[u] = __shfl_sync(0xffffffffU, place[u], s % 32);
                        meta.key[u] = __shfl_sync(0xffffffffU, place_scale[u], s % 32);
                        meta.value[u] = __shfl_sync(0xffffffffU, place_scale[2 + u], s % 32);
                    }
                    if (lane == 0) {
                        scales[warp][s % STAGES] = meta;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int row = lane / 8 + 4 * i;
                        const bool valid = key0 + row < length;
                        const size_t offset = valid ? static_cast<size_t>(at[i / 4] + row % 16) * 128 + (lane % 8) * 16 : 0;
                        const uint32_t to = row * 128 + (((lane % 8) ^ swizzle(row)) * 16);
                        copy16(dst + to, p.keys + offset, valid);
                        copy16(dst + S::OPERAND + to, p.values + offset, valid);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int row = lane / 16 + 2 * i;
                        const bool valid = key0 + row < length;
                        const size_t offset = valid ? ((static_cast<size_t>(entry) * p.keys_most + key0 + row) * p.kv_heads + kv_head) * 256 + (lane % 16) * 16 : 0;
                        const uint32_t to = row * 256 + (((lane % 16) ^ swizzle(row)) * 16);
                        copy16(dst + to, p.keys + offset, valid);
                        copy16(dst + S::OPERAND + to, p.values + offset, valid);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        float o[MT][16][4];
        float m[MT][2], l[MT][2];
        float unit = 0.0F;              // the largest value scale so far: weights are relative to it
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int q = 0; q < 16; ++q) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[mt][q][e] = 0.0F;
                }
            }
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.0F;
        }
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            issue(s);
        }
        for (int s = 0; s < steps; ++s) {
            __syncwarp();               // every lane has read the slot that is filled next
            issue(s + STAGES - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t keys = ring + (s % STAGES) * S::STAGE;
            const uint32_t values = keys + S::OPERAND;
            const int key0 = first_key + s * S::TILE;

            // S = Q K^T
            float score[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        score[mt][t][e] = 0.0F;
                    }
                }
            }
            constexpr int KLOADS = S::ROW_BYTES / 64;       // 16-byte units of a key that a thread takes
            constexpr int STEPS_PER_LOAD = KSTEPS / KLOADS;
#pragma unroll
            for (int j = 0; j < KLOADS; ++j) {
                uint4 words[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    words[t] = lds128(keys + (8 * t + g) * S::ROW_BYTES + (((c + 4 * j) ^ swizzle(g)) * 16));
                }
#pragma unroll
                for (int i = 0; i < STEPS_PER_LOAD; ++i) {
                    const int k = j * STEPS_PER_LOAD + i;
                    uint4 a[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        if constexpr (MT == 1) {
                            a[mt] = qa[k];
                        } else {
                            a[mt] = lds128(S::RING + ((mt * KSTEPS + k) * 32 + lane) * 16);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint32_t* w = reinterpret_cast<const uint32_t*>(&words[t]);
                        uint32_t b0, b1;
                        if constexpr (SOURCE == BF16) {
                            b0 = w[2 * i];
                            b1 = w[2 * i + 1];
                        } else {
                            widen<SOURCE>(w[i], b0, b1);
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16816<SOURCE>(score[mt][t], a[mt], b0, b1);
                        }
                    }
                }
            }

            // softmax
            float key_scale[KU], value_scale[KU];
            float shrink = 1.0F;
            if constexpr (SOURCE == BF16) {
                key_scale[0] = value_scale[0] = 1.0F;
            } else {
                const Scales meta = scales[warp][s % STAGES];
                // (a group of keys behind the end repeats the scales of the last one)
                const float largest = fmaxf(meta.value[0], meta.value[1]);
                if (largest > unit) {
                    shrink = unit / largest;
                    unit = largest;
                }
                const float inverse = unit > 0.0F ? WEIGHT_UNIT / unit : 0.0F;
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    key_scale[u] = meta.key[u];
                    value_scale[u] = meta.value[u] * inverse;
                }
            }
            uint4 weights[MT][KU];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float alpha[2];
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    float top = -INFINITY;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const float f = factor[mt][side] * key_scale[t / 2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float x = score[mt][t][2 * side + e] * f;
                            score[mt][t][2 * side + e] = key0 + 8 * t + 2 * c + e < limit[mt][side] ? x : -INFINITY;
                            top = fmaxf(top, score[mt][t][2 * side + e]);
                        }
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffU, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffU, top, 2));
                    const float now = fmaxf(m[mt][side], top);
                    const float reference = now == -INFINITY ? 0.0F : now;          // no key so far: all weights are exp2(-inf) = 0
                    alpha[side] = exp2_approx(m[mt][side] - reference);
                    m[mt][side] = now;
                    float sum = 0.0F;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float weight = exp2_approx(score[mt][t][2 * side + e] - reference);
                            sum += weight;
                            score[mt][t][2 * side + e] = SOURCE == BF16 ? weight : weight * value_scale[t / 2];
                        }
                    }
                    l[mt][side] = l[mt][side] * alpha[side] + sum;
                    alpha[side] *= shrink;
                }
                if (__any_sync(0xffffffffU, alpha[0] != 1.0F || alpha[1] != 1.0F)) {
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        o[mt][q][0] *= alpha[0];
                        o[mt][q][1] *= alpha[0];
                        o[mt][q][2] *= alpha[1];
                        o[mt][q][3] *= alpha[1];
                    }
                }
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    const float(&x)[4] = score[mt][2 * u];
                    const float(&y)[4] = score[mt][2 * u + 1];
                    if constexpr (SOURCE == BF16) {
                        weights[mt][u] = make_uint4(sm100::pack_bf16x2(x[0], x[1]), sm100::pack_bf16x2(x[2], x[3]), sm100::pack_bf16x2(y[0], y[1]),
                                                    sm100::pack_bf16x2(y[2], y[3]));
                    } else {
                        weights[mt][u] = make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]));
                    }
                }
            }

            // O += P V
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                constexpr int VLOADS = S::ROW_BYTES / 128;
#pragma unroll
                for (int h = 0; h < VLOADS; ++h) {
                    uint4 rows4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 16 * u + 8 * (e / 2) + 2 * c + e % 2;
                        rows4[e] = lds128(values + row * S::ROW_BYTES + (((delta + 8 * h) ^ swizzle(row)) * 16));
                    }
                    const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&rows4[0]);
                    const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&rows4[1]);
                    const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&rows4[2]);
                    const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&rows4[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (SOURCE == BF16) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t b0 = __byte_perm(w0[i], w1[i], e == 0 ? 0x5410 : 0x7632);
                                const uint32_t b1 = __byte_perm(w2[i], w3[i], e == 0 ? 0x5410 : 0x7632);
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    mma16816<SOURCE>(o[mt][8 * h + 2 * i + e], weights[mt][u], b0, b1);
                                }
                            }
                        } else {
                            uint32_t b0[4], b1[4];
                            widen<SOURCE>(__byte_perm(w0[i], w1[i], 0x5140), b0[0], b0[1]);
                            widen<SOURCE>(__byte_perm(w0[i], w1[i], 0x7362), b0[2], b0[3]);
                            widen<SOURCE>(__byte_perm(w2[i], w3[i], 0x5140), b1[0], b1[1]);
                            widen<SOURCE>(__byte_perm(w2[i], w3[i], 0x7362), b1[2], b1[3]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    mma16816<SOURCE>(o[mt][4 * i + e], weights[mt][u], b0[e], b1[e]);
                                }
                            }
                        }
                    }
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- the four warps' parts of the item ----------------------------------------------------------
        __syncthreads();                // every ring is idle: the merge buffer takes its place
        float* merge = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                float sum = l[mt][side];
                sum += __shfl_xor_sync(0xffffffffU, sum, 1);
                sum += __shfl_xor_sync(0xffffffffU, sum, 2);
                const int row = mt * 16 + g + side * 8;
                if (c == 0) {
                    merge_m[warp][row] = m[mt][side];
                    merge_l[warp][row] = sum;
                }
                float* dst = merge + (warp * S::ROWS + row) * HEAD;
                // column e of n-tile q is head column 16 delta(e) + q (8 bits), 8 (delta(e) + 8 (q / 8)) + q % 8 (bf16); delta(2 c) = c, delta(2 c + 1) = c + 4
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = c + 4 * e;
#pragma unroll
                    for (int q = 0; q < 16; q += 4) {
                        const int column = SOURCE == BF16 ? 8 * (d + 8 * (q / 8)) + q % 8 : 16 * d + q;
                        *reinterpret_cast<float4*>(dst + column) =
                            make_float4(o[mt][q][2 * side + e], o[mt][q + 1][2 * side + e], o[mt][q + 2][2 * side + e], o[mt][q + 3][2 * side + e]);
                    }
                }
            }
        }
        if (lane == 0) {
            merge_unit[warp] = SOURCE == BF16 ? 1.0F : unit / WEIGHT_UNIT;
        }
        __syncthreads();
        const bool whole = tile_begin == 0 && tile_end == entry_tiles;
        const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
        constexpr int PER_ROW = THREADS / 16;           // threads to a row
#pragma unroll
        for (int pass = 0; pass < MT; ++pass) {
            const int row = pass * 16 + threadIdx.x / PER_ROW;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                top = fmaxf(top, merge_m[w][row]);
            }
            const float reference = top == -INFINITY ? 0.0F : top;
            float sum = 0.0F, share[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                share[w] = exp2_approx(merge_m[w][row] - reference);
                sum += merge_l[w][row] * share[w];
                share[w] *= merge_unit[w];
            }
            const float inverse = sum == 0.0F ? 0.0F : 1.0F / sum;
            const float lse2 = sum == 0.0F ? -INFINITY : reference + log2f(sum);
            const int absolute = row_base + row;
            if (whole && absolute < rows && threadIdx.x % PER_ROW == 0) {
                p.lse[lse_offset(p, entry, kv_head, absolute)] = lse2 * LN2;
            }
            if (!whole && threadIdx.x % PER_ROW == 0) {
                p.part_lse[static_cast<size_t>(slot) * S::ROWS + row] = lse2;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int column = ((k * PER_ROW) + threadIdx.x % PER_ROW) * 4;
                float4 sum4 = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(merge + (w * S::ROWS + row) * HEAD + column);
                    sum4.x += x.x * share[w];
                    sum4.y += x.y * share[w];
                    sum4.z += x.z * share[w];
                    sum4.w += x.w * share[w];
                }
                sum4 = make_float4(sum4.x * inverse, sum4.y * inverse, sum4.z * inverse, sum4.w * inverse);
                if (!whole) {
                    *reinterpret_cast<float4*>(p.part_out + (static_cast<size_t>(slot) * S::ROWS + row) * HEAD + column) = sum4;
                } else if (absolute < rows) {
                    *reinterpret_cast<uint2*>(p.out + row_offset(p, entry, kv_head, absolute) + column) =
                        make_uint2(sm100::pack_bf16x2(sum4.x, sum4.y), sm100::pack_bf16x2(sum4.z, sum4.w));
                }
            }
        }
        position = item_first + tile_end;
        first_segment = false;
    }
}

// Joins the parts of the items that several CTAs worked on, in the order of their keys, and writes the rows of entries without any key.
// A block takes one row of one item.
__global__ void __launch_bounds__(THREADS) flash_decode_combine_kernel(const __grid_constant__ DecodeParams p, int tile, int block_rows, int ctas) {
    __shared__ long long scratch[WARPS];
    const int rows = p.group * p.tokens;
    const int entry = blockIdx.y;
    const int kv_head = blockIdx.x / rows;
    const int row = blockIdx.x % rows;
    const int item = kv_head * p.row_blocks + row / block_rows;
    sm100::grid_dependency_wait();
    const long long tiles = tiles_of(p, entry, tile);
    __nv_bfloat16* out = p.out + row_offset(p, entry, kv_head, row);
    if (tiles == 0) {
        out[threadIdx.x] = __float2bfloat16(0.0F);
        if (threadIdx.x == 0) {
            p.lse[lse_offset(p, entry, kv_head, row)] = -INFINITY;
        }
        return;
    }
    const long long total = sum_tiles(p, p.batch, tile, scratch);
    const long long first = sum_tiles(p, entry, tile, scratch) + item * tiles;
    // the CTA whose range holds a tile: the last one that starts at or before it
    auto holder = [&](long long at) {
        int cta = static_cast<int>(at * ctas / total);
        while (cta + 1 < ctas && range_start(total, ctas, cta + 1) <= at) {
            ++cta;
        }
        while (range_start(total, ctas, cta) > at) {
            --cta;
        }
        return cta;
    };
    const int cta_first = holder(first), cta_last = holder(first + tiles - 1);
    if (cta_first == cta_last) {
        return;                         // written by that CTA
    }
    auto slot_of = [&](int cta) { return 2 * cta + (range_start(total, ctas, cta) >= first ? 0 : 1); };
    const int inside = row % block_rows;
    float top = -INFINITY;
    for (int cta = cta_first; cta <= cta_last; ++cta) {
        if (range_start(total, ctas, cta) < range_start(total, ctas, cta + 1)) {
            top = fmaxf(top, p.part_lse[static_cast<size_t>(slot_of(cta)) * block_rows + inside]);
        }
    }
    const float reference = top == -INFINITY ? 0.0F : top;
    float sum = 0.0F, value = 0.0F;
    for (int cta = cta_first; cta <= cta_last; ++cta) {
        if (range_start(total, ctas, cta) < range_start(total, ctas, cta + 1)) {
            const size_t slot = static_cast<size_t>(slot_of(cta)) * block_rows + inside;
            const float weight = exp2_approx(p.part_lse[slot] - reference);
            sum += weight;
            value += weight * p.part_out[slot * HEAD + threadIdx.x];
        }
    }
    out[threadIdx.x] = __float2bfloat16(sum == 0.0F ? 0.0F : value / sum);
    if (threadIdx.x == 0) {
        p.lse[lse_offset(p, entry, kv_head, row)] = sum == 0.0F ? -INFINITY : (reference + log2f(sum)) * LN2;
    }
}

template <int SOURCE, int MT>
void launch_decode(DecodeParams& p, cudaStream_t stream) {
    using S = Shape<SOURCE, MT>;
    static bool done[16] = {};
    int device = 0;
    CUDA_CHECK(cudaGetDevice(&device));
    if (device >= 16 || !done[device]) {
        CUDA_CHECK(cudaFuncSetAttribute(flash_decode_kernel<SOURCE, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
        if (device < 16) {
            done[device] = true;
        }
    }
    p.row_blocks = (p.group * p.tokens + S::ROWS - 1) / S::ROWS;
    const long long most = static_cast<long long>((p.keys_most + S::TILE - 1) / S::TILE) * p.batch * p.kv_heads * p.row_blocks;
    const int ctas = static_cast<int>(std::min<long long>(CTAS, most));
    p.part_lse = p.part_out + static_cast<size_t>(2 * CTAS) * S::ROWS * HEAD;
    launch_chained(flash_decode_kernel<SOURCE, MT>, dim3(ctas), dim3(THREADS), S::BYTES, stream, p);
    launch_chained(flash_decode_combine_kernel, dim3(p.kv_heads * p.group * p.tokens, p.batch), dim3(THREADS), 0, stream, p, S::TILE, S::ROWS, ctas);
}

template <int SOURCE>
void launch_rows(DecodeParams& p, cudaStream_t stream) {
    if (p.group * p.tokens <= 16) {
        launch_decode<SOURCE, 1>(p, stream);
    } else {
        launch_decode<SOURCE, 2>(p, stream);
    }
}

}  // namespace

namespace internal {

std::size_t few_rows_workspace_bytes(long long rows) {
    return static_cast<std::size_t>(2 * CTAS) * (rows <= 16 ? 16 : 32) * (HEAD + 1) * sizeof(float);
}

void launch_few_rows_cross(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* query, const __nv_bfloat16* key, const __nv_bfloat16* value,
                           const int* key_lengths, void* workspace, int batch, int tokens, int keys, int query_heads, int key_value_heads, float scale,
                           cudaStream_t stream) {
    DecodeParams p{};
    p.query = query;
    p.keys = reinterpret_cast<const uint8_t*>(key);
    p.values = reinterpret_cast<const uint8_t*>(value);
    p.lengths = key_lengths;
    p.out = output;
    p.lse = logsumexp;
    p.part_out = static_cast<float*>(workspace);
    p.batch = batch;
    p.tokens = tokens;
    p.heads = query_heads;
    p.kv_heads = key_value_heads;
    p.group = query_heads / key_value_heads;
    p.keys_most = keys;
    p.causal = 0;
    p.scale = scale;
    launch_rows<BF16>(p, stream);
}

int flash_decode_device_status(bool reset) {
    int status = 0;
    CUDA_CHECK(cudaDeviceSynchronize());
    CUDA_CHECK(cudaMemcpyFromSymbol(&status, flash_decode_status, sizeof(int)));
    if (reset && status != 0) {
        const int zero = 0;
        CUDA_CHECK(cudaMemcpyToSymbol(flash_decode_status, &zero, sizeof(int)));
    }
    return status;
}

}  // namespace internal

std::size_t flash_decode_workspace_bytes(int tokens, int query_heads, int key_value_heads) {
    if (tokens <= 0 || query_heads <= 0 || key_value_heads <= 0) {
        return 0;
    }
    return internal::few_rows_workspace_bytes(static_cast<long long>(tokens) * (query_heads / key_value_heads));
}

void flash_decode_cuda(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* query, const void* key_cache, const void* value_cache,
                       const float* key_scale, const float* value_scale, const int* block_table, const int* cache_lengths, void* workspace,
                       std::size_t workspace_bytes, int batch_size, int tokens, int query_heads, int key_value_heads, int head_size, int page_size,
                       int pages_per_sequence, int cache_blocks, FlashCacheType type, float scale, cudaStream_t stream) {
    internal::check_flash_cache_shape(batch_size, tokens, key_value_heads, head_size, page_size, pages_per_sequence, cache_blocks, type);
    if (query_heads <= 0 || query_heads % key_value_heads != 0) {
        throw std::invalid_argument("flash decode requires query_heads to be divisible by key_value_heads");
    }
    if (tokens > FLASH_DECODE_MAX_TOKENS) {
        throw std::invalid_argument("flash decode takes at most 64 new tokens of a sequence");
    }
    if (!(scale > 0.0F)) {
        throw std::invalid_argument("flash decode requires a positive softmax scale");
    }
    if (batch_size > 65535 || static_cast<long long>(batch_size) * tokens * query_heads > 0x7fffffffLL) {
        throw std::invalid_argument("flash decode shape exceeds the supported index range");
    }
    internal::check_flash_pointers({output, query, key_cache, value_cache, workspace}, {logsumexp, key_scale, value_scale, block_table, cache_lengths});
    if (workspace_bytes < flash_decode_workspace_bytes(tokens, query_heads, key_value_heads)) {
        throw std::invalid_argument("flash decode workspace is too small");
    }
    DecodeParams p{};
    p.query = query;
    p.keys = static_cast<const uint8_t*>(key_cache);
    p.values = static_cast<const uint8_t*>(value_cache);
    p.key_scale = key_scale;
    p.value_scale = value_scale;
    p.table = block_table;
    p.lengths = cache_lengths;
    p.out = output;
    p.lse = logsumexp;
    p.part_out = static_cast<float*>(workspace);
    p.batch = batch_size;
    p.tokens = tokens;
    p.heads = query_heads;
    p.kv_heads = key_value_heads;
    p.group = query_heads / key_value_heads;
    p.page = page_size;
    p.pages = pages_per_sequence;
    p.blocks = cache_blocks;
    p.keys_most = page_size * pages_per_sequence;
    p.causal = 1;
    p.scale = scale;
    if (type == FlashCacheType::INT8) {
        launch_rows<INT8>(p, stream);
    } else {
        launch_rows<E4M3>(p, stream);
    }
}

}  // namespace dscuda
