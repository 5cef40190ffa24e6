// Grouped-query attention of a few query rows over many keys (D = 128), for single tokens and short drafts:
//
//   * over the paged 8-bit cache that flash_cache.cu writes: int8 or e4m3 codes [blocks, Hkv, page, 128] with one fp32 scale
//     for each page and head;
//   * over an encoder's states in bf16, [B, Tk, Hkv, 128], each entry with its own length.
//
// The rows of one key/value head are its group's heads times the new tokens (row = token * group + head), in blocks of 8, 16 or 32,
// so a key is fetched once for a block.  Per key x and row r: s = scale * ks * (q . x), online softmax, O += p * vs * v.
//
// Bound: HBM, 256 bytes per cached token and head (8 bits) against 4 * 128 FLOP per row.  With 16 rows that is 32 FLOP per byte,
// far below the tensor core's ratio, so the products run on mma.sync (m16n8k16, fp32 sums): 16 rows fit its tile, its operands
// come from registers where the codes are widened on the way, and at the copy rate it is a third busy.  tcgen05 wants the
// widened tile written back to shared memory, 192 KB of traffic a tile: measured over 8 sequences of 20000-40000 positions it took 140 us for 32
// rows (this form 116 at the time, 118-125 by now) and 154 for 64 (213: the cache is read twice), over 32 sequences of 500-4000 114 us for
// 64 rows (96).  That was with f16 operands; the 8-bit kinds, which could read the codes as they lie but want the rows as several 8-bit terms, were
// not tried.  Steps of single tokens and short drafts are what this is for, so the one form serves all.
//
// Measured: 32 sequences of 1-8192 tokens, 32 query heads on 8, 46.5-47.5 us (floor 38.3); 4 drafted tokens at 20000-40000, 64 on 8, 118-125 us (floor 72.7);
// 8 items of 128 keys 4.4 us (one launch; 6.5 in parts).  With 32 rows no unit is the bound (DRAM 47 %, tensor 46 %, issue 39 %): the forms of 32 rows take 255
// registers and spill 28-48 bytes, so that two CTAs, eight warps, are all an SM holds, and these do not cover the latency of a step.
//
// Operands.  Codes become f16 (exact for both types: int8 through 1024 + u - 1152, e4m3 by conversion) and so does Q, each row
// multiplied by a power of two that brings its largest element to 2^13..2^14; P is rounded to f16 (half a step is 2^-11 of it), relative to the
// largest value scale met so far and times 2^7, so that small weights of long rows keep their bits (the smallest step is 2^-31 of the largest weight).  bf16 states are multiplied as they
// are, P rounded to bf16.  Sums, maxima and the softmax are fp32.
//
// Products.  S^T = K Q^T and O^T = V^T P^T: the keys, and then the head columns, are the 16 rows of an instruction, the query rows its 8
// columns, so that 1 to 8 query rows waste nothing (with the rows on the 16-row side a step of four heads took twice the tensor instructions and
// twice the softmax: 74 us for 32 ragged sequences where this form took 52).  The 8 x 8 blocks of P^T are turned by movmatrix.
// The order of head columns inside a product is free as long as both factors agree, so a thread takes 16 consecutive bytes of a key
// (four k-steps of its fragment) instead of a gather, and of a value 16 consecutive bytes of four keys.  Rows in shared memory are
// swizzled by ((r & 7) >> 1) | ((r & 1) << 2) in 16-byte units, which makes both read patterns free of bank conflicts.
//
// Work split: tiles of 4 warps x 32 (16) keys of all (sequence, head, row block) items laid end to end and cut into equal ranges, one
// per CTA.  A warp streams its own keys through its own ring (cp.async, no barriers between warps); the four merge at the end of an
// item.  An item that one CTA sees whole is written at once, parts go to the workspace, and the CTA with an item's first tile leaves a
// note of who holds them; flash_decode_combine_kernel joins them.  Where no item can be long each stays with a CTA of its own (stays_whole).  No atomics: results do
// not depend on the order in which CTAs run.
#include "flash_attention.h"
#include "cuda_common.h"
#include "attention_internal.h"
#include "sm100_primitives.cuh"
#include "../common/launch.h"

#include <cuda_fp16.h>
#include <algorithm>
#include <cstdint>
#include <stdexcept>

namespace dscuda {
namespace {

using sm100::exp2_approx;

constexpr int HEAD = 128;
constexpr int KSTEPS = HEAD / 16;
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int MOST_CTAS = 3 * 148;
constexpr int MERGE_PITCH = HEAD + 4;       // floats between rows of the merge buffer
constexpr float LOG2E = 1.4426950408889634F;
constexpr float LN2 = 0.6931471805599453F;
constexpr float WEIGHT_UNIT = 128.0F;       // f16 weights are stored times this
constexpr float RESCALE_THRESHOLD = 8.0F;   // log2 units by which a score may pass the reference before the sums are rescaled; f16 holds 2^8 * 128
constexpr unsigned ITEM_TILES = 2;          // what an item costs beside its tiles (Q, pipeline fill, merge), in tiles; 16 sequences of 500-4000 tokens: 28.4 us a layer step with 1, 27.6 with 2 or 3

enum Source { INT8 = 0, E4M3 = 1, BF16 = 2 };

__device__ int flash_decode_status = 0;

// Who holds the parts of an item: `count` CTAs from `first` on, the first one in its slot 2 * first + `slot`, the others in 2 * cta.
// count 1: written already.
struct PartNote {
    int first;
    int count_slot;                     // 2 * count + slot
};

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
    float* part_out;                    // [2 * MOST_CTAS][rows of a block][128], normalised
    float* part_lse;                    // [2 * MOST_CTAS][rows of a block], log2 domain
    PartNote* notes;                    // [B][items]
    int batch, tokens, heads, kv_heads, group;
    unsigned group_inverse;             // ceil(2^32 / group), 0 for a group of 1
    int page, pages, blocks;
    int keys_most;                      // pages * page, or Tk
    int row_blocks;
    int causal;                         // token t sees keys < length - tokens + 1 + t
    int whole;                          // a CTA to an item, no parts
    float scale;
};

// NB: blocks of 8 query rows of an item.
template <int SOURCE, int NB>
struct Shape {
    static constexpr int ROWS = 8 * NB;
    static constexpr int KEYS = SOURCE == BF16 ? 16 : 32;          // of a warp's step (16 with four blocks of rows: 135 us for 123)
    static constexpr int TILE = WARPS * KEYS;
    static constexpr int ROW_BYTES = SOURCE == BF16 ? 256 : 128;
    static constexpr int OPERAND = KEYS * ROW_BYTES;
    static constexpr int STAGE = 2 * OPERAND;
    static constexpr int CTAS_PER_SM = NB == 1 ? 3 : 2;
    static constexpr int STAGES = NB == 1 ? 2 : 3;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int QUERY = NB > 2 ? NB * KSTEPS * 256 : 0;   // fragments of Q, when registers do not hold them
    static constexpr int MERGE = WARPS * ROWS * MERGE_PITCH * 4;   // in the ring's place, between items
    static constexpr int BYTES = RING + QUERY;
    static_assert(MERGE <= RING, "merge buffer");
    static_assert(CTAS_PER_SM * (BYTES + 2048) <= 227 * 1024, "CTAs of an SM");
};

struct Scales {
    float key[2], value[2];             // of the step's one or two groups of 16 keys
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// 16 bytes, or 16 zeros: what lies behind the end of a sequence may be anything
__device__ __forceinline__ void copy16_if(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

template <int SOURCE>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], const uint2& b) {
    if constexpr (SOURCE == BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    }
}

// Turns an 8 x 8 block of 16-bit values: lane (g, c) gives columns 2 c, 2 c + 1 of row g and gets those of the transposed block.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
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
        asm("{\n\t"
            ".reg .b16 l, h;\n\t"
            "mov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, h;\n\t"
            "}\n"
            : "=r"(lo), "=r"(hi)
            : "r"(word));
    }
}

__device__ __forceinline__ uint32_t swizzle(int row) {
    return static_cast<uint32_t>(((row & 7) >> 1) | ((row & 1) << 2));
}

__device__ __forceinline__ int length_of(const DecodeParams& p, int b) {
    const int length = p.lengths == nullptr ? p.keys_most : p.lengths[b];
    return min(max(length, 0), p.keys_most);
}

// What an item of `length` keys counts when the ranges are cut: its tiles and ITEM_TILES in front of them.
__device__ __forceinline__ unsigned item_cost(int length, int tile) {
    return length > 0 ? (length + tile - 1) / tile + ITEM_TILES : 0;
}

// row / group: exact for row * group < 2^32 (a row is below 64 * group, a group at most 4096).
__device__ __forceinline__ int token_of(const DecodeParams& p, int row) {
    return p.group_inverse == 0 ? row : static_cast<int>(__umulhi(static_cast<unsigned>(row), p.group_inverse));
}

// The address of a query or output row: row = token * group + head of the group.
__device__ __forceinline__ size_t row_offset(const DecodeParams& p, int b, int kv_head, int row) {
    const int token = token_of(p, row);
    return ((static_cast<size_t>(b) * p.tokens + token) * p.heads + kv_head * p.group + (row - token * p.group)) * HEAD;
}

__device__ __forceinline__ size_t lse_offset(const DecodeParams& p, int b, int kv_head, int row) {
    const int token = token_of(p, row);
    return (static_cast<size_t>(b) * p.heads + kv_head * p.group + (row - token * p.group)) * p.tokens + token;
}

// Equal ranges of tiles: the first total % ctas CTAs take one more than the others.
struct Ranges {
    unsigned each = 0, more = 0;
    Ranges() = default;
    __device__ Ranges(unsigned total, unsigned ctas) : each(total / ctas), more(total % ctas) {}
    __device__ unsigned start(unsigned cta) const { return each * cta + min(cta, more); }
    __device__ unsigned holder(unsigned tile) const { return tile < (each + 1) * more ? tile / (each + 1) : more + (tile - (each + 1) * more) / each; }
};

// An item of an entry without keys: zeros and -inf.
template <int ROWS>
__device__ void write_empty_rows(const DecodeParams& p, int entry, int item) {
    const int kv_head = item / p.row_blocks;
    const int row_base = (item - kv_head * p.row_blocks) * ROWS;
    const int rows = min(ROWS, p.group * p.tokens - row_base);
    for (int unit = threadIdx.x; unit < rows * (HEAD / 8); unit += THREADS) {
        const int row = row_base + unit / (HEAD / 8);
        reinterpret_cast<uint4*>(p.out + row_offset(p, entry, kv_head, row))[unit % (HEAD / 8)] = make_uint4(0, 0, 0, 0);
        if (unit % (HEAD / 8) == 0) {
            p.lse[lse_offset(p, entry, kv_head, row)] = -INFINITY;
        }
    }
}

template <int SOURCE, int NB>
__global__ void __launch_bounds__(THREADS, Shape<SOURCE, NB>::CTAS_PER_SM) flash_decode_kernel(const __grid_constant__ DecodeParams p) {
    using S = Shape<SOURCE, NB>;
    constexpr int KEYS = S::KEYS;
    constexpr int STAGES = S::STAGES;
    constexpr int KU = KEYS / 16;                       // blocks of 16 keys of a step
    constexpr bool QUERY_IN_REGISTERS = S::QUERY == 0;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Scales scales[WARPS][STAGES];
    __shared__ float merge_m[WARPS][S::ROWS], merge_l[WARPS][S::ROWS], merge_unit[WARPS];

    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const int g = lane / 4;
    const int c = lane % 4;
    const uint32_t delta = static_cast<uint32_t>((g >> 1) | ((g & 1) << 2));        // which 16-byte unit of a value row this lane takes
    const uint32_t ring = warp * STAGES * S::STAGE;     // offset of the warp's ring
    const uint32_t smem_base = sm100::smem_u32(smem);
    auto lds128 = [&](uint32_t offset) { return *reinterpret_cast<const uint4*>(smem + offset); };
    constexpr int LANES = S::ROW_BYTES / 16;            // lanes that copy a row
    constexpr int COPY_ROWS = 32 / LANES;               // rows of one instruction
    // rows lane / LANES + COPY_ROWS * i: their place in a stage repeats after 8 rows
    uint32_t copy_to[8 / COPY_ROWS];
#pragma unroll
    for (int i = 0; i < 8 / COPY_ROWS; ++i) {
        const int row = lane / LANES + COPY_ROWS * i;
        copy_to[i] = smem_base + ring + row * S::ROW_BYTES + (((lane % LANES) ^ swizzle(row)) * 16);
    }

    sm100::grid_dependency_wait();
    // ---- the CTA's range of tiles, and the entry that holds its first one; every warp for itself --------------
    const unsigned items = p.kv_heads * p.row_blocks;
    Ranges ranges;
    unsigned position, end, entry_first = 0;
    int entry = 0;
    if (p.whole != 0) {
        entry = static_cast<int>(blockIdx.x / items);
        const unsigned item = blockIdx.x - entry * items;
        const int length = length_of(p, entry);
        if (length == 0) {
            write_empty_rows<S::ROWS>(p, entry, static_cast<int>(item));
            return;
        }
        position = item * item_cost(length, S::TILE);
        end = position + item_cost(length, S::TILE);
    } else {
        unsigned total = 0, own = 0;
        for (int base = 0; base < p.batch; base += 32) {
            own = base + lane < p.batch ? item_cost(length_of(p, base + lane), S::TILE) * items : 0;
            total += __reduce_add_sync(0xffffffffU, own);
        }
        const unsigned ctas = min(total, gridDim.x);
        if (blockIdx.x >= ctas) {
            return;
        }
        ranges = Ranges(total, ctas);
        position = ranges.start(blockIdx.x);
        end = ranges.start(blockIdx.x + 1);
        for (int base = 0;; base += 32) {
            if (p.batch > 32) {
                own = base + lane < p.batch ? item_cost(length_of(p, base + lane), S::TILE) * items : 0;
            }
            unsigned inclusive = own;
#pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const unsigned other = __shfl_up_sync(0xffffffffU, inclusive, offset);
                inclusive += lane >= offset ? other : 0;
            }
            const unsigned mine = __ballot_sync(0xffffffffU, position < entry_first + inclusive);
            if (mine != 0) {
                const int source = __ffs(mine) - 1;
                entry = base + source;
                entry_first += __shfl_sync(0xffffffffU, inclusive - own, source);
                break;
            }
            entry_first += __shfl_sync(0xffffffffU, inclusive, 31);
        }
    }

    bool first_segment = true;
    while (position < end) {
        const int length = length_of(p, entry);
        const unsigned cost = item_cost(length, S::TILE);
        if (position >= entry_first + cost * items) {
            entry_first += cost * items;
            ++entry;
            continue;
        }
        const unsigned item = (position - entry_first) / cost;
        const unsigned first_tile = entry_first + item * cost + ITEM_TILES;         // position of the item's first tile
        const int entry_tiles = static_cast<int>(cost - ITEM_TILES);
        const int tile_begin = static_cast<int>(max(position, first_tile) - first_tile);
        const int tile_end = min(entry_tiles, static_cast<int>(end) - static_cast<int>(first_tile));
        position = first_tile + max(tile_end, 0);
        if (tile_end <= tile_begin) {
            continue;                   // the range ends in front of the item's tiles
        }
        const int kv_head = static_cast<int>(item) / p.row_blocks;
        const int row_base = (static_cast<int>(item) - kv_head * p.row_blocks) * S::ROWS;
        const int rows = p.group * p.tokens;

        // ---- Q on its way, in front of the keys in the queue of the memory: lane (g, c) has row g of each block of 8 ------------
        uint4 raw[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int row = row_base + nb * 8 + g;
            const uint4* src = reinterpret_cast<const uint4*>(p.query + (row < rows ? row_offset(p, entry, kv_head, row) : 0));
            // 8-bit: k-step 4 j + i holds columns 16 (c + 4 j) + 4 i .. + 3; bf16: k-step 2 j + i columns 8 (c + 4 j) + 4 i .. + 3
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                raw[nb][u] = row < rows ? src[SOURCE == BF16 ? c + 4 * u : 2 * (c + 4 * (u / 2)) + u % 2] : make_uint4(0, 0, 0, 0);
            }
        }

        // ---- the warp's keys: steps of KEYS, one to a tile ------------------------------------------------
        const int first_key = tile_begin * S::TILE + warp * KEYS;
        const int steps = min(tile_end - tile_begin, max(0, (length - first_key + S::TILE - 1) / S::TILE));
        uint32_t place[KU] = {};                        // lane l: where step (s / 32) * 32 + l finds its groups of 16 keys
        Scales place_scales = {};
        auto issue = [&](int s) {
            if (s < steps) {
                const int key0 = first_key + s * S::TILE;
                const uint32_t slot = (s % STAGES) * S::STAGE;
                if constexpr (SOURCE != BF16) {
                    if (s % 32 == 0) {
                        const int key = key0 + lane * S::TILE;
                        if (s + lane < steps) {
#pragma unroll
                            for (int u = 0; u < KU; ++u) {
                                const int k = min(key + 16 * u, length - 1);
                                const int logical = k / p.page;
                                int page = p.table[static_cast<size_t>(entry) * p.pages + logical];
                                if (page < 0 || page >= p.blocks) {
                                    atomicExch(&flash_decode_status, sm100::STATUS_BAD_INDEX);
                                    page = 0;
                                }
                                const uint32_t head_page = static_cast<uint32_t>(page) * p.kv_heads + kv_head;
                                place[u] = head_page * p.page + (k / 16 * 16 - logical * p.page);
                                place_scales.key[u] = p.key_scale[head_page];
                                place_scales.value[u] = p.value_scale[head_page];
                            }
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (int u = 0; u < KU; ++u) {
                        const uint32_t at = __shfl_sync(0xffffffffU, place[u], s % 32);
                        const size_t offset = static_cast<size_t>(at) * 128 + lane * 16;        // rows of a group lie one after the other
                        const uint8_t *k = p.keys + offset, *v = p.values + offset;
                        const int left = length - key0 - 16 * u;
                        if (__all_sync(0xffffffffU, left >= 16)) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t to = copy_to[i % 2] + slot + (16 * u + 8 * (i / 2)) * 128;
                                copy16(to, k + i * 512);
                                copy16(to + S::OPERAND, v + i * 512);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t to = copy_to[i % 2] + slot + (16 * u + 8 * (i / 2)) * 128;
                                const bool valid = lane / 8 + 4 * i < left;
                                copy16_if(to, valid ? k + i * 512 : p.keys, valid);
                                copy16_if(to + S::OPERAND, valid ? v + i * 512 : p.values, valid);
                            }
                        }
                    }
                    if (lane == s % 32) {
                        scales[warp][s % STAGES] = place_scales;        // (behind the copies, which need not wait for them)
                    }
                } else {
                    const size_t pitch = static_cast<size_t>(p.kv_heads) * 256;
                    const size_t offset = (static_cast<size_t>(entry) * p.keys_most + key0 + lane / 16) * pitch + kv_head * 256 + (lane % 16) * 16;
                    const uint8_t *k = p.keys + offset, *v = p.values + offset;
                    const int left = length - key0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t to = copy_to[i % 4] + slot + 8 * (i / 4) * 256;
                        const bool valid = lane / 16 + 2 * i < left;
                        copy16_if(to, valid ? k + 2 * i * pitch : p.keys, valid);
                        copy16_if(to + S::OPERAND, valid ? v + 2 * i * pitch : p.values, valid);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();                // the last item's merge buffer has been read
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            issue(s);
        }

        // ---- Q: B fragments in the column order of the codes ----------------
        uint2 query[QUERY_IN_REGISTERS ? NB : 1][KSTEPS];
        float factor[NB][2];            // scale * log2(e) * 2^-shift of rows 2 c and 2 c + 1
        int limit[NB][2];               // keys that they see
        int least = 0x7fffffff;         // the fewest that a row sees
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            uint32_t pairs[KSTEPS * 2];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                pairs[4 * u] = raw[nb][u].x;
                pairs[4 * u + 1] = raw[nb][u].y;
                pairs[4 * u + 2] = raw[nb][u].z;
                pairs[4 * u + 3] = raw[nb][u].w;
            }
            float down = p.scale * LOG2E;
            if (SOURCE != BF16) {
                float largest = 0.0F;
#pragma unroll
                for (int e = 0; e < KSTEPS * 2; ++e) {
                    largest = fmaxf(largest, fmaxf(fabsf(__uint_as_float(pairs[e] << 16)), fabsf(__uint_as_float(pairs[e] & 0xffff0000U))));
                }
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffU, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffU, largest, 2));
                const int exponent = static_cast<int>(__float_as_uint(largest) >> 23) - 127;
                const int shift = largest > 0.0F && exponent < 128 ? min(13 - exponent, 120) : 0;
                const float up = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
                down *= __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll
                for (int e = 0; e < KSTEPS * 2; ++e) {
                    pairs[e] = pack_f16x2(__uint_as_float(pairs[e] << 16) * up, __uint_as_float(pairs[e] & 0xffff0000U) * up);
                }
            }
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                const int column = row_base + nb * 8 + 2 * c + side;
                factor[nb][side] = __shfl_sync(0xffffffffU, down, 8 * c + 4 * side);
                // (rows that do not exist have Q = 0 and are not written)
                limit[nb][side] = p.causal && column < rows ? length - p.tokens + 1 + token_of(p, column) : length;
                least = min(least, limit[nb][side]);
            }
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
                if constexpr (QUERY_IN_REGISTERS) {
                    query[nb][k] = make_uint2(pairs[2 * k], pairs[2 * k + 1]);
                } else if (warp == nb % WARPS) {
                    *reinterpret_cast<uint2*>(smem + S::RING + ((nb * KSTEPS + k) * 32 + lane) * 8) = make_uint2(pairs[2 * k], pairs[2 * k + 1]);
                }
            }
        }
        least = __reduce_min_sync(0xffffffffU, least);
        if constexpr (!QUERY_IN_REGISTERS) {
            __syncthreads();
        }
        auto query_fragment = [&](int nb, int k) {
            if constexpr (QUERY_IN_REGISTERS) {
                return query[nb][k];
            } else {
                return *reinterpret_cast<const uint2*>(smem + S::RING + ((nb * KSTEPS + k) * 32 + lane) * 8);
            }
        };

        float o[NB][8][4];              // O^T: m-tile j holds head columns 2 j and 2 j + 1 of the lane's unit; query rows 2 c and 2 c + 1
        float2 m[NB], l[NB];            // reference and sum of rows 2 c and 2 c + 1 (the sum over this lane's keys)
        float unit = 0.0F;              // the largest value scale so far: weights are relative to it
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[nb][j][e] = 0.0F;
                }
            }
            m[nb] = make_float2(-INFINITY, -INFINITY);
            l[nb] = make_float2(0.0F, 0.0F);
        }
        for (int s = 0; s < steps; ++s) {
            __syncwarp();               // every lane has read the slot that is filled next
            issue(s + STAGES - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t keys = ring + (s % STAGES) * S::STAGE;
            const uint32_t values = keys + S::OPERAND;
            const int key0 = first_key + s * S::TILE;

            // S^T = K Q^T: lane (g, c) gets keys g and g + 8 of a block of 16, query rows 2 c and 2 c + 1
            float score[KU][NB][4];
#pragma unroll
            for (int u = 0; u < KU; ++u) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        score[u][nb][e] = 0.0F;
                    }
                }
            }
            constexpr int KLOADS = S::ROW_BYTES / 64;       // 16-byte units of a key that a thread takes
            constexpr int STEPS_PER_LOAD = KSTEPS / KLOADS;
#pragma unroll
            for (int j = 0; j < KLOADS; ++j) {
                uint4 words[KU][2];
#pragma unroll
                for (int u = 0; u < KU; ++u) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        words[u][h] = lds128(keys + (16 * u + 8 * h + g) * S::ROW_BYTES + (((c + 4 * j) ^ swizzle(g)) * 16));
                    }
                }
#pragma unroll
                for (int i = 0; i < STEPS_PER_LOAD; ++i) {
                    const int k = j * STEPS_PER_LOAD + i;
#pragma unroll
                    for (int u = 0; u < KU; ++u) {
                        const uint32_t *w0 = reinterpret_cast<const uint32_t*>(&words[u][0]), *w1 = reinterpret_cast<const uint32_t*>(&words[u][1]);
                        uint32_t a[4];
                        if constexpr (SOURCE == BF16) {
                            a[0] = w0[2 * i];
                            a[1] = w1[2 * i];
                            a[2] = w0[2 * i + 1];
                            a[3] = w1[2 * i + 1];
                        } else {
                            widen<SOURCE>(w0[i], a[0], a[2]);
                            widen<SOURCE>(w1[i], a[1], a[3]);
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            mma16816<SOURCE>(score[u][nb], a, query_fragment(nb, k));
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
                const float largest = fmaxf(meta.value[0], meta.value[KU - 1]);
                if (largest > unit) {
                    shrink = unit / largest;
                    unit = largest;
                }
                const float inverse = unit > 0.0F ? __fdividef(WEIGHT_UNIT, unit) : 0.0F;
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    key_scale[u] = meta.key[u];
                    value_scale[u] = meta.value[u] * inverse;
                }
            }
            // x = score * f - reference for the pair of query rows at once.  The reference m of a row lags its maximum by up to the threshold: the
            // lanes of a row compare notes, and the sums are rescaled, only when one of them passes it.
            float2 f[KU][NB];
#pragma unroll
            for (int u = 0; u < KU; ++u) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    f[u][nb] = make_float2(factor[nb][0] * key_scale[u], factor[nb][1] * key_scale[u]);
                }
            }
            if (__any_sync(0xffffffffU, key0 + KEYS > least)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int u = 0; u < KU; ++u) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = score[u][nb][e] * (e % 2 == 0 ? f[u][nb].x : f[u][nb].y);
                            score[u][nb][e] = key0 + 16 * u + 8 * (e / 2) + g < limit[nb][e % 2] ? x : -INFINITY;
                        }
                        f[u][nb] = make_float2(1.0F, 1.0F);         // (a scale of zero must not meet the infinity)
                    }
                }
            }
            float2 top[NB];
            bool moved = shrink != 1.0F;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                top[nb] = make_float2(-INFINITY, -INFINITY);
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    top[nb].x = fmaxf(top[nb].x, fmaxf(score[u][nb][0], score[u][nb][2]) * f[u][nb].x);
                    top[nb].y = fmaxf(top[nb].y, fmaxf(score[u][nb][1], score[u][nb][3]) * f[u][nb].y);
                }
                moved |= top[nb].x > m[nb].x + RESCALE_THRESHOLD || top[nb].y > m[nb].y + RESCALE_THRESHOLD;
            }
            if (__any_sync(0xffffffffU, moved)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int offset = 4; offset < 32; offset <<= 1) {
                        top[nb].x = fmaxf(top[nb].x, __shfl_xor_sync(0xffffffffU, top[nb].x, offset));
                        top[nb].y = fmaxf(top[nb].y, __shfl_xor_sync(0xffffffffU, top[nb].y, offset));
                    }
                    const float2 now = make_float2(fmaxf(m[nb].x, top[nb].x), fmaxf(m[nb].y, top[nb].y));
                    // no key so far: the sums are zero
                    float2 alpha = make_float2(now.x == -INFINITY ? 1.0F : exp2_approx(m[nb].x - now.x), now.y == -INFINITY ? 1.0F : exp2_approx(m[nb].y - now.y));
                    m[nb] = now;
                    l[nb] = make_float2(l[nb].x * alpha.x, l[nb].y * alpha.y);
                    alpha = make_float2(alpha.x * shrink, alpha.y * shrink);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        o[nb][j][0] *= alpha.x;
                        o[nb][j][1] *= alpha.y;
                        o[nb][j][2] *= alpha.x;
                        o[nb][j][3] *= alpha.y;
                    }
                }
            }
            uint2 weights[KU][NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                // a row without any key so far: all its weights are exp2(-inf) = 0
                const float2 minus = make_float2(m[nb].x == -INFINITY ? 0.0F : -m[nb].x, m[nb].y == -INFINITY ? 0.0F : -m[nb].y);
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    uint32_t packed[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 x = sm100::fma2(make_float2(score[u][nb][2 * h], score[u][nb][2 * h + 1]), f[u][nb], minus);
                        const float2 weight = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                        l[nb] = sm100::add2(l[nb], weight);
                        if constexpr (SOURCE == BF16) {
                            packed[h] = sm100::pack_bf16x2(weight.x, weight.y);
                        } else {
                            const float2 scaled = sm100::mul2(weight, make_float2(value_scale[u], value_scale[u]));
                            packed[h] = pack_f16x2(scaled.x, scaled.y);
                        }
                    }
                    weights[u][nb] = make_uint2(turn8x8(packed[0]), turn8x8(packed[1]));
                }
            }

            // O^T += V^T P^T
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
                    const uint32_t *w0 = reinterpret_cast<const uint32_t*>(&rows4[0]), *w1 = reinterpret_cast<const uint32_t*>(&rows4[1]);
                    const uint32_t *w2 = reinterpret_cast<const uint32_t*>(&rows4[2]), *w3 = reinterpret_cast<const uint32_t*>(&rows4[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (SOURCE == BF16) {
                            const uint32_t a[4] = {__byte_perm(w0[i], w1[i], 0x5410), __byte_perm(w0[i], w1[i], 0x7632), __byte_perm(w2[i], w3[i], 0x5410),
                                                   __byte_perm(w2[i], w3[i], 0x7632)};
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                mma16816<SOURCE>(o[nb][4 * h + i], a, weights[u][nb]);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                // columns 4 i + 2 e and + 1 of four keys
                                uint32_t a[4];
                                widen<SOURCE>(__byte_perm(w0[i], w1[i], e == 0 ? 0x5140 : 0x7362), a[0], a[1]);
                                widen<SOURCE>(__byte_perm(w2[i], w3[i], e == 0 ? 0x5140 : 0x7362), a[2], a[3]);
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb) {
                                    mma16816<SOURCE>(o[nb][2 * i + e], a, weights[u][nb]);
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
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                float sum = side == 0 ? l[nb].x : l[nb].y;
#pragma unroll
                for (int offset = 4; offset < 32; offset <<= 1) {
                    sum += __shfl_xor_sync(0xffffffffU, sum, offset);
                }
                const int row = nb * 8 + 2 * c + side;
                if (g == 0) {
                    merge_m[warp][row] = side == 0 ? m[nb].x : m[nb].y;
                    merge_l[warp][row] = sum;
                }
                float* dst = merge + (warp * S::ROWS + row) * MERGE_PITCH;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int column = SOURCE == BF16 ? 8 * (delta + 8 * (j / 4)) + 2 * (j % 4) : 16 * delta + 2 * j;
                    *reinterpret_cast<float4*>(dst + column) = make_float4(o[nb][j][side], o[nb][j][2 + side], o[nb][j + 1][side], o[nb][j + 1][2 + side]);
                }
            }
        }
        if (lane == 0) {
            merge_unit[warp] = SOURCE == BF16 ? 1.0F : unit / WEIGHT_UNIT;
        }
        __syncthreads();
        const bool whole = tile_begin == 0 && tile_end == entry_tiles;
        const unsigned slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
        if (tile_begin == 0 && threadIdx.x == 0 && p.whole == 0) {
            const int holders = static_cast<int>(ranges.holder(first_tile + entry_tiles - 1) - blockIdx.x) + 1;
            p.notes[static_cast<size_t>(entry) * items + item] = {static_cast<int>(blockIdx.x), 2 * holders + (first_segment ? 0 : 1)};
        }
        constexpr int PER_ROW = THREADS / 8;            // threads to a row
#pragma unroll
        for (int pass = 0; pass < NB; ++pass) {
            const int row = pass * 8 + threadIdx.x / PER_ROW;
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
            if (absolute < rows) {
                if (threadIdx.x % PER_ROW == 0) {
                    if (whole) {
                        p.lse[lse_offset(p, entry, kv_head, absolute)] = lse2 * LN2;
                    } else {
                        p.part_lse[static_cast<size_t>(slot) * S::ROWS + row] = lse2;
                    }
                }
                const size_t out_row = row_offset(p, entry, kv_head, absolute);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int column = ((k * PER_ROW) + threadIdx.x % PER_ROW) * 4;
                    float4 sum4 = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) {
                        const float4 x = *reinterpret_cast<const float4*>(merge + (w * S::ROWS + row) * MERGE_PITCH + column);
                        sum4.x += x.x * share[w];
                        sum4.y += x.y * share[w];
                        sum4.z += x.z * share[w];
                        sum4.w += x.w * share[w];
                    }
                    sum4 = make_float4(sum4.x * inverse, sum4.y * inverse, sum4.z * inverse, sum4.w * inverse);
                    if (whole) {
                        *reinterpret_cast<uint2*>(p.out + out_row + column) = make_uint2(sm100::pack_bf16x2(sum4.x, sum4.y), sm100::pack_bf16x2(sum4.z, sum4.w));
                    } else {
                        *reinterpret_cast<float4*>(p.part_out + (static_cast<size_t>(slot) * S::ROWS + row) * HEAD + column) = sum4;
                    }
                }
            }
        }
        first_segment = false;
    }
}

// Joins the parts of the items that several CTAs worked on, in the order of their keys, and writes the rows of entries without any key.  SHARE
// warps take a row, a lane four of its columns; each warp joins a run of the row's parts, four (eight) of them on the way at once, and the
// first one joins the runs.  One warp to a row joined the 58 parts of 2 x 8 rows over 7354 keys (two kernels) in 15.4 us, four
// join them in 7.6.
template <int SHARE>
__global__ void __launch_bounds__(THREADS) flash_decode_combine_kernel(const __grid_constant__ DecodeParams p, int block_rows) {
    static_assert(SHARE == 1 || SHARE == WARPS, "a warp or a CTA to a row");
    __shared__ float4 run_value[SHARE > 1 ? WARPS : 1][32];
    __shared__ float2 run_sum[WARPS];                               // reference (log2 domain) and sum of a warp's run
    const int rows = p.group * p.tokens;
    const int warp = threadIdx.x / 32;
    const int index = SHARE == 1 ? blockIdx.x * WARPS + warp : blockIdx.x;      // kv_head * rows + row
    const int lane = threadIdx.x % 32;
    const int entry = blockIdx.y;
    if (index >= p.kv_heads * rows) {
        return;
    }
    const int kv_head = index / rows;
    const int row = index - kv_head * rows;
    const int block = row / block_rows;
    sm100::grid_dependency_wait();
    const int length = length_of(p, entry);
    const PartNote note = p.notes[(static_cast<size_t>(entry) * p.kv_heads + kv_head) * p.row_blocks + block];
    uint2* out = reinterpret_cast<uint2*>(p.out + row_offset(p, entry, kv_head, row)) + lane;
    float* lse = p.lse + lse_offset(p, entry, kv_head, row);
    if (length == 0) {
        if (SHARE == 1 || warp == 0) {
            *out = make_uint2(0, 0);
            if (lane == 0) {
                *lse = -INFINITY;
            }
        }
        return;
    }
    const int count = note.count_slot / 2;
    if (count <= 1) {
        return;                         // written by the CTA that saw all of it
    }
    const int inside = row - block * block_rows;
    auto slot_row = [&](int part) {
        return static_cast<size_t>(2 * (note.first + part) + (part == 0 ? note.count_slot % 2 : 0)) * block_rows + inside;
    };
    // one pass, some parts at a time: their logarithms and columns are on the way together
    constexpr int AT_ONCE = SHARE == 1 ? 4 : 8;
    const int begin = SHARE == 1 ? 0 : count * warp / SHARE, end = SHARE == 1 ? count : count * (warp + 1) / SHARE;
    float top = -INFINITY, sum = 0.0F;
    float4 value = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
    for (int base = begin; base < end; base += AT_ONCE) {
        float lse2[AT_ONCE];
        float4 x[AT_ONCE];
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const size_t at = slot_row(min(base + n, end - 1));
            lse2[n] = p.part_lse[at];
            x[n] = *reinterpret_cast<const float4*>(p.part_out + at * HEAD + lane * 4);
        }
        float now = top;
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            lse2[n] = base + n < end ? lse2[n] : -INFINITY;
            now = fmaxf(now, lse2[n]);
        }
        const float reference = now == -INFINITY ? 0.0F : now;
        const float shrink = exp2_approx(top - reference);
        sum *= shrink;
        value = make_float4(value.x * shrink, value.y * shrink, value.z * shrink, value.w * shrink);
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const float weight = exp2_approx(lse2[n] - reference);
            sum += weight;
            value = make_float4(fmaf(weight, x[n].x, value.x), fmaf(weight, x[n].y, value.y), fmaf(weight, x[n].z, value.z), fmaf(weight, x[n].w, value.w));
        }
        top = now;
    }
    if constexpr (SHARE > 1) {
        run_value[warp][lane] = value;
        if (lane == 0) {
            run_sum[warp] = make_float2(top, sum);
        }
        __syncthreads();
        if (warp != 0) {
            return;
        }
        float now = -INFINITY;
#pragma unroll
        for (int w = 0; w < SHARE; ++w) {
            now = fmaxf(now, run_sum[w].x);
        }
        const float reference = now == -INFINITY ? 0.0F : now;
        sum = 0.0F;
        value = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
        for (int w = 0; w < SHARE; ++w) {
            const float weight = exp2_approx(run_sum[w].x - reference);
            const float4 x = run_value[w][lane];
            sum = fmaf(weight, run_sum[w].y, sum);
            value = make_float4(fmaf(weight, x.x, value.x), fmaf(weight, x.y, value.y), fmaf(weight, x.z, value.z), fmaf(weight, x.w, value.w));
        }
        top = now;
    }
    const float inverse = sum == 0.0F ? 0.0F : 1.0F / sum;
    *out = make_uint2(sm100::pack_bf16x2(value.x * inverse, value.y * inverse), sm100::pack_bf16x2(value.z * inverse, value.w * inverse));
    if (lane == 0) {
        *lse = sum == 0.0F ? -INFINITY : (top + log2f(sum)) * LN2;
    }
}

// Whether every item stays whole, with a CTA of its own and no second kernel: up to so many keys the time of the longest item is below that of the parts and
// their joining.  us, parts and whole, lengths down to a third or less: 8 items of up to 128 keys 6.5 and 4.4, 384 7.3 and 6.3, 512 7.3 and 7.1, 700 7.4 and 8.1 (16 rows: 384 8.8 and
// 8.1, 512 8.7 and 9.5); 32 items of up to 400 keys 9.4 and 6.8, 640 8.7 and 8.0; 64 of 900 10.3 and 10.4; 128 of 512
// 10.8 and 8.2, 768 12.5 and 10.0, bf16 states of 1000 13.0 and 13.6; 200 of 1000 15.0 and 14.0, 1500 16.6 and 16.4, 2000 18.3 and 21.4; 512 of 512 17.8 and 15.7, 800
// 19.6 and 19.3, 1200 25.6 and 27.1.  More items bear longer ones, as the parts' CTAs have several each to go over; from more items than CTAs run at once on, whole items
// need a second wave.  The longest is what the caller's table or tensor holds: lengths are not known here, so a wide table over short sequences takes the parts.
bool stays_whole(long long items, int keys_most, int at_once) {
    return keys_most <= (items > at_once ? 768 : items >= 200 ? 1280 : items >= 96 ? 896 : items >= 32 ? 704 : 384);
}

// Rows up to which each has a CTA of the joining kernel.  Both kernels with a warp and a CTA to a row: 8 rows over 40000 keys 52.3 and 15.8 us, 128 over
// 3000 12.6 and 10.2, 1024 over 5000 21.8 and 22.1, 2048 over 600 14.8 and 16.8.
constexpr long long WIDE_COMBINE_ROWS = 512;

// Blocks of 8 query rows that an item has.
int blocks_of_rows(long long rows) {
    return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}

template <int SOURCE, int NB>
void launch_decode(DecodeParams& p, cudaStream_t stream) {
    using S = Shape<SOURCE, NB>;
    const int rows = p.group * p.tokens;
    if (p.group > 4096) {
        throw std::invalid_argument("flash attention over few rows takes at most 4096 query heads to a key head");
    }
    p.group_inverse = p.group == 1 ? 0 : static_cast<unsigned>(((1ULL << 32) + p.group - 1) / p.group);
    p.row_blocks = (rows + S::ROWS - 1) / S::ROWS;
    const long long most = static_cast<long long>((p.keys_most + S::TILE - 1) / S::TILE + ITEM_TILES) * p.batch * p.kv_heads * p.row_blocks;
    if (most > 0x7fffffffLL) {
        throw std::invalid_argument("flash attention over few rows: the shape exceeds the supported index range");
    }
    static bool done[16] = {};
    int device = 0;
    CUDA_CHECK(cudaGetDevice(&device));
    if (device >= 16 || !done[device]) {
        CUDA_CHECK(cudaFuncSetAttribute(flash_decode_kernel<SOURCE, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
        if (device < 16) {
            done[device] = true;
        }
    }
    const long long items = static_cast<long long>(p.batch) * p.kv_heads * p.row_blocks;
    p.whole = stays_whole(items, p.keys_most, 148 * S::CTAS_PER_SM);
    if (p.whole != 0) {
        launch_chained(flash_decode_kernel<SOURCE, NB>, dim3(static_cast<unsigned>(items)), dim3(THREADS), S::BYTES, stream, p);
        return;
    }
    const int ctas = static_cast<int>(std::min<long long>(148LL * S::CTAS_PER_SM, most));
    p.part_lse = p.part_out + static_cast<size_t>(2 * MOST_CTAS) * S::ROWS * HEAD;
    p.notes = reinterpret_cast<PartNote*>(p.part_lse + static_cast<size_t>(2 * MOST_CTAS) * S::ROWS);
    launch_chained(flash_decode_kernel<SOURCE, NB>, dim3(ctas), dim3(THREADS), S::BYTES, stream, p);
    if (static_cast<long long>(p.kv_heads) * rows * p.batch <= WIDE_COMBINE_ROWS) {
        launch_chained(flash_decode_combine_kernel<WARPS>, dim3(p.kv_heads * rows, p.batch), dim3(THREADS), 0, stream, p, S::ROWS);
    } else {
        launch_chained(flash_decode_combine_kernel<1>, dim3((p.kv_heads * rows + WARPS - 1) / WARPS, p.batch), dim3(THREADS), 0, stream, p, S::ROWS);
    }
}

template <int SOURCE>
void launch_rows(DecodeParams& p, cudaStream_t stream) {
    switch (blocks_of_rows(static_cast<long long>(p.group) * p.tokens)) {
        case 1:
            return launch_decode<SOURCE, 1>(p, stream);
        case 2:
            return launch_decode<SOURCE, 2>(p, stream);
        default:
            return launch_decode<SOURCE, 4>(p, stream);
    }
}

}  // namespace

namespace internal {

std::size_t few_rows_workspace_bytes(int batch, int key_value_heads, long long rows) {
    const std::size_t block = 8 * static_cast<std::size_t>(blocks_of_rows(rows));
    const std::size_t items = static_cast<std::size_t>(batch) * key_value_heads * ((rows + block - 1) / block);
    return 2 * MOST_CTAS * block * (HEAD + 1) * sizeof(float) + items * sizeof(PartNote);
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

std::size_t flash_decode_workspace_bytes(int batch_size, int tokens, int query_heads, int key_value_heads) {
    if (batch_size <= 0 || tokens <= 0 || query_heads <= 0 || key_value_heads <= 0) {
        return 0;
    }
    return internal::few_rows_workspace_bytes(batch_size, key_value_heads, static_cast<long long>(tokens) * (query_heads / key_value_heads));
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
    if (workspace_bytes < flash_decode_workspace_bytes(batch_size, tokens, query_heads, key_value_heads)) {
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
