// Cross attention forward (D = 128, grouped-query) on tcgen05: the queries of a decoder over an encoder's states, each entry with its own
// number of valid keys, no causal mask.
//
// Rows.  All query heads of a key head see the same keys, so their queries are the rows of one matrix, row = token * group + head: a TMA box
// of {64 columns, group heads, tokens} lays them out that way (a group that does not divide 128 leaves the last rows of a tile
// unused).  Short queries fill their tiles and a key tile is fetched once for a whole group.
//
// A CTA takes one 128-row tile of one (entry, key head): S = Q K^T into tensor memory, online softmax with one thread to a row, P back into tensor memory
// as bf16 (P aliases S) and O += P V.  It holds half of an SM's tensor memory, shared memory and registers, so that two CTAs share an SM: one's softmax runs
// beside the other's products, and one's beginning and end beside the other's loop.  (A CTA of two alternating tiles, which fetches K and V
// once for both, took the same 398 us for the longest case, 4 x 2048 tokens of 32 heads over 2048-4096 keys, but 48.5 for 36.5 on 64 tokens over 1500 keys with 256
// heads, 29.5 for 22.5 on 584 tokens over 12 keys, 82 for 73 on 835 x 7 rows over 982 ragged keys.)  K and V stream through one tile's place, four chunks of 16 KB: a
// chunk's successor is on its way as soon as the products that read it are done.
//
// Warps 0-3 are the softmax, warp 4 issues the MMAs, warp 5 the loads; warps 6 and 7 clear the value rows behind an entry's length (a weight of zero
// does not keep their NaN out of P V).  The second warpgroup hands registers to the softmax, which holds a row of scores.  Two CTAs to an SM leave the compiler 128
// registers at launch, and it spills 132 bytes of a thread's state around the scores.
//
// Small problems: where the tiles would leave SMs idle the loop over the keys is cut into parts for the CTAs of a cluster, which join their fp32 sums
// through distributed shared memory (loop_parts.cuh).
//
// Few rows to a key head (single tokens) go to flash_decode.cu instead, which splits the keys over the SMs.
//
// P is rounded to bf16 (half a step is 2^-8 of each weight); sums, maxima and O are fp32.  Every wait is bounded.
#include "flash_attention.h"
#include "cuda_common.h"
#include "attention_internal.h"
#include "sm100_primitives.cuh"
#include "loop_parts.cuh"
#include "../common/launch.h"
#include "../common/tensor_map.h"

#include <stdexcept>

namespace dscuda {
namespace {

using namespace sm100;

constexpr int HEAD = 128;
constexpr int TILE = 128;                   // rows of a query tile, keys of a key tile
constexpr int CHUNK = 128 * 128;            // 16 KB: 128 rows x 64 bf16, or 64 keys x 128
constexpr int CHUNKS = 4;                   // of a key tile: two of K, two of V
constexpr int Q_BYTES = 2 * CHUNK;
constexpr int MISC_BYTES = 2048;
constexpr int SMEM_BYTES = Q_BYTES + CHUNKS * CHUNK + MISC_BYTES + 1024;
constexpr int THREADS = 256;
constexpr int MMA_WARP = 4;
constexpr int LOAD_WARP = 5;
constexpr int TAIL_WARP = 6;
constexpr int TMEM_COLUMNS = 256;           // S | O
constexpr float RESCALE_THRESHOLD = 8.0F;   // log2 units; below it the old row maximum is kept
constexpr float LOG2E = 1.4426950408889634F;
constexpr float LN2 = 0.6931471805599453F;

__device__ int cross_forward_status = 0;

struct CrossForwardParams {
    CUtensorMap q;              // group rows, box {64, group, tokens of a tile}
    CUtensorMap k;              // [B][Tk][Hkv * 128], boxes of 128 rows
    CUtensorMap v;              // boxes of 64 rows
    CUtensorMap out;            // like q
    float* lse;                 // [B, Hq, Tq]
    const int* lengths;         // null: Tk
    __nv_bfloat16* output;      // [B, Tq, Hq, 128]
    int tokens, keys, heads, group;
    int tile_tokens;            // tokens of a query tile
    int parts;                  // CTAs (a cluster) that share the keys of a query tile
    float scale, scale_log2;
};

struct Barriers {
    uint64_t q_full;
    uint64_t s_full;
    uint64_t p_full;
    uint64_t p_half;
    uint64_t staged;            // the output rows are in shared memory
    uint64_t full[CHUNKS];
    uint64_t empty[CHUNKS];
    uint64_t tail_full[2];      // the last tile's value chunks, before the rows behind the length are cleared
    uint32_t tmem_base;
    int abort_flag;
    int gave_up;
    float2 row_sums[TILE];      // parts: reference (log2 domain) and sum of each row
};
static_assert(sizeof(Barriers) <= MISC_BYTES, "barrier block too large");

__global__ void __launch_bounds__(THREADS, 2) cross_forward_kernel(const __grid_constant__ CrossForwardParams p) {
    extern __shared__ uint8_t smem_raw[];
    const int entry = blockIdx.z;
    const int kv_head = blockIdx.y;
    const int part = blockIdx.x % p.parts;              // also the rank in the cluster
    const int token0 = blockIdx.x / p.parts * p.tile_tokens;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023U) & ~1023U;
    uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t tile_smem = smem_base + Q_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(smem + Q_BYTES + CHUNKS * CHUNK);
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&bars->q_full), 1);
        mbar_init(smem_u32(&bars->s_full), 1);
        mbar_init(smem_u32(&bars->p_full), TILE);
        mbar_init(smem_u32(&bars->p_half), TILE);
        mbar_init(smem_u32(&bars->staged), TILE);
        mbar_init(smem_u32(&bars->tail_full[0]), 1);
        mbar_init(smem_u32(&bars->tail_full[1]), 1);
        for (int i = 0; i < CHUNKS; ++i) {
            mbar_init(smem_u32(&bars->full[i]), 1);
            mbar_init(smem_u32(&bars->empty[i]), 1);
        }
        bars->abort_flag = 0;
        // after an earlier launch ran into a time limit nothing is done; the CTAs of a cluster stay to the end all the same
        bars->gave_up = *reinterpret_cast<volatile int*>(&cross_forward_status);
        mbar_init_fence();
    }
    if (warp == MMA_WARP) {
        tmem_alloc(smem_u32(&bars->tmem_base), TMEM_COLUMNS);
        tmem_relinquish();
    }
    if (warp == LOAD_WARP && lane == 0) {
        tma_prefetch_descriptor(&p.q);
        tma_prefetch_descriptor(&p.k);
        tma_prefetch_descriptor(&p.v);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    grid_dependency_wait();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    const int length = p.lengths == nullptr ? p.keys : min(max(p.lengths[entry], 0), p.keys);
    const int all_tiles = (length + TILE - 1) / TILE;
    const int first_tile = part_begin(all_tiles, part, p.parts);
    const bool dead = *reinterpret_cast<volatile int*>(&bars->gave_up) != 0;
    const int tile_count = dead ? 0 : part_begin(all_tiles, part + 1, p.parts) - first_tile;
    const int left = length - first_tile * TILE;        // keys from the first tile on
    // what lies between the length and the end of the entry's states may be anything; behind that end the loads give zeros
    const int tail_keys = length < p.keys ? min(left - (tile_count - 1) * TILE, TILE) : TILE;

    constexpr int REG_LO = 48;
    constexpr int REG_HI = 208;
    static_assert(4 * REG_HI + 4 * REG_LO <= 8 * 128, "register redistribution exceeds the CTA's allocation");
    if (warp >= 4) {
        reg_dealloc<REG_LO>();
        if (warp >= TAIL_WARP) {
            if (tail_keys < TILE && tile_count > 0) {
                const int half = warp - TAIL_WARP;
                if (__all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->tail_full[half]), 0, abort_flag, &cross_forward_status))) {
                    uint8_t* chunk = smem + Q_BYTES + (2 + half) * CHUNK;
                    const int first = min(max(tail_keys - half * 64, 0), 64);
                    clear_rows(chunk, first, 64, lane);
                    clear_rows(chunk + CHUNK / 2, first, 64, lane);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(smem_u32(&bars->full[2 + half]));
                    }
                }
            }
        } else if (warp == LOAD_WARP) {
            if (lane == 0 && tile_count > 0) {
                const uint32_t q_bar = smem_u32(&bars->q_full);
                mbar_arrive_expect_tx(q_bar, 2 * p.group * p.tile_tokens * 128);
                for (int c = 0; c < 2; ++c) {
                    tma_load_4d(smem_base + c * CHUNK, &p.q, q_bar, c * 64, kv_head * p.group, token0, entry);
                }
                bool alive = true;
#pragma unroll 1
                for (int j = 0; j < tile_count && alive; ++j) {
                    const int key = (first_tile + j) * TILE;
                    const bool tail = tail_keys < TILE && j + 1 == tile_count;
#pragma unroll 1
                    for (int c = 0; c < CHUNKS && alive; ++c) {
                        if (j > 0 && !mbar_wait(smem_u32(&bars->empty[c]), (j - 1) & 1, abort_flag, &cross_forward_status)) {
                            alive = false;
                            break;
                        }
                        const uint32_t dst = tile_smem + c * CHUNK;
                        const uint32_t bar = smem_u32(tail && c >= 2 ? &bars->tail_full[c - 2] : &bars->full[c]);
                        mbar_arrive_expect_tx(bar, CHUNK);
                        if (c < 2) {
                            tma_load_3d(dst, &p.k, bar, kv_head * HEAD + c * 64, key, entry);
                        } else {
                            tma_load_3d(dst, &p.v, bar, kv_head * HEAD, key + (c - 2) * 64, entry);
                            tma_load_3d(dst + CHUNK / 2, &p.v, bar, kv_head * HEAD + 64, key + (c - 2) * 64, entry);
                        }
                    }
                }
            }
        } else if (tile_count > 0) {
            // ---- MMA: the whole warp runs the loop, the elected lane executes the instructions ----
            const uint32_t leader = elect_one();
            constexpr uint32_t IDESC_QK = make_idesc_bf16(TILE, TILE, false, false);
            constexpr uint32_t IDESC_PV = make_idesc_bf16(TILE, HEAD, false, true);
            auto wait = [&](uint64_t* barrier, int parity) {
                return __all_sync(0xffffffffU, mbar_wait(smem_u32(barrier), parity, abort_flag, &cross_forward_status)) != 0;
            };
            auto issue_qk = [&](int j) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (!wait(&bars->full[c], j & 1)) {
                        return false;
                    }
                    tc_fence_after_sync();
                    const uint32_t q_chunk = smem_base + c * CHUNK, k_chunk = tile_smem + c * CHUNK;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ss_elect(tmem_base, make_kmajor_desc(q_chunk + k * 32), make_kmajor_desc(k_chunk + k * 32), IDESC_QK,
                                     (c | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->s_full), leader);
                mma_commit_elect(smem_u32(&bars->empty[0]), leader);
                mma_commit_elect(smem_u32(&bars->empty[1]), leader);
                return true;
            };
            auto issue_pv = [&](int j) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!wait(&bars->full[2 + half], j & 1) || !wait(half == 0 ? &bars->p_half : &bars->p_full, j & 1)) {
                        return false;
                    }
                    tc_fence_after_sync();
                    const uint32_t v_chunk = tile_smem + (2 + half) * CHUNK;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ts_elect(tmem_base + TILE, tmem_base + half * 32 + k * 8, make_smem_desc(v_chunk + k * 2048, CHUNK / 2, 1024), IDESC_PV,
                                     (j | half | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->empty[2]), leader);
                mma_commit_elect(smem_u32(&bars->empty[3]), leader);
                return true;
            };
            bool alive = wait(&bars->q_full, 0) && issue_qk(0);
            for (int j = 0; j < tile_count && alive; ++j) {
                alive = issue_pv(j);
                if (alive && j + 1 < tile_count) {
                    alive = issue_qk(j + 1);
                }
            }
            if (alive) {
                mma_commit_elect(smem_u32(&bars->s_full), leader);      // O is final
            }
        }
    } else {
        // ---- softmax and output: a thread to a row ----
        reg_alloc<REG_HI>();
        const int r = threadIdx.x % TILE;
        const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base;
        const uint32_t o_tmem = tmem_base + lane_base + TILE;
        const int token = token0 + r / p.group;
        const bool valid = r < p.tile_tokens * p.group && token < p.tokens;
        float* lse = p.lse + (static_cast<size_t>(entry) * p.heads + kv_head * p.group + r % p.group) * p.tokens + token;
        float m_ref = 0.0F;
        float l_sum = 0.0F;
        bool alive = true;

        for (int j = 0; j < tile_count; ++j) {
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->s_full), j & 1, abort_flag, &cross_forward_status));
            if (!alive) {
                break;
            }
            tc_fence_after_sync();
            uint32_t sb[TILE];
#pragma unroll
            for (int c = 0; c < TILE / 32; ++c) {
                tmem_ld_x32(s_tmem + c * 32, sb + c * 32);
            }
            tmem_wait_ld();
            if (j == tile_count - 1) {
                const int present = left - j * TILE;
#pragma unroll
                for (int n = 0; n < TILE; ++n) {
                    sb[n] = n < present ? sb[n] : 0xff800000U;
                }
            }
            float mx0 = __uint_as_float(sb[0]), mx1 = __uint_as_float(sb[1]), mx2 = __uint_as_float(sb[2]), mx3 = __uint_as_float(sb[3]);
#pragma unroll
            for (int n = 4; n + 7 < TILE; n += 8) {
                mx0 = max3(mx0, __uint_as_float(sb[n]), __uint_as_float(sb[n + 1]));
                mx1 = max3(mx1, __uint_as_float(sb[n + 2]), __uint_as_float(sb[n + 3]));
                mx2 = max3(mx2, __uint_as_float(sb[n + 4]), __uint_as_float(sb[n + 5]));
                mx3 = max3(mx3, __uint_as_float(sb[n + 6]), __uint_as_float(sb[n + 7]));
            }
            mx0 = max3(mx0, __uint_as_float(sb[TILE - 4]), __uint_as_float(sb[TILE - 3]));
            mx1 = max3(mx1, __uint_as_float(sb[TILE - 2]), __uint_as_float(sb[TILE - 1]));
            const float tile_max = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
            if (j == 0) {
                m_ref = tile_max;
            } else {
                const bool grow = (tile_max - m_ref) * p.scale_log2 > RESCALE_THRESHOLD;
                if (__any_sync(0xffffffffU, grow)) {
                    float alpha = 1.0F;
                    if (grow) {
                        alpha = exp2_approx((m_ref - tile_max) * p.scale_log2);
                        m_ref = tile_max;
                        l_sum *= alpha;
                    }
                    // S(j) complete implies P(j-1) V complete: O is quiescent here
#pragma unroll
                    for (int c = 0; c < HEAD / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld_x32(o_tmem + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        }
                        tmem_st_x32(o_tmem + c * 32, o);
                    }
                }
            }
            const float bias = -m_ref * p.scale_log2;
            float2 sums = make_float2(0.0F, 0.0F);
            const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
            const float2 bias2 = make_float2(bias, bias);
#pragma unroll
            for (int c = 0; c < TILE / 32; ++c) {
                uint32_t packed[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float2 x = fma2(make_float2(__uint_as_float(sb[c * 32 + 2 * e]), __uint_as_float(sb[c * 32 + 2 * e + 1])), scale2, bias2);
                    const float2 pr = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                    sums = add2(sums, pr);
                    packed[e] = pack_bf16x2(pr.x, pr.y);
                }
                tmem_st_x16(s_tmem + c * 16, packed);
                if (c == 1) {
                    tmem_wait_st();
                    tc_fence_before_sync();
                    mbar_arrive(smem_u32(&bars->p_half));
                }
            }
            l_sum += sums.x + sums.y;
            tmem_wait_st();
            tc_fence_before_sync();
            mbar_arrive(smem_u32(&bars->p_full));
        }
        if (alive && tile_count > 0) {
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->s_full), tile_count & 1, abort_flag, &cross_forward_status));
        }
        if (alive && !dead && p.parts > 1) {
            // the part's sums into the place of K and V, which is idle by now
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < HEAD / 32 && tile_count > 0; ++c) {
                uint32_t o[32];
                tmem_ld_x32(o_tmem + c * 32, o);
                tmem_wait_ld();
                result_store32(smem + Q_BYTES, r, c * 32, o);
            }
            bars->row_sums[r] = tile_count > 0 ? make_float2(m_ref * p.scale_log2, l_sum) : make_float2(-INFINITY, 0.0F);
        } else if (alive && !dead) {
            // rows of 64 columns into Q's chunks (idle by now), from where a TMA store takes them
            tc_fence_after_sync();
            const float inverse = tile_count > 0 ? 1.0F / l_sum : 0.0F;
#pragma unroll
            for (int c = 0; c < HEAD / 32; ++c) {
                uint32_t o[32];
                if (tile_count > 0) {
                    tmem_ld_x32(o_tmem + c * 32, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        o[e] = 0;
                    }
                }
                uint8_t* row = smem + c / 2 * CHUNK + r * 128;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint4 vec;
                    vec.x = pack_bf16x2(__uint_as_float(o[8 * u]) * inverse, __uint_as_float(o[8 * u + 1]) * inverse);
                    vec.y = pack_bf16x2(__uint_as_float(o[8 * u + 2]) * inverse, __uint_as_float(o[8 * u + 3]) * inverse);
                    vec.z = pack_bf16x2(__uint_as_float(o[8 * u + 4]) * inverse, __uint_as_float(o[8 * u + 5]) * inverse);
                    vec.w = pack_bf16x2(__uint_as_float(o[8 * u + 6]) * inverse, __uint_as_float(o[8 * u + 7]) * inverse);
                    *reinterpret_cast<uint4*>(row + ((((c % 2) * 4 + u) ^ (r & 7)) * 16)) = vec;
                }
            }
            if (valid) {
                *lse = tile_count > 0 ? m_ref * p.scale + logf(l_sum) : -INFINITY;
            }
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&bars->staged));
            if (r == 0 && mbar_wait(smem_u32(&bars->staged), 0, abort_flag, &cross_forward_status)) {
                for (int c = 0; c < 2; ++c) {
                    tma_store_4d(&p.out, smem_base + c * CHUNK, c * 64, kv_head * p.group, token0, entry);
                }
                tma_store_commit();
                tma_store_wait_read();
            }
        }
    }

    // ---- parts: each CTA its share of the rows ----
    if (p.parts > 1) {
        __syncwarp();
        cluster_sync_all();
        const int rows = min(p.tile_tokens, p.tokens - token0) * p.group;
        const int row_end = dead ? 0 : part_begin(rows, part + 1, p.parts);
        constexpr int WARPS = THREADS / 32;
        for (int first = part_begin(rows, part, p.parts) + warp; first < row_end; first += SUM_ROWS * WARPS) {
            // lane 8 k + n: reference and sum of part n (of at most 8) for the warp's k-th row
            float2 sums = make_float2(-INFINITY, 0.0F);
            const int mine = first + lane / 8 * WARPS;
            if (lane % 8 < p.parts && lane / 8 < SUM_ROWS && mine < row_end) {
                sums = cluster_load2(map_to_cta(smem_u32(&bars->row_sums[mine]), lane % 8));
            }
            float top = sums.x;
#pragma unroll
            for (int offset = 4; offset > 0; offset >>= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffU, top, offset));
            }
            const float reference = top == -INFINITY ? 0.0F : top;
            float weight = exp2_approx(sums.x - reference);
            float total = weight * sums.y;
#pragma unroll
            for (int offset = 4; offset > 0; offset >>= 1) {
                total += __shfl_xor_sync(0xffffffffU, total, offset);
            }
            weight = total == 0.0F ? 0.0F : weight / total;
            float4 value[SUM_ROWS];
            cluster_sums(value, tile_smem, lane, parts_without(all_tiles, p.parts), p.parts, first, WARPS, row_end,
                         [&](int k, int other) { return __shfl_sync(0xffffffffU, weight, 8 * k + other); });
#pragma unroll
            for (int k = 0; k < SUM_ROWS; ++k) {
                const int row = first + k * WARPS;
                if (row < row_end) {
                    const int token = token0 + row / p.group;
                    const int head = kv_head * p.group + row % p.group;
                    reinterpret_cast<uint2*>(p.output + ((static_cast<size_t>(entry) * p.tokens + token) * p.heads + head) * HEAD)[lane] =
                        make_uint2(pack_bf16x2(value[k].x, value[k].y), pack_bf16x2(value[k].z, value[k].w));
                    if (lane == 8 * k) {
                        p.lse[(static_cast<size_t>(entry) * p.heads + head) * p.tokens + token] = total == 0.0F ? -INFINITY : reference * LN2 + logf(total);
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync_all();             // nobody leaves while others read
    }

    // ---- teardown: every path reaches this point ----
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag != 0) {
        for (int k = 0; k < 64; ++k) {
            __nanosleep(1000);
        }
    }
    if (warp == MMA_WARP) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, TMEM_COLUMNS);
    }
}


// Microseconds of a key tile in a CTA that has an SM to itself and in one of two that share it, and what a cluster costs beside its tiles (more when two of them
// share their SMs): 3000 keys under 160 rows 44.2 us whole, 29.4, 22.3, 16.5, 13.9 in 2, 4, 6, 8 parts; 637 keys 10.2 whole, 11.3 in 5.
constexpr double TILE_US = 1.7;
constexpr double PAIR_US = 2.36;
constexpr double JOIN_US = 7.0;
constexpr double PAIR_JOIN_US = 10.0;

// Parts that the loop over `tiles` key tiles is cut into for `ctas` query tiles.
int key_parts(long long ctas, long long tiles, const ClusterCounts& counts) {
    const long long rest = ctas % (2 * SMS);
    double best_us = static_cast<double>(tiles) * (static_cast<double>(ctas / (2 * SMS)) * PAIR_US + (rest == 0 ? 0.0 : rest <= SMS ? TILE_US : PAIR_US));
    int best = 1;
    for (int parts = 2; parts <= 8 && parts <= tiles; ++parts) {
        if (ctas > 2LL * counts.of[parts]) {            // (the device counts one CTA to an SM)
            break;
        }
        const bool alone = ctas <= counts.of[parts];
        const double us = static_cast<double>((tiles + parts - 1) / parts) * (alone ? TILE_US : PAIR_US) + (alone ? JOIN_US : PAIR_JOIN_US);
        if (us < best_us) {
            best = parts;
            best_us = us;
        }
    }
    return best;
}

const ClusterCounts& configure() {
    static PerDevice<ClusterCounts> devices;
    return devices.get([] {
        CUDA_CHECK(cudaFuncSetAttribute(cross_forward_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        return cluster_counts(cross_forward_kernel, THREADS, SMEM_BYTES, 8);
    });
}

// Rows to a key head up to which flash_decode.cu's kernels take the call.
constexpr long long FEW_ROWS = 32;

}  // namespace

namespace internal {

void check_flash_cross_shape(int batch_size, int query_length, int key_length, int query_heads, int key_value_heads, int head_size, float scale) {
    if (head_size != HEAD) {
        throw std::invalid_argument("flash cross attention requires head_size 128");
    }
    if (batch_size <= 0 || query_length <= 0 || key_length <= 0) {
        throw std::invalid_argument("flash cross attention requires positive batch and lengths");
    }
    if (query_heads <= 0 || key_value_heads <= 0 || query_heads % key_value_heads != 0) {
        throw std::invalid_argument("flash cross attention requires query_heads to be divisible by key_value_heads");
    }
    if (query_heads / key_value_heads > 64) {
        throw std::invalid_argument("flash cross attention takes at most 64 query heads to a key head");
    }
    if (!(scale > 0.0F)) {
        throw std::invalid_argument("flash cross attention requires a positive softmax scale");
    }
    if (static_cast<long long>(batch_size) * query_length > 0x7fffffffLL || static_cast<long long>(batch_size) * key_length > 0x7fffffffLL ||
        query_length > (1 << 30) || key_length > (1 << 30) || static_cast<long long>(query_length) * query_heads > 0x7fffffffLL ||
        query_heads > 65535 || batch_size > 65535) {
        throw std::invalid_argument("flash cross attention shape exceeds the supported index range");
    }
}

int cross_forward_device_status(bool reset) {
    int status = 0;
    CUDA_CHECK(cudaDeviceSynchronize());
    CUDA_CHECK(cudaMemcpyFromSymbol(&status, cross_forward_status, sizeof(int)));
    if (reset && status != 0) {
        const int zero = 0;
        CUDA_CHECK(cudaMemcpyToSymbol(cross_forward_status, &zero, sizeof(int)));
    }
    return status;
}

}  // namespace internal

std::size_t flash_cross_forward_workspace_bytes(int batch_size, int query_length, int key_length, int query_heads, int key_value_heads) {
    if (batch_size <= 0 || query_length <= 0 || key_length <= 0 || query_heads <= 0 || key_value_heads <= 0) {
        return 0;
    }
    const long long rows = static_cast<long long>(query_length) * (query_heads / key_value_heads);
    return rows <= FEW_ROWS ? internal::few_rows_workspace_bytes(batch_size, key_value_heads, rows) : 0;
}

void flash_cross_forward_cuda(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* query, const __nv_bfloat16* key,
                              const __nv_bfloat16* value, const int* key_lengths, void* workspace, std::size_t workspace_bytes, int batch_size,
                              int query_length, int key_length, int query_heads, int key_value_heads, int head_size, float scale,
                              cudaStream_t stream) {
    internal::check_flash_cross_shape(batch_size, query_length, key_length, query_heads, key_value_heads, head_size, scale);
    internal::check_flash_pointers({output, query, key, value}, {logsumexp});
    if (key_lengths != nullptr) {
        internal::check_flash_pointers({}, {key_lengths});
    }
    const std::size_t needed = flash_cross_forward_workspace_bytes(batch_size, query_length, key_length, query_heads, key_value_heads);
    if (needed > 0) {
        internal::check_flash_pointers({workspace}, {});
        if (workspace_bytes < needed) {
            throw std::invalid_argument("flash cross attention workspace is too small");
        }
    }
    const int group = query_heads / key_value_heads;
    if (static_cast<long long>(query_length) * group <= FEW_ROWS) {
        internal::launch_few_rows_cross(output, logsumexp, query, key, value, key_lengths, workspace, batch_size, query_length, key_length, query_heads,
                                        key_value_heads, scale, stream);
        return;
    }
    CrossForwardParams p{};
    p.tile_tokens = TILE / group;
    p.q = make_bf16_group_rows_map(query, batch_size, query_length, query_heads, group, p.tile_tokens);
    p.out = make_bf16_group_rows_map(output, batch_size, query_length, query_heads, group, p.tile_tokens);
    p.k = make_bf16_batched_tile_map(key, batch_size, key_length, static_cast<std::uint64_t>(key_value_heads) * HEAD, TILE);
    p.v = make_bf16_batched_tile_map(value, batch_size, key_length, static_cast<std::uint64_t>(key_value_heads) * HEAD, 64);
    p.lse = logsumexp;
    p.lengths = key_lengths;
    p.tokens = query_length;
    p.keys = key_length;
    p.heads = query_heads;
    p.group = group;
    p.scale = scale;
    p.scale_log2 = scale * LOG2E;
    p.output = output;
    const long long row_tiles = (query_length + p.tile_tokens - 1LL) / p.tile_tokens;
    p.parts = key_parts(row_tiles * key_value_heads * batch_size, (key_length + TILE - 1LL) / TILE, configure());
    launch_chained_clusters(cross_forward_kernel, dim3(static_cast<unsigned>(row_tiles) * p.parts, key_value_heads, batch_size), p.parts, dim3(THREADS), SMEM_BYTES,
                            stream, p);
}

}  // namespace dscuda
