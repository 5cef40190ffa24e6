// Gradients of the cross attention (D = 128, grouped-query) on tcgen05.
//
// With rows r = (token, head of the group) of one (entry, key head), P = exp(scale * Q K^T - lse) and dP = dO V^T:
//     delta[r] = sum_d dO[r,d] O[r,d]        dS = P (dP - delta) scale
//     dV = P^T dO        dK = dS^T Q          dQ = dS K
// dK and dV of a key head are sums over all rows of its group, so the heads of a group need no step of their own.
//
// One call launches:
//   1. cross_query_kernel: a CTA keeps 128 rows (Q, dO) and goes over the keys in tiles of 128: S = Q K^T, dP = dO V^T, dQ += dS K.  It forms delta from the
//      O rows first, and leaves lse * log2(e) and delta in row order for the next kernel.  Where a softmax sits on few keys, the rounding of O in delta is the largest error
//      of dS (2 keys: 0.4 % of dQ and dK, against 0.17 % of the last rounding).  Up to 128 keys, one tile, delta = sum_k P dP is formed from the tile itself and free
//      of it; longer entries keep that error, as two passes over the keys would be the price.  One key has no gradient at all (its weight is 1 whatever the score), where P (dP - delta) would leave what two
//      orders of the same sum differ by: dQ leaves as zeros (a step inside the loop cost 1-3 % here), and the key side sets dS to zero.
//   2. cross_key_kernel: a CTA keeps 128 keys (K, V) and goes over the rows in tiles of at most 64: S^T = K Q^T, dP^T = V dO^T, one thread to a
//      key (two, half the rows each), P^T and dS^T back into tensor memory as bf16 A operands, dV += P^T dO, dK += dS^T Q.  Tensor memory: dV 128, dK
//      128, two pairs of 64-column scores, so the scores of the next tile are computed while the softmax works on this one.
// Short loops over many tiles take the forms of cross_query_short.cu and cross_backward_short.cu.
// Where a grid of whole loops would leave SMs idle the loops are cut into parts for the CTAs of a cluster, which add their fp32 sums in order through
// distributed shared memory (loop_parts.cuh).
// S and dP are computed twice (1792 instead of 1280 FLOP per pair).  The alternative of the causal backward, dS stored once and streamed
// back, moves 4 bytes per pair through HBM, 0.62 ps at the measured copy rate, against 0.31 ps for the 512 FLOP at the measured tensor rate.
//
// Every gradient element has one writer and a fixed order of sums: results are the same bits from call to call.  P and dS are rounded to
// bf16 (half a step is 2^-8); everything else is fp32.
//
// Rows that do not exist (a group that does not divide 64, tokens behind the last) carry lse = +inf, which makes their P zero, and zeros for Q and
// dO.  Keys behind an entry's length cost nothing in the key kernel (one thread owns a key, its sums are replaced by zeros at the end); the
// query kernel clears them in shared memory, because dS K multiplies them by zeros.  Every wait is bounded.
#include "flash_attention.h"
#include "cuda_common.h"
#include "attention_internal.h"
#include "sm100_primitives.cuh"
#include "cross_backward.cuh"
#include "loop_parts.cuh"
#include "../common/launch.h"
#include "../common/tensor_map.h"

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <stdexcept>

namespace dscuda {
namespace {

using namespace cross;

constexpr double QUERY_TILE_US = 1.15;      // a key tile of the query kernel's loop
constexpr double KEY_TILE_US = 0.75;        // a row tile of the key kernel's loop
constexpr int MOST_KEY_PARTS = 16;          // few keys under many rows: the backward of 64 keys under 4096 x 3 rows 45 us with 8 parts, 38 with 16

__device__ int cross_backward_status = 0;

// ---------------------------------------------------------------------------
// dK, dV
// ---------------------------------------------------------------------------
namespace keyside {
constexpr int STAGES = 4;
constexpr int STAGE_BYTES = 4 * SUB_CHUNK;          // Q and dO of 64 rows
constexpr int RESIDENT_BYTES = 4 * BIG_CHUNK;       // K and V of 128 keys
constexpr int MISC_BYTES = 2560;
constexpr int SMEM_BYTES = RESIDENT_BYTES + STAGES * STAGE_BYTES + MISC_BYTES + 1024;
constexpr uint32_t TMEM_DV = 0;
constexpr uint32_t TMEM_DK = 128;
constexpr uint32_t TMEM_S = 256;                    // two pairs of S^T and dP^T, 64 columns each

struct Barriers {
    uint64_t resident_full;
    uint64_t stage_full[STAGES];
    uint64_t stage_empty[STAGES];
    uint64_t s_full[2];             // tensor core -> softmax, per score pair
    uint64_t dp_full[2];
    uint64_t p_full[2];             // softmax -> tensor core
    uint64_t ds_full[2];
    uint64_t final_full;
    uint64_t staged[2];             // dV, dK rows are in shared memory
    uint32_t tmem_base;
    int abort_flag;
    int gave_up;
    alignas(16) float lse2[STAGES][SUB];
    alignas(16) float delta[STAGES][SUB];
};
static_assert(sizeof(Barriers) <= MISC_BYTES, "barrier block too large");
static_assert(2 * RESULT_BYTES <= STAGES * STAGE_BYTES, "the parts' sums take the streamed tiles' place");
static_assert(offsetof(Barriers, lse2) % 16 == 0 && offsetof(Barriers, delta) % 16 == 0, "16-byte loads of the per-row constants");
}  // namespace keyside

__global__ void __launch_bounds__(THREADS, 1) cross_key_kernel(const __grid_constant__ CrossBackwardParams p) {
    using namespace keyside;
    extern __shared__ uint8_t smem_raw[];
    const int entry = blockIdx.z;
    const int kv_head = blockIdx.y;
    const int part = blockIdx.x % p.key_parts;          // also the rank in the cluster
    const int key_start = blockIdx.x / p.key_parts * BIG;
    const int rows_per_tile = p.sub_tokens * p.group;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023U) & ~1023U;
    uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t k_smem = smem_base;
    const uint32_t v_smem = smem_base + 2 * BIG_CHUNK;
    const uint32_t stage_smem = smem_base + RESIDENT_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(smem + RESIDENT_BYTES + STAGES * STAGE_BYTES);
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&bars->resident_full), 1);
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(smem_u32(&bars->stage_full[i]), 2);       // the loads and the per-row constants
            mbar_init(smem_u32(&bars->stage_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&bars->s_full[i]), 1);
            mbar_init(smem_u32(&bars->dp_full[i]), 1);
            mbar_init(smem_u32(&bars->p_full[i]), SOFTMAX_THREADS);
            mbar_init(smem_u32(&bars->ds_full[i]), SOFTMAX_THREADS);
            mbar_init(smem_u32(&bars->staged[i]), BIG);
        }
        mbar_init(smem_u32(&bars->final_full), 1);
        bars->abort_flag = 0;
        // after an earlier launch ran into a time limit nothing is done; the CTAs of a cluster stay to the end all the same
        bars->gave_up = *reinterpret_cast<volatile int*>(&cross_backward_status);
        mbar_init_fence();
    }
    if (warp == MMA_WARP) {
        tmem_alloc(smem_u32(&bars->tmem_base), TMEM_COLUMNS);
        tmem_relinquish();
    }
    if (rows_per_tile < SUB && warp < MMA_WARP) {
        // rows that no load fills: dV += P^T dO and dK += dS^T Q multiply them by zeros
        for (int chunk = warp; chunk < STAGES * 4; chunk += MMA_WARP) {
            clear_rows(smem + RESIDENT_BYTES + chunk * SUB_CHUNK, rows_per_tile, SUB, lane);
        }
        fence_proxy_async_smem();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    grid_dependency_wait();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    const int length = length_of(p, entry);
    // keys behind the length have gradients of zero: no tiles for them
    const int all_tiles = (p.tokens + p.sub_tokens - 1) / p.sub_tokens;
    const int first_tile = part_begin(all_tiles, part, p.key_parts);
    const bool dead = *reinterpret_cast<volatile int*>(&bars->gave_up) != 0;
    const int tile_count = key_start < length && !dead ? part_begin(all_tiles, part + 1, p.key_parts) - first_tile : 0;

    if (warp == LOAD_WARP) {
        if (tile_count > 0 && lane == 0) {
            const uint32_t bar = smem_u32(&bars->resident_full);
            mbar_arrive_expect_tx(bar, RESIDENT_BYTES);
            for (int c = 0; c < 2; ++c) {
                tma_load_3d(k_smem + c * BIG_CHUNK, &p.k, bar, kv_head * HEAD + c * 64, key_start, entry);
                tma_load_3d(v_smem + c * BIG_CHUNK, &p.v, bar, kv_head * HEAD + c * 64, key_start, entry);
            }
        }
        const float2* constants = p.rows + (static_cast<size_t>(entry) * p.kv_heads + kv_head) * p.tokens * p.group;
        bool alive = true;
        for (int t = 0; t < tile_count; ++t) {
            const int stage = t % STAGES;
            const int use = t / STAGES;
            if (use > 0) {
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->stage_empty[stage]), (use - 1) & 1, abort_flag, &cross_backward_status));
                if (!alive) {
                    break;
                }
            }
            const int token = (first_tile + t) * p.sub_tokens;
            const uint32_t full = smem_u32(&bars->stage_full[stage]);
            if (lane == 0) {
                mbar_arrive_expect_tx(full, 4 * rows_per_tile * 128);
                const uint32_t dst = stage_smem + stage * STAGE_BYTES;
                for (int c = 0; c < 2; ++c) {
                    tma_load_4d(dst + c * SUB_CHUNK, &p.q_sub, full, c * 64, kv_head * p.group, token, entry);
                    tma_load_4d(dst + (2 + c) * SUB_CHUNK, &p.do_sub, full, c * 64, kv_head * p.group, token, entry);
                }
            }
            const int present = min(rows_per_tile, (p.tokens - token) * p.group);
#pragma unroll
            for (int e = 0; e < SUB / 32; ++e) {
                const int n = e * 32 + lane;
                const float2 both = n < present ? constants[static_cast<size_t>(token) * p.group + n] : make_float2(INFINITY, 0.0F);
                bars->lse2[stage][n] = both.x;
                bars->delta[stage][n] = both.y;
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(full);
            }
        }
    } else if (warp == MMA_WARP) {
        if (tile_count > 0) {
            const uint32_t leader = elect_one();
            constexpr uint32_t IDESC_SCORE = make_idesc_bf16(BIG, SUB, false, false);
            constexpr uint32_t IDESC_GRAD = make_idesc_bf16(BIG, HEAD, false, true);
            bool alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->resident_full), 0, abort_flag, &cross_backward_status));
            // S^T(t) = K Q_t^T and dP^T(t) = V dO_t^T
            auto issue_scores = [&](int t) {
                const int stage = t % STAGES;
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->stage_full[stage]), (t / STAGES) & 1, abort_flag, &cross_backward_status));
                if (!alive) {
                    return;
                }
                tc_fence_after_sync();
                const uint32_t q_smem = stage_smem + stage * STAGE_BYTES;
                const uint32_t scores = tmem_base + TMEM_S + (t & 1) * 128;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ss_elect(scores, make_kmajor_desc(k_smem + c * BIG_CHUNK + k * 32), make_kmajor_desc(q_smem + c * SUB_CHUNK + k * 32), IDESC_SCORE,
                                     (c | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->s_full[t & 1]), leader);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ss_elect(scores + 64, make_kmajor_desc(v_smem + c * BIG_CHUNK + k * 32), make_kmajor_desc(q_smem + (2 + c) * SUB_CHUNK + k * 32),
                                     IDESC_SCORE, (c | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->dp_full[t & 1]), leader);
            };
            if (alive) {
                issue_scores(0);
            }
            for (int t = 0; t < tile_count && alive; ++t) {
                const int stage = t % STAGES;
                const uint32_t parity = (t >> 1) & 1;
                if (t + 1 < tile_count) {
                    issue_scores(t + 1);
                    if (!alive) {
                        break;
                    }
                }
                const uint32_t q_smem = stage_smem + stage * STAGE_BYTES;
                const uint32_t scores = tmem_base + TMEM_S + (t & 1) * 128;
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->p_full[t & 1]), parity, abort_flag, &cross_backward_status));
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                // rows 32 g .. 32 g + 31 are packed into columns 32 g .. 32 g + 15 of their score tile
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    mma_ts_elect(tmem_base + TMEM_DV, scores + (k / 2) * 32 + (k % 2) * 8, make_smem_desc(q_smem + 2 * SUB_CHUNK + k * 2048, SUB_CHUNK, 1024),
                                 IDESC_GRAD, (t | k) != 0 ? 1U : 0U, leader);
                }
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->ds_full[t & 1]), parity, abort_flag, &cross_backward_status));
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    mma_ts_elect(tmem_base + TMEM_DK, scores + 64 + (k / 2) * 32 + (k % 2) * 8, make_smem_desc(q_smem + k * 2048, SUB_CHUNK, 1024), IDESC_GRAD,
                                 (t | k) != 0 ? 1U : 0U, leader);
                }
                mma_commit_elect(smem_u32(&bars->stage_empty[stage]), leader);
            }
            if (alive) {
                mma_commit_elect(smem_u32(&bars->final_full), leader);
            }
        }
    } else {
        const int group = warp / 4;
        const int r = threadIdx.x % BIG;
        const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
        const float ds_scale = length == 1 ? 0.0F : p.scale;       // (the weight of a single key is 1 whatever the score)
        bool alive = true;
        for (int t = 0; t < tile_count; ++t) {
            const int stage = t % STAGES;
            const uint32_t parity = (t >> 1) & 1;
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->stage_full[stage]), (t / STAGES) & 1, abort_flag, &cross_backward_status) &&
                                                mbar_wait(smem_u32(&bars->s_full[t & 1]), parity, abort_flag, &cross_backward_status));
            if (!alive) {
                break;
            }
            tc_fence_after_sync();
            const uint32_t s_tmem = tmem_base + lane_base + TMEM_S + (t & 1) * 128 + group * 32;
            const float4* lse4 = reinterpret_cast<const float4*>(bars->lse2[stage] + group * 32);
            const float4* delta4 = reinterpret_cast<const float4*>(bars->delta[stage] + group * 32);
            uint32_t sb[32];
            float prob[32];
            tmem_ld_x32(s_tmem, sb);
            tmem_wait_ld();
            uint32_t packed[16];
#pragma unroll
            for (int n = 0; n < 32; n += 4) {
                const float4 l = lse4[n / 4];
                prob[n] = exp2_approx(fmaf(__uint_as_float(sb[n]), p.scale_log2, -l.x));
                prob[n + 1] = exp2_approx(fmaf(__uint_as_float(sb[n + 1]), p.scale_log2, -l.y));
                prob[n + 2] = exp2_approx(fmaf(__uint_as_float(sb[n + 2]), p.scale_log2, -l.z));
                prob[n + 3] = exp2_approx(fmaf(__uint_as_float(sb[n + 3]), p.scale_log2, -l.w));
                packed[n / 2] = pack_bf16x2(prob[n], prob[n + 1]);
                packed[n / 2 + 1] = pack_bf16x2(prob[n + 2], prob[n + 3]);
            }
            tmem_st_x16(s_tmem, packed);
            tmem_wait_st();
            tc_fence_before_sync();
            mbar_arrive(smem_u32(&bars->p_full[t & 1]));

            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->dp_full[t & 1]), parity, abort_flag, &cross_backward_status));
            if (!alive) {
                break;
            }
            tc_fence_after_sync();
            tmem_ld_x32(s_tmem + 64, sb);
            tmem_wait_ld();
#pragma unroll
            for (int n = 0; n < 32; n += 4) {
                const float4 d = delta4[n / 4];
                packed[n / 2] = pack_bf16x2(prob[n] * (__uint_as_float(sb[n]) - d.x) * ds_scale, prob[n + 1] * (__uint_as_float(sb[n + 1]) - d.y) * ds_scale);
                packed[n / 2 + 1] =
                    pack_bf16x2(prob[n + 2] * (__uint_as_float(sb[n + 2]) - d.z) * ds_scale, prob[n + 3] * (__uint_as_float(sb[n + 3]) - d.w) * ds_scale);
            }
            tmem_st_x16(s_tmem + 64, packed);
            tmem_wait_st();
            tc_fence_before_sync();
            mbar_arrive(smem_u32(&bars->ds_full[t & 1]));
        }
        if (alive && tile_count > 0) {
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->final_full), 0, abort_flag, &cross_backward_status));
        }
        if (alive && !dead) {
            // group 0 stores dV through V's place, group 1 dK through K's
            tc_fence_after_sync();
            const bool keep = key_start + r < length;
            uint8_t* stage = smem + (group == 0 ? 2 * BIG_CHUNK : 0);
            if (p.key_parts > 1) {
                // into the streamed tiles' place, dV in front of dK
#pragma unroll
                for (int c = 0; c < HEAD / 32 && tile_count > 0; ++c) {
                    uint32_t values[32];
                    tmem_ld_x32(tmem_base + lane_base + (group == 0 ? TMEM_DV : TMEM_DK) + c * 32, values);
                    tmem_wait_ld();
                    result_store32(smem + RESIDENT_BYTES + group * RESULT_BYTES, r, c * 32, values);
                }
            } else {
#pragma unroll
                for (int c = 0; c < HEAD / 32; ++c) {
                    uint32_t values[32];
                    if (tile_count > 0) {
                        tmem_ld_x32(tmem_base + lane_base + (group == 0 ? TMEM_DV : TMEM_DK) + c * 32, values);
                        tmem_wait_ld();
                    }
                    stage_bf16x32(stage + (c / 2) * BIG_CHUNK, r, c % 2, values, keep && tile_count > 0);
                }
                fence_proxy_async_smem();
                mbar_arrive(smem_u32(&bars->staged[group]));
                if (r == 0 && mbar_wait(smem_u32(&bars->staged[group]), 0, abort_flag, &cross_backward_status)) {
                    for (int c = 0; c < 2; ++c) {
                        tma_store_3d(group == 0 ? &p.dv : &p.dk, (group == 0 ? v_smem : k_smem) + c * BIG_CHUNK, kv_head * HEAD + c * 64, key_start, entry);
                    }
                    tma_store_commit();
                    tma_store_wait_read();
                }
            }
        }
    }

    if (p.key_parts > 1) {
        // each CTA its share of the 2 x 128 rows of dV and dK
        __syncwarp();
        cluster_sync_all();
        constexpr int WARPS = THREADS / 32;
        const int row_end = dead ? 0 : part_begin(2 * BIG, part + 1, p.key_parts);
        for (int first = part_begin(2 * BIG, part, p.key_parts) + warp; first < row_end; first += SUM_ROWS * WARPS) {
            float4 sums[SUM_ROWS];
            // (dK lies behind dV, so that row 128 + k of the two together is row k of dK)
            cluster_sums(sums, stage_smem, lane, 0, key_start < length ? p.key_parts : 0, first, WARPS, row_end, [](int, int) { return 1.0F; });
#pragma unroll
            for (int k = 0; k < SUM_ROWS; ++k) {
                const int row = first + k * WARPS;
                const int key = key_start + row % BIG;
                if (row < row_end && key < p.keys) {
                    const uint2 packed = make_uint2(pack_bf16x2(sums[k].x, sums[k].y), pack_bf16x2(sums[k].z, sums[k].w));
                    reinterpret_cast<uint2*>((row < BIG ? p.dv_out : p.dk_out) + ((static_cast<size_t>(entry) * p.keys + key) * p.kv_heads + kv_head) * HEAD)[lane] =
                        key < length ? packed : make_uint2(0, 0);
                }
            }
        }
        __syncwarp();
        cluster_sync_all();             // nobody leaves while others read
    }

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

// ---------------------------------------------------------------------------
// dQ: 128 rows resident (Q in shared memory, dO in tensor memory), tiles of 128 keys.  Order of the tensor core: S(j+1) | dQ(j) | dP(j+1).
// K(j) is read by S(j) and again by dQ(j), a tile and a half later: three slots, the last of which first holds O; V in two, the second of which first holds dO.
// ---------------------------------------------------------------------------
namespace queryside {
constexpr int KEYS = 128;
constexpr int Q_BYTES = 2 * BIG_CHUNK;
constexpr int TILE_BYTES = 2 * BIG_CHUNK;
constexpr int K_SLOTS = 3;
constexpr int V_SLOTS = 2;
constexpr int MISC_BYTES = 2560;
constexpr int SMEM_BYTES = Q_BYTES + (K_SLOTS + V_SLOTS) * TILE_BYTES + MISC_BYTES + 1024;
constexpr uint32_t TMEM_S = 0;
constexpr uint32_t TMEM_DP = 128;
constexpr uint32_t TMEM_DQ = 256;
constexpr uint32_t TMEM_DO = 384;

struct Barriers {
    uint64_t resident_full;
    uint64_t do_copied;
    uint64_t k_full[K_SLOTS];
    uint64_t k_empty[K_SLOTS];
    uint64_t v_full[V_SLOTS];
    uint64_t v_empty[V_SLOTS];
    uint64_t tail_full[2];
    uint64_t s_full;
    uint64_t dp_full;
    uint64_t s_free;
    uint64_t ds_full;
    uint64_t final_full;
    uint64_t staged;
    uint64_t delta_full;
    uint32_t tmem_base;
    int abort_flag;
    int gave_up;
    float delta[2][2][BIG];     // each half's share of sum_d dO O, and with one key tile of sum_k P dP
};
static_assert(sizeof(Barriers) <= MISC_BYTES, "barrier block too large");
static_assert(RESULT_BYTES <= K_SLOTS * TILE_BYTES, "the part's sums take K's place");
}  // namespace queryside

__global__ void __launch_bounds__(THREADS, 1) cross_query_kernel(const __grid_constant__ CrossBackwardParams p) {
    using namespace queryside;
    extern __shared__ uint8_t smem_raw[];
    const int entry = blockIdx.z;
    const int kv_head = blockIdx.y;
    const int part = blockIdx.x % p.query_parts;        // also the rank in the cluster
    const int token0 = blockIdx.x / p.query_parts * p.big_tokens;
    const int rows_per_tile = p.big_tokens * p.group;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023U) & ~1023U;
    uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t k_ring = smem_base + Q_BYTES;
    const uint32_t v_ring = k_ring + K_SLOTS * TILE_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(smem + Q_BYTES + (K_SLOTS + V_SLOTS) * TILE_BYTES);
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&bars->resident_full), 1);
        mbar_init(smem_u32(&bars->do_copied), SOFTMAX_THREADS);
        for (int i = 0; i < K_SLOTS; ++i) {
            mbar_init(smem_u32(&bars->k_full[i]), 1);
            mbar_init(smem_u32(&bars->k_empty[i]), 1);
        }
        for (int i = 0; i < V_SLOTS; ++i) {
            mbar_init(smem_u32(&bars->v_full[i]), 1);
            mbar_init(smem_u32(&bars->v_empty[i]), 1);
        }
        mbar_init(smem_u32(&bars->tail_full[0]), 1);
        mbar_init(smem_u32(&bars->tail_full[1]), 1);
        mbar_init(smem_u32(&bars->s_full), 1);
        mbar_init(smem_u32(&bars->dp_full), 1);
        mbar_init(smem_u32(&bars->s_free), SOFTMAX_THREADS);
        mbar_init(smem_u32(&bars->ds_full), SOFTMAX_THREADS);
        mbar_init(smem_u32(&bars->final_full), 1);
        mbar_init(smem_u32(&bars->staged), SOFTMAX_THREADS);
        mbar_init(smem_u32(&bars->delta_full), SOFTMAX_THREADS);
        bars->abort_flag = 0;
        // after an earlier launch ran into a time limit nothing is done; the CTAs of a cluster stay to the end all the same
        bars->gave_up = *reinterpret_cast<volatile int*>(&cross_backward_status);
        mbar_init_fence();
    }
    if (warp == MMA_WARP) {
        tmem_alloc(smem_u32(&bars->tmem_base), TMEM_COLUMNS);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    grid_dependency_wait();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    const int length = length_of(p, entry);
    const int all_tiles = (length + KEYS - 1) / KEYS;
    const int first_tile = part_begin(all_tiles, part, p.query_parts);
    const bool dead = *reinterpret_cast<volatile int*>(&bars->gave_up) != 0;
    const int tile_count = dead ? 0 : part_begin(all_tiles, part + 1, p.query_parts) - first_tile;
    const int left = length - first_tile * KEYS;        // keys from the first tile on

    if (warp == LOAD_WARP) {
        if (tile_count > 0) {
            const int last = tile_count - 1;
            const bool ragged = length < p.keys && tile_count * KEYS > left;
            bool alive = true;
            auto load_v = [&](int j) {
                const int slot = j % V_SLOTS;
                if (j == 1) {
                    alive = mbar_wait(smem_u32(&bars->do_copied), 0, abort_flag, &cross_backward_status);
                } else if (j >= V_SLOTS) {
                    alive = mbar_wait(smem_u32(&bars->v_empty[slot]), (j / V_SLOTS - 1) & 1, abort_flag, &cross_backward_status);
                }
                if (!alive) {
                    return;
                }
                const uint32_t full = smem_u32(ragged && j == last ? &bars->tail_full[1] : &bars->v_full[slot]);
                mbar_arrive_expect_tx(full, TILE_BYTES);
                for (int c = 0; c < 2; ++c) {
                    tma_load_3d(v_ring + slot * TILE_BYTES + c * BIG_CHUNK, &p.v, full, kv_head * HEAD + c * 64, (first_tile + j) * KEYS, entry);
                }
            };
            auto load_k = [&](int j) {
                const int slot = j % K_SLOTS;
                if (j == K_SLOTS - 1) {
                    alive = mbar_wait(smem_u32(&bars->do_copied), 0, abort_flag, &cross_backward_status);
                } else if (j >= K_SLOTS) {
                    alive = mbar_wait(smem_u32(&bars->k_empty[slot]), (j / K_SLOTS - 1) & 1, abort_flag, &cross_backward_status);
                }
                if (!alive) {
                    return;
                }
                const uint32_t full = smem_u32(ragged && j == last ? &bars->tail_full[0] : &bars->k_full[slot]);
                mbar_arrive_expect_tx(full, TILE_BYTES);
                for (int c = 0; c < 2; ++c) {
                    tma_load_3d(k_ring + slot * TILE_BYTES + c * BIG_CHUNK, &p.k, full, kv_head * HEAD + c * 64, (first_tile + j) * KEYS, entry);
                }
            };
            auto clear_tail = [&](int which, uint32_t offset, uint64_t* full) {
                __syncwarp();
                if (!__all_sync(0xffffffffU, alive && mbar_wait(smem_u32(&bars->tail_full[which]), 0, abort_flag, &cross_backward_status))) {
                    alive = false;
                    return;
                }
                for (int c = 0; c < 2; ++c) {
                    clear_rows(smem + offset + c * BIG_CHUNK, left - last * KEYS, KEYS, lane);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(full));
                }
            };
            if (lane == 0) {
                const uint32_t bar = smem_u32(&bars->resident_full);
                mbar_arrive_expect_tx(bar, 6 * rows_per_tile * 128);
                for (int c = 0; c < 2; ++c) {
                    tma_load_4d(smem_base + c * BIG_CHUNK, &p.q_big, bar, c * 64, kv_head * p.group, token0, entry);
                    tma_load_4d(k_ring + (K_SLOTS - 1) * TILE_BYTES + c * BIG_CHUNK, &p.o_big, bar, c * 64, kv_head * p.group, token0, entry);
                    tma_load_4d(v_ring + TILE_BYTES + c * BIG_CHUNK, &p.do_big, bar, c * 64, kv_head * p.group, token0, entry);
                }
                for (int j = 0; j < tile_count && alive; ++j) {
                    load_k(j);
                    if (alive && j < last) {
                        load_v(j);
                    }
                }
            }
            if (ragged) {
                clear_tail(0, Q_BYTES + (last % K_SLOTS) * TILE_BYTES, &bars->k_full[last % K_SLOTS]);
            }
            if (lane == 0 && alive) {
                load_v(last);
            }
            if (ragged) {
                clear_tail(1, Q_BYTES + (K_SLOTS + last % V_SLOTS) * TILE_BYTES, &bars->v_full[last % V_SLOTS]);
            }
        }
    } else if (warp == MMA_WARP) {
        if (tile_count > 0) {
            const uint32_t leader = elect_one();
            constexpr uint32_t IDESC_SCORE = make_idesc_bf16(BIG, KEYS, false, false);
            constexpr uint32_t IDESC_DQ = make_idesc_bf16(BIG, HEAD, false, true);
            bool alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->resident_full), 0, abort_flag, &cross_backward_status));
            auto issue_s = [&](int j) {
                const int slot = j % K_SLOTS;
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->k_full[slot]), (j / K_SLOTS) & 1, abort_flag, &cross_backward_status));
                if (alive && j > 0) {
                    alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->s_free), (j - 1) & 1, abort_flag, &cross_backward_status));
                }
                if (!alive) {
                    return;
                }
                tc_fence_after_sync();
                const uint32_t k_smem = k_ring + slot * TILE_BYTES;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ss_elect(tmem_base + TMEM_S, make_kmajor_desc(smem_base + c * BIG_CHUNK + k * 32), make_kmajor_desc(k_smem + c * BIG_CHUNK + k * 32),
                                     IDESC_SCORE, (c | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->s_full), leader);
            };
            auto issue_dp = [&](int j) {
                const int slot = j % V_SLOTS;
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->v_full[slot]), (j / V_SLOTS) & 1, abort_flag, &cross_backward_status));
                if (!alive) {
                    return;
                }
                tc_fence_after_sync();
                const uint32_t v_smem = v_ring + slot * TILE_BYTES;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ts_elect(tmem_base + TMEM_DP, tmem_base + TMEM_DO + c * 32 + k * 8, make_kmajor_desc(v_smem + c * BIG_CHUNK + k * 32), IDESC_SCORE,
                                     (c | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->v_empty[slot]), leader);
                mma_commit_elect(smem_u32(&bars->dp_full), leader);
            };
            if (alive) {
                issue_s(0);
            }
            if (alive) {
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->do_copied), 0, abort_flag, &cross_backward_status));
            }
            if (alive) {
                tc_fence_after_sync();
                issue_dp(0);
            }
            for (int j = 0; j < tile_count && alive; ++j) {
                if (j + 1 < tile_count) {
                    issue_s(j + 1);
                    if (!alive) {
                        break;
                    }
                }
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->ds_full), j & 1, abort_flag, &cross_backward_status));
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                const uint32_t k_smem = k_ring + (j % K_SLOTS) * TILE_BYTES;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    mma_ts_elect(tmem_base + TMEM_DQ, tmem_base + TMEM_DP + (k / 4) * 64 + (k % 4) * 8, make_smem_desc(k_smem + k * 2048, BIG_CHUNK, 1024), IDESC_DQ,
                                 (j | k) != 0 ? 1U : 0U, leader);
                }
                mma_commit_elect(smem_u32(&bars->k_empty[j % K_SLOTS]), leader);
                if (j + 1 < tile_count) {
                    issue_dp(j + 1);
                }
            }
            if (alive) {
                mma_commit_elect(smem_u32(&bars->final_full), leader);
            }
        }
    } else {
        const int half = warp / 4;
        const int r = threadIdx.x % BIG;
        const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
        const int token = token0 + r / p.group;
        const bool valid = r < rows_per_tile && token < p.tokens;
        float lse2 = INFINITY;
        if (valid) {
            lse2 = p.lse[(static_cast<size_t>(entry) * p.kv_heads * p.group + kv_head * p.group + r % p.group) * p.tokens + token] * LOG2E;
        }
        float delta = 0.0F;
        bool alive = true;
        if (tile_count > 0) {
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->resident_full), 0, abort_flag, &cross_backward_status));
            if (alive) {
                // dO chunk `half`, row r, into 32 packed columns of tensor memory (without the 128-byte swizzle)
                uint32_t values[32];
                const uint8_t* row = smem + Q_BYTES + (K_SLOTS + 1) * TILE_BYTES + half * BIG_CHUNK + r * 128;
#pragma unroll
                for (int unit = 0; unit < 8; ++unit) {
                    const uint4 v = *reinterpret_cast<const uint4*>(row + ((unit ^ (r & 7)) * 16));
                    values[unit * 4 + 0] = v.x;
                    values[unit * 4 + 1] = v.y;
                    values[unit * 4 + 2] = v.z;
                    values[unit * 4 + 3] = v.w;
                }
                tmem_st_x32(tmem_base + lane_base + TMEM_DO + half * 32, values);
                const uint8_t* out = smem + Q_BYTES + (K_SLOTS - 1) * TILE_BYTES + half * BIG_CHUNK + r * 128;
                float share = 0.0F;
#pragma unroll
                for (int unit = 0; unit < 8; ++unit) {
                    const uint4 v = *reinterpret_cast<const uint4*>(out + ((unit ^ (r & 7)) * 16));
                    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        share = fmaf(__uint_as_float(values[unit * 4 + e] << 16), __uint_as_float(words[e] << 16), share);
                        share = fmaf(__uint_as_float(values[unit * 4 + e] & 0xffff0000U), __uint_as_float(words[e] & 0xffff0000U), share);
                    }
                }
                bars->delta[0][half][r] = share;
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&bars->do_copied));
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->do_copied), 0, abort_flag, &cross_backward_status));
                delta = bars->delta[0][0][r] + bars->delta[0][1][r];
            }
        }
        // (the last part always has a tile of an entry that has any)
        float2* row = valid && half == 0 && part + 1 == p.query_parts && tile_count > 0
                          ? p.rows + ((static_cast<size_t>(entry) * p.kv_heads + kv_head) * p.tokens + token) * p.group + r % p.group
                          : nullptr;
        if (row != nullptr && alive) {
            *row = make_float2(lse2, delta);
        }
        const uint32_t s_tmem = tmem_base + lane_base + TMEM_S + half * 64;
        const uint32_t dp_tmem = tmem_base + lane_base + TMEM_DP + half * 64;
        for (int j = 0; j < tile_count && alive; ++j) {
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->s_full), j & 1, abort_flag, &cross_backward_status));
            if (!alive) {
                break;
            }
            tc_fence_after_sync();
            uint32_t sb[64];
            tmem_ld_x32(s_tmem, sb);
            tmem_ld_x32(s_tmem + 32, sb + 32);
            tmem_wait_ld();
            tc_fence_before_sync();
            mbar_arrive(smem_u32(&bars->s_free));
            float prob[64];             // P * scale
#pragma unroll
            for (int n = 0; n < 64; ++n) {
                prob[n] = exp2_approx(fmaf(__uint_as_float(sb[n]), p.scale_log2, -lse2)) * p.scale;
            }
            if (j + 1 == tile_count) {
                const int present = left - j * KEYS - half * 64;
#pragma unroll
                for (int n = 0; n < 64; ++n) {
                    prob[n] = n < present ? prob[n] : 0.0F;
                }
            }
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->dp_full), j & 1, abort_flag, &cross_backward_status));
            if (!alive) {
                break;
            }
            tc_fence_after_sync();
            tmem_ld_x32(dp_tmem, sb);
            tmem_ld_x32(dp_tmem + 32, sb + 32);
            tmem_wait_ld();
            if (all_tiles == 1) {
                float share = 0.0F;
#pragma unroll
                for (int n = 0; n < 64; ++n) {
                    share = fmaf(prob[n], __uint_as_float(sb[n]), share);
                }
                bars->delta[1][half][r] = share;
                mbar_arrive(smem_u32(&bars->delta_full));
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->delta_full), 0, abort_flag, &cross_backward_status));
                if (!alive) {
                    break;
                }
                delta = (bars->delta[1][0][r] + bars->delta[1][1][r]) / p.scale;
                if (row != nullptr) {
                    row->y = delta;
                }
            }
            uint32_t packed[32];
#pragma unroll
            for (int n = 0; n < 64; n += 2) {
                packed[n / 2] = pack_bf16x2(prob[n] * (__uint_as_float(sb[n]) - delta), prob[n + 1] * (__uint_as_float(sb[n + 1]) - delta));
            }
            tmem_st_x32(dp_tmem, packed);
            tmem_wait_st();
            tc_fence_before_sync();
            mbar_arrive(smem_u32(&bars->ds_full));
        }
        if (alive && tile_count > 0) {
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->final_full), 0, abort_flag, &cross_backward_status));
        }
        if (alive && !dead) {
            tc_fence_after_sync();
            if (p.query_parts > 1) {
#pragma unroll
                for (int c = 0; c < 2 && tile_count > 0; ++c) {
                    uint32_t values[32];
                    tmem_ld_x32(tmem_base + lane_base + TMEM_DQ + half * 64 + c * 32, values);
                    tmem_wait_ld();
                    result_store32(smem + Q_BYTES, r, half * 64 + c * 32, values);     // into K's place
                }
            } else {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t values[32];
                    if (tile_count > 0) {
                        tmem_ld_x32(tmem_base + lane_base + TMEM_DQ + half * 64 + c * 32, values);
                        tmem_wait_ld();
                    }
                    stage_bf16x32(smem + half * BIG_CHUNK, r, c, values, length > 1);
                }
                fence_proxy_async_smem();
                mbar_arrive(smem_u32(&bars->staged));
                if (threadIdx.x == 0 && mbar_wait(smem_u32(&bars->staged), 0, abort_flag, &cross_backward_status)) {
                    for (int c = 0; c < 2; ++c) {
                        tma_store_4d(&p.dq, smem_base + c * BIG_CHUNK, c * 64, kv_head * p.group, token0, entry);
                    }
                    tma_store_commit();
                    tma_store_wait_read();
                }
            }
        }
    }

    if (p.query_parts > 1) {
        // each CTA its share of the rows; parts without tiles have left nothing
        __syncwarp();
        cluster_sync_all();
        constexpr int WARPS = THREADS / 32;
        const int rows = min(p.big_tokens, p.tokens - token0) * p.group;
        const int row_end = dead ? 0 : part_begin(rows, part + 1, p.query_parts);
        for (int first = part_begin(rows, part, p.query_parts) + warp; first < row_end; first += SUM_ROWS * WARPS) {
            float4 sums[SUM_ROWS];
            cluster_sums(sums, k_ring, lane, parts_without(all_tiles, p.query_parts), p.query_parts, first, WARPS, row_end, [](int, int) { return 1.0F; });
#pragma unroll
            for (int k = 0; k < SUM_ROWS; ++k) {
                const int row = first + k * WARPS;
                if (row < row_end) {
                    reinterpret_cast<uint2*>(p.dq_out + ((static_cast<size_t>(entry) * p.tokens + token0 + row / p.group) * p.kv_heads * p.group + kv_head * p.group +
                                                         row % p.group) * HEAD)[lane] =
                        length > 1 ? make_uint2(pack_bf16x2(sums[k].x, sums[k].y), pack_bf16x2(sums[k].z, sums[k].w)) : make_uint2(0, 0);
                }
            }
        }
        __syncwarp();
        cluster_sync_all();             // nobody leaves while others read
    }

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

struct Clusters {
    ClusterCounts query, key;
};

struct Plan {
    int query_parts, key_parts;
    bool query_short, key_short;
};

Plan make_plan(int batch, int queries, int keys, int heads, int kv_heads, const Clusters& clusters) {
    const int group = heads / kv_heads;
    const long long key_tiles = (keys + BIG - 1LL) / BIG;
    const long long row_tiles = (queries + BIG / group - 1LL) / (BIG / group);
    const long long sub_tiles = (queries + SUB / group - 1LL) / (SUB / group);
    const long long pairs = static_cast<long long>(batch) * kv_heads;
    const int key_parts = loop_parts(key_tiles * pairs, sub_tiles, KEY_TILE_US, clusters.key);
    const int query_parts = loop_parts(row_tiles * pairs, key_tiles, QUERY_TILE_US, clusters.query);
    return {query_parts, key_parts, query_parts == 1 && cross_query_short_takes(row_tiles * pairs, key_tiles), key_parts == 1 && cross_key_short_takes(key_tiles * pairs, sub_tiles)};
}

const Clusters& configure() {
    static PerDevice<Clusters> devices;
    return devices.get([] {
        CUDA_CHECK(cudaFuncSetAttribute(cross_key_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, keyside::SMEM_BYTES));
        CUDA_CHECK(cudaFuncSetAttribute(cross_key_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        CUDA_CHECK(cudaFuncSetAttribute(cross_query_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, queryside::SMEM_BYTES));
        return Clusters{cluster_counts(cross_query_kernel, THREADS, queryside::SMEM_BYTES, 8),
                        cluster_counts(cross_key_kernel, THREADS, keyside::SMEM_BYTES, MOST_KEY_PARTS)};
    });
}

}  // namespace

namespace internal {

int cross_backward_device_status(bool reset) {
    int status = 0;
    CUDA_CHECK(cudaDeviceSynchronize());
    CUDA_CHECK(cudaMemcpyFromSymbol(&status, cross_backward_status, sizeof(int)));
    if (reset && status != 0) {
        const int zero = 0;
        CUDA_CHECK(cudaMemcpyToSymbol(cross_backward_status, &zero, sizeof(int)));
    }
    return status;
}

}  // namespace internal

std::size_t flash_cross_backward_workspace_bytes(int batch_size, int query_length, int key_length, int query_heads, int key_value_heads) {
    if (batch_size <= 0 || query_length <= 0 || key_length <= 0 || query_heads <= 0 || key_value_heads <= 0) {
        return 0;
    }
    return static_cast<std::size_t>(batch_size) * query_length * query_heads * sizeof(float2);
}

void flash_cross_backward_cuda(__nv_bfloat16* query_gradient, __nv_bfloat16* key_gradient, __nv_bfloat16* value_gradient,
                               const __nv_bfloat16* output_gradient, const __nv_bfloat16* output, const float* logsumexp, const __nv_bfloat16* query,
                               const __nv_bfloat16* key, const __nv_bfloat16* value, const int* key_lengths, void* workspace,
                               std::size_t workspace_bytes, int batch_size, int query_length, int key_length, int query_heads, int key_value_heads,
                               int head_size, float scale, cudaStream_t stream) {
    internal::check_flash_cross_shape(batch_size, query_length, key_length, query_heads, key_value_heads, head_size, scale);
    internal::check_flash_pointers({query_gradient, key_gradient, value_gradient, output_gradient, output, query, key, value, workspace}, {logsumexp});
    if (key_lengths != nullptr) {
        internal::check_flash_pointers({}, {key_lengths});
    }
    if (workspace_bytes < flash_cross_backward_workspace_bytes(batch_size, query_length, key_length, query_heads, key_value_heads)) {
        throw std::invalid_argument("flash cross attention backward workspace is too small");
    }
    CrossBackwardParams p{};
    p.group = query_heads / key_value_heads;
    p.sub_tokens = SUB / p.group;
    p.big_tokens = BIG / p.group;
    const std::uint64_t wide = static_cast<std::uint64_t>(key_value_heads) * HEAD;
    p.q_sub = make_bf16_group_rows_map(query, batch_size, query_length, query_heads, p.group, p.sub_tokens);
    p.do_sub = make_bf16_group_rows_map(output_gradient, batch_size, query_length, query_heads, p.group, p.sub_tokens);
    p.q_big = make_bf16_group_rows_map(query, batch_size, query_length, query_heads, p.group, p.big_tokens);
    p.do_big = make_bf16_group_rows_map(output_gradient, batch_size, query_length, query_heads, p.group, p.big_tokens);
    p.o_big = make_bf16_group_rows_map(output, batch_size, query_length, query_heads, p.group, p.big_tokens);
    p.dq = make_bf16_group_rows_map(query_gradient, batch_size, query_length, query_heads, p.group, p.big_tokens);
    p.k = make_bf16_batched_tile_map(key, batch_size, key_length, wide, BIG);
    p.v = make_bf16_batched_tile_map(value, batch_size, key_length, wide, BIG);
    p.dk = make_bf16_batched_tile_map(key_gradient, batch_size, key_length, wide, BIG);
    p.dv = make_bf16_batched_tile_map(value_gradient, batch_size, key_length, wide, BIG);
    if ((key_length + BIG - 1LL) / BIG * key_value_heads * batch_size > 0x7fffffffLL) {
        throw std::invalid_argument("flash cross attention shape exceeds the supported index range");
    }
    const Plan plan = make_plan(batch_size, query_length, key_length, query_heads, key_value_heads, configure());
    p.rows = static_cast<float2*>(workspace);
    p.dq_out = query_gradient;
    p.dk_out = key_gradient;
    p.dv_out = value_gradient;
    p.query_parts = plan.query_parts;
    p.key_parts = plan.key_parts;
    p.lse = logsumexp;
    p.lengths = key_lengths;
    p.tokens = query_length;
    p.keys = key_length;
    p.kv_heads = key_value_heads;
    p.scale = scale;
    p.scale_log2 = scale * LOG2E;
    p.batch = batch_size;
    p.key_tiles = (key_length + BIG - 1) / BIG;
    if (plan.query_short) {
        launch_cross_query_short(p, stream);
    } else {
        launch_chained_clusters(cross_query_kernel, dim3((query_length + p.big_tokens - 1) / p.big_tokens * plan.query_parts, key_value_heads, batch_size),
                                plan.query_parts, dim3(THREADS), queryside::SMEM_BYTES, stream, p);
    }
    if (plan.key_short) {
        launch_cross_key_short(p, stream);
        return;
    }
    launch_chained_clusters(cross_key_kernel, dim3((key_length + BIG - 1) / BIG * plan.key_parts, key_value_heads, batch_size), plan.key_parts, dim3(THREADS),
                            keyside::SMEM_BYTES, stream, p);
}

}  // namespace dscuda
