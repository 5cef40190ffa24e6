// Gradients of the cross attention (D = 128, grouped-query) on tcgen05.
//
// With rows r = (token, head of the group) of one (entry, key head), P = exp(scale * Q K^T - lse) and dP = dO V^T:
//     delta[r] = sum_d dO[r,d] O[r,d]        dS = P (dP - delta) scale
//     dV = P^T dO        dK = dS^T Q          dQ = dS K
// dK and dV of a key head are sums over all rows of its group, so the heads of a group need no step of their own.
//
// One call launches:
//   1. cross_delta_kernel: delta and lse * log2(e) in row order, one pair to a row.
//   2. cross_query_kernel: a CTA keeps 128 rows and goes over the keys in tiles of 128: S = Q K^T, dP = dO V^T, dQ += dS K.  With few keys the
//      rounding of O in delta would be the largest error of dS (2 keys: 0.4 % of dQ and dK, against 0.17 % of the last rounding); where one tile
//      holds all keys, delta = sum_k P dP is formed from the tile itself and left for the next kernel as well.
//   3. cross_key_kernel: a CTA keeps 128 keys (K, V) and goes over the rows in tiles of at most 64: S^T = K Q^T, dP^T = V dO^T, one thread to a
//      key (two, half the rows each), P^T and dS^T back into tensor memory as bf16 A operands, dV += P^T dO, dK += dS^T Q.  Tensor memory: dV 128, dK
//      128, two pairs of 64-column scores, so the scores of the next tile are computed while the softmax works on this one.
// S and dP are computed twice (1792 instead of 1280 FLOP per pair).  The alternative of the causal backward, dS stored once and streamed
// back, moves 4 bytes per pair through HBM, 0.62 ps at the measured copy rate, against 0.31 ps for the 512 FLOP at the measured tensor rate.
//
// Every gradient element has one writer and a fixed order of sums: results are the same bits from call to call.  P and dS are rounded to
// bf16 (half a step is 2^-9); everything else is fp32.
//
// Rows that do not exist (a group that does not divide 64, tokens behind the last) carry lse = +inf, which makes their P zero, and zeros for Q and
// dO.  Keys behind an entry's length cost nothing in the key kernel (one thread owns a key, its sums are replaced by zeros at the end); the
// query kernel clears them in shared memory, because dS K multiplies them by zeros.  Every wait is bounded.
#include "flash_attention.h"
#include "cuda_common.h"
#include "attention_internal.h"
#include "sm100_primitives.cuh"
#include "../common/launch.h"
#include "../common/tensor_map.h"

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <stdexcept>

namespace dscuda {
namespace {

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

__device__ int cross_backward_status = 0;

struct CrossBackwardParams {
    CUtensorMap q_sub, do_sub;          // group rows, box {64, group, tokens of a 64-row tile}
    CUtensorMap q_big, do_big;          // the same for 128-row tiles
    CUtensorMap k, v;                   // [B][Tk][Hkv * 128], boxes of 128 rows
    CUtensorMap dq;                     // like q_big
    CUtensorMap dk, dv;                 // like k
    float2* rows;                       // [B, Hkv, Tq, group]: lse * log2(e), delta
    const int* lengths;                 // null: Tk
    int tokens, keys, kv_heads, group;
    int sub_tokens, big_tokens;         // tokens of a query tile of each kind
    float scale, scale_log2;
};

__device__ __forceinline__ int length_of(const CrossBackwardParams& p, int entry) {
    return p.lengths == nullptr ? p.keys : min(max(p.lengths[entry], 0), p.keys);
}

// ---------------------------------------------------------------------------
// delta and lse * log2(e) in row order; half a warp to a row
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) cross_delta_kernel(float2* rows, const __nv_bfloat16* dout, const __nv_bfloat16* out, const float* lse,
                                                          long long count, int tokens, int heads, int group) {
    const int lane = threadIdx.x % 32;
    const int half = lane / 16;
    const int part = lane % 16;
    const long long stride = static_cast<long long>(gridDim.x) * 16;
    grid_dependency_wait();
    for (long long base = static_cast<long long>(blockIdx.x) * 16 + threadIdx.x / 32 * 2; base < count; base += stride) {
        const long long row = base + half;              // (entry, token, head)
        float sum = 0.0F;
        if (row < count) {
            const uint4 a = reinterpret_cast<const uint4*>(dout + row * HEAD)[part];
            const uint4 b = reinterpret_cast<const uint4*>(out + row * HEAD)[part];
            const __nv_bfloat162* a2 = reinterpret_cast<const __nv_bfloat162*>(&a);
            const __nv_bfloat162* b2 = reinterpret_cast<const __nv_bfloat162*>(&b);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 x = __bfloat1622float2(a2[e]), y = __bfloat1622float2(b2[e]);
                sum += x.x * y.x + x.y * y.y;
            }
        }
#pragma unroll
        for (int offset = 8; offset > 0; offset >>= 1) {
            sum += __shfl_xor_sync(0xffffffffU, sum, offset);
        }
        if (part == 0 && row < count) {
            const int head = static_cast<int>(row % heads);
            const long long at = row / heads;
            const long long entry = at / tokens;
            const int token = static_cast<int>(at % tokens);
            const int kv_heads = heads / group;
            rows[((entry * kv_heads + head / group) * tokens + token) * group + head % group] =
                make_float2(lse[(entry * heads + head) * tokens + token] * LOG2E, sum);
        }
    }
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

// ---------------------------------------------------------------------------
// dK, dV
// ---------------------------------------------------------------------------
namespace keyside {
constexpr int STAGES = 4;
constexpr int STAGE_BYTES = 4 * SUB_CHUNK;          // Q and dO of 64 rows
constexpr int RESIDENT_BYTES = 4 * BIG_CHUNK;       // K and V of 128 keys
constexpr int MISC_BYTES = 3072;
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
    alignas(16) float lse2[STAGES][SUB];
    alignas(16) float delta[STAGES][SUB];
};
static_assert(sizeof(Barriers) <= MISC_BYTES, "barrier block too large");
static_assert(offsetof(Barriers, lse2) % 16 == 0 && offsetof(Barriers, delta) % 16 == 0, "16-byte loads of the per-row constants");
}  // namespace keyside

__global__ void __launch_bounds__(THREADS, 1) cross_key_kernel(const __grid_constant__ CrossBackwardParams p) {
    using namespace keyside;
    extern __shared__ uint8_t smem_raw[];
    if (*reinterpret_cast<volatile int*>(&cross_backward_status) != 0) {
        grid_dependency_wait();
        return;
    }
    const int entry = blockIdx.z;
    const int kv_head = blockIdx.y;
    const int key_start = blockIdx.x * BIG;
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
    const int tile_count = key_start < length ? (p.tokens + p.sub_tokens - 1) / p.sub_tokens : 0;

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
            const int token = t * p.sub_tokens;
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
                packed[n / 2] = pack_bf16x2(prob[n] * (__uint_as_float(sb[n]) - d.x) * p.scale, prob[n + 1] * (__uint_as_float(sb[n + 1]) - d.y) * p.scale);
                packed[n / 2 + 1] =
                    pack_bf16x2(prob[n + 2] * (__uint_as_float(sb[n + 2]) - d.z) * p.scale, prob[n + 3] * (__uint_as_float(sb[n + 3]) - d.w) * p.scale);
            }
            tmem_st_x16(s_tmem + 64, packed);
            tmem_wait_st();
            tc_fence_before_sync();
            mbar_arrive(smem_u32(&bars->ds_full[t & 1]));
        }
        if (alive && tile_count > 0) {
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->final_full), 0, abort_flag, &cross_backward_status));
        }
        if (alive) {
            // group 0 stores dV through V's place, group 1 dK through K's
            tc_fence_after_sync();
            const bool keep = key_start + r < length;
            uint8_t* stage = smem + (group == 0 ? 2 * BIG_CHUNK : 0);
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
// K(j) is read by S(j) and again by dQ(j), a tile and a half later: three slots; V in two.
// ---------------------------------------------------------------------------
namespace queryside {
constexpr int KEYS = 128;
constexpr int Q_BYTES = 2 * BIG_CHUNK;
constexpr int TILE_BYTES = 2 * BIG_CHUNK;
constexpr int K_SLOTS = 3;
constexpr int V_SLOTS = 2;                          // the second one first holds dO
constexpr int MISC_BYTES = 2048;
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
    float delta[2][BIG];        // one key tile: each half's share of sum_k P dP
};
static_assert(sizeof(Barriers) <= MISC_BYTES, "barrier block too large");
}  // namespace queryside

__global__ void __launch_bounds__(THREADS, 1) cross_query_kernel(const __grid_constant__ CrossBackwardParams p) {
    using namespace queryside;
    extern __shared__ uint8_t smem_raw[];
    if (*reinterpret_cast<volatile int*>(&cross_backward_status) != 0) {
        grid_dependency_wait();
        return;
    }
    const int entry = blockIdx.z;
    const int kv_head = blockIdx.y;
    const int token0 = blockIdx.x * p.big_tokens;
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
    const int tile_count = (length + KEYS - 1) / KEYS;

    if (warp == LOAD_WARP) {
        if (tile_count > 0) {
            const int last = tile_count - 1;
            const bool ragged = length < p.keys && tile_count * KEYS > length;
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
                    tma_load_3d(v_ring + slot * TILE_BYTES + c * BIG_CHUNK, &p.v, full, kv_head * HEAD + c * 64, j * KEYS, entry);
                }
            };
            auto load_k = [&](int j) {
                const int slot = j % K_SLOTS;
                if (j >= K_SLOTS) {
                    alive = mbar_wait(smem_u32(&bars->k_empty[slot]), (j / K_SLOTS - 1) & 1, abort_flag, &cross_backward_status);
                }
                if (!alive) {
                    return;
                }
                const uint32_t full = smem_u32(ragged && j == last ? &bars->tail_full[0] : &bars->k_full[slot]);
                mbar_arrive_expect_tx(full, TILE_BYTES);
                for (int c = 0; c < 2; ++c) {
                    tma_load_3d(k_ring + slot * TILE_BYTES + c * BIG_CHUNK, &p.k, full, kv_head * HEAD + c * 64, j * KEYS, entry);
                }
            };
            auto clear_tail = [&](int which, uint32_t offset, uint64_t* full) {
                __syncwarp();
                if (!__all_sync(0xffffffffU, alive && mbar_wait(smem_u32(&bars->tail_full[which]), 0, abort_flag, &cross_backward_status))) {
                    alive = false;
                    return;
                }
                for (int c = 0; c < 2; ++c) {
                    clear_rows(smem + offset + c * BIG_CHUNK, length - last * KEYS, KEYS, lane);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(full));
                }
            };
            if (lane == 0) {
                const uint32_t bar = smem_u32(&bars->resident_full);
                mbar_arrive_expect_tx(bar, 4 * rows_per_tile * 128);
                for (int c = 0; c < 2; ++c) {
                    tma_load_4d(smem_base + c * BIG_CHUNK, &p.q_big, bar, c * 64, kv_head * p.group, token0, entry);
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
        const size_t row_index = ((static_cast<size_t>(entry) * p.kv_heads + kv_head) * p.tokens + token) * p.group + r % p.group;
        float2 constants = make_float2(INFINITY, 0.0F);
        if (valid) {
            constants = p.rows[row_index];
        }
        const float lse2 = constants.x;
        float delta = constants.y;
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
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&bars->do_copied));
            }
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
                const int left = length - j * KEYS - half * 64;
#pragma unroll
                for (int n = 0; n < 64; ++n) {
                    prob[n] = n < left ? prob[n] : 0.0F;
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
            if (tile_count == 1) {
                float share = 0.0F;
#pragma unroll
                for (int n = 0; n < 64; ++n) {
                    share = fmaf(prob[n], __uint_as_float(sb[n]), share);
                }
                bars->delta[half][r] = share;
                mbar_arrive(smem_u32(&bars->delta_full));
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->delta_full), 0, abort_flag, &cross_backward_status));
                if (!alive) {
                    break;
                }
                delta = (bars->delta[0][r] + bars->delta[1][r]) / p.scale;
                if (valid && half == 0) {
                    p.rows[row_index].y = delta;
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
        if (alive) {
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t values[32];
                if (tile_count > 0) {
                    tmem_ld_x32(tmem_base + lane_base + TMEM_DQ + half * 64 + c * 32, values);
                    tmem_wait_ld();
                }
                stage_bf16x32(smem + half * BIG_CHUNK, r, c, values, tile_count > 0);
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

void configure() {
    static bool done[16] = {};
    int device = 0;
    CUDA_CHECK(cudaGetDevice(&device));
    if (device < 16 && done[device]) {
        return;
    }
    CUDA_CHECK(cudaFuncSetAttribute(cross_key_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, keyside::SMEM_BYTES));
    CUDA_CHECK(cudaFuncSetAttribute(cross_query_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, queryside::SMEM_BYTES));
    if (device < 16) {
        done[device] = true;
    }
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
    p.dq = make_bf16_group_rows_map(query_gradient, batch_size, query_length, query_heads, p.group, p.big_tokens);
    p.k = make_bf16_batched_tile_map(key, batch_size, key_length, wide, BIG);
    p.v = make_bf16_batched_tile_map(value, batch_size, key_length, wide, BIG);
    p.dk = make_bf16_batched_tile_map(key_gradient, batch_size, key_length, wide, BIG);
    p.dv = make_bf16_batched_tile_map(value_gradient, batch_size, key_length, wide, BIG);
    p.rows = static_cast<float2*>(workspace);
    p.lengths = key_lengths;
    p.tokens = query_length;
    p.keys = key_length;
    p.kv_heads = key_value_heads;
    p.scale = scale;
    p.scale_log2 = scale * LOG2E;
    configure();
    const long long rows = static_cast<long long>(batch_size) * query_length * query_heads;
    const unsigned blocks = static_cast<unsigned>(std::min((rows + 15) / 16, 148LL * 16));
    launch_chained(cross_delta_kernel, dim3(blocks), dim3(256), 0, stream, static_cast<float2*>(workspace), output_gradient, output, logsumexp, rows,
                   query_length, query_heads, p.group);
    launch_chained(cross_query_kernel, dim3((query_length + p.big_tokens - 1) / p.big_tokens, key_value_heads, batch_size), dim3(THREADS),
                   queryside::SMEM_BYTES, stream, p);
    launch_chained(cross_key_kernel, dim3((key_length + BIG - 1) / BIG, key_value_heads, batch_size), dim3(THREADS), keyside::SMEM_BYTES, stream, p);
}

}  // namespace dscuda
