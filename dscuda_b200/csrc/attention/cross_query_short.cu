// dQ of the cross attention for short loops (few keys under many rows), the first kernel of cross_backward.cu otherwise: the same products and sums in the same
// order.  A CTA goes over several items (128 rows of a key head and entry): the Q, O and dO of the next one arrive while this one's products run and its dQ
// leaves.  That takes the room of a K and a V tile, and the items are dealt out in fixed turns, so long loops and few items stay with the other form.  Where one
// tile holds all keys O is not read at all (delta comes from the tile).
//
// dQ kernel, us, this form and the other: 3506 x 4 rows over 20 keys, 16 heads and entries 58.9 and 92.2 (36 of HBM traffic), 584 rows over 12 keys, 208 heads 31.8
// and 49.8, 1024 x 4 rows over 256 keys (two tiles), 64 heads 86 and 119, 1024 x 4 over 576 (five), 32 heads 78.6 and 86.0, 4096 x 4 over 1024 (eight), 16 heads 211
// and 215; with three items to a CTA 858 x 4 over 555 keys 39.0 and 37.1.
#include "attention_internal.h"
#include "cuda_common.h"
#include "cross_backward.cuh"
#include "loop_parts.cuh"
#include "../common/launch.h"

#include <cstdint>

namespace dscuda {
namespace {

using namespace cross;

__device__ int cross_query_short_status = 0;

constexpr int KEYS = 128;
constexpr int ROWS_BYTES = 2 * BIG_CHUNK;           // 128 rows or keys
constexpr int Q_SLOTS = 2;
constexpr int K_SLOTS = 2;
constexpr int O_OFFSET = Q_SLOTS * ROWS_BYTES;
constexpr int DO_OFFSET = O_OFFSET + ROWS_BYTES;
constexpr int K_OFFSET = DO_OFFSET + ROWS_BYTES;
constexpr int V_OFFSET = K_OFFSET + K_SLOTS * ROWS_BYTES;
constexpr int MISC_OFFSET = V_OFFSET + ROWS_BYTES;
constexpr int MISC_BYTES = 2048;
constexpr int SMEM_BYTES = MISC_OFFSET + MISC_BYTES + 1024;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of a CTA");
constexpr uint32_t TMEM_S = 0;
constexpr uint32_t TMEM_DP = 128;
constexpr uint32_t TMEM_DQ = 256;
constexpr uint32_t TMEM_DO = 384;

struct Barriers {
    uint64_t q_full[Q_SLOTS];
    uint64_t q_empty[Q_SLOTS];          // the item's dQ has left from Q's place
    uint64_t o_full;                    // O and dO
    uint64_t do_copied;
    uint64_t k_full[K_SLOTS];
    uint64_t k_empty[K_SLOTS];
    uint64_t v_full;
    uint64_t v_empty;
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
    float delta[2][BIG];                // each half's share of sum_d dO O, with one key tile of sum_k P dP
};
static_assert(sizeof(Barriers) <= MISC_BYTES, "barrier block too large");

struct Item {
    int entry, kv_head, token0, length;
};

__global__ void __launch_bounds__(THREADS, 1) cross_query_short_kernel(const __grid_constant__ CrossBackwardParams p) {
    extern __shared__ uint8_t smem_raw[];
    const int rows_per_tile = p.big_tokens * p.group;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023U) & ~1023U;
    uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
    Barriers* bars = reinterpret_cast<Barriers*>(smem + MISC_OFFSET);
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&bars->q_full[i]), 1);
            mbar_init(smem_u32(&bars->q_empty[i]), 1);
            mbar_init(smem_u32(&bars->k_full[i]), 1);
            mbar_init(smem_u32(&bars->k_empty[i]), 1);
            mbar_init(smem_u32(&bars->tail_full[i]), 1);
        }
        mbar_init(smem_u32(&bars->o_full), 1);
        mbar_init(smem_u32(&bars->do_copied), SOFTMAX_THREADS);
        mbar_init(smem_u32(&bars->v_full), 1);
        mbar_init(smem_u32(&bars->v_empty), 1);
        mbar_init(smem_u32(&bars->s_full), 1);
        mbar_init(smem_u32(&bars->dp_full), 1);
        mbar_init(smem_u32(&bars->s_free), SOFTMAX_THREADS);
        mbar_init(smem_u32(&bars->ds_full), SOFTMAX_THREADS);
        mbar_init(smem_u32(&bars->final_full), 1);
        mbar_init(smem_u32(&bars->staged), SOFTMAX_THREADS);
        mbar_init(smem_u32(&bars->delta_full), SOFTMAX_THREADS);
        bars->abort_flag = 0;
        // after an earlier launch ran into a time limit nothing is done
        bars->gave_up = *reinterpret_cast<volatile int*>(&cross_query_short_status);
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
    const int row_tiles = (p.tokens + p.big_tokens - 1) / p.big_tokens;
    const long long items = *reinterpret_cast<volatile int*>(&bars->gave_up) != 0 ? 0 : static_cast<long long>(row_tiles) * p.kv_heads * p.batch;
    auto item_at = [&](long long index) {
        const int pair = static_cast<int>(index / row_tiles), entry = pair / p.kv_heads;
        return Item{entry, pair - entry * p.kv_heads, static_cast<int>(index - static_cast<long long>(pair) * row_tiles) * p.big_tokens, length_of(p, entry)};
    };
    // Each role goes over the CTA's items.  `n` counts those with keys, `base` their key tiles.

    if (warp == LOAD_WARP) {
        bool alive = true;
        int n = 0, base = 0, tails = 0;
        for (long long index = blockIdx.x; index < items && alive; index += gridDim.x) {
            const Item at = item_at(index);
            if (at.length == 0) {
                continue;
            }
            const int tile_count = (at.length + KEYS - 1) / KEYS;
            const int last = tile_count - 1;
            const bool ragged = at.length < p.keys && tile_count * KEYS > at.length;
            auto wait = [&](uint64_t* barrier, int parity) { return mbar_wait(smem_u32(barrier), parity & 1, abort_flag, &cross_query_short_status); };
            auto load_rows = [&](uint32_t offset, const CUtensorMap* map, uint32_t bar) {
                for (int c = 0; c < 2; ++c) {
                    tma_load_4d(smem_base + offset + c * BIG_CHUNK, map, bar, c * 64, at.kv_head * p.group, at.token0, at.entry);
                }
            };
            auto load_keys = [&](uint32_t offset, const CUtensorMap* map, uint64_t* full, int j) {
                const uint32_t bar = smem_u32(full);
                mbar_arrive_expect_tx(bar, ROWS_BYTES);
                for (int c = 0; c < 2; ++c) {
                    tma_load_3d(smem_base + offset + c * BIG_CHUNK, map, bar, at.kv_head * HEAD + c * 64, j * KEYS, at.entry);
                }
            };
            auto load_k = [&](int j) {
                const int slot = (base + j) % K_SLOTS, use = (base + j) / K_SLOTS;
                alive = use == 0 || wait(&bars->k_empty[slot], use - 1);
                if (alive) {
                    load_keys(K_OFFSET + slot * ROWS_BYTES, &p.k, ragged && j == last ? &bars->tail_full[0] : &bars->k_full[slot], j);
                }
            };
            auto load_v = [&](int j) {
                alive = base + j == 0 || wait(&bars->v_empty, base + j - 1);
                if (alive) {
                    load_keys(V_OFFSET, &p.v, ragged && j == last ? &bars->tail_full[1] : &bars->v_full, j);
                }
            };
            auto clear_tail = [&](int which, uint32_t offset, uint64_t* full) {
                __syncwarp();
                if (!__all_sync(0xffffffffU, alive && wait(&bars->tail_full[which], tails))) {
                    alive = false;
                    return;
                }
                for (int c = 0; c < 2; ++c) {
                    clear_rows(smem + offset + c * BIG_CHUNK, at.length - last * KEYS, KEYS, lane);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(full));
                }
            };
            if (lane == 0) {
                alive = n < Q_SLOTS || wait(&bars->q_empty[n % Q_SLOTS], n / Q_SLOTS - 1);
                if (alive) {
                    const uint32_t bar = smem_u32(&bars->q_full[n % Q_SLOTS]);
                    mbar_arrive_expect_tx(bar, 2 * rows_per_tile * 128);
                    load_rows(n % Q_SLOTS * ROWS_BYTES, &p.q_big, bar);
                    alive = n == 0 || wait(&bars->do_copied, n - 1);
                }
                if (alive) {
                    const uint32_t bar = smem_u32(&bars->o_full);
                    mbar_arrive_expect_tx(bar, (tile_count > 1 ? 4 : 2) * rows_per_tile * 128);
                    load_rows(DO_OFFSET, &p.do_big, bar);
                    if (tile_count > 1) {
                        load_rows(O_OFFSET, &p.o_big, bar);
                    }
                }
                for (int j = 0; j < tile_count && alive; ++j) {
                    load_k(j);
                    if (alive && j < last) {
                        load_v(j);
                    }
                }
            }
            const int k_slot = (base + last) % K_SLOTS;
            if (ragged) {
                clear_tail(0, K_OFFSET + k_slot * ROWS_BYTES, &bars->k_full[k_slot]);
            }
            if (lane == 0 && alive) {
                load_v(last);
            }
            if (ragged) {
                clear_tail(1, V_OFFSET, &bars->v_full);
                ++tails;
            }
            alive = __all_sync(0xffffffffU, alive);
            ++n;
            base += tile_count;
        }
    } else if (warp == MMA_WARP) {
        const uint32_t leader = elect_one();
        constexpr uint32_t IDESC_SCORE = make_idesc_bf16(BIG, KEYS, false, false);
        constexpr uint32_t IDESC_DQ = make_idesc_bf16(BIG, HEAD, false, true);
        bool alive = true;
        int n = 0, base = 0;
        for (long long index = blockIdx.x; index < items && alive; index += gridDim.x) {
            const Item at = item_at(index);
            if (at.length == 0) {
                continue;
            }
            const int tile_count = (at.length + KEYS - 1) / KEYS;
            const uint32_t q_smem = smem_base + n % Q_SLOTS * ROWS_BYTES;
            auto wait = [&](uint64_t* barrier, int parity) {
                return __all_sync(0xffffffffU, mbar_wait(smem_u32(barrier), parity & 1, abort_flag, &cross_query_short_status)) != 0;
            };
            // S(t) = Q K_t^T, once the softmax has taken the scores of the tile before
            auto issue_s = [&](int t) {
                alive = wait(&bars->k_full[t % K_SLOTS], t / K_SLOTS) && (t == 0 || wait(&bars->s_free, t - 1));
                if (!alive) {
                    return;
                }
                tc_fence_after_sync();
                const uint32_t k_smem = smem_base + K_OFFSET + t % K_SLOTS * ROWS_BYTES;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ss_elect(tmem_base + TMEM_S, make_kmajor_desc(q_smem + c * BIG_CHUNK + k * 32), make_kmajor_desc(k_smem + c * BIG_CHUNK + k * 32),
                                     IDESC_SCORE, (c | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->s_full), leader);
            };
            auto issue_dp = [&](int t) {
                alive = wait(&bars->v_full, t);
                if (!alive) {
                    return;
                }
                tc_fence_after_sync();
                const uint32_t v_smem = smem_base + V_OFFSET;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ts_elect(tmem_base + TMEM_DP, tmem_base + TMEM_DO + c * 32 + k * 8, make_kmajor_desc(v_smem + c * BIG_CHUNK + k * 32), IDESC_SCORE,
                                     (c | k) != 0 ? 1U : 0U, leader);
                    }
                }
                mma_commit_elect(smem_u32(&bars->v_empty), leader);
                mma_commit_elect(smem_u32(&bars->dp_full), leader);
            };
            alive = wait(&bars->q_full[n % Q_SLOTS], n / Q_SLOTS);
            if (alive) {
                issue_s(base);              // (beside the softmax warps' work on the last item's dQ)
            }
            if (alive) {
                alive = wait(&bars->do_copied, n);
            }
            if (alive) {
                tc_fence_after_sync();
                issue_dp(base);
            }
            for (int t = base; t < base + tile_count && alive; ++t) {
                if (t + 1 < base + tile_count) {
                    issue_s(t + 1);
                    if (!alive) {
                        break;
                    }
                }
                // (all softmax threads have read the last item's dQ when they hand over the first dS of this one)
                alive = wait(&bars->ds_full, t);
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                const uint32_t k_smem = smem_base + K_OFFSET + t % K_SLOTS * ROWS_BYTES;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    mma_ts_elect(tmem_base + TMEM_DQ, tmem_base + TMEM_DP + (k / 4) * 64 + (k % 4) * 8, make_smem_desc(k_smem + k * 2048, BIG_CHUNK, 1024), IDESC_DQ,
                                 t > base || k != 0 ? 1U : 0U, leader);
                }
                mma_commit_elect(smem_u32(&bars->k_empty[t % K_SLOTS]), leader);
                if (t + 1 < base + tile_count) {
                    issue_dp(t + 1);
                }
            }
            if (alive) {
                mma_commit_elect(smem_u32(&bars->final_full), leader);
            }
            ++n;
            base += tile_count;
        }
    } else {
        const int half = warp / 4;
        const int r = threadIdx.x % BIG;
        const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base + TMEM_S + half * 64;
        const uint32_t dp_tmem = tmem_base + lane_base + TMEM_DP + half * 64;
        const int my_token = r / p.group, my_head = r - my_token * p.group;
        auto wait = [&](uint64_t* barrier, int parity) {
            return __all_sync(0xffffffffU, mbar_wait(smem_u32(barrier), parity & 1, abort_flag, &cross_query_short_status)) != 0;
        };
        bool alive = true;
        int n = 0, base = 0, single = 0;
        for (long long index = blockIdx.x; index < items && alive; index += gridDim.x) {
            const Item at = item_at(index);
            if (at.length == 0) {
                // rows of an entry without keys: half a warp to a row
                const int rows = min(p.big_tokens, p.tokens - at.token0) * p.group;
                for (int row = warp * 2 + lane / 16; row < rows; row += 2 * MMA_WARP) {
                    reinterpret_cast<uint4*>(p.dq_out + ((static_cast<size_t>(at.entry) * p.tokens + at.token0 + row / p.group) * p.kv_heads * p.group +
                                                         at.kv_head * p.group + row % p.group) * HEAD)[lane % 16] = make_uint4(0, 0, 0, 0);
                }
                continue;
            }
            const int tile_count = (at.length + KEYS - 1) / KEYS;
            const int token = at.token0 + my_token;
            const bool valid = r < rows_per_tile && token < p.tokens;
            float lse2 = INFINITY;
            if (valid) {
                lse2 = p.lse[(static_cast<size_t>(at.entry) * p.kv_heads * p.group + at.kv_head * p.group + my_head) * p.tokens + token] * LOG2E;
            }
            alive = wait(&bars->o_full, n);
            if (!alive) {
                break;
            }
            {
                // dO chunk `half`, row r, into 32 packed columns of tensor memory (without the 128-byte swizzle); the last item's products with dO are done
                uint32_t values[32];
                const uint8_t* row = smem + DO_OFFSET + half * BIG_CHUNK + r * 128;
                const uint8_t* out = smem + O_OFFSET + half * BIG_CHUNK + r * 128;
#pragma unroll
                for (int unit = 0; unit < 8; ++unit) {
                    const uint4 v = *reinterpret_cast<const uint4*>(row + ((unit ^ (r & 7)) * 16));
                    values[unit * 4 + 0] = v.x;
                    values[unit * 4 + 1] = v.y;
                    values[unit * 4 + 2] = v.z;
                    values[unit * 4 + 3] = v.w;
                }
                tmem_st_x32(tmem_base + lane_base + TMEM_DO + half * 32, values);
                if (tile_count > 1) {
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
                    bars->delta[half][r] = share;
                }
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&bars->do_copied));
            }
            alive = wait(&bars->do_copied, n);
            if (!alive) {
                break;
            }
            float delta = tile_count > 1 ? bars->delta[0][r] + bars->delta[1][r] : 0.0F;
            float2* row = valid && half == 0
                              ? p.rows + ((static_cast<size_t>(at.entry) * p.kv_heads + at.kv_head) * p.tokens + token) * p.group + my_head
                              : nullptr;
            if (row != nullptr && tile_count > 1) {
                *row = make_float2(lse2, delta);
            }
            for (int j = 0; j < tile_count; ++j) {
                alive = wait(&bars->s_full, base + j);
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
                for (int k = 0; k < 64; ++k) {
                    prob[k] = exp2_approx(fmaf(__uint_as_float(sb[k]), p.scale_log2, -lse2)) * p.scale;
                }
                if (j + 1 == tile_count) {
                    const int present = at.length - j * KEYS - half * 64;
#pragma unroll
                    for (int k = 0; k < 64; ++k) {
                        prob[k] = k < present ? prob[k] : 0.0F;
                    }
                }
                alive = wait(&bars->dp_full, base + j);
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                tmem_ld_x32(dp_tmem, sb);
                tmem_ld_x32(dp_tmem + 32, sb + 32);
                tmem_wait_ld();
                if (tile_count == 1) {
                    // the exact delta, from the tile that holds all keys
                    float share = 0.0F;
#pragma unroll
                    for (int k = 0; k < 64; ++k) {
                        share = fmaf(prob[k], __uint_as_float(sb[k]), share);
                    }
                    bars->delta[half][r] = share;
                    mbar_arrive(smem_u32(&bars->delta_full));
                    alive = wait(&bars->delta_full, single);
                    ++single;
                    if (!alive) {
                        break;
                    }
                    delta = (bars->delta[0][r] + bars->delta[1][r]) / p.scale;
                    if (row != nullptr) {
                        *row = make_float2(lse2, delta);
                    }
                }
                uint32_t packed[32];
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    packed[k / 2] = pack_bf16x2(prob[k] * (__uint_as_float(sb[k]) - delta), prob[k + 1] * (__uint_as_float(sb[k + 1]) - delta));
                }
                tmem_st_x32(dp_tmem, packed);
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&bars->ds_full));
            }
            if (alive) {
                alive = wait(&bars->final_full, n);
            }
            if (!alive) {
                break;
            }
            tc_fence_after_sync();
            // dQ leaves through Q's place
            const int place = n % Q_SLOTS * ROWS_BYTES;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t values[32];
                tmem_ld_x32(tmem_base + lane_base + TMEM_DQ + half * 64 + c * 32, values);
                tmem_wait_ld();
                stage_bf16x32(smem + place + half * BIG_CHUNK, r, c, values, at.length > 1);     // (one key: its weight is 1 whatever the score)
            }
            tc_fence_before_sync();
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&bars->staged));
            if (threadIdx.x == 0 && mbar_wait(smem_u32(&bars->staged), n & 1, abort_flag, &cross_query_short_status)) {
                for (int c = 0; c < 2; ++c) {
                    tma_store_4d(&p.dq, smem_base + place + c * BIG_CHUNK, c * 64, at.kv_head * p.group, at.token0, at.entry);
                }
                tma_store_commit();
                tma_store_wait_read();
                mbar_arrive(smem_u32(&bars->q_empty[n % Q_SLOTS]));
            }
            __syncwarp();
            ++n;
            base += tile_count;
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
    CUDA_CHECK(cudaFuncSetAttribute(cross_query_short_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
    if (device < 16) {
        done[device] = true;
    }
}

}  // namespace

namespace internal {

int cross_query_short_device_status(bool reset) {
    int status = 0;
    CUDA_CHECK(cudaDeviceSynchronize());
    CUDA_CHECK(cudaMemcpyFromSymbol(&status, cross_query_short_status, sizeof(int)));
    if (reset && status != 0) {
        const int zero = 0;
        CUDA_CHECK(cudaMemcpyToSymbol(cross_query_short_status, &zero, sizeof(int)));
    }
    return status;
}

}  // namespace internal

bool cross_query_short_takes(long long items, long long key_tiles) {
    return items > (key_tiles <= 2 ? 2 : 4) * SMS && key_tiles <= 8;
}

void launch_cross_query_short(const CrossBackwardParams& p, cudaStream_t stream) {
    configure();
    launch_chained(cross_query_short_kernel, dim3(static_cast<unsigned>(SMS)), dim3(THREADS), SMEM_BYTES, stream, p);
}

}  // namespace dscuda
