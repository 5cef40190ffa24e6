// dK and dV of the cross attention for short loops (few rows under many keys), the second kernel of cross_backward.cu otherwise: the same products and sums in the
// same order.  A CTA goes over several items (128 keys of a head and entry): the K and V of the next one arrive, and its first scores run, while this one's
// gradients leave, where a CTA to an item spends most of its time on its beginning and end.  The price is a stage of rows less, and items in a fixed
// share, so long loops stay with the other form.  Backward, us, this form and the other: 12 tokens x 7 heads (2 row tiles) over 5942 keys 47.9 and 58.5, 64 tokens
// (1) over 1500 keys and 256 heads 130 and 187, 448 tokens (7) 183 and 207, 256 x 4 rows (16) 67.8 and 67.6, 858 x 4 rows (54) 84.9 and 83.4, 1665 x 4
// rows (105) 316 and 304; with fewer than two items to a CTA 584 tokens (10) over 12 keys and 208 heads 75.2 and 74.5.
#include "attention_internal.h"
#include "cuda_common.h"
#include "cross_backward.cuh"
#include "loop_parts.cuh"
#include "../common/launch.h"

#include <cstdint>

namespace dscuda {
namespace {

using namespace cross;

__device__ int cross_backward_short_status = 0;

constexpr int STAGES = 3;
constexpr int STAGE_BYTES = 4 * SUB_CHUNK;          // Q and dO of 64 rows
constexpr int RESIDENT_BYTES = 4 * BIG_CHUNK;       // K and V of 128 keys
constexpr int RESIDENTS = 2;
constexpr int STREAM_OFFSET = RESIDENTS * RESIDENT_BYTES;
constexpr int MISC_OFFSET = STREAM_OFFSET + STAGES * STAGE_BYTES;
constexpr int MISC_BYTES = 2048;
constexpr int SMEM_BYTES = MISC_OFFSET + MISC_BYTES + 1024;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of a CTA");
constexpr uint32_t TMEM_DV = 0;
constexpr uint32_t TMEM_DK = 128;
constexpr uint32_t TMEM_S = 256;                    // two pairs of S^T and dP^T, 64 columns each

struct Barriers {
    uint64_t resident_full[RESIDENTS];
    uint64_t resident_empty[RESIDENTS];
    uint64_t stage_full[STAGES];
    uint64_t stage_empty[STAGES];
    uint64_t s_full[2];
    uint64_t dp_full[2];
    uint64_t p_full[2];
    uint64_t ds_full[2];
    uint64_t final_full;
    uint64_t staged[2];
    uint32_t tmem_base;
    int abort_flag;
    int gave_up;
    alignas(16) float lse2[STAGES][SUB];
    alignas(16) float delta[STAGES][SUB];
};
static_assert(sizeof(Barriers) <= MISC_BYTES, "barrier block too large");

// The tensor core's share of a row tile, by the elected lane: S^T = K Q^T with dP^T = V dO^T behind it ..
__device__ __forceinline__ void issue_tile_scores(uint32_t scores, uint32_t k_smem, uint32_t v_smem, uint32_t q_smem, uint64_t* s_full, uint64_t* dp_full, uint32_t leader) {
    constexpr uint32_t IDESC = make_idesc_bf16(BIG, SUB, false, false);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            mma_ss_elect(scores, make_kmajor_desc(k_smem + c * BIG_CHUNK + k * 32), make_kmajor_desc(q_smem + c * SUB_CHUNK + k * 32), IDESC, (c | k) != 0 ? 1U : 0U, leader);
        }
    }
    mma_commit_elect(smem_u32(s_full), leader);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            mma_ss_elect(scores + 64, make_kmajor_desc(v_smem + c * BIG_CHUNK + k * 32), make_kmajor_desc(q_smem + (2 + c) * SUB_CHUNK + k * 32), IDESC,
                         (c | k) != 0 ? 1U : 0U, leader);
        }
    }
    mma_commit_elect(smem_u32(dp_full), leader);
}

// .. and sums += weights^T rows (dV += P^T dO, dK += dS^T Q); rows 32 g .. 32 g + 31 are packed into columns 32 g .. 32 g + 15 of their score tile.
__device__ __forceinline__ void issue_gradient(uint32_t sums, uint32_t weights, uint32_t rows_smem, bool first, uint32_t leader) {
    constexpr uint32_t IDESC = make_idesc_bf16(BIG, HEAD, false, true);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        mma_ts_elect(sums, weights + (k / 2) * 32 + (k % 2) * 8, make_smem_desc(rows_smem + k * 2048, SUB_CHUNK, 1024), IDESC, !first || k != 0 ? 1U : 0U, leader);
    }
}

// A thread's key and 32 rows: P from the scores and the rows' logarithms, kept in fp32 and written back in bf16 ..
__device__ __forceinline__ void weights_of_rows(float (&prob)[32], uint32_t s_tmem, const float* lse2, float scale_log2) {
    const float4* lse4 = reinterpret_cast<const float4*>(lse2);
    uint32_t sb[32], packed[16];
    tmem_ld_x32(s_tmem, sb);
    tmem_wait_ld();
#pragma unroll
    for (int n = 0; n < 32; n += 4) {
        const float4 l = lse4[n / 4];
        prob[n] = exp2_approx(fmaf(__uint_as_float(sb[n]), scale_log2, -l.x));
        prob[n + 1] = exp2_approx(fmaf(__uint_as_float(sb[n + 1]), scale_log2, -l.y));
        prob[n + 2] = exp2_approx(fmaf(__uint_as_float(sb[n + 2]), scale_log2, -l.z));
        prob[n + 3] = exp2_approx(fmaf(__uint_as_float(sb[n + 3]), scale_log2, -l.w));
        packed[n / 2] = pack_bf16x2(prob[n], prob[n + 1]);
        packed[n / 2 + 1] = pack_bf16x2(prob[n + 2], prob[n + 3]);
    }
    tmem_st_x16(s_tmem, packed);
    tmem_wait_st();
}

// .. and dS = P (dP - delta) scale.
__device__ __forceinline__ void score_gradients(const float (&prob)[32], uint32_t dp_tmem, const float* delta, float scale) {
    const float4* delta4 = reinterpret_cast<const float4*>(delta);
    uint32_t sb[32], packed[16];
    tmem_ld_x32(dp_tmem, sb);
    tmem_wait_ld();
#pragma unroll
    for (int n = 0; n < 32; n += 4) {
        const float4 d = delta4[n / 4];
        packed[n / 2] = pack_bf16x2(prob[n] * (__uint_as_float(sb[n]) - d.x) * scale, prob[n + 1] * (__uint_as_float(sb[n + 1]) - d.y) * scale);
        packed[n / 2 + 1] = pack_bf16x2(prob[n + 2] * (__uint_as_float(sb[n + 2]) - d.z) * scale, prob[n + 3] * (__uint_as_float(sb[n + 3]) - d.w) * scale);
    }
    tmem_st_x16(dp_tmem, packed);
    tmem_wait_st();
}

// A CTA's items (128 keys of a head and entry), the grid's size apart: those with keys lie in front of those without, so that a CTA's share of either is known without
// asking the others.  Every warp walks for itself.
struct KeyItems {
    int entry, kv_head, key_start, length;

    __device__ KeyItems(const CrossBackwardParams& params, int first, int warp_lane) : p(params), lane(warp_lane), index(first) {
        load();
    }

    __device__ bool next() {
        index += gridDim.x;
        return find();
    }

    __device__ bool find() {
        for (;;) {
            const int inside = index - before;
            const unsigned mine = __ballot_sync(0xffffffffU, inside < inclusive);
            if (mine != 0) {
                const int source = __ffs(mine) - 1;
                const int of_entry = __shfl_sync(0xffffffffU, own, source);
                const int offset = inside - (__shfl_sync(0xffffffffU, inclusive, source) - of_entry);
                length = __shfl_sync(0xffffffffU, own_length, source);
                entry = base + source;
                const int tiles = of_entry / p.kv_heads;
                kv_head = offset / tiles;
                key_start = (offset - kv_head * tiles + (empty ? (length + BIG - 1) / BIG : 0)) * BIG;
                return true;
            }
            before += __shfl_sync(0xffffffffU, inclusive, 31);
            base += 32;
            if (base >= p.batch) {
                if (empty) {
                    return false;
                }
                empty = true;
                base = 0;
            }
            load();
        }
    }

private:
    __device__ void load() {
        const bool there = base + lane < p.batch;
        own_length = there ? length_of(p, base + lane) : 0;
        const int tiles = (own_length + BIG - 1) / BIG;
        own = !there ? 0 : (empty ? p.key_tiles - tiles : tiles) * p.kv_heads;
        inclusive = own;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xffffffffU, inclusive, offset);
            inclusive += lane >= offset ? other : 0;
        }
    }

    const CrossBackwardParams& p;
    int lane, index;
    int base = 0, before = 0;           // entries base .. base + 31 are looked at, `before` items lie in front of theirs
    bool empty = false;                 // among the items without keys
    int own, own_length, inclusive;     // of entry base + lane
};
__global__ void __launch_bounds__(THREADS, 1) cross_key_short_kernel(const __grid_constant__ CrossBackwardParams p) {
    extern __shared__ uint8_t smem_raw[];
    const int rows_per_tile = p.sub_tokens * p.group;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023U) & ~1023U;
    uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t stage_smem = smem_base + STREAM_OFFSET;
    Barriers* bars = reinterpret_cast<Barriers*>(smem + MISC_OFFSET);
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < RESIDENTS; ++i) {
            mbar_init(smem_u32(&bars->resident_full[i]), 1);
            mbar_init(smem_u32(&bars->resident_empty[i]), 2);   // the stores of dV and dK from its place
        }
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
        // after an earlier launch ran into a time limit nothing is done
        bars->gave_up = *reinterpret_cast<volatile int*>(&cross_backward_short_status);
        mbar_init_fence();
    }
    if (warp == MMA_WARP) {
        tmem_alloc(smem_u32(&bars->tmem_base), TMEM_COLUMNS);
        tmem_relinquish();
    }
    if (rows_per_tile < SUB && warp < MMA_WARP) {
        // rows that no load fills: dV += P^T dO and dK += dS^T Q multiply them by zeros
        for (int chunk = warp; chunk < STAGES * 4; chunk += MMA_WARP) {
            clear_rows(smem + STREAM_OFFSET + chunk * SUB_CHUNK, rows_per_tile, SUB, lane);
        }
        fence_proxy_async_smem();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    grid_dependency_wait();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    const int tile_count = (p.tokens + p.sub_tokens - 1) / p.sub_tokens;
    const bool dead = *reinterpret_cast<volatile int*>(&bars->gave_up) != 0;
    // Each role goes over the CTA's items: `n` counts those with keys, `base` their tiles.
    auto over_items = [&](auto&& work) {
        int n = 0;
        KeyItems at(p, blockIdx.x, lane);
        for (bool more = !dead && at.find(); more; more = at.next()) {
            if (!work(at, n, n * tile_count)) {
                break;
            }
            n += at.key_start < at.length;
        }
    };
    if (warp == LOAD_WARP) {
        bool alive = true;
        over_items([&](const auto& at, const int n, const int base) {
            if (at.key_start >= at.length) {
                return false;               // only the softmax warps have to do with items without keys, which come last
            }
            const int buffer = n % RESIDENTS;
            if (n >= RESIDENTS) {
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->resident_empty[buffer]), (n / RESIDENTS - 1) & 1, abort_flag, &cross_backward_short_status));
                if (!alive) {
                    return false;
                }
            }
            if (lane == 0) {
                const uint32_t bar = smem_u32(&bars->resident_full[buffer]);
                const uint32_t dst = smem_base + buffer * RESIDENT_BYTES;
                mbar_arrive_expect_tx(bar, RESIDENT_BYTES);
                for (int c = 0; c < 2; ++c) {
                    tma_load_3d(dst + c * BIG_CHUNK, &p.k, bar, at.kv_head * HEAD + c * 64, at.key_start, at.entry);
                    tma_load_3d(dst + (2 + c) * BIG_CHUNK, &p.v, bar, at.kv_head * HEAD + c * 64, at.key_start, at.entry);
                }
            }
            const float2* constants = p.rows + (static_cast<size_t>(at.entry) * p.kv_heads + at.kv_head) * p.tokens * p.group;
            for (int t = 0; t < tile_count; ++t) {
                const int stage = (base + t) % STAGES;
                const int use = (base + t) / STAGES;
                if (use > 0) {
                    alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->stage_empty[stage]), (use - 1) & 1, abort_flag, &cross_backward_short_status));
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
                        tma_load_4d(dst + c * SUB_CHUNK, &p.q_sub, full, c * 64, at.kv_head * p.group, token, at.entry);
                        tma_load_4d(dst + (2 + c) * SUB_CHUNK, &p.do_sub, full, c * 64, at.kv_head * p.group, token, at.entry);
                    }
                }
                const int present = min(rows_per_tile, (p.tokens - token) * p.group);
#pragma unroll
                for (int e = 0; e < SUB / 32; ++e) {
                    const int row = e * 32 + lane;
                    const float2 both = row < present ? constants[static_cast<size_t>(token) * p.group + row] : make_float2(INFINITY, 0.0F);
                    bars->lse2[stage][row] = both.x;
                    bars->delta[stage][row] = both.y;
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(full);
                }
            }
            return alive;
        });
    } else if (warp == MMA_WARP) {
        const uint32_t leader = elect_one();
        bool alive = true;
        over_items([&](const auto& at, const int n, const int base) {
            if (at.key_start >= at.length) {
                return false;               // only the softmax warps have to do with items without keys, which come last
            }
            const uint32_t k_smem = smem_base + n % RESIDENTS * RESIDENT_BYTES;
            const uint32_t v_smem = k_smem + 2 * BIG_CHUNK;
            alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->resident_full[n % RESIDENTS]), (n / RESIDENTS) & 1, abort_flag, &cross_backward_short_status));
            // S^T(t) = K Q_t^T and dP^T(t) = V dO_t^T
            auto issue_scores = [&](int t) {
                const int stage = t % STAGES;
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->stage_full[stage]), (t / STAGES) & 1, abort_flag, &cross_backward_short_status));
                if (!alive) {
                    return;
                }
                tc_fence_after_sync();
                const uint32_t q_smem = stage_smem + stage * STAGE_BYTES;
                const uint32_t scores = tmem_base + TMEM_S + (t & 1) * 128;
                issue_tile_scores(scores, k_smem, v_smem, q_smem, &bars->s_full[t & 1], &bars->dp_full[t & 1], leader);
            };
            if (alive) {
                issue_scores(base);         // (beside the softmax warps' work on the last item's results)
            }
            for (int t = base; t < base + tile_count && alive; ++t) {
                const int stage = t % STAGES;
                const uint32_t parity = (t >> 1) & 1;
                if (t + 1 < base + tile_count) {
                    issue_scores(t + 1);
                    if (!alive) {
                        break;
                    }
                }
                const uint32_t q_smem = stage_smem + stage * STAGE_BYTES;
                const uint32_t scores = tmem_base + TMEM_S + (t & 1) * 128;
                // (all softmax threads have read the last item's dV and dK when they hand over the first P of this one)
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->p_full[t & 1]), parity, abort_flag, &cross_backward_short_status));
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                issue_gradient(tmem_base + TMEM_DV, scores, q_smem + 2 * SUB_CHUNK, t == base, leader);
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->ds_full[t & 1]), parity, abort_flag, &cross_backward_short_status));
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                issue_gradient(tmem_base + TMEM_DK, scores + 64, q_smem, t == base, leader);
                mma_commit_elect(smem_u32(&bars->stage_empty[stage]), leader);
            }
            if (alive) {
                mma_commit_elect(smem_u32(&bars->final_full), leader);
            }
            return alive;
        });
    } else {
        const int group = warp / 4;                     // 0 stores dV, 1 dK
        const int r = threadIdx.x % BIG;
        const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
        bool alive = true;
        over_items([&](const auto& at, const int n, const int base) {
            if (at.key_start >= at.length) {
                // half a warp to a row
                __nv_bfloat16* out = group == 0 ? p.dv_out : p.dk_out;
                for (int k = warp % 4 * 32 + lane / 16; k < warp % 4 * 32 + 32; k += 2) {
                    if (at.key_start + k < p.keys) {
                        reinterpret_cast<uint4*>(out + ((static_cast<size_t>(at.entry) * p.keys + at.key_start + k) * p.kv_heads + at.kv_head) * HEAD)[lane % 16] =
                            make_uint4(0, 0, 0, 0);
                    }
                }
                return true;
            }
            for (int t = base; t < base + tile_count; ++t) {
                const int stage = t % STAGES;
                const uint32_t parity = (t >> 1) & 1;
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->stage_full[stage]), (t / STAGES) & 1, abort_flag, &cross_backward_short_status) &&
                                                    mbar_wait(smem_u32(&bars->s_full[t & 1]), parity, abort_flag, &cross_backward_short_status));
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                const uint32_t s_tmem = tmem_base + lane_base + TMEM_S + (t & 1) * 128 + group * 32;
                float prob[32];
                weights_of_rows(prob, s_tmem, bars->lse2[stage] + group * 32, p.scale_log2);
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&bars->p_full[t & 1]));

                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->dp_full[t & 1]), parity, abort_flag, &cross_backward_short_status));
                if (!alive) {
                    break;
                }
                tc_fence_after_sync();
                score_gradients(prob, s_tmem + 64, bars->delta[stage] + group * 32, at.length == 1 ? 0.0F : p.scale);      // (one key: its weight is 1 whatever the score)
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&bars->ds_full[t & 1]));
            }
            if (alive) {
                alive = __all_sync(0xffffffffU, mbar_wait(smem_u32(&bars->final_full), n & 1, abort_flag, &cross_backward_short_status));
            }
            if (!alive) {
                return false;
            }
            tc_fence_after_sync();
            // dV leaves through V's place, dK through K's
            const int buffer = n % RESIDENTS;
            const int offset = buffer * RESIDENT_BYTES + (group == 0 ? 2 * BIG_CHUNK : 0);
            const bool keep = at.key_start + r < at.length;
#pragma unroll
            for (int c = 0; c < HEAD / 32; ++c) {
                uint32_t values[32];
                tmem_ld_x32(tmem_base + lane_base + (group == 0 ? TMEM_DV : TMEM_DK) + c * 32, values);
                tmem_wait_ld();
                stage_bf16x32(smem + offset + (c / 2) * BIG_CHUNK, r, c % 2, values, keep);
            }
            tc_fence_before_sync();
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&bars->staged[group]));
            if (r == 0 && mbar_wait(smem_u32(&bars->staged[group]), n & 1, abort_flag, &cross_backward_short_status)) {
                for (int c = 0; c < 2; ++c) {
                    tma_store_3d(group == 0 ? &p.dv : &p.dk, smem_base + offset + c * BIG_CHUNK, at.kv_head * HEAD + c * 64, at.key_start, at.entry);
                }
                tma_store_commit();
                tma_store_wait_read();
                mbar_arrive(smem_u32(&bars->resident_empty[buffer]));
            }
            __syncwarp();
            return alive;
        });
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
    CUDA_CHECK(cudaFuncSetAttribute(cross_key_short_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
    if (device < 16) {
        done[device] = true;
    }
}

}  // namespace

namespace internal {

int cross_backward_short_device_status(bool reset) {
    int status = 0;
    CUDA_CHECK(cudaDeviceSynchronize());
    CUDA_CHECK(cudaMemcpyFromSymbol(&status, cross_backward_short_status, sizeof(int)));
    if (reset && status != 0) {
        const int zero = 0;
        CUDA_CHECK(cudaMemcpyToSymbol(cross_backward_short_status, &zero, sizeof(int)));
    }
    return status;
}

}  // namespace internal

bool cross_key_short_takes(long long items, long long row_tiles) {
    return items > 2 * SMS && row_tiles <= 12;
}

void launch_cross_key_short(const CrossBackwardParams& p, cudaStream_t stream) {
    configure();
    launch_chained(cross_key_short_kernel, dim3(static_cast<unsigned>(SMS)), dim3(THREADS), SMEM_BYTES, stream, p);
}

}  // namespace dscuda
