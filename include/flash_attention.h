// Causal D=128 grouped-query attention forward.  Drop-in for the reference's
// include/flash_attention.h:12-24 (same name, arguments and layouts).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstddef>

namespace dscuda {

// Q/O are BF16 [B,T,Hq,128], K/V are BF16 [B,T,Hkv,128], the natural-log LSE is
// FP32 [B,Hq,T].  Hq must be divisible by Hkv and head_size must be 128.  The
// reference demands T % 64 == 0 (kernels/attention/flash_attention/
// sm89_forward.cu:226-228); this implementation accepts any T >= 1.
// Launch-only on `stream`: no allocation, no synchronisation, capturable in a
// CUDA graph.  Throws std::invalid_argument / std::runtime_error.
void flash_attention_forward_cuda(
    __nv_bfloat16* output,
    float* logsumexp,
    const __nv_bfloat16* query,
    const __nv_bfloat16* key,
    const __nv_bfloat16* value,
    int batch_size,
    int sequence_length,
    int query_heads,
    int key_value_heads,
    int head_size,
    float scale,
    cudaStream_t stream = nullptr);

// ---------------------------------------------------------------------------
// Steps of a grouped-query layer around the forward above (no counterpart in the reference).  The same contract: launch-only on
// `stream`, std::invalid_argument / std::runtime_error.
// ---------------------------------------------------------------------------

// Rotary embedding with one to four position axes (time, height, width ...).  query [rows, Hq, W], key [rows, Hk, W] (either may be
// null with its output), W = 64 or 128; a row of all heads is contiguous, rows lie `*_stride` elements apart, so the parts of a
// fused projection can be given as they are.  Outputs are written with their own strides and may be the inputs (the same pointer
// and stride).  Element i pairs with i + W/2; sections[a] pairs belong to axis a, in order, W/2 in all.  The angle of pair i
// of axis a is positions[a][row] * theta^(-2i/W), or with `restart` theta^(-j / sections[a]) for the j-th pair of its section.
// positions [axes, rows] int32 on the device, sections on the host.  `inverse` turns back: the gradient of the forward.
void flash_rope_cuda(
    __nv_bfloat16* query_output,
    __nv_bfloat16* key_output,
    const __nv_bfloat16* query,
    const __nv_bfloat16* key,
    const int* positions,
    long long rows,
    int query_heads,
    int key_heads,
    int head_size,
    long long query_output_stride,
    long long key_output_stride,
    long long query_stride,
    long long key_stride,
    int axes,
    const int* sections,
    bool restart,
    bool inverse,
    float theta,
    cudaStream_t stream = nullptr);

// The paged cache in 8 bits: keys and values each as codes [cache_blocks, Hkv, page_size, 128] with one FP32 scale for each page and
// head, [cache_blocks, Hkv]; value = code * scale, with the scales that flash_cache_append_cuda writes.  page_size is a multiple of 16.
enum class FlashCacheType : int {
    INT8 = 0,           // codes -127..127
    E4M3 = 1,           // codes up to +-448
};

constexpr int FLASH_DECODE_MAX_TOKENS = 64;

// Writes new tokens.  Token t of sequence b goes to position start_positions[b] + t (0 when null), page
// block_table[b][position / page_size]; token_counts [B] (or null): sequence b appends only its first token_counts[b] of the T rows.
// key, value [B,T,Hkv,128], a token's heads contiguous, tokens `*_stride` elements apart (entries T * stride).
// A page's scale covers the values it holds: need = max|new| * (1/127 or 1/448 as FP32), or 0 when that maximum is below 2^-100; a page that starts
// with a new token takes `need`, another max(its scale, need), and where that raises the scale its older codes are rounded again to
// the new one.  code = round-half-even(x * (1 / scale)).  NaN becomes 0, an infinity the largest code; neither counts for the scale.
// What a page held at and behind the first new position is given up, whether it is written over or not (its codes do not follow the scale).  A
// page must not be written twice in one call, for two sequences or for one.  A position or page number outside the cache is not written
// and sets the device status to 3 (an entry without tokens has no position, whatever its start).
void flash_cache_append_cuda(
    void* key_cache,
    void* value_cache,
    float* key_scale,
    float* value_scale,
    const __nv_bfloat16* key,
    const __nv_bfloat16* value,
    const int* block_table,
    const int* start_positions,
    const int* token_counts,
    int batch_size,
    int tokens,
    int key_value_heads,
    int head_size,
    long long key_stride,
    long long value_stride,
    int page_size,
    int pages_per_sequence,
    int cache_blocks,
    FlashCacheType type,
    cudaStream_t stream = nullptr);

// Bytes of the decode's workspace.
std::size_t flash_decode_workspace_bytes(int batch_size, int tokens, int query_heads, int key_value_heads);

// Attention of the newest T tokens (at most FLASH_DECODE_MAX_TOKENS) over that cache.  query, output [B,T,Hq,128], logsumexp [B,Hq,T].
// cache_lengths [B] counts the new tokens too: token t sees the first cache_lengths[b] - T + 1 + t positions.  A row that sees
// none gets zeros and -inf.  Lengths are read as at least 0 and at most pages_per_sequence * page_size; a page number
// outside [0, cache_blocks) is read as page 0 and sets the device status to 3.  Calls that may run at the same time need
// workspaces of their own.
// How the work is cut depends on what the table can hold (batch, heads and pages_per_sequence * page_size): where that is short (384 to 1280 positions) a sequence stays
// with one CTA to a head and row block and there is one launch, otherwise its parts are joined by a second kernel.  So a table trimmed to the longest sequence
// is the faster one for short sequences, and the same sequence may get other last bits in a table of another width; the same arguments get the same bits.
void flash_decode_cuda(
    __nv_bfloat16* output,
    float* logsumexp,
    const __nv_bfloat16* query,
    const void* key_cache,
    const void* value_cache,
    const float* key_scale,
    const float* value_scale,
    const int* block_table,
    const int* cache_lengths,
    void* workspace,
    std::size_t workspace_bytes,
    int batch_size,
    int tokens,
    int query_heads,
    int key_value_heads,
    int head_size,
    int page_size,
    int pages_per_sequence,
    int cache_blocks,
    FlashCacheType type,
    float scale,
    cudaStream_t stream = nullptr);

// Cross attention: every query sees the first key_lengths[b] of its entry's Tk keys (all when key_lengths is null; lengths are read as
// at least 0 and at most Tk).  query, output [B,Tq,Hq,128], key, value [B,Tk,Hkv,128], logsumexp [B,Hq,Tq].  An entry without keys gets
// zeros and -inf.  What lies behind an entry's length is never used, NaN included.  Calls that may run at the same time need
// workspaces of their own; the size may be 0 (then workspace may be null).  How the work is cut depends on the sizes, Tk among them, not on the lengths: another
// padding may give other last bits, the same arguments give the same.
std::size_t flash_cross_forward_workspace_bytes(int batch_size, int query_length, int key_length, int query_heads, int key_value_heads);

void flash_cross_forward_cuda(
    __nv_bfloat16* output,
    float* logsumexp,
    const __nv_bfloat16* query,
    const __nv_bfloat16* key,
    const __nv_bfloat16* value,
    const int* key_lengths,
    void* workspace,
    std::size_t workspace_bytes,
    int batch_size,
    int query_length,
    int key_length,
    int query_heads,
    int key_value_heads,
    int head_size,
    float scale,
    cudaStream_t stream = nullptr);

// Its gradients, BF16 in the shapes of query, key and value, overwritten; those of keys behind an entry's length are zero, and so are those of the queries and the
// key of an entry with a single key, whose weight is 1 whatever the score.  In entries of more than 128 keys the rounding of `output` reaches the gradients
// (through delta: 0.4 % of them where a softmax sits on two keys).  No atomics: two calls on the same inputs return the same bits.
std::size_t flash_cross_backward_workspace_bytes(int batch_size, int query_length, int key_length, int query_heads, int key_value_heads);

void flash_cross_backward_cuda(
    __nv_bfloat16* query_gradient,
    __nv_bfloat16* key_gradient,
    __nv_bfloat16* value_gradient,
    const __nv_bfloat16* output_gradient,
    const __nv_bfloat16* output,
    const float* logsumexp,
    const __nv_bfloat16* query,
    const __nv_bfloat16* key,
    const __nv_bfloat16* value,
    const int* key_lengths,
    void* workspace,
    std::size_t workspace_bytes,
    int batch_size,
    int query_length,
    int key_length,
    int query_heads,
    int key_value_heads,
    int head_size,
    float scale,
    cudaStream_t stream = nullptr);

}  // namespace dscuda
