// Declarations shared between the attention translation units and the C-ABI
// bridges; not part of the public headers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "flash_attention.h"

#include <cstddef>
#include <initializer_list>

namespace dscuda {
namespace internal {

// Throws std::invalid_argument unless the arguments describe a supported
// non-absorbed prefill problem (128/64/128 head sizes, positive sizes and scale,
// index ranges that fit the kernels).
void check_prefill_shape(const int* cu_seqlens, int batch_size, int max_sequence_length, int total_tokens, int heads,
                         int nope_size, int rope_size, int value_size, float scale);

void launch_prefill_forward(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* q_nope, const __nv_bfloat16* q_pe,
                            const __nv_bfloat16* k_nope, const __nv_bfloat16* k_pe, const __nv_bfloat16* v, const int* cu_seqlens,
                            int batch_size, int max_sequence_length, int total_tokens, int heads, float scale,
                            cudaStream_t stream);

// Throws std::invalid_argument for null pointers and for tensors that are not 16-byte (the first list) or 4-byte aligned.
void check_flash_pointers(std::initializer_list<const void*> wide, std::initializer_list<const void*> narrow);

// Throws std::invalid_argument unless the arguments describe an 8-bit paged cache that the kernels can index.
void check_flash_cache_shape(int batch_size, int tokens, int key_value_heads, int head_size, int page_size, int pages_per_sequence,
                             int cache_blocks, FlashCacheType type);

// Throws std::invalid_argument unless the arguments describe a supported cross attention.
void check_flash_cross_shape(int batch_size, int query_length, int key_length, int query_heads, int key_value_heads, int head_size, float scale);

// Cross attention of few query rows to a key head (group * tokens) on the kernels of flash_decode.cu, and its workspace.
std::size_t few_rows_workspace_bytes(int batch, int key_value_heads, long long rows);
void launch_few_rows_cross(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* query, const __nv_bfloat16* key, const __nv_bfloat16* value,
                           const int* key_lengths, void* workspace, int batch, int tokens, int keys, int query_heads, int key_value_heads, float scale,
                           cudaStream_t stream);

// Per-translation-unit sticky status words (0 = fine).  Reading synchronises.
int forward_device_status(bool reset);
int absorbed_backward_device_status(bool reset);
int decode_device_status(bool reset);
int projection_device_status(bool reset);
int backward_device_status(bool reset);
int append_device_status(bool reset);
int flash_cache_device_status(bool reset);
int flash_decode_device_status(bool reset);
int cross_forward_device_status(bool reset);
int cross_backward_device_status(bool reset);
int cross_backward_short_device_status(bool reset);
int cross_query_short_device_status(bool reset);

}  // namespace internal
}  // namespace dscuda
