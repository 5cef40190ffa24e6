// extern "C" surface of libdscuda_flash_attention_bench.so; same symbols as the
// reference's benchmarks/bindings/flash_attention_bridge.cu:13-30.
#include "flash_attention.h"
#include "../attention/attention_internal.h"

#include <cstddef>
#include <exception>
#include <string>

namespace {
thread_local std::string last_error;
}

extern "C" const char* dscuda_flash_last_error() {
    return last_error.c_str();
}

extern "C" int dscuda_flash_forward(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* query, const __nv_bfloat16* key,
                                    const __nv_bfloat16* value, int batch, int sequence, int query_heads, int key_value_heads,
                                    int dimension, float scale, cudaStream_t stream) {
    try {
        dscuda::flash_attention_forward_cuda(output, logsumexp, query, key, value, batch, sequence, query_heads, key_value_heads,
                                             dimension, scale, stream);
        return 0;
    } catch (const std::exception& error) {
        last_error = error.what();
        return 1;
    }
}

namespace {

template <class Call>
int guarded(Call&& call) {
    try {
        call();
        return 0;
    } catch (const std::exception& error) {
        last_error = error.what();
        return 1;
    }
}

}  // namespace

extern "C" int dscuda_flash_rope(__nv_bfloat16* query_output, __nv_bfloat16* key_output, const __nv_bfloat16* query, const __nv_bfloat16* key,
                                 const int* positions, long long rows, int query_heads, int key_heads, int dimension,
                                 long long query_output_stride, long long key_output_stride, long long query_stride, long long key_stride, int axes,
                                 const int* sections, int restart, int inverse, float theta, cudaStream_t stream) {
    return guarded([&] {
        dscuda::flash_rope_cuda(query_output, key_output, query, key, positions, rows, query_heads, key_heads, dimension, query_output_stride,
                                key_output_stride, query_stride, key_stride, axes, sections, restart != 0, inverse != 0, theta, stream);
    });
}

extern "C" int dscuda_flash_cache_append(void* key_cache, void* value_cache, float* key_scale, float* value_scale, const __nv_bfloat16* key,
                                         const __nv_bfloat16* value, const int* block_table, const int* start_positions, const int* token_counts,
                                         int batch, int tokens, int key_value_heads, int dimension, long long key_stride, long long value_stride,
                                         int page_size, int pages, int cache_blocks, int type, cudaStream_t stream) {
    return guarded([&] {
        dscuda::flash_cache_append_cuda(key_cache, value_cache, key_scale, value_scale, key, value, block_table, start_positions, token_counts, batch,
                                        tokens, key_value_heads, dimension, key_stride, value_stride, page_size, pages, cache_blocks,
                                        static_cast<dscuda::FlashCacheType>(type), stream);
    });
}

extern "C" std::size_t dscuda_flash_decode_workspace_bytes(int batch, int tokens, int query_heads, int key_value_heads) {
    return dscuda::flash_decode_workspace_bytes(batch, tokens, query_heads, key_value_heads);
}

extern "C" int dscuda_flash_decode(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* query, const void* key_cache,
                                   const void* value_cache, const float* key_scale, const float* value_scale, const int* block_table,
                                   const int* lengths, void* workspace, std::size_t workspace_bytes, int batch, int tokens, int query_heads,
                                   int key_value_heads, int dimension, int page_size, int pages, int cache_blocks, int type, float scale,
                                   cudaStream_t stream) {
    return guarded([&] {
        dscuda::flash_decode_cuda(output, logsumexp, query, key_cache, value_cache, key_scale, value_scale, block_table, lengths, workspace,
                                  workspace_bytes, batch, tokens, query_heads, key_value_heads, dimension, page_size, pages, cache_blocks,
                                  static_cast<dscuda::FlashCacheType>(type), scale, stream);
    });
}

extern "C" std::size_t dscuda_flash_cross_forward_workspace_bytes(int batch, int query_length, int key_length, int query_heads, int key_value_heads) {
    return dscuda::flash_cross_forward_workspace_bytes(batch, query_length, key_length, query_heads, key_value_heads);
}

extern "C" int dscuda_flash_cross_forward(__nv_bfloat16* output, float* logsumexp, const __nv_bfloat16* query, const __nv_bfloat16* key,
                                          const __nv_bfloat16* value, const int* key_lengths, void* workspace, std::size_t workspace_bytes,
                                          int batch, int query_length, int key_length, int query_heads, int key_value_heads, int dimension,
                                          float scale, cudaStream_t stream) {
    return guarded([&] {
        dscuda::flash_cross_forward_cuda(output, logsumexp, query, key, value, key_lengths, workspace, workspace_bytes, batch, query_length, key_length,
                                         query_heads, key_value_heads, dimension, scale, stream);
    });
}

extern "C" std::size_t dscuda_flash_cross_backward_workspace_bytes(int batch, int query_length, int key_length, int query_heads, int key_value_heads) {
    return dscuda::flash_cross_backward_workspace_bytes(batch, query_length, key_length, query_heads, key_value_heads);
}

extern "C" int dscuda_flash_cross_backward(__nv_bfloat16* dquery, __nv_bfloat16* dkey, __nv_bfloat16* dvalue, const __nv_bfloat16* dout,
                                           const __nv_bfloat16* output, const float* logsumexp, const __nv_bfloat16* query,
                                           const __nv_bfloat16* key, const __nv_bfloat16* value, const int* key_lengths, void* workspace,
                                           std::size_t workspace_bytes, int batch, int query_length, int key_length, int query_heads,
                                           int key_value_heads, int dimension, float scale, cudaStream_t stream) {
    return guarded([&] {
        dscuda::flash_cross_backward_cuda(dquery, dkey, dvalue, dout, output, logsumexp, query, key, value, key_lengths, workspace, workspace_bytes,
                                          batch, query_length, key_length, query_heads, key_value_heads, dimension, scale, stream);
    });
}

extern "C" int dscuda_flash_device_status(int reset) {
    using namespace dscuda::internal;
    try {
        // every word is read (and reset); the first that is not 0 is reported
        int status = 0;
        for (int (*word)(bool) : {forward_device_status, flash_cache_device_status, flash_decode_device_status, cross_forward_device_status,
                                  cross_backward_device_status, cross_backward_short_device_status, cross_query_short_device_status}) {
            const int value = word(reset != 0);
            status = status != 0 ? status : value;
        }
        return status;
    } catch (const std::exception& error) {
        last_error = error.what();
        return -1;
    }
}
