// paged_internal.h -- launch-side structures shared by the paged-cache kernels and their C ABI.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "odf_internal.h"
#include "odf_paged_sm100.h"

namespace odf {

// One layer of a cache as the kernels see it (strides in bytes, validated, resolved).
struct PagedView {
    uint8_t* k;
    uint8_t* v;
    int64_t k_page, k_head, k_slot;
    int64_t v_page, v_head, v_slot;
    const int32_t* table;
    int64_t table_stride;
    int32_t max_pages, num_pages, page_size, heads_kv;
    FastDiv fd_page;  // by page_size
    const float* k_scale;
    const float* v_scale;
    int* status;
};

struct DecodeArgs {
    PagedView c;
    // the cache's strides in 16-byte units
    uint32_t k16_page, k16_head, k16_slot, v16_page, v16_head, v16_slot;
    const int32_t* lens;
    int32_t batch, heads_q, group;
    int32_t row_tiles, items_per_seq;  // items of one sequence: kv-heads x blocks of query heads
    FastDiv fd_items;                  // by items_per_seq
    int32_t window, sinks;             // window 0 = every key
    const void* q;
    int64_t q_b, q_h;  // elements
    void* o;
    int64_t o_b, o_h;  // elements
    float* lse;
    void* workspace;
    int32_t o_bf16, sm_count;
    float scale;
    float softcap, inv_softcap;
    int32_t has_alibi, alibi_generated;
    float alibi_slopes[ODF_MAX_EXPLICIT_SLOPES];
};

struct AppendArgs {
    PagedView c;
    const void* k;
    const void* v;
    int64_t k_b, k_h, k_t, v_b, v_h, v_t;  // elements
    const int32_t* starts;
    const int32_t* counts;
    int32_t batch, tokens, sm_count;
    FastDiv fd_tokens, fd_heads;
};

// Pages are copied as runs of consecutive bytes: a page is heads x slots rows of head_dim
// elements, joined into longer runs where the strides allow.
struct CopyArgs {
    uint8_t* base[2];                 // K and V
    int64_t page[2], layer[2];        // bytes
    int64_t outer_stride[2], inner_stride[2];  // bytes between runs
    int32_t outer[2], inner[2];       // runs per page: outer x inner
    int64_t run_bytes[2];
    int32_t layers;
    const int32_t* pairs;             // host
    int64_t n_pairs;
};

// Whether the slices of a decode call, as the kernel counts them, stay within its 32 bits (no CUDA call).  Reads the
// cache's sizes, batch, group, window and sinks.
bool decode_work_fits(const DecodeArgs& a, int32_t head_dim, int32_t kv_dtype);
int launch_paged_decode(DecodeArgs& a, int32_t head_dim, int32_t kv_dtype, cudaStream_t stream, const char** err);
int launch_paged_append(AppendArgs& a, int32_t head_dim, int32_t kv_dtype, cudaStream_t stream, const char** err);
int launch_page_copy(const CopyArgs& a, cudaStream_t stream, const char** err);
size_t decode_workspace_bytes(int32_t head_dim);

}  // namespace odf
