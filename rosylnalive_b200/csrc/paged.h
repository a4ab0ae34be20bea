// paged.h -- the paged serving step's operators (internal launch interface): the page plan and release, the q/k/v
// append and the attention of new tokens over the paged cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qwen.h"

namespace lrm {

// Codes in the error word (meanings in lrm_cuda.h).
constexpr uint32_t kErrAttnRequest = 0x4001, kErrAttnPage = 0x4002;
constexpr uint32_t kErrPlanRequest = 0x5001, kErrPlanPages = 0x5002, kErrPlanTokens = 0x5003, kErrPlanFree = 0x5004,
                   kErrPlanTable = 0x5005;
constexpr uint32_t kErrReleaseRequest = 0x5011, kErrReleaseCount = 0x5012, kErrReleasePage = 0x5014;
constexpr uint32_t kErrAppendRow = 0x6001;

constexpr int kMaxRequests = 65535, kMaxSeqs = 1 << 17, kMaxSeqPages = 1 << 20, kMaxPoolPages = 1 << 26,
              kMaxStepTokens = 1 << 24;

// Page plan, and with keep_len set the release (cu_seqlens, kv_len, tok_pos, slot_map and max_tokens unused then).
struct PageStepArgs {
    const int32_t *slots, *new_len, *keep_len, *seq_len;
    int32_t *page_table, *free_list;
    const int32_t *free_count;
    int32_t *cu_seqlens, *kv_len, *tok_pos, *slot_map, *seq_len_out, *free_count_out;
    int requests, max_seqs, pages_per_seq, kv_pages, max_tokens;
    uint32_t *err;
};
cudaError_t launch_page_step(const PageStepArgs &a, cudaStream_t st);

struct QkvAppendArgs {
    const __nv_bfloat16 *qkv, *q_norm, *k_norm;  // the gains null: no norm
    const float *cos_t, *sin_t;                  // null: no rotation
    const int32_t *tok_pos, *slot_map;
    __nv_bfloat16 *q_out, *pool;
    int64_t ld_qkv, ld_q;
    int tokens, q_heads, kv_heads, rope_rows;
    int64_t places;  // kv_pages * 16
    float eps;
    uint32_t *err;
};
cudaError_t launch_qkv_append(const QkvAppendArgs &a, cudaStream_t st);

struct PagedAttnArgs {
    const __nv_bfloat16 *q, *pool;
    const int32_t *page_table, *slots, *cu_seqlens, *kv_len;
    __nv_bfloat16 *out;
    uint8_t *workspace;
    int64_t ld_q, ld_out;
    int requests, tokens, q_heads, kv_heads, max_seqs, pages_per_seq, kv_pages;
    float scale_log2;
    uint32_t *err;
};
// Bytes of workspace for `tokens` rows on a device of `sms` SMs.
uint64_t paged_attention_workspace(int tokens, int q_heads, int kv_heads, int sms);
cudaError_t launch_paged_attention(const PagedAttnArgs &a, int sms, cudaStream_t st);

}  // namespace lrm
