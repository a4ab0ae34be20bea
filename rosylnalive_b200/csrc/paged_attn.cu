// paged_attn.cu -- attention of each request's new tokens over its cached keys (lrm_op_paged_attention).
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(scale log2(e) q.k_j - m), m the running maximum: one pass over the keys.
// One warp a (token, query head): 4 dims a lane, a key at a time.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "internal.h"
#include "paged.h"
#include "ptx.cuh"

namespace lrm {
namespace {

__global__ void __launch_bounds__(128) paged_attn_kernel(PagedAttnArgs a) {
    const int lane = threadIdx.x & 31, h = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int t = blockIdx.x;
    // the request of row t: the last one that starts at or before it (requests without tokens start where the next does)
    int lo = 0, hi = a.requests;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu_seqlens[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    const int start = a.cu_seqlens[lo], end = a.cu_seqlens[lo + 1];
    if (t < start || t >= end || h >= a.q_heads) return;
    const int slot = a.slots[lo], kv = a.kv_len[lo];
    if (start < 0 || end > a.tokens || slot < 0 || slot >= a.max_seqs || kv < end - start ||
        kv > (int64_t)a.pages_per_seq * kPageTokens) {
        if (lane == 0) atomicCAS(a.err, 0u, kErrAttnRequest);
        return;
    }
    const int pos = kv - (end - t);
    const int kvh = h / (a.q_heads / a.kv_heads);
    float q[4], o[4] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < 4; ++e) q[e] = __bfloat162float(a.q[(size_t)t * a.ld_q + h * kHeadDim + 4 * lane + e]);
    for (int j = 0; j <= pos; ++j) {
        const int pg = a.page_table[(size_t)slot * a.pages_per_seq + j / kPageTokens];
        const bool good = pg >= 0 && pg < a.kv_pages;
        if (!good && lane == 0) atomicCAS(a.err, 0u, kErrAttnPage);
        const __nv_bfloat16 *k = a.pool + (size_t)(good ? pg : 0) * kv_page_elems(a.kv_heads) +
                                 (size_t)kvh * 2 * kPageTokens * kHeadDim + (j % kPageTokens) * kHeadDim + 4 * lane;
        float s = 0.f;
        for (int e = 0; e < 4; ++e) s += good ? q[e] * __bfloat162float(k[e]) : 0.f;
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= a.scale_log2;
        const float m2 = fmaxf(m, s), f = m == -INFINITY ? 0.f : exp2f(m - m2);
        const float p = exp2f(s - (m2 == -INFINITY ? 0.f : m2));
        m = m2;
        l = l * f + p;
        for (int e = 0; e < 4; ++e)
            o[e] = o[e] * f + (good ? p * __bfloat162float(k[kPageTokens * kHeadDim + e]) : 0.f);
    }
    for (int e = 0; e < 4; ++e)
        a.out[(size_t)t * a.ld_out + h * kHeadDim + 4 * lane + e] = __float2bfloat16_rn(o[e] / l);
}

}  // namespace

uint64_t paged_attention_workspace(int tokens, int q_heads, int kv_heads, int sms) { return 16; }

cudaError_t launch_paged_attention(const PagedAttnArgs &a, int sms, cudaStream_t st) {
    paged_attn_kernel<<<dim3(a.tokens, (a.q_heads + 3) / 4), 128, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace lrm
