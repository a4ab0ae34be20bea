// paged_step.cu -- the bookkeeping and the append of a paged serving step (include/lrm_cuda.h, "a paged serving step on
// the device"): lrm_op_page_plan, lrm_op_page_release, lrm_op_qkv_append, and the argument checks of
// lrm_op_paged_attention (its kernels are in paged_attn.cu).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <exception>
#include <string>

#include "../../include/lrm_cuda.h"
#include "internal.h"
#include "paged.h"
#include "ptx.cuh"

namespace lrm {
uint32_t *device_error_word();
int device_sms();
lrm_status op_fail(lrm_status s, const std::string &m);
lrm_status op_cuda(cudaError_t e, const char *what);

namespace {

// ---- page plan and release --------------------------------------------------------------------------------------
//
// Request i has n_i new tokens (the plan) and c_i pages to take (plan: ceil((len + n) / 16) - ceil(len / 16)) or to
// give back (release: ceil(len / 16) - ceil(keep / 16)). With exclusive sums N and C over the requests, token t of
// request i is row N_i + t of the step and page j of request i is entry count - 1 - (C_i + j) of the free list (plan)
// or count + C_i + j (release). So everything follows from one scan over the requests, and the rest is one binary
// search a token or page.
//
// One cluster does it all: every CTA scans all requests (1024 a pass, their prefixes in shared memory), so no CTA waits
// for another's sums, and the tokens and pages are dealt out over the cluster's threads. First pass: totals and checks
// only; nothing is written before the whole step is known to be sound. seq_len and free_count may be updated in
// place, so the new values are written behind a cluster barrier that every CTA reaches after its last read of them.
// Sums saturate at 2^30 (min(a + b, 2^30) is associative for non-negative terms), far above every limit.
constexpr int kPlanThreads = 1024;
constexpr uint32_t kSat = 1u << 30;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kSat); }
__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

struct PlanShared {
    uint32_t n0[kPlanThreads], c0[kPlanThreads];  // exclusive sums of this pass's requests, the earlier passes' included
    int slot[kPlanThreads], held[kPlanThreads];   // held: pages of the old length (plan) or of the kept one (release)
    int past[kPlanThreads];
    uint32_t warp_n[32], warp_c[32];
    uint32_t n_end, c_end;  // sums through this pass
    int code;               // the first broken rule's code (lowest wins), 0 for none
    int shared_code;        // rank 0: codes found by the dealt-out checks of every CTA
};

template <bool kRelease>
__device__ __forceinline__ void scan_pass(const PageStepArgs &a, PlanShared &s, uint32_t *seen, int base, uint32_t n_base,
                                          uint32_t c_base, bool check) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int i = base + tid;
    int slot = -1, past = 0, held = 0, code = 0;
    uint32_t n = 0, c = 0;
    if (i < a.requests) slot = a.slots[i];
    if (slot != -1) {
        const int cap = a.pages_per_seq * kPageTokens;
        if (slot < 0 || slot >= a.max_seqs) {
            code = kRelease ? kErrReleaseRequest : kErrPlanRequest;
            slot = -1;
        } else {
            if (check) {
                const uint32_t bit = 1u << (slot & 31);
                if (atomicOr(&seen[slot >> 5], bit) & bit) code = kRelease ? kErrReleaseRequest : kErrPlanRequest;
            }
            past = a.seq_len[slot];
            const int x = kRelease ? a.keep_len[i] : a.new_len[i];
            const bool bad = past < 0 || past > cap || x < 0 || (kRelease ? x > past : x > cap - past);
            if (bad) {
                code = kRelease ? kErrReleaseRequest : kErrPlanRequest;
                past = 0;
            } else if (kRelease) {
                held = pages_of(x);
                c = pages_of(past) - held;
                n = x;  // the kept length, for the last step
            } else {
                held = pages_of(past);
                n = x;
                c = pages_of(past + x) - held;
            }
        }
    }
    if (code) atomicMin((unsigned int *)&s.code, (unsigned int)code);
    s.slot[tid] = slot;
    s.held[tid] = held;
    s.past[tid] = kRelease ? (int)n : past;
    if (kRelease) n = 0;
    uint32_t in = n, ic = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t un = __shfl_up_sync(0xffffffffu, in, o), uc = __shfl_up_sync(0xffffffffu, ic, o);
        if (lane >= o) {
            in = sat_add(in, un);
            ic = sat_add(ic, uc);
        }
    }
    if (lane == 31) {
        s.warp_n[warp] = in;
        s.warp_c[warp] = ic;
    }
    __syncthreads();
    uint32_t bn = n_base, bc = c_base;
    {
        // each warp adds up the totals of the warps before it
        uint32_t wn = lane < warp ? s.warp_n[lane] : 0, wc = lane < warp ? s.warp_c[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            wn = sat_add(wn, __shfl_xor_sync(0xffffffffu, wn, o));
            wc = sat_add(wc, __shfl_xor_sync(0xffffffffu, wc, o));
        }
        bn = sat_add(bn, wn);
        bc = sat_add(bc, wc);
    }
    const uint32_t en = sat_add(bn, in), ec = sat_add(bc, ic);
    s.n0[tid] = en - n;  // exact while the sums are below the saturation, which the checks make sure of before any use
    s.c0[tid] = ec - c;
    if (tid == kPlanThreads - 1) {
        s.n_end = en;
        s.c_end = ec;
    }
    __syncthreads();
}

// The request of this pass that holds item x: the last one whose exclusive sum is <= x. Requests of no items share
// their sum with the next one, so the last is the one that holds it.
__device__ __forceinline__ int find_request(const uint32_t *sum, uint32_t x) {
    int lo = 0;
#pragma unroll
    for (int step = kPlanThreads / 2; step > 0; step >>= 1)
        if (sum[lo + step] <= x) lo += step;
    return lo;
}

__device__ __forceinline__ void cluster_or_code(int *code, int value) {
    asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(ptx::mapa(code, 0)), "r"(value)
                 : "memory");
}
__device__ __forceinline__ int cluster_read_code(const int *code) {
    int v;
    asm volatile("ld.relaxed.cluster.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ptx::mapa(code, 0)) : "memory");
    return v;
}

template <bool kRelease>
__global__ void __launch_bounds__(kPlanThreads) page_step_kernel(PageStepArgs a) {
    __shared__ PlanShared s;
    extern __shared__ uint32_t seen[];  // one bit a slot: the slots listed so far
    const int tid = threadIdx.x;
    const int rank = (int)ptx::cluster_ctarank(), ranks = (int)gridDim.x;
    const int passes = (a.requests + kPlanThreads - 1) / kPlanThreads;
    const int count = *a.free_count;
    for (int w = tid; w < (a.max_seqs + 31) / 32; w += kPlanThreads) seen[w] = 0;
    if (tid == 0) {
        s.code = -1;  // as unsigned, above every code
        s.shared_code = 0;
    }
    __syncthreads();
    uint32_t n_total = 0, c_total = 0;
    for (int p = 0; p < passes; ++p) {
        scan_pass<kRelease>(a, s, seen, p * kPlanThreads, n_total, c_total, true);
        n_total = s.n_end;
        c_total = s.c_end;
        if (p + 1 < passes) __syncthreads();
    }
    int code = s.code == -1 ? 0 : s.code;
    const bool bad_count = count < 0 || count > a.kv_pages;
    if (kRelease) {
        if (!code && (bad_count || c_total > (uint32_t)(a.kv_pages - count))) code = kErrReleaseCount;
    } else {
        if (!code && bad_count) code = kErrPlanFree;
        if (!code && c_total > (uint32_t)count) code = kErrPlanPages;
        if (!code && n_total > (uint32_t)a.max_tokens) code = kErrPlanTokens;
    }
    if (ranks > 1) ptx::cluster_sync();  // rank 0's shared_code is initialised
    // The page ids that change hands, checked before any is used (dealt out over the cluster).
    if (!code) {
        bool bad = false;
        if (!kRelease) {
            for (uint32_t j = rank * kPlanThreads + tid; j < c_total; j += ranks * kPlanThreads)
                bad |= (uint32_t)a.free_list[count - 1 - (int)j] >= (uint32_t)a.kv_pages;
        } else {
            uint32_t done = 0;
            for (int p = 0; p < passes; ++p) {
                if (passes > 1) {
                    __syncthreads();
                    scan_pass<kRelease>(a, s, seen, p * kPlanThreads, 0, done, false);
                }
                for (uint32_t j = done + rank * kPlanThreads + tid; j < s.c_end; j += ranks * kPlanThreads) {
                    const int r = find_request(s.c0, j);
                    const int64_t at = (int64_t)s.slot[r] * a.pages_per_seq + s.held[r] + (int)(j - s.c0[r]);
                    bad |= (uint32_t)a.page_table[at] >= (uint32_t)a.kv_pages;
                }
                done = s.c_end;
            }
        }
        if (bad) cluster_or_code(&s.shared_code, kRelease ? kErrReleasePage : kErrPlanFree);
    }
    if (ranks > 1)
        ptx::cluster_sync();
    else
        __syncthreads();
    if (!code) code = cluster_read_code(&s.shared_code);

    if (code) {  // nothing is taken or given back
        if (rank == 0 && tid == 0) {
            atomicCAS(a.err, 0u, (uint32_t)code);
            if (a.free_count_out != a.free_count) *a.free_count_out = count;
        }
        const int t0 = rank * kPlanThreads + tid, step = ranks * kPlanThreads;
        if (!kRelease) {
            for (int i = t0; i <= a.requests; i += step) a.cu_seqlens[i] = 0;
            for (int i = t0; i < a.requests; i += step) a.kv_len[i] = 0;
            for (int t = t0; t < a.max_tokens; t += step) {
                a.tok_pos[t] = 0;
                a.slot_map[t] = -1;
            }
        }
        if (a.seq_len_out != a.seq_len)
            for (int i = t0; i < a.requests; i += step) {
                const int slot = a.slots[i];
                if (slot >= 0 && slot < a.max_seqs) a.seq_len_out[slot] = a.seq_len[slot];
            }
        if (ranks > 1) ptx::cluster_sync();  // rank 0's shared memory has been read
        return;
    }

    uint32_t n_done = 0, c_done = 0;
    for (int p = 0; p < passes; ++p) {
        if (passes > 1) {
            __syncthreads();
            scan_pass<kRelease>(a, s, seen, p * kPlanThreads, n_done, c_done, false);
        }
        const int i = p * kPlanThreads + tid;
        if (!kRelease && i < a.requests && p % ranks == rank) {
            const uint32_t n1 = tid + 1 < kPlanThreads ? s.n0[tid + 1] : s.n_end;
            a.cu_seqlens[i] = (int)s.n0[tid];
            a.kv_len[i] = s.past[tid] + (int)(n1 - s.n0[tid]);  // 0 + 0 for padding
            if (i == a.requests - 1) a.cu_seqlens[a.requests] = (int)n_total;
        }
        for (uint32_t j = c_done + rank * kPlanThreads + tid; j < s.c_end; j += ranks * kPlanThreads) {
            const int r = find_request(s.c0, j);
            const int64_t at = (int64_t)s.slot[r] * a.pages_per_seq + s.held[r] + (int)(j - s.c0[r]);
            if (kRelease)
                a.free_list[count + (int)j] = a.page_table[at];
            else
                a.page_table[at] = a.free_list[count - 1 - (int)j];
        }
        if (!kRelease)
            for (uint32_t t = n_done + rank * kPlanThreads + tid; t < s.n_end; t += ranks * kPlanThreads) {
                const int r = find_request(s.n0, t);
                const int pos = s.past[r] + (int)(t - s.n0[r]), pg = pos / kPageTokens;
                // a page taken just now is read from the free list: its table entry may not be written yet
                const int id = pg < s.held[r] ? a.page_table[(int64_t)s.slot[r] * a.pages_per_seq + pg]
                                              : a.free_list[count - 1 - (int)(s.c0[r] + (pg - s.held[r]))];
                const bool good = (uint32_t)id < (uint32_t)a.kv_pages;
                if (!good) atomicCAS(a.err, 0u, kErrPlanTable);
                a.tok_pos[t] = pos;
                a.slot_map[t] = good ? id * kPageTokens + pos % kPageTokens : -1;
            }
        n_done = s.n_end;
        c_done = s.c_end;
    }
    if (!kRelease)
        for (uint32_t t = n_total + rank * kPlanThreads + tid; t < (uint32_t)a.max_tokens; t += ranks * kPlanThreads) {
            a.tok_pos[t] = 0;
            a.slot_map[t] = -1;
        }
    // Every CTA is done with the old lengths and count: the new ones may take their place.
    if (ranks > 1)
        ptx::cluster_sync();
    else
        __syncthreads();
    if (rank == 0 && tid == 0) *a.free_count_out = kRelease ? count + (int)c_total : count - (int)c_total;
    for (int p = rank; p < passes; p += ranks) {
        const int i = p * kPlanThreads + tid;
        if (i >= a.requests) continue;
        const int slot = a.slots[i];
        if (slot < 0) continue;
        a.seq_len_out[slot] = kRelease ? a.keep_len[i] : a.kv_len[i];  // kv_len[i]: this thread's own write
    }
}

// ---- q/k/v append -----------------------------------------------------------------------------------------------
//
// y = x * gain / sqrt(mean(x^2) + eps), then (y_d, y_{d+64}) -> (y_d c - y_{d+64} s, y_{d+64} c + y_d s) for q and k.
// Every byte is read once and written once (bound: HBM copy), so a half-warp takes a head (16 lanes x 16 bytes): the
// sum of squares is 4 shuffles, RoPE's partner dims are 8 lanes away, and a store is 256 contiguous bytes. A block of
// four warps takes one row; a half-warp's kBatch heads are loaded before the first is used, and its cos / sin row
// stays in registers for all of them.
constexpr int kAppendThreads = 128, kBatch = 4;

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}

__global__ void __launch_bounds__(kAppendThreads) qkv_append_kernel(QkvAppendArgs a) {
    const int t = blockIdx.x;
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;  // 8 half-warps
    const int heads = a.q_heads + 2 * a.kv_heads, qk = a.q_heads + a.kv_heads;
    const int place = a.slot_map[t];
    const int pos = a.cos_t ? a.tok_pos[t] : 0;
    if (place == -1) return;
    if (place < 0 || place >= a.places || (a.cos_t && (pos < 0 || pos >= a.rope_rows))) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0u, kErrAppendRow);
        return;
    }
    const __nv_bfloat16 *row = a.qkv + (size_t)t * a.ld_qkv + 8 * l;
    float cs[8], sn[8];  // of this lane's 8 dims; sin's sign is that of its term
    if (a.cos_t) {
        const size_t at = (size_t)pos * 64 + 8 * (l & 7);
        const float sign = l < 8 ? -1.f : 1.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float4 c = __ldg(reinterpret_cast<const float4 *>(a.cos_t + at) + u);
            const float4 n = __ldg(reinterpret_cast<const float4 *>(a.sin_t + at) + u);
            cs[4 * u] = c.x, cs[4 * u + 1] = c.y, cs[4 * u + 2] = c.z, cs[4 * u + 3] = c.w;
            sn[4 * u] = sign * n.x, sn[4 * u + 1] = sign * n.y, sn[4 * u + 2] = sign * n.z, sn[4 * u + 3] = sign * n.w;
        }
    }
    __nv_bfloat16 *page = a.pool + (size_t)(place / kPageTokens) * kv_page_elems(a.kv_heads) +
                          (place % kPageTokens) * kHeadDim + 8 * l;
    for (int h0 = 0; h0 < heads; h0 += 8 * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int h = h0 + b * 8 + half;
            raw[b] = h < heads ? *reinterpret_cast<const uint4 *>(row + h * kHeadDim) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int h = h0 + b * 8 + half;
            uint4 o = raw[b];
            if (__any_sync(0xffffffffu, h < qk)) {  // the warp's two heads; a v head keeps its bits
                float x[8] = {bf_lo(o.x), bf_hi(o.x), bf_lo(o.y), bf_hi(o.y), bf_lo(o.z), bf_hi(o.z), bf_lo(o.w), bf_hi(o.w)};
                if (a.q_norm) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
                    for (int m = 8; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
                    const float r = 1.f / sqrtf(ss * (1.f / kHeadDim) + a.eps);
                    const uint4 g = __ldg(reinterpret_cast<const uint4 *>((h < a.q_heads ? a.q_norm : a.k_norm) + 8 * l));
                    const float w[8] = {bf_lo(g.x), bf_hi(g.x), bf_lo(g.y), bf_hi(g.y), bf_lo(g.z), bf_hi(g.z), bf_lo(g.w), bf_hi(g.w)};
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] *= r * w[e];
                }
                if (a.cos_t) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = x[e] * cs[e] + __shfl_xor_sync(0xffffffffu, x[e], 8) * sn[e];
                }
                if (h < qk && (a.q_norm || a.cos_t))
                    o = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
            }
            if (h < a.q_heads)
                *reinterpret_cast<uint4 *>(a.q_out + (size_t)t * a.ld_q + h * kHeadDim + 8 * l) = o;
            else if (h < heads) {
                const int kv = h < qk ? 0 : 1, hk = h - a.q_heads - kv * a.kv_heads;
                *reinterpret_cast<uint4 *>(page + (size_t)(hk * 2 + kv) * (kPageTokens * kHeadDim)) = o;
            }
        }
    }
}

// Nothing is thrown across the ABI: an exception (a message that cannot be allocated) becomes a status.
template <class F>
lrm_status guarded(F &&f) noexcept {
    try {
        return f();
    } catch (...) {
        return LRM_ERR_OUT_OF_MEMORY;
    }
}

bool in(int64_t v, int64_t lo, int64_t hi) { return v >= lo && v <= hi; }

}  // namespace

cudaError_t launch_page_step(const PageStepArgs &a, cudaStream_t st) {
    // One CTA for steps of up to 1024 requests and 4096 tokens; a cluster of 8 above, where the dealt-out writes pay
    // for the cluster's start and barriers.
    const bool big = a.requests > kPlanThreads || (!a.keep_len && a.max_tokens > 4 * kPlanThreads);
    const unsigned ctas = big ? 8 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = (size_t)((a.max_seqs + 31) / 32) * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return a.keep_len ? cudaLaunchKernelEx(&cfg, page_step_kernel<true>, a)
                      : cudaLaunchKernelEx(&cfg, page_step_kernel<false>, a);
}

cudaError_t launch_qkv_append(const QkvAppendArgs &a, cudaStream_t st) {
    qkv_append_kernel<<<a.tokens, kAppendThreads, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace lrm

using namespace lrm;

extern "C" {

lrm_status lrm_op_page_plan(void *stream, const lrm_page_plan_desc *d) {
    return guarded([&]() -> lrm_status {
        if (!d) return op_fail(LRM_ERR_ARGUMENT, "descriptor is null");
        if (!in(d->requests, 1, kMaxRequests) || !in(d->max_seqs, 1, kMaxSeqs) || !in(d->pages_per_seq, 1, kMaxSeqPages) ||
            !in(d->kv_pages, 1, kMaxPoolPages) || !in(d->max_tokens, 1, kMaxStepTokens))
            return op_fail(LRM_ERR_ARGUMENT, "page plan: a size is outside its limits");
        const uint64_t p[] = {d->slots,  d->new_len, d->seq_len, d->page_table,  d->free_list,     d->free_count, d->cu_seqlens,
                              d->kv_len, d->tok_pos, d->slot_map, d->seq_len_out, d->free_count_out};
        for (uint64_t x : p)
            if (!x || (x & 3)) return op_fail(LRM_ERR_ARGUMENT, "page plan: pointers must be non-null and 4-byte aligned");
        PageStepArgs a = {};
        a.slots = (const int32_t *)d->slots;
        a.new_len = (const int32_t *)d->new_len;
        a.seq_len = (const int32_t *)d->seq_len;
        a.page_table = (int32_t *)d->page_table;
        a.free_list = (int32_t *)d->free_list;
        a.free_count = (const int32_t *)d->free_count;
        a.cu_seqlens = (int32_t *)d->cu_seqlens;
        a.kv_len = (int32_t *)d->kv_len;
        a.tok_pos = (int32_t *)d->tok_pos;
        a.slot_map = (int32_t *)d->slot_map;
        a.seq_len_out = (int32_t *)d->seq_len_out;
        a.free_count_out = (int32_t *)d->free_count_out;
        a.requests = d->requests;
        a.max_seqs = d->max_seqs;
        a.pages_per_seq = d->pages_per_seq;
        a.kv_pages = d->kv_pages;
        a.max_tokens = d->max_tokens;
        if (!(a.err = device_error_word())) return LRM_ERR_CUDA;
        return op_cuda(launch_page_step(a, (cudaStream_t)stream), "page plan");
    });
}

lrm_status lrm_op_page_release(void *stream, const lrm_page_release_desc *d) {
    return guarded([&]() -> lrm_status {
        if (!d) return op_fail(LRM_ERR_ARGUMENT, "descriptor is null");
        if (!in(d->requests, 1, kMaxRequests) || !in(d->max_seqs, 1, kMaxSeqs) || !in(d->pages_per_seq, 1, kMaxSeqPages) ||
            !in(d->kv_pages, 1, kMaxPoolPages))
            return op_fail(LRM_ERR_ARGUMENT, "page release: a size is outside its limits");
        const uint64_t p[] = {d->slots,     d->keep_len,   d->seq_len,     d->page_table,
                              d->free_list, d->free_count, d->seq_len_out, d->free_count_out};
        for (uint64_t x : p)
            if (!x || (x & 3))
                return op_fail(LRM_ERR_ARGUMENT, "page release: pointers must be non-null and 4-byte aligned");
        PageStepArgs a = {};
        a.slots = (const int32_t *)d->slots;
        a.keep_len = (const int32_t *)d->keep_len;
        a.seq_len = (const int32_t *)d->seq_len;
        a.page_table = (int32_t *)d->page_table;
        a.free_list = (int32_t *)d->free_list;
        a.free_count = (const int32_t *)d->free_count;
        a.seq_len_out = (int32_t *)d->seq_len_out;
        a.free_count_out = (int32_t *)d->free_count_out;
        a.requests = d->requests;
        a.max_seqs = d->max_seqs;
        a.pages_per_seq = d->pages_per_seq;
        a.kv_pages = d->kv_pages;
        if (!(a.err = device_error_word())) return LRM_ERR_CUDA;
        return op_cuda(launch_page_step(a, (cudaStream_t)stream), "page release");
    });
}

lrm_status lrm_op_qkv_append(void *stream, const lrm_qkv_append_desc *d) {
    return guarded([&]() -> lrm_status {
        if (!d) return op_fail(LRM_ERR_ARGUMENT, "descriptor is null");
        if (d->head_dim != kHeadDim) return op_fail(LRM_ERR_ARGUMENT, "q/k/v append needs head_dim 128");
        if (!in(d->tokens, 1, kMaxStepTokens) || !in(d->q_heads, 1, 65535) || !in(d->kv_heads, 1, 65535) ||
            !in(d->kv_pages, 1, kMaxPoolPages))
            return op_fail(LRM_ERR_ARGUMENT, "q/k/v append: a size is outside its limits");
        const int64_t q_cols = (int64_t)d->q_heads * kHeadDim, cols = q_cols + (int64_t)2 * d->kv_heads * kHeadDim;
        if (!in(d->ld_qkv, cols, 1 << 30) || !in(d->ld_q, q_cols, 1 << 30) || (d->ld_qkv & 7) || (d->ld_q & 7))
            return op_fail(LRM_ERR_ARGUMENT, "q/k/v append: row strides must hold a row and be multiples of 8");
        if (!d->q_norm != !d->k_norm || !d->cos != !d->sin)
            return op_fail(LRM_ERR_ARGUMENT, "q/k/v append: give both gains or none, and both of cos and sin or none");
        if (!d->qkv || !d->slot_map || !d->q_out || !d->pool || (d->cos && !d->tok_pos))
            return op_fail(LRM_ERR_ARGUMENT, "q/k/v append: null pointer");
        if (((d->qkv | d->q_norm | d->k_norm | d->cos | d->sin | d->q_out | d->pool) & 15) || ((d->tok_pos | d->slot_map) & 3))
            return op_fail(LRM_ERR_ARGUMENT, "q/k/v append: a pointer is not aligned (16 bytes; 4 for tok_pos and slot_map)");
        if (d->cos && d->rope_rows < 1) return op_fail(LRM_ERR_ARGUMENT, "q/k/v append: the RoPE table has no rows");
        if (d->q_norm && !(d->eps >= 0.f && isfinite(d->eps)))
            return op_fail(LRM_ERR_ARGUMENT, "q/k/v append: eps must be finite and not negative");
        QkvAppendArgs a = {};
        a.qkv = (const __nv_bfloat16 *)d->qkv;
        a.q_norm = (const __nv_bfloat16 *)d->q_norm;
        a.k_norm = (const __nv_bfloat16 *)d->k_norm;
        a.cos_t = (const float *)d->cos;
        a.sin_t = (const float *)d->sin;
        a.tok_pos = (const int32_t *)d->tok_pos;
        a.slot_map = (const int32_t *)d->slot_map;
        a.q_out = (__nv_bfloat16 *)d->q_out;
        a.pool = (__nv_bfloat16 *)d->pool;
        a.ld_qkv = d->ld_qkv;
        a.ld_q = d->ld_q;
        a.tokens = d->tokens;
        a.q_heads = d->q_heads;
        a.kv_heads = d->kv_heads;
        a.rope_rows = d->rope_rows;
        a.places = (int64_t)d->kv_pages * kPageTokens;
        a.eps = d->eps;
        if (!(a.err = device_error_word())) return LRM_ERR_CUDA;
        return op_cuda(launch_qkv_append(a, (cudaStream_t)stream), "q/k/v append");
    });
}

uint64_t lrm_op_paged_attention_workspace(int32_t tokens, int32_t q_heads, int32_t kv_heads) {
    if (!in(tokens, 1, kMaxStepTokens) || !in(kv_heads, 1, 65535) || !in(q_heads, 1, 65535) || q_heads % kv_heads ||
        q_heads / kv_heads > 128)
        return 0;
    return paged_attention_workspace(tokens, q_heads, kv_heads, device_sms());
}

lrm_status lrm_op_paged_attention(void *stream, const lrm_paged_attn_desc *d) {
    return guarded([&]() -> lrm_status {
        if (!d) return op_fail(LRM_ERR_ARGUMENT, "descriptor is null");
        if (d->head_dim != kHeadDim) return op_fail(LRM_ERR_ARGUMENT, "paged attention needs head_dim 128");
        if (!in(d->q_heads, 1, 65535) || !in(d->kv_heads, 1, 65535) || d->q_heads % d->kv_heads ||
            d->q_heads / d->kv_heads > 128)
            return op_fail(LRM_ERR_ARGUMENT, "paged attention: kv_heads must divide q_heads, at most 128 a KV head");
        if (!in(d->requests, 1, kMaxRequests) || !in(d->tokens, 1, kMaxStepTokens) || !in(d->max_seqs, 1, kMaxSeqs) ||
            !in(d->pages_per_seq, 1, kMaxSeqPages) || !in(d->kv_pages, 1, kMaxPoolPages) ||
            (int64_t)d->kv_pages * d->kv_heads >= (1 << 30))
            return op_fail(LRM_ERR_ARGUMENT, "paged attention: a size is outside its limits");
        const int64_t cols = (int64_t)d->q_heads * kHeadDim;
        if (!in(d->ld_q, cols, 1 << 30) || !in(d->ld_out, cols, 1 << 30) || (d->ld_q & 7) || (d->ld_out & 7))
            return op_fail(LRM_ERR_ARGUMENT, "paged attention: row strides must hold a row and be multiples of 8");
        if (!d->q || !d->pool || !d->page_table || !d->slots || !d->cu_seqlens || !d->kv_len || !d->out || !d->workspace)
            return op_fail(LRM_ERR_ARGUMENT, "paged attention: null pointer");
        if (((d->q | d->pool | d->out | d->workspace) & 15) || ((d->page_table | d->slots | d->cu_seqlens | d->kv_len) & 3))
            return op_fail(LRM_ERR_ARGUMENT,
                           "paged attention: a pointer is not aligned (16 bytes; 4 for the int32 arrays)");
        if (!(d->scale > 0.f) || !isfinite(d->scale * 1.4426950408889634f))
            return op_fail(LRM_ERR_ARGUMENT, "paged attention: the scale must be positive and finite");
        PagedAttnArgs a = {};
        a.q = (const __nv_bfloat16 *)d->q;
        a.pool = (const __nv_bfloat16 *)d->pool;
        a.page_table = (const int32_t *)d->page_table;
        a.slots = (const int32_t *)d->slots;
        a.cu_seqlens = (const int32_t *)d->cu_seqlens;
        a.kv_len = (const int32_t *)d->kv_len;
        a.out = (__nv_bfloat16 *)d->out;
        a.workspace = (uint8_t *)d->workspace;
        a.ld_q = d->ld_q;
        a.ld_out = d->ld_out;
        a.requests = d->requests;
        a.tokens = d->tokens;
        a.q_heads = d->q_heads;
        a.kv_heads = d->kv_heads;
        a.max_seqs = d->max_seqs;
        a.pages_per_seq = d->pages_per_seq;
        a.kv_pages = d->kv_pages;
        a.scale_log2 = d->scale * 1.4426950408889634f;
        if (!(a.err = device_error_word())) return LRM_ERR_CUDA;
        return op_cuda(launch_paged_attention(a, device_sms(), (cudaStream_t)stream), "paged attention");
    });
}

}  // extern "C"
