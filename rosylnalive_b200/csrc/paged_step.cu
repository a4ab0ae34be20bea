// paged_step.cu -- the bookkeeping and the append of a paged serving step (include/lrm_cuda.h, "a paged serving step on
// the device"): lrm_op_page_plan, lrm_op_page_release, lrm_op_qkv_append, and the argument checks of
// lrm_op_paged_attention (its kernels are in paged_attn.cu).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
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
// or count + C_i + j (release). So everything follows from one scan over the requests, and the rest is a binary search
// and a few loads and stores, by one thread for two or four pages that are given back or for the tokens of a quad (rows 4k ..
// 4k+3 of the step), whose stores are then 16 bytes: of a large step the number of stores is what counts (65536 tokens on
// one CTA: 20 us, 44 with single words). A small one is bound by latency, the fetch of instructions included: loops
// stay rolled where their loads do not have to overlap, and a single CTA takes its tokens one by one.
//
// One cluster does it all, each CTA a contiguous part of the requests (1024 a pass, their prefixes in shared memory):
//   1. load and check the part, and sum it up; a bit a slot, kept by CTA slot % ranks, finds a slot listed twice;
//   2. each CTA writes its sums to all others' shared memory: its first token and page, and whether the step is sound;
//   3. the page ids that change hands are checked; the CTAs agree on that too, before anything is written;
//   4. write the part's outputs, tokens, pages and lengths.
// A slot is listed once, so no CTA reads a length that another writes, and the new lengths may take the old ones' place;
// free_count is read by all before the second barrier and written after it. What bounds it is latency: two dependent
// loads, three barriers and the stores: 3.2 us for 64 requests of one token (3.9 with lengths of their own), 9.2 us for 1024
// of 64 (a cluster in which every CTA scans all requests took 15 us for 2000 requests and 36 thousand tokens, this one 10).
// A step that fits one pass of one CTA (kCluster false) leaves out the exchange between the CTAs.
// Sums saturate at 2^30 (min(a + b, 2^30) is associative for non-negative terms), far above every limit.
constexpr int kPlanThreads = 1024, kPlanCtas = 8;
constexpr uint32_t kSat = 1u << 30;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kSat); }
__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

struct PlanShared {
    uint32_t n0[kPlanThreads], c0[kPlanThreads];  // exclusive sums of this pass's requests, from the call's first on
    int slot[kPlanThreads], held[kPlanThreads];   // held: pages of the old length (plan) or of the kept one (release)
    int past[kPlanThreads];
    uint32_t d0[kPlanThreads];  // exclusive sums of the most quads that the requests' tokens touch (plan), per pass
    uint32_t warp_n[32], warp_c[32], warp_d[32];
    uint32_t n_end, c_end, d_end;  // sums through this pass
    uint32_t code;          // of this part, 0: sound
    uint32_t part_n[kPlanCtas], part_c[kPlanCtas], part_code[kPlanCtas], part_id[kPlanCtas];  // written by each CTA
};

struct Request {
    int slot, x, past;  // x: new_len or keep_len
};

template <bool kRelease>
__device__ __forceinline__ Request load_request(const PageStepArgs &a, int i, int end) {
    Request q = {-1, 0, 0};
    if (i < end) {
        q.slot = a.slots[i];
        q.x = kRelease ? a.keep_len[i] : a.new_len[i];
        if (q.slot >= 0 && q.slot < a.max_seqs) q.past = a.seq_len[q.slot];
    }
    return q;
}

// A pass of up to 1024 requests, one a thread: checks and sums. With `seen` (the first time), slots listed twice.
template <bool kRelease, bool kCluster>
__device__ __forceinline__ void scan_pass(const PageStepArgs &a, PlanShared &s, uint32_t *seen, const Request &q,
                                          uint32_t n_base, uint32_t c_base, int ranks) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int slot = q.slot, past = q.past, held = 0;
    const int x = q.x;
    uint32_t n = 0, c = 0, d = 0;
    bool bad = false;
    if (slot != -1) {
        const int cap = a.pages_per_seq * kPageTokens;
        if (slot < 0 || slot >= a.max_seqs) {
            bad = true;
            slot = -1;
        } else {
            if (seen) {
                const int owner = kCluster ? slot % ranks : 0, at = kCluster ? slot / ranks : slot;
                uint32_t old;
                asm volatile("atom.relaxed.cluster.shared::cluster.or.b32 %0, [%1], %2;"
                             : "=r"(old)
                             : "r"(ptx::mapa(seen + (at >> 5), owner)), "r"(1u << (at & 31))
                             : "memory");
                bad = old >> (at & 31) & 1;
            }
            if (past < 0 || past > cap || x < 0 || (kRelease ? x > past : x > cap - past)) {
                bad = true;
                past = 0;
            } else if (kRelease) {
                held = pages_of(x);
                c = pages_of(past) - held;
            } else {
                held = pages_of(past);
                n = x;
                c = pages_of(past + x) - held;
                d = kCluster && x ? (x + 6) / 4 : 0;
            }
        }
    }
    if (bad) s.code = kRelease ? kErrReleaseRequest : kErrPlanRequest;
    s.slot[tid] = slot;
    s.held[tid] = held;
    s.past[tid] = kRelease ? x : past;
    uint32_t in = n, ic = c, id = d;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t un = __shfl_up_sync(0xffffffffu, in, o), uc = __shfl_up_sync(0xffffffffu, ic, o);
        const uint32_t ud = kRelease || !kCluster ? 0 : __shfl_up_sync(0xffffffffu, id, o);
        if (lane >= o) {
            in = sat_add(in, un);
            ic = sat_add(ic, uc);
            id += ud;
        }
    }
    if (lane == 31) {
        s.warp_n[warp] = in;
        s.warp_c[warp] = ic;
        s.warp_d[warp] = id;
    }
    __syncthreads();
    // each warp adds up the totals of the warps before it
    uint32_t wn = lane < warp ? s.warp_n[lane] : 0, wc = lane < warp ? s.warp_c[lane] : 0;
    uint32_t wd = lane < warp ? s.warp_d[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        wn = sat_add(wn, __shfl_xor_sync(0xffffffffu, wn, o));
        wc = sat_add(wc, __shfl_xor_sync(0xffffffffu, wc, o));
        if (!kRelease && kCluster) wd += __shfl_xor_sync(0xffffffffu, wd, o);
    }
    const uint32_t en = sat_add(sat_add(n_base, wn), in), ec = sat_add(sat_add(c_base, wc), ic);
    s.n0[tid] = en - n;  // exact while the sums are below the saturation, which the checks make sure of before any use
    s.c0[tid] = ec - c;
    if (!kRelease && kCluster) s.d0[tid] = wd + id - d;
    if (tid == kPlanThreads - 1) {
        s.n_end = en;
        s.c_end = ec;
        s.d_end = wd + id;
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

template <bool kRelease, bool kCluster>
__global__ void __launch_bounds__(kPlanThreads, 1) page_step_kernel(const __grid_constant__ PageStepArgs a) {
    __shared__ PlanShared s;
    extern __shared__ uint32_t seen[];  // one bit for each slot of this CTA: listed so far
    const int tid = threadIdx.x;
    const int rank = kCluster ? (int)ptx::cluster_ctarank() : 0, ranks = kCluster ? kPlanCtas : 1;
    auto sync = [&]() {
        if (kCluster)
            ptx::cluster_sync();
        else
            __syncthreads();
    };
    // to[rank] of every CTA, read by them after the next sync
    auto tell = [&](uint32_t *to, uint32_t v) {
        asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], %1;" ::"r"(ptx::mapa(to + rank, tid)), "r"(v) : "memory");
    };
    const int part = (a.requests + ranks - 1) / ranks;
    const int r0 = min(a.requests, rank * part), r1 = min(a.requests, r0 + part);
    const int passes = kCluster ? max(1, (r1 - r0 + kPlanThreads - 1) / kPlanThreads) : 1;
    const int count = *a.free_count;
    auto load = [&](int p) { return load_request<kRelease>(a, r0 + p * kPlanThreads + tid, r1); };
    const Request first = load(0);
    for (int w = tid; w < (a.max_seqs / ranks + 32) / 32; w += kPlanThreads) seen[w] = 0;
    if (tid == 0) s.code = 0;
    sync();
    uint32_t n_part = 0, c_part = 0;
    for (int p = 0; p < passes; ++p) {
        if (p) __syncthreads();
        scan_pass<kRelease, kCluster>(a, s, seen, p ? load(p) : first, n_part, c_part, ranks);
        n_part = s.n_end;
        c_part = s.c_end;
    }
    // This part's first token and page, and the whole call's sums.
    uint32_t n_base = 0, c_base = 0, n_total = n_part, c_total = c_part, code = s.code;
    if (kCluster) {
        if (tid < ranks) {
            tell(s.part_n, n_part);
            tell(s.part_c, c_part);
            tell(s.part_code, code);
        }
        sync();
        n_total = c_total = code = 0;
#pragma unroll
        for (int r = 0; r < ranks; ++r) {
            if (r == rank) {
                n_base = n_total;
                c_base = c_total;
            }
            n_total = sat_add(n_total, s.part_n[r]);
            c_total = sat_add(c_total, s.part_c[r]);
            code |= s.part_code[r];
        }
    }
    const bool bad_count = count < 0 || count > a.kv_pages;
    if (kRelease) {
        if (!code && (bad_count || c_total > (uint32_t)(a.kv_pages - count))) code = kErrReleaseCount;
    } else {
        if (!code && bad_count) code = kErrPlanFree;
        if (!code && c_total > (uint32_t)count) code = kErrPlanPages;
        if (!code && n_total > (uint32_t)a.max_tokens) code = kErrPlanTokens;
    }
    // The page ids that change hands, checked before any is used; the first ones are kept for the write.
    // (`code` is the same in all threads of the cluster.)
    auto entry = [&](int r, uint32_t j) {  // of the page table, for page j of the call, which is request r's
        return (int64_t)s.slot[r] * a.pages_per_seq + s.held[r] + (int)(j - s.c0[r]);
    };
    // of a thread, in a row (releases: of 1500 requests 11.5 us, with 8 13.8; of 40 on one CTA 3.4, with 4 3.6, with 1 4.1)
    constexpr int kIds = kRelease ? (kCluster ? 4 : 2) : 1;
    auto ids_of = [&](uint32_t j, uint32_t end, int(&id)[kIds]) {
        if (j >= end) return;
        if (kRelease) {
            int r = find_request(s.c0, j);
            // the next request's first page, and where page j of the table would be in this one
            uint32_t next = r + 1 < kPlanThreads ? s.c0[r + 1] : end;
            int64_t at = entry(r, j);
#pragma unroll
            for (int k = 0; k < kIds; ++k) {
                if (j + k >= end) break;
                while (j + k >= next) {
                    ++r;
                    next = r + 1 < kPlanThreads ? s.c0[r + 1] : end;
                    at = entry(r, j);
                }
                id[k] = a.page_table[at + k];
            }
        } else {
            id[0] = a.free_list[count - 1 - (int)j];
        }
    };
    int kept[kIds] = {};  // this thread's first ids
    if (!code) {
        bool bad = false;
        uint32_t nb = n_base, cb = c_base;
        for (int p = 0; p < passes; ++p) {
            if (passes > 1) {
                __syncthreads();
                scan_pass<kRelease, kCluster>(a, s, nullptr, load(p), nb, cb, ranks);
            } else if (kCluster) {  // the sums made above only need their base
                s.n0[tid] += n_base;
                s.c0[tid] += c_base;
                if (tid == 0) {
                    s.n_end += n_base;
                    s.c_end += c_base;
                }
                __syncthreads();
            }
#pragma unroll 1
            for (uint32_t j0 = cb; j0 < s.c_end; j0 += kIds * kPlanThreads) {
                int id[kIds] = {};
                ids_of(j0 + kIds * tid, s.c_end, id);
#pragma unroll
                for (int k = 0; k < kIds; ++k) {
                    bad |= (uint32_t)id[k] >= (uint32_t)a.kv_pages;
                    if (j0 == cb) kept[k] = id[k];
                }
            }
            nb = s.n_end;
            cb = s.c_end;
        }
        bad = __syncthreads_or(bad);
        const uint32_t id_code = bad ? kRelease ? kErrReleasePage : kErrPlanFree : 0;
        if (!kCluster)
            code = id_code;
        else if (tid < ranks)
            tell(s.part_id, id_code);
        if (kCluster) {
            sync();
            for (int r = 0; r < ranks && !code; ++r) code = s.part_id[r];
        }
    }

    const int t0 = rank * kPlanThreads + tid, step = ranks * kPlanThreads;
    if (code) {  // nothing is taken or given back
        if (rank == 0 && tid == 0) {
            atomicCAS(a.err, 0u, code);
            if (a.free_count_out != a.free_count) *a.free_count_out = count;
        }
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
        return;
    }

    const bool out_of_line = ((uintptr_t)a.tok_pos | (uintptr_t)a.slot_map) & 15;
    uint32_t nb = n_base, cb = c_base;
    for (int p = 0; p < passes; ++p) {
        if (passes > 1) {
            __syncthreads();
            scan_pass<kRelease, kCluster>(a, s, nullptr, load(p), nb, cb, ranks);
        }
        const int i = r0 + p * kPlanThreads + tid;
        const uint32_t n_end = s.n_end, c_end = s.c_end;
        if (i < r1) {
            int len = s.past[tid];  // release: the kept length
            if (!kRelease) {
                const uint32_t n1 = tid + 1 < kPlanThreads ? s.n0[tid + 1] : n_end;
                len += (int)(n1 - s.n0[tid]);  // 0 + 0 for padding
                a.cu_seqlens[i] = (int)s.n0[tid];
                a.kv_len[i] = len;
            }
            if (s.slot[tid] >= 0) a.seq_len_out[s.slot[tid]] = len;
        }
#pragma unroll 1
        for (uint32_t j0 = cb; j0 < c_end; j0 += kIds * kPlanThreads) {
            const uint32_t j = j0 + kIds * tid;
            int id[kIds];
#pragma unroll
            for (int k = 0; k < kIds; ++k) id[k] = kept[k];
            if (j0 != cb || passes > 1) ids_of(j, c_end, id);
            if (!kRelease) {
                if (j < c_end) a.page_table[entry(find_request(s.c0, j), j)] = id[0];
            } else {
#pragma unroll
                for (int k = 0; k < kIds; ++k)
                    if (j + k < c_end) a.free_list[count + (int)(j + k)] = id[k];
            }
        }
        // a page taken just now is read from the free list: its table entry may not be written yet
        auto place_of = [&](int r, int pos) {
            const int pg = pos / kPageTokens;
            const int id = pg < s.held[r] ? a.page_table[(int64_t)s.slot[r] * a.pages_per_seq + pg]
                                          : a.free_list[count - 1 - (int)(s.c0[r] + (pg - s.held[r]))];
            if ((uint32_t)id < (uint32_t)a.kv_pages) return id * kPageTokens + pos % kPageTokens;
            atomicCAS(a.err, 0u, kErrPlanTable);
            return -1;
        };
        if (!kRelease && !kCluster) {
#pragma unroll 1
            for (uint32_t t = tid; t < n_end; t += kPlanThreads) {
                const int r = find_request(s.n0, t), pos = s.past[r] + (int)(t - s.n0[r]);
                a.tok_pos[t] = pos;
                a.slot_map[t] = place_of(r, pos);
            }
        } else if (!kRelease) {
#pragma unroll 1
            for (uint32_t x = tid; x < s.d_end; x += kPlanThreads) {
                const int r = find_request(s.d0, x);
                const uint32_t n0 = s.n0[r], n1 = r + 1 < kPlanThreads ? s.n0[r + 1] : n_end;
                const uint32_t quad = n0 / 4 + (x - s.d0[r]), hi = min(4 * quad + 4, n1);
                uint32_t t = max(4 * quad, n0);
                int pos = s.past[r] + (int)(t - n0);
                if (t + 4 == hi && pos % kPageTokens <= kPageTokens - 4 && !out_of_line) {
                    const int at = place_of(r, pos), up = at < 0 ? 0 : 1;
                    *reinterpret_cast<int4 *>(a.tok_pos + t) = make_int4(pos, pos + 1, pos + 2, pos + 3);
                    *reinterpret_cast<int4 *>(a.slot_map + t) = make_int4(at, at + up, at + 2 * up, at + 3 * up);
                } else {
#pragma unroll 1
                    for (; t < hi; ++t, ++pos) {
                        a.tok_pos[t] = pos;
                        a.slot_map[t] = place_of(r, pos);
                    }
                }
            }
        }
        nb = n_end;
        cb = c_end;
    }
    if (!kRelease)
        for (uint32_t t = n_total + t0; t < (uint32_t)a.max_tokens; t += step) {
            a.tok_pos[t] = 0;
            a.slot_map[t] = -1;
        }
    if (rank == 0 && tid == 0) {
        *a.free_count_out = kRelease ? count + (int)c_total : count - (int)c_total;
        if (!kRelease) a.cu_seqlens[a.requests] = (int)n_total;
    }
}

// ---- q/k/v append -----------------------------------------------------------------------------------------------
//
// y = x * gain / sqrt(mean(x^2) + eps), then (y_d, y_{d+64}) -> (y_d c - y_{d+64} s, y_{d+64} c + y_d s) for q and k.
// Every byte is read once and written once (bound: HBM copy). A quarter-warp takes a head, a lane dims 8l..8l+7 and the
// same 64 further: RoPE's pairs are in one lane, the sum of squares is 3 shuffles, loads and stores are 16 bytes, and
// the arithmetic runs on pairs (f32x2), since with scalar instructions their issue takes longer than the copy.
// A block takes up to 48 heads (blockIdx.y) of every gridDim.x-th row. A thread copies its own bytes of a row to its own
// places of shared memory, kStages - 1 rows ahead (so there is no barrier), and loads the cos / sin of the next row while
// it computes this one. 32768 rows of 48 heads: 95 us, 5.65 TB/s (115 us with a block a row, 133 us so and with scalar
// arithmetic); 64 rows: 2.8 us. 4 stages of 4 blocks an SM and 3 of 5 are alike, 2 of 6 take 119 us.
constexpr int kAppendThreads = 128, kBatch = 3, kStages = 4, kAppendBlocks = 4;  // blocks of an SM
constexpr int kAppendHeads = kAppendThreads / 8, kUnitHeads = kAppendHeads * kBatch;
constexpr int kAppendSmem = kStages * kBatch * kAppendThreads * 32;

struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 pair(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ F2 pair(uint32_t bf16x2) {
    return pair(__uint_as_float(bf16x2 << 16), __uint_as_float(bf16x2 & 0xFFFF0000u));
}
__device__ __forceinline__ float2 split(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(F2 a) {
    const float2 f = split(a);
    __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<uint32_t *>(&h);
}

struct Place {
    int place, pos;
};

__global__ void __launch_bounds__(kAppendThreads, kAppendBlocks)
    qkv_append_kernel(const __grid_constant__ QkvAppendArgs a) {
    extern __shared__ uint4 buf[];  // [stage][batch][2][thread]
    const int tid = threadIdx.x, l = tid & 7, step = gridDim.x;
    const int heads = a.q_heads + 2 * a.kv_heads, qk = a.q_heads + a.kv_heads;
    const int h0 = blockIdx.y * kUnitHeads + (tid >> 3);  // this quarter-warp's first head
    auto fetch = [&](int64_t t, int stage) {
        if (t < a.tokens) {
            const __nv_bfloat16 *from = a.qkv + t * a.ld_qkv + (int64_t)h0 * kHeadDim + 8 * l;
            const uint32_t to = ptx::smem_u32(buf + stage * kBatch * 2 * kAppendThreads + tid);
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (h0 + b * kAppendHeads < heads)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (b * 2 + i) * kAppendThreads * 16),
                                     "l"(from + b * kAppendHeads * kHeadDim + i * 64)
                                     : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto place_of = [&](int64_t t) {
        Place p = {-1, 0};
        if (t < a.tokens) {
            p.place = a.slot_map[t];
            if (a.cos_t) p.pos = a.tok_pos[t];
        }
        return p;
    };
    auto good = [&](const Place &p) {
        return p.place >= 0 && p.place < a.places && (!a.cos_t || (p.pos >= 0 && p.pos < a.rope_rows));
    };
    F2 gain[8];  // of this lane's dims
    auto gain_of = [&](const __nv_bfloat16 *of) {
        const uint4 *g = reinterpret_cast<const uint4 *>(of + 8 * l);
        const uint4 g0 = __ldg(g), g1 = __ldg(g + 8);
        gain[0] = pair(g0.x), gain[1] = pair(g0.y), gain[2] = pair(g0.z), gain[3] = pair(g0.w);
        gain[4] = pair(g1.x), gain[5] = pair(g1.y), gain[6] = pair(g1.z), gain[7] = pair(g1.w);
    };
    float4 cs[2], sn[2], cs_next[2], sn_next[2];  // of dims 8l..8l+7
    auto rope_of = [&](const Place &p, float4 *c, float4 *n) {
        if (a.cos_t && good(p)) {
            const size_t at = (size_t)p.pos * 64 + 8 * l;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                c[i] = __ldg(reinterpret_cast<const float4 *>(a.cos_t + at) + i);
                n[i] = __ldg(reinterpret_cast<const float4 *>(a.sin_t + at) + i);
            }
        }
    };

    int64_t t = blockIdx.x;
    Place now = place_of(t), next = place_of(t + step);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(t + (int64_t)i * step, i);
    rope_of(now, cs, sn);
    bool gain_is_k = false;
    if (a.q_norm) gain_of(a.q_norm);
    for (int stage = 0; t < a.tokens; t += step) {
        fetch(t + (int64_t)(kStages - 1) * step, (stage + kStages - 1) % kStages);
        const Place after = place_of(t + 2 * (int64_t)step);
        rope_of(next, cs_next, sn_next);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        if (good(now)) {
            __nv_bfloat16 *page = a.pool + (size_t)(now.place / kPageTokens) * kv_page_elems(a.kv_heads) +
                                  (now.place % kPageTokens) * kHeadDim + 8 * l;
            __nv_bfloat16 *q_to = a.q_out + t * a.ld_q + (int64_t)h0 * kHeadDim + 8 * l;
            const F2 co[4] = {pair(cs[0].x, cs[0].y), pair(cs[0].z, cs[0].w), pair(cs[1].x, cs[1].y), pair(cs[1].z, cs[1].w)};
            const F2 si[4] = {pair(sn[0].x, sn[0].y), pair(sn[0].z, sn[0].w), pair(sn[1].x, sn[1].y), pair(sn[1].z, sn[1].w)};
            const F2 minus = pair(-1.f, -1.f);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int h = h0 + b * kAppendHeads;
                const uint4 *from = buf + (stage * kBatch + b) * 2 * kAppendThreads + tid;
                uint4 o0 = make_uint4(0, 0, 0, 0), o1 = o0;
                if (h < heads) o0 = from[0], o1 = from[kAppendThreads];
                // the warp's four heads; a v head keeps its bits
                if (__any_sync(0xffffffffu, h < qk) && (a.q_norm || a.cos_t)) {
                    F2 x[4] = {pair(o0.x), pair(o0.y), pair(o0.z), pair(o0.w)};
                    F2 y[4] = {pair(o1.x), pair(o1.y), pair(o1.z), pair(o1.w)};
                    if (a.q_norm) {
                        if ((h >= a.q_heads) != gain_is_k) {
                            gain_is_k = h >= a.q_heads;
                            gain_of(gain_is_k ? a.k_norm : a.q_norm);
                        }
                        F2 sum = x[0] * x[0];
#pragma unroll
                        for (int e = 1; e < 4; ++e) sum = fma2(x[e], x[e], sum);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum = fma2(y[e], y[e], sum);
                        float ss = split(sum).x + split(sum).y;
#pragma unroll
                        for (int m = 4; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
                        const float r = rsqrtf(ss * (1.f / kHeadDim) + a.eps);  // off by 2 ulp at most
                        const F2 rr = pair(r, r);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = x[e] * (rr * gain[e]), y[e] = y[e] * (rr * gain[4 + e]);
                    }
                    if (a.cos_t) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const F2 v = x[e], yn = y[e] * minus;
                            x[e] = fma2(yn, si[e], v * co[e]);
                            y[e] = fma2(y[e], co[e], v * si[e]);
                        }
                    }
                    if (h < qk) {
                        o0 = make_uint4(pack_bf16(x[0]), pack_bf16(x[1]), pack_bf16(x[2]), pack_bf16(x[3]));
                        o1 = make_uint4(pack_bf16(y[0]), pack_bf16(y[1]), pack_bf16(y[2]), pack_bf16(y[3]));
                    }
                }
                __nv_bfloat16 *to = q_to + b * kAppendHeads * kHeadDim;
                if (h >= a.q_heads) {
                    const int kv = h < qk ? 0 : 1, hk = h - a.q_heads - kv * a.kv_heads;
                    to = page + (int64_t)(hk * 2 + kv) * (kPageTokens * kHeadDim);
                }
                if (h < heads) {
                    *reinterpret_cast<uint4 *>(to) = o0;
                    *reinterpret_cast<uint4 *>(to + 64) = o1;
                }
            }
        } else if (now.place != -1 && tid == 0) {
            atomicCAS(a.err, 0u, kErrAppendRow);
        }
        now = next;
        next = after;
#pragma unroll
        for (int i = 0; i < 2; ++i) cs[i] = cs_next[i], sn[i] = sn_next[i];
        stage = (stage + 1) % kStages;
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
    // Up to a size one CTA is faster, above it a cluster of 8. Times in us, one CTA against the cluster, with 1000 cached
    // tokens a request: plans of 64 requests and tokens 3.2, 6.1; of 1024 4.6, 6.1; of 512 requests and 4096 tokens 5.5, 6.4,
    // and 6144 tokens 8.4, 7.1; of 64 requests and 4096 tokens 6.3, 7.1. A release's time goes by its pages, which only the
    // device knows; the host knows how many there can be. All of 40 requests' 2520 pages 4.6, 6.3; of 64's 4032 5.0, 6.4; of
    // 256's 16,128 12.7, 6.7; of 768's 48,384 33.5, 9.1. A release of few pages is 3 us faster on one CTA, whatever it could be.
    const int64_t most_pages = std::min<int64_t>((int64_t)a.requests * a.pages_per_seq, a.kv_pages);
    const bool big = a.keep_len ? a.requests > 768 || most_pages > 8192 : a.requests > kPlanThreads || a.max_tokens > 5 * 1024;
    const unsigned ctas = big ? kPlanCtas : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = (size_t)((a.max_seqs / ctas + 32) / 32) * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = big ? 1 : 0;
    const auto kernel = a.keep_len ? big ? page_step_kernel<true, true> : page_step_kernel<true, false>
                        : big      ? page_step_kernel<false, true>
                                   : page_step_kernel<false, false>;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

cudaError_t launch_qkv_append(const QkvAppendArgs &a, cudaStream_t st) {
    const int groups = (a.q_heads + 2 * a.kv_heads + kUnitHeads - 1) / kUnitHeads;
    const int blocks = std::max(1, device_sms() * kAppendBlocks / groups);
    qkv_append_kernel<<<dim3(std::min(a.tokens, blocks), groups), kAppendThreads, kAppendSmem, st>>>(a);
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
    uint64_t bytes = 0;
    guarded([&] {  // without a device the message of that may not be allocated
        bytes = paged_attention_workspace(tokens, q_heads, kv_heads, device_sms());
        return LRM_OK;
    });
    return bytes;
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
        const int sms = device_sms();
        if (d->workspace_bytes < 0 ||
            (uint64_t)d->workspace_bytes < paged_attention_workspace(a.tokens, a.q_heads, a.kv_heads, sms))
            return op_fail(LRM_ERR_ARGUMENT, "paged attention: the workspace is smaller than "
                                             "lrm_op_paged_attention_workspace says");
        if (!(a.err = device_error_word())) return LRM_ERR_CUDA;
        return op_cuda(launch_paged_attention(a, sms, (cudaStream_t)stream), "paged attention");
    });
}

}  // extern "C"
