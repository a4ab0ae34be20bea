// paged_attn.cu -- attention of each request's new tokens over its cached keys (lrm_op_paged_attention), on the
// 5th-generation tensor cores (tcgen05, TMEM, TMA).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(scale log2(e) q.k_j - m),   m a running reference maximum:
// one pass over the keys, with the statistics and the accumulator in fp32. For the product with v, p is two bf16 values (16
// bits) in items of up to 32 rows. In larger ones it is rounded to bf16, as in the prefill attention: a second product would
// add 320 cycles to a tile's 740 of MMAs a slot, and a second P does not fit beside S and O in tensor memory.
//
// The work is cut evenly over one persistent CTA an SM (paged_sched.h): single tokens, verify chunks and prefill chunks
// of any lengths fill the GPU alike. An item is up to 2 * floor(128 / group) tokens of one request and KV head. Its rows
// are (token, query head) pairs, token-major, so the query heads that share a KV head share its tiles whatever the group
// size, and one TMA box brings their q. 128 rows make a "slot" with S, P and O in half of tensor memory:
//   wide    (more than 128 rows): each tile of K and V is used by both slots' rows;
//   narrow  (33 to 128 rows): one set of rows; the even key tiles go to slot 0 and the odd ones to slot 1, so one
//           slot's products run under the other's softmax; the two states merge at the end;
//   few     (up to 32 rows): as narrow, with keys and rows swapped (below).
// Tiles of wide and narrow items have 80 keys: S (80 columns) and P (40, two bf16 a column) then lie side by side in the
// 128 that O leaves of a slot, so the next S is computed while the softmax still works on this one. With 128 keys, P over
// S, every S waited for the P V before it: 1,000 rows over 121,000 keys took 1.465 million cycles, with 80 keys 1.383 (and
// 1.25 with what came after).
// Warps of a CTA:
//   0, 3    TMA producers: q of an item and K's tiles, and V's tiles, in the order of their use through a ring of five
//           32 KiB stages (5 or 8 pages of 16 tokens, one box a page and 64 dims), running ahead into the next item;
//           warp 3 also cleans V;
//   1       tensor-core issuer (one thread);
//   2       scheduler: walks the CTA's range and hands the items to the others through a ring of four;
//   4..11   softmax, one warpgroup a slot, thread = row (few: thread = key).
// Keys that a row does not see: their scores are replaced before the maximum, and their v, which the product multiplies
// by 0, must not be infinite or NaN. So in tiles where some row's mask bites (the last tokens' own tiles, "dirty") warp 3
// tests v of the keys that not all rows see, and zeroes what is not finite; if a key of the request itself was hit, the
// epilogue adds its original values to the rows that see it.
// Items that a cut passes through leave (m, sum p, unnormalised o) in the workspace, at most two a CTA, and
// paged_combine_kernel merges them. Within a range the last item is walked first: CTAs that share a head's keys then
// all start at key 0 of an item and stream the same tiles at about the same time, from L2.
// Every wait is bounded and reports to the error word.
//
// What bounds it and what it measured (device time, both kernels; 8 KV heads, two query heads each unless said):
//   HBM       64 single tokens over 4096 to 4352 keys: 171 us, 6.48 TB/s, 0.99 of a copy's rate.
//   HBM and the start: 32 x 5 tokens over 100 to 6000 keys, 32 query heads: 39.4 to 41 us by the board, 4.2 TB/s. 3.5 us pass
//             before the first load (the lengths' and page table's loads, the cut, and code that no CTA has fetched yet), 4
//             after the last; every item's own 4,000 cycles are there too.
//   softmax   1,000 tokens over 121,000 keys: 1.25 million cycles, tensor pipe active in 67 percent of them, the
//             exponentials' unit in 67; 820 us at 1.53 GHz. Over seconds the board's 1000 W allow 1.36 GHz and it takes 1,010:
//             a GEMM's sustained rate, at the same clock, would be 701.
//   the same and what an item costs beside its tiles (9,000 cycles of 36,000): 16 x 2048 tokens without a past 320 us.
//   latency   one token over 900 keys: 10.7 us.
// Tried and slower: two issuing warps (their MMAs interleave badly); four softmax warpgroups (spills); a part of the
// exponentials as polynomials on the FMA pipes (the warps' issue is as full as that unit).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "internal.h"
#include "paged.h"
#include "paged_sched.h"
#include "ptx.cuh"

namespace lrm {
namespace {

constexpr int TK = sched::kTileKeys, TKF = sched::kFewTileKeys, KV_ST = sched::kRing, SLOTS = 2, ITEMS = 4, DIRTY = 8;
constexpr int P_COL = 80;  // P's columns in tensor memory, behind S's (two bf16 a column): 80 + 40 of the slot's first 128
constexpr int SUB = 128 * 64 * 2;  // one [128 rows][64] bf16 swizzled sub-tile
constexpr int TILE = 2 * SUB;      // [128 rows][128]
static_assert(TK + TK / 2 <= 128 && TK % kPageTokens == 0 && TK % 16 == 0, "S and P of a tile lie side by side");
constexpr int kThreads = 384;
constexpr int kRegsLaunch = 168;  // 65536 / 384, rounded down to the allocation unit of 8
constexpr int kRegsControl = 72, kRegsSoftmax = 216;
static_assert(128 * kRegsControl + 256 * kRegsSoftmax <= kThreads * kRegsLaunch, "register split exceeds the launch");
constexpr float kRescaleThreshold = 8.0f;  // log2 units: the reference maximum moves only when a tile exceeds it by more
constexpr int kFewRows = sched::kFewRows;  // items of up to this many rows run with keys and rows swapped
constexpr int FEW_SUB = kFewRows * 128;  // half of the dims of up to 32 rows of q
constexpr int FEW_P_SUB = 2 * FEW_SUB, FEW_P = 2 * FEW_P_SUB;  // half of the keys (all) of P, two lines a row, in a slot
constexpr uint32_t kErrWaitProducer = 0x4010, kErrWaitIssuer = 0x4011, kErrWaitSoftmax = 0x4012, kErrWaitScheduler = 0x4013;

// One item's share of a CTA's range: key tiles [kb, ke) of it.
struct Item {
    int tok0, ntok;     // its token rows in q and out; ntok 0 ends the list
    int kvh, pos0;      // KV head; position of its first token
    int kb, ke;
    int npages, dest;   // pages of the request; dest -1: the whole item, else the partial slot 0 or 1
    int dirty, pad;     // its tiles from this one on are not seen whole by some row
    int64_t table;      // the request's first page-table entry
};

// An item whose last keys lie in later CTAs' ranges, left by the CTA that holds its first: partial slot 1 of this CTA
// and slots 0 of the next `follow` CTAs make it up. ntok 0: none.
struct alignas(16) Record {
    int tok0, ntok, kvh, follow;
};

// A value that is the same in all lanes, so that the compiler knows it is.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// A request's tokens and keys when it is sound and has any, else n = 0.
struct Request {
    int start, n, kv, slot;
};

// A walk over a CTA's range from its last item to its first: item i of `items` of request r's KV head h, and the share's end
// in it, in units; units of the range that are left.
struct Walk {
    Request q;
    sched::Item cost;
    int r, h, i, items, end;
    int pushed;  // items handed out so far
    uint64_t left;
    Record rec;
};

struct Control {
    uint64_t q_full[2], q_empty[2], fin, o_free;  // q: even and odd items
    uint64_t kv_full[KV_ST], kv_empty[KV_ST];
    uint64_t s_full[SLOTS], s_free[SLOTS], p_full[SLOTS], o_done[SLOTS];  // a phase each product of the slot
    uint64_t item_full[ITEMS], item_empty[ITEMS];
    uint64_t v_clean[DIRTY];  // dirty tile n's v is clean: barrier n % DIRTY
    int z[2][32];  // the producers': z coordinates of a window of pages (one int behind it is read, and not used)
    int kv_issued[KV_ST], q_issued[2];  // the last ring item copied to a stage, the last item's q to a place; from 1, 0: none
    int gave_up;                        // the issuer did not get to the end of the items
    Item items[ITEMS];
    uint64_t warp_sum[kThreads / 32];
    uint64_t started;
    Walk walk;  // of the scheduler, behind the range's last item
    uint32_t tmem;
    int poison[sched::kMarks];  // the item (counted from 1) in which v of a visible key was zeroed, by item % kMarks
    union {
        float ml[SLOTS][128][2];  // narrow: the slots' states
        struct {                  // few
            union {
                alignas(16) float max[SLOTS][kFewRows][4];  // a tile's maxima, by row and warp (read as float4)
                float l[SLOTS][4][kFewRows];    // sums of p, by warp and row
            };
            float m[SLOTS][kFewRows], neg[SLOTS][kFewRows], alpha[SLOTS][kFewRows];
        } few;
    };
};
static_assert(sched::kSoftmaxPolls > sched::kIssuerWaits * sched::kPolls, "the softmax's warps give up together");
static_assert(offsetof(Control, few) % 16 == 0, "few.max is read as float4");
constexpr int SMEM_BYTES = (SLOTS + KV_ST) * TILE + (int)sizeof(Control);
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");
static_assert(SLOTS * FEW_P <= TILE && 2 * 2 * FEW_SUB <= TILE, "q of two few-row items in one tile, their P in the other");

struct Params {
    PagedAttnArgs a;
    sched::Shape shape;
    int group, tt, rows_cap;  // query heads a KV head; tokens a slot; rows of a partial slot
    int few_tok;              // tokens of a few-row item's q box
    int inv_group;            // ceil(2^16 / group): r * inv_group >> 16 = r / group for r < 256
    float *part_o, *part_ml;
    Record *records;
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ void add2(float &d0, float &d1, float a0, float a1) {
    asm("{\n\t.reg .b64 a, d;\n\tmov.b64 d, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\t"
        "add.rn.f32x2 d, d, a;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(d0), "+f"(d1)
        : "f"(a0), "f"(a1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// ptx::mbar_wait with the first poll (which by itself waits some time) on the straight path and the loop behind it out of
// the way. Three roles' code shares an SM sub-partition's instruction buffers, so code that is not straight costs some 5
// cycles an instruction in fetches: with the polls unrolled (60 KB of code for thirty waits) every role stalled on them.
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, uint32_t *err, uint32_t code) {
    if (__builtin_expect(try_wait(bar, parity), 1)) return true;
    const uint32_t polls = code == kErrWaitSoftmax ? sched::kSoftmaxPolls : sched::kPolls;
#pragma unroll 1
    for (uint32_t i = 0; i < polls; ++i)
        if (try_wait(bar, parity)) return true;
    atomicCAS(err, 0u, code);
    return false;
}
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, uint32_t *err, uint32_t code) {
    return wait_bar(ptx::smem_u32(bar), parity, err, code);
}

// tma_load_3d of a page's 64 dims from `x` on, with shared addresses as they are.
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(x), "r"(0), "r"(z)
        : "memory");
}

__device__ __forceinline__ bool finite_bf16(uint32_t h) { return (h & 0x7F80u) != 0x7F80u; }

struct RawRequest {
    int start, end, kv, slot;
};
__device__ __forceinline__ RawRequest fetch_request(const PagedAttnArgs &a, int r) {
    return RawRequest{a.cu_seqlens[r], a.cu_seqlens[r + 1], a.kv_len[r], a.slots[r]};
}
__device__ __forceinline__ Request check_request(const PagedAttnArgs &a, const RawRequest &w, bool report) {
    const int64_t n = (int64_t)w.end - w.start;
    const bool ok = w.start >= 0 && n > 0 && w.end <= a.tokens && w.slot >= 0 && w.slot < a.max_seqs && w.kv >= n &&
                    w.kv <= (int64_t)a.pages_per_seq * kPageTokens;
    if (report && !ok && n != 0) atomicCAS(a.err, 0u, kErrAttnRequest);
    return Request{w.start, ok ? (int)n : 0, w.kv, w.slot};
}
__device__ __forceinline__ Request load_request(const PagedAttnArgs &a, int r, bool report) {
    return check_request(a, fetch_request(a, r), report);
}

// Tests v of keys [from, to) of a tile, one a lane of a warp, and zeroes what is not finite. Keys up to `last_seen` are seen
// by some row: if one of them is hit, `poison` is set.
__device__ __forceinline__ void clean_v(uint8_t *tile, int from, int to, int lane, int last_seen, volatile int *poison,
                                        int id) {
    const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll 1
    for (int key = from + lane; key < to; key += 32) {
        const uint32_t row = ptx::smem_u32(tile) + key * 128;
        __nv_bfloat162 acc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = zero;
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {  // 16-byte chunks in an order that differs by lane: no bank conflicts
            const uint4 v = ptx::ld_shared_v4(row + (i >> 3) * SUB + (((i + lane) & 7) << 4));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)  // 0 * v + acc: NaN once v is infinite or NaN
                acc[e] = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&w[e]), zero, acc[e]);
        }
        const float2 f = __bfloat1622float2(__hadd2(__hadd2(acc[0], acc[1]), __hadd2(acc[2], acc[3])));
        if (f.x != f.x || f.y != f.y) {
            if (key <= last_seen) *poison = id;
#pragma unroll 1
            for (int i = 0; i < 64; ++i) {
                const uint32_t at = row + (i >> 5) * SUB + (i & 31) * 4;
                uint32_t w;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
                if (!finite_bf16(w)) w &= 0xFFFF0000u;
                if (!finite_bf16(w >> 16)) w &= 0x0000FFFFu;
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(w) : "memory");
            }
        }
    }
    ptx::fence_proxy_async();  // the tensor core reads the tile through the async proxy
}

// Adds the values that clean_v zeroed to one slot's O (128 columns at `t`, this warp's lanes), from the cache: this
// lane's row sees keys lo .. hi, of which the slot has those of tiles tile0, tile0 + step, ... Rare, so it is kept out of the
// kernel's instruction stream.
__device__ __noinline__ void add_poison(const PagedAttnArgs &a, int64_t table, int kvh, int lo, int hi, int tk, int tile0,
                                        int step, uint32_t t) {
#pragma unroll 1
    for (int c = 0; c < kHeadDim; c += 16) {
        uint32_t o[16];
        ptx::tmem_ld16(t + c, o);
        ptx::tmem_ld_wait();
#pragma unroll 1
        for (int key = lo; key <= hi; ++key) {
            if ((key / tk - tile0) % step != 0) continue;  // the other slot's tile
            const int pg = a.page_table[table + key / kPageTokens];
            if (pg < 0 || pg >= a.kv_pages) continue;
            const __nv_bfloat16 *v = a.pool + (size_t)pg * kv_page_elems(a.kv_heads) +
                                     (size_t)(kvh * 2 + 1) * (kPageTokens * kHeadDim) + (key % kPageTokens) * kHeadDim + c;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = __bfloat162float(v[e]);
                if (!(fabsf(x) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
            }
        }
        __syncwarp();
        ptx::tmem_st16(t + c, o);
    }
    ptx::tmem_st_wait();
}

// Within each group of four lanes: v[j] becomes lane j's v[own lane]. A thread holds 64 bytes of its own row; after
// this, v[j] is 16 bytes of row j of the group, and the four lanes' 16 bytes are 64 contiguous ones.
__device__ __forceinline__ void quad_transpose(uint4 (&v)[4], int lane) {
#pragma unroll
    for (int step = 1; step <= 2; step *= 2) {
        const bool up = lane & step;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = step == 1 ? 2 * i : i, y = x + step;
            uint4 t = up ? v[x] : v[y];
            t.x = __shfl_xor_sync(0xffffffffu, t.x, step);
            t.y = __shfl_xor_sync(0xffffffffu, t.y, step);
            t.z = __shfl_xor_sync(0xffffffffu, t.z, step);
            t.w = __shfl_xor_sync(0xffffffffu, t.w, step);
            if (up)
                v[x] = t;
            else
                v[y] = t;
        }
    }
}

// ---- items of few rows ------------------------------------------------------------------------------------------
//
// With 1 to 32 rows (single tokens, short drafts) most of a 128-row tile would be empty and a thread would walk 128
// scores alone. So keys and rows change places: the keys fill the MMA's 128 rows, S^T = K Q^T has 16 or 32 columns, one a
// row, and a thread holds one key's scores. The running maximum of a row is the same in all threads of a slot's
// warpgroup and moves only when some score exceeds it by 2^8, which one barrier with an OR finds out; only then (and at
// an item's first tile) are the tile's maxima reduced over threads. P goes to shared memory as the B operand of
// O^T = V^T P^T; sums of p stay per thread until the end. A tile costs 1,400 cycles, which hide under the 2,800 that its K
// and V take as one SM's share of HBM.
// Each row of P has two rows of bf16 here, its first 16 bits and the rest: together off by 2^-15 of p at most, so that a
// single token is as precise as with lrm_op_decode_attention, whose p is fp32. Groups of eight rows alternate (eight rows,
// the eight rests, ...), so O^T's columns do too, and up to eight rows still make one MMA of 16 columns. (p rounded to bf16
// alone: 64 single tokens over 4096 keys off by 2.3e-3 in norm instead of 1.66e-3, which is the output's own rounding; 32 x 5
// drafted tokens 39.2 us instead of 39.4, on another board 40.0 and 41.0, 8 x 511 among 56 decodes 54.4 instead of 54.9,
// single tokens alike. The rests in eight MMAs of their own: 32 x 5 42.7 us where it is 41.2, 64 x 4096 173.9 and 172.5.)
struct RoleState {
    Control *c;
    const Params *p;
    uint8_t *pt;  // this slot's P
    uint32_t tmem;
    int s, quarter, lane, cta, k;
};

__device__ __forceinline__ bool barrier_or(int id, int count, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((int)x), "r"(id), "r"(count)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void tmem_ld8(uint32_t t, float (&x)[8]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(x);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(t));
}
__device__ __forceinline__ void tmem_st8(uint32_t t, const float (&x)[8]) {
    const uint32_t *r = reinterpret_cast<const uint32_t *>(x);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(t), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// The sum of the values that clean_v zeroed in dim d of keys lo .. hi in tiles tile0, tile0 + step, ... (infinite or NaN, or
// 0 if there are none).
__device__ __noinline__ float poison_sum(const PagedAttnArgs &a, int64_t table, int kvh, int lo, int hi, int tk, int tile0,
                                         int step, int d) {
    float sum = 0.f;
#pragma unroll 1
    for (int key = lo; key <= hi; ++key) {
        if ((key / tk - tile0) % step != 0) continue;  // the other slot's tile
        const int pg = a.page_table[table + key / kPageTokens];
        if (pg < 0 || pg >= a.kv_pages) continue;
        const float x = __bfloat162float(a.pool[(size_t)pg * kv_page_elems(a.kv_heads) +
                                                (size_t)(kvh * 2 + 1) * (kPageTokens * kHeadDim) +
                                                (key % kPageTokens) * kHeadDim + d]);
        if (!(fabsf(x) < INFINITY)) sum += x;
    }
    return sum;
}

__device__ __forceinline__ void load8(const float *shared, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(shared)[0], b = reinterpret_cast<const float4 *>(shared)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// What is left of p beside its first 16 bits (the difference is exact). Where p is above 0 this is at least bf16's smallest
// number, so that it times an infinite v is that infinity and no NaN.
__device__ __forceinline__ float rest(float p) {
    const float hi = __uint_as_float(__float_as_uint(p) & 0xFFFF0000u);
    return fmaxf(p - hi, fminf(p, 0x1p-133f));
}

// Eight rows' scores of this thread's key; rows that do not see it (those before `from`) as -inf.
__device__ __forceinline__ void load_scores(uint32_t t, int from, float (&x)[8]) {
    tmem_ld8(t, x);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e >= from ? x[e] : -INFINITY;
}

// An item's tiles in one slot and its epilogue, eight rows at a time in rolled loops (code that the instruction cache
// holds). Columns of the slot's tensor memory: S^T at 0, O^T at 128, the thread's sums of p at 192 (not beside S^T, which the
// next item's first scores may overwrite while this item is still read out).
// done: products of the items before, a slot
__device__ __forceinline__ bool few_item(const RoleState &r, const Item &it, uint32_t &steps, uint32_t (&done)[SLOTS]) {
    Control &c = *r.c;
    const PagedAttnArgs &a = r.p->a;
    const int s = r.s, lane = r.lane, group = r.p->group, nt = it.ke - it.kb, rows = it.ntok * group;
    const int key = r.quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(r.quarter * 32) << 16, tS = r.tmem + 256 * s + lanes, tO = tS + 128, tL = tS + 192;
    const float sc = a.scale_log2;
    // P[row][key] with keys contiguous, 64 a 128-byte swizzled line; rows g .. g + 7 at lines 2g .. 2g + 7, their rests behind
    const uint32_t pt = ptx::smem_u32(r.pt) + (key >> 6) * FEW_P_SUB, pk = (key & 63) * 2;
#pragma unroll 1
    for (int j = s; j < nt; j += 2, ++steps) {
        if (!wait_bar(&c.s_full[s], steps & 1, a.err, kErrWaitSoftmax)) return false;
        ptx::tc_fence_after();
        const int key0 = (it.kb + j) * TKF;
        const bool first = j == s, dirty = key0 + TKF - 1 > it.pos0;  // dirty: some row does not see the whole tile
        // rows are token-major, so the key is seen from this row on
        const int from = dirty ? min(max(key0 + key - it.pos0, 0), 64) * group : 0;
        bool over = false;
        if (!first) {
#pragma unroll 1
            for (int g = 0; g < rows; g += 8) {
                float x[8], m[8];
                load8(&c.few.m[s][g], m);
                load_scores(tS + g, from - g, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) over |= g + e < rows && x[e] * sc > m[e] + kRescaleThreshold;
            }
        }
        if (first || barrier_or(6 + s, 128, over)) {
#pragma unroll 1
            for (int g = 0; g < rows; g += 8) {
                float x[8];
                load_scores(tS + g, from - g, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = warp_max(x[e]);
                    if (lane == e) c.few.max[s][g + e][r.quarter] = w;
                }
            }
            ptx::named_barrier(6 + s, 128);
            if (key < kFewRows) {  // thread = row
                const float4 w = *reinterpret_cast<const float4 *>(c.few.max[s][key]);
                const float mx = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)) * sc, old = c.few.m[s][key];
                const bool up = first || mx > old + kRescaleThreshold;
                c.few.alpha[s][key] = up ? ptx::ex2(old - mx) : 1.f;  // 0 when no key was seen before
                if (up) {
                    c.few.m[s][key] = mx;
                    c.few.neg[s][key] = mx == -INFINITY ? 0.f : -mx;  // a row that has seen no key yet: p = 0
                }
            }
            ptx::named_barrier(6 + s, 128);
            if (!first) {
                // O is quiescent once the slot's product before has been added
                if (!wait_bar(&c.o_done[s], (steps - 1) & 1, a.err, kErrWaitSoftmax)) return false;
                ptx::tc_fence_after();
#pragma unroll 1
                for (int g = 0; g < rows; g += 8) {
                    float o[16], l[8], alpha[8];
                    load8(&c.few.alpha[s][g], alpha);
                    ptx::tmem_ld16(tO + 2 * g, reinterpret_cast<uint32_t(&)[16]>(o));
                    tmem_ld8(tL + g, l);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[e] *= alpha[e];
                        o[e + 8] *= alpha[e];
                        l[e] *= alpha[e];
                    }
                    ptx::tmem_st16(tO + 2 * g, reinterpret_cast<uint32_t(&)[16]>(o));
                    tmem_st8(tL + g, l);
                }
                ptx::tmem_st_wait();
            }
        }
        // P's place is free once the slot's product before has read it
        if (steps > 0 && !wait_bar(&c.o_done[s], (steps - 1) & 1, a.err, kErrWaitSoftmax)) return false;
#pragma unroll 1
        for (int g = 0; g < rows; g += 8) {
            float x[8], l[8], neg[8];
            load8(&c.few.neg[s][g], neg);
            tmem_ld8(tL + g, l);
            load_scores(tS + g, from - g, x);
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = ptx::ex2(fmaf(x[e], sc, neg[e]));
                l[e] = first ? x[e] : l[e] + x[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __byte_perm(__float_as_uint(x[2 * e]), __float_as_uint(x[2 * e + 1]), 0x7632);
            const uint32_t row = pt + g * 256;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(row + part * 1024 + e * 128 + (pk ^ (e << 4))),
                                 "h"((uint16_t)(w[e / 2] >> (e & 1 ? 16 : 0))));
                if (part == 0) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = pack2(rest(x[2 * e]), rest(x[2 * e + 1]));
                }
            }
            tmem_st8(tL + g, l);
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&c.s_free[s]);
        ptx::fence_proxy_async();  // P is read through the async proxy
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&c.p_full[s]);
    }

    const bool two = nt > 1;  // the second slot has a state
    done[0] += (nt + 1) / 2;
    done[1] += nt / 2;
    // This warp's sums of each row's p, while the last product runs: eight rows over 32 lanes, each step halving the rows
    // that a lane holds.
    if (nt > s) {
#pragma unroll 1
        for (int g = 0; g < rows; g += 8) {
            float l[8];
            tmem_ld8(tL + g, l);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int o = 4; o > 0; o /= 2) {
                const bool up = lane & o;
#pragma unroll
                for (int e = 0; e < o; ++e) {
                    const float give = up ? l[e] : l[e + o], keep = up ? l[e + o] : l[e];
                    l[e] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
            }
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], 8);
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], 16);
            if (lane < 8) c.few.l[s][r.quarter][g + lane] = l[0];
        }
    }
    // This slot's last product first: the other's barrier is then at its own last one's phase. (Both warpgroups are through
    // with their tiles behind these waits, so neither waits in vain at the barriers below.)
    bool ok = nt <= s || wait_bar(&c.o_done[s], (done[s] - 1) & 1, a.err, kErrWaitSoftmax);
    if (ok && nt > 1 - s) ok = wait_bar(&c.o_done[1 - s], (done[1 - s] - 1) & 1, a.err, kErrWaitSoftmax);
    if (!ok) return false;
    ptx::tc_fence_after();
    if (c.poison[r.k % sched::kMarks] == r.k + 1) {
        if (nt > s)
#pragma unroll 1
            for (int e = 0; e < rows; ++e) {
                uint32_t o;
                const uint32_t at = tO + 2 * (e & ~7) + (e & 7);  // row e's column
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(o) : "r"(at));
                ptx::tmem_ld_wait();
                const int last = min(it.pos0 + (e * r.p->inv_group >> 16), it.ke * TKF - 1);
                o = __float_as_uint(__uint_as_float(o) + poison_sum(a, it.table, it.kvh, max(it.kb * TKF, it.pos0 + 1), last,
                                                                    TKF, it.kb + s, 2, key));
                asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(at), "r"(o) : "memory");
            }
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::named_barrier(1, 256);
        ptx::tc_fence_after();
    }
    ptx::named_barrier(1, 256);
    // Lane e: row e's place in the output and its weights of the two slots' O.
    const float m0 = c.few.m[0][lane], m1 = c.few.m[1][lane];
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        l0 += c.few.l[0][q][lane];
        l1 += c.few.l[1][q][lane];
    }
    ptx::named_barrier(1, 256);  // read by both before either may write there again
    if (!two) l1 = 0.f;
    const float mt = l0 == 0.f ? m1 : (l1 == 0.f ? m0 : fmaxf(m0, m1));
    float w0 = l0 == 0.f ? 0.f : ptx::ex2(m0 - mt), w1 = l1 == 0.f ? 0.f : ptx::ex2(m1 - mt);
    const float lt = (l0 == 0.f ? 0.f : w0 * l0) + (l1 == 0.f ? 0.f : w1 * l1);
    const size_t part = ((size_t)r.cta * 2 + (it.dest > 0)) * r.p->rows_cap;
    const int tok = lane * r.p->inv_group >> 16;
    int64_t at;  // of the row in out, or in the partial results
    if (it.dest < 0) {
        const float inv = 1.f / lt;
        w0 *= inv;
        w1 *= inv;
        at = (int64_t)(it.tok0 + tok) * a.ld_out + (int64_t)(it.kvh * group + lane - tok * group) * kHeadDim;
    } else {
        at = (int64_t)(part + lane) * kHeadDim;
        if (s == 0 && r.quarter == 0 && lane < rows)
            *reinterpret_cast<float2 *>(r.p->part_ml + (part + lane) * 2) = make_float2(mt, lt);
    }
    // Every other eight rows are this warpgroup's to write; thread = dim.
#pragma unroll 1
    for (int g = 8 * s; g < rows; g += 16) {
        float o[16], o1[16];
        ptx::tmem_ld16(r.tmem + lanes + 128 + 2 * g, reinterpret_cast<uint32_t(&)[16]>(o));
        if (two) ptx::tmem_ld16(r.tmem + lanes + 256 + 128 + 2 * g, reinterpret_cast<uint32_t(&)[16]>(o1));
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[e] += o[e + 8];  // the rests' share
            o[e] *= __shfl_sync(0xffffffffu, w0, g + e);
            const float v1 = __shfl_sync(0xffffffffu, w1, g + e);
            if (two) o[e] = fmaf(o1[e] + o1[e + 8], v1, o[e]);
            const int64_t to = __shfl_sync(0xffffffffu, at, g + e) + key;
            if (g + e < rows) {
                if (it.dest < 0)
                    a.out[to] = __float2bfloat16_rn(o[e]);
                else
                    r.p->part_o[to] = o[e];
            }
        }
    }
    ptx::tc_fence_before();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&c.o_free);
    return true;
}

// The share of the walk's item that lies in the range, taken off its units.
__device__ __forceinline__ Item take_share(const Params &p, const sched::Cut &cut, uint64_t u1, int cta, Walk &w) {
    Item it;
    const sched::Share share = sched::share_of(w.cost, w.end, w.left);
    const int span = SLOTS * p.tt, tk = w.cost.tile == sched::kFew.tile ? TKF : TK;
    it.kb = share.kb;
    it.ke = share.ke;
    it.table = (int64_t)w.q.slot * p.a.pages_per_seq;
    if (it.ke > it.kb)  // the producers' first load of page ids would miss otherwise
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.a.page_table + it.table + it.kb * (tk / kPageTokens)));
    it.tok0 = w.q.start + w.i * span;
    it.ntok = min(span, w.q.n - w.i * span);
    it.kvh = w.h;
    it.pos0 = w.q.kv - w.q.n + w.i * span;
    it.npages = (w.q.kv + kPageTokens - 1) / kPageTokens;
    it.dirty = max(0, (tk == TK ? (it.pos0 + 1) / TK : (it.pos0 + 1) / TKF) - it.kb);
    it.dest = share.dest;
    if (it.dest == 1 && it.ke > it.kb)  // the range's last item, begun here: the rest of it lies behind the range
        w.rec = Record{it.tok0, it.ntok, w.h, sched::cta_of(cut, u1 - 1 + (uint64_t)(w.cost.units - w.end)) - cta};
    w.left -= (uint64_t)(w.end - share.begin);
    return it;
}

__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tq_few,
                      const __grid_constant__ CUtensorMap tkv, const __grid_constant__ Params p) {
    ptx::griddep_wait();
    ptx::griddep_launch();
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sQ = smem;                // SLOTS tiles
    uint8_t *sKV = sQ + SLOTS * TILE;  // KV_ST tiles: ring item 2j is K_j, 2j + 1 is V_j
    Control &c = *reinterpret_cast<Control *>(sKV + KV_ST * TILE);
    const PagedAttnArgs &a = p.a;
    uint32_t *err = a.err;
    // (the shuffle tells the compiler that the warp index, and so the role, is the same in all lanes)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
    const int cta = blockIdx.x;
    const sched::Shape &shape = p.shape;
    // This thread's requests, `per` of them. The first one's lengths are on their way while the CTA sets itself up.
    const int per = a.requests <= kThreads ? 1 : (a.requests + kThreads - 1) / kThreads;
    const int r0 = min(a.requests, tid * per), r1 = min(a.requests, r0 + per);
    RawRequest raw = {0, 0, 0, 0};
    if (r0 < r1) raw = fetch_request(a, r0);
    if (ptx::smem_u32(smem) & 1023) {  // the swizzled tiles and their descriptors need 1024-byte alignment
        if (tid == 0) {
            atomicCAS(err, 0u, kErrWaitScheduler);
            p.records[cta] = Record{0, 0, 0, 0};
        }
        return;
    }

    if (warp == 2) {
        if (lane == 0) {
            ptx::mbar_init(&c.q_full[0], 1);
            ptx::mbar_init(&c.q_full[1], 1);
            ptx::mbar_init(&c.q_empty[0], 1);
            ptx::mbar_init(&c.q_empty[1], 1);
            ptx::mbar_init(&c.fin, 1);
            ptx::mbar_init(&c.started, 1);
            ptx::mbar_init(&c.o_free, 8);
            for (int s = 0; s < KV_ST; ++s) {
                ptx::mbar_init(&c.kv_full[s], 1);
                ptx::mbar_init(&c.kv_empty[s], 1);
            }
            for (int s = 0; s < SLOTS; ++s) {
                ptx::mbar_init(&c.s_full[s], 1);
                ptx::mbar_init(&c.s_free[s], 4);
                ptx::mbar_init(&c.p_full[s], 4);
                ptx::mbar_init(&c.o_done[s], 1);
            }
            for (int s = 0; s < sched::kMarks; ++s) c.poison[s] = 0;
            for (int s = 0; s < KV_ST; ++s) c.kv_issued[s] = 0;
            c.q_issued[0] = c.q_issued[1] = c.gave_up = 0;
            for (int s = 0; s < DIRTY; ++s) ptx::mbar_init(&c.v_clean[s], 1);
            for (int s = 0; s < ITEMS; ++s) {
                ptx::mbar_init(&c.item_full[s], 1);
                ptx::mbar_init(&c.item_empty[s], 11);  // two producers, the issuer, eight softmax warps
            }
            ptx::fence_barrier_init();
        }
    } else if (warp == 1) {
        ptx::tmem_alloc(&c.tmem, 512);
        ptx::tmem_relinquish();
    } else if (warp == 0 && lane == 0) {
        ptx::prefetch_tmap(&tq);
        ptx::prefetch_tmap(&tq_few);
        ptx::prefetch_tmap(&tkv);
    }

    // ---- this CTA's range ----
    // Units of each thread's requests, their exclusive sums over the threads, and the request of the range's last unit.
    Request mine = check_request(a, raw, cta == 0);
    uint64_t head = mine.n ? sched::head_units(shape, mine.n, mine.kv) : 0;
    uint64_t own = head * (uint64_t)a.kv_heads;
#pragma unroll 1
    for (int r = r0 + 1; r < r1; ++r) {
        const Request q = load_request(a, r, cta == 0);
        if (q.n) own += sched::head_units(shape, q.n, q.kv) * (uint64_t)a.kv_heads;
    }
    uint64_t incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) c.warp_sum[warp] = incl;
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    uint64_t before = incl - own, units = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += c.warp_sum[w];
        units += c.warp_sum[w];
    }
    const uint32_t tmem = __shfl_sync(0xffffffffu, c.tmem, 0);
    const sched::Cut cut = sched::make_cut(units, (int)gridDim.x, sched::kLeastUnits);
    const bool idle = cta >= cut.ctas;
    const uint64_t u0 = sched::begin(cut, cta), u1 = sched::begin(cut, cta + 1);
    if (!idle && before <= u1 - 1 && u1 - 1 < before + own) {
        // The thread whose requests hold the range's last unit hands out that item, so that the rest can begin.
        Walk w;
        w.r = r0;
        uint64_t at = before, sum = head * (uint64_t)a.kv_heads;  // units before request r, and of it
#pragma unroll 1
        while (u1 - 1 >= at + sum) {
            at += sum;
            mine = load_request(a, ++w.r, false);
            head = mine.n ? sched::head_units(shape, mine.n, mine.kv) : 0;
            sum = head * (uint64_t)a.kv_heads;
        }
        w.q = mine;
        w.h = (int)sched::quotient(u1 - 1 - at, head);
        const uint64_t off = u1 - 1 - at - (uint64_t)w.h * head;
        w.items = sched::items_of(shape, mine.n);
        w.i = sched::item_at(shape, mine.n, mine.kv, off, w.items);
        w.cost = sched::item_of(shape, mine.n, mine.kv, w.i, w.items);
        w.end = (int)(off - sched::units_before(shape, mine.n, mine.kv, w.i)) + 1;
        w.left = u1 - u0;
        w.rec = Record{0, 0, 0, 0};
        const Item it = take_share(p, cut, u1, cta, w);
        w.pushed = it.ke > it.kb;  // a share of the item's own cost alone has no tiles
        if (w.pushed) {
            c.items[0] = it;
            ptx::mbar_arrive(&c.item_full[0]);
        }
        c.walk = w;
        ptx::mbar_arrive(&c.started);
    }
    __syncwarp();

    if (idle) {
        if (tid == 0) p.records[cta] = Record{0, 0, 0, 0};
    } else if (warp < 4) {
        ptx::setmaxnreg_dec<kRegsControl>();
        if (warp == 2) {
            // ---- scheduler ----
            if (lane == 0) {
                bool ok = wait_bar(&c.started, 0, err, kErrWaitScheduler);
                Walk w = c.walk;
                while (ok) {
                    Item it = {};
                    if (w.left > 0) {
                        // the item before: of this head, else of the head before, else of the request before
                        if (w.i > 0) {
                            --w.i;
                        } else {
                            if (w.h > 0) {
                                --w.h;
                            } else {
                                do w.q = load_request(a, --w.r, false);
                                while (!w.q.n);
                                w.h = a.kv_heads - 1;
                                w.items = sched::items_of(shape, w.q.n);
                            }
                            w.i = w.items - 1;
                        }
                        w.cost = sched::item_of(shape, w.q.n, w.q.kv, w.i, w.items);
                        w.end = w.cost.units;
                        it = take_share(p, cut, u1, cta, w);
                        if (it.ke == it.kb) continue;
                    }
                    const int k = w.pushed++;
                    ok = wait_bar(&c.item_empty[k % ITEMS], ((k / ITEMS) & 1) ^ 1, err, kErrWaitScheduler);
                    if (!ok) break;
                    c.items[k % ITEMS] = it;
                    ptx::mbar_arrive(&c.item_full[k % ITEMS]);
                    if (it.ntok == 0) break;  // the end
                }
                p.records[cta] = ok ? w.rec : Record{0, 0, 0, 0};
            }
        } else if (warp == 0 || warp == 3) {
            // ---- TMA producers: warp 0 q and the tiles of K, warp 3 those of V ----
            // A stage's barrier counts phases of both; the ring's order is also the order in which the tiles are released,
            // and a producer's next tile is at most 5 items on, so its wait cannot be a phase behind.
            const int kv = warp == 3;
            const int oob = a.kv_pages * a.kv_heads * 2;  // past the tensor map: read as zeros, without a memory access
            int ring = 0, q_free = 0;  // ring items of the items before this one; items known to be through with q
            int cleaned = 0;           // dirty tiles so far
            bool few_before = false;
            for (int k = 0;; ++k) {
                bool ok = wait_bar(&c.item_full[k % ITEMS], (k / ITEMS) & 1, err, kErrWaitProducer);
                if (__any_sync(0xffffffffu, !ok)) break;
                const Item &item = c.items[k % ITEMS];
                const int tok0 = uniform(item.tok0), ntok = uniform(item.ntok), kvh = uniform(item.kvh);
                const int kb = uniform(item.kb), nt = uniform(item.ke) - kb, npages = uniform(item.npages);
                const int32_t *pages = a.page_table + item.table;
                const int pos0 = item.pos0, item_dirty = item.dirty;
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&c.item_empty[k % ITEMS]);
                if (ntok == 0) break;
                const bool few = ntok * p.group <= kFewRows, wide = ntok > p.tt;
                const int tile_pages = few ? TKF / kPageTokens : TK / kPageTokens, window = 32 / tile_pages;
                // The z coordinates (K or V block of page and head) of a window of tiles, one a lane.
                // Its page ids are loaded ahead and first used when they are needed (for the first ones, once q is on its way).
                auto fetch = [&](int t) {
                    const int pg = (kb + t) * tile_pages + lane;
                    return pg < npages ? pages[pg] : 0;
                };
                auto place = [&](int t, int id) {
                    if ((kb + t) * tile_pages + lane >= npages) return oob;  // keys past the request, which no row sees
                    if ((uint32_t)id < (uint32_t)a.kv_pages) return (id * a.kv_heads + kvh) * 2 + kv;
                    atomicCAS(err, 0u, kErrAttnPage);
                    return oob;
                };
                int id = fetch(0);
                if (!kv) {
                    // Two few-row items in a row use different places for q, so the second one's q is loaded while the
                    // first still runs; otherwise q's place is free once the item before is through. Even and odd items
                    // have a barrier each: one that is waited for late, behind two items, would have lost its phase.
                    for (const int need = few && few_before ? k - 1 : k; ok && q_free < need; ++q_free)
                        ok = wait_bar(&c.q_empty[q_free & 1], (q_free >> 1) & 1, err, kErrWaitProducer);
                    if (__any_sync(0xffffffffu, !ok)) break;
                    few_before = few;
                    if (ptx::elect_one()) {
                        uint64_t *bar = &c.q_full[k & 1];
                        c.q_issued[k & 1] = k + 1;
                        if (few) {
                            uint8_t *dst = sQ + (k & 1) * 2 * FEW_SUB;
                            ptx::mbar_arrive_expect_tx(bar, p.few_tok * p.group * 256);
                            ptx::tma_load_3d(dst, &tq_few, bar, 0, kvh * p.group, tok0);
                            ptx::tma_load_3d(dst + FEW_SUB, &tq_few, bar, 64, kvh * p.group, tok0);
                        } else {
                            ptx::mbar_arrive_expect_tx(bar, (wide ? 2 : 1) * p.tt * p.group * 256);
#pragma unroll 1
                            for (int s = 0; s < (wide ? 2 : 1); ++s) {
                                ptx::tma_load_3d(sQ + s * TILE, &tq, bar, 0, kvh * p.group, tok0 + s * p.tt);
                                ptx::tma_load_3d(sQ + s * TILE + SUB, &tq, bar, 64, kvh * p.group, tok0 + s * p.tt);
                            }
                        }
                    }
                    __syncwarp();
                }
                const int lead = wide ? sched::kLeadWide : sched::kLead, dirty = kv ? uniform(item_dirty) : nt;
                // Dirty tile j's keys that the first token does not see. (Those past the request's pages are zeros.)
                auto clean = [&](int j) {
                    const int x = ring + sched::v_place(j, nt, lead), key0 = (kb + j) * tile_pages * kPageTokens;
                    if (!wait_bar(&c.kv_full[x % KV_ST], sched::fill_parity(x), err, kErrWaitProducer)) ok = false;
                    clean_v(sKV + (x % KV_ST) * TILE, max(0, pos0 + 1 - key0),
                            min(tile_pages * kPageTokens, npages * kPageTokens - key0), lane, pos0 + ntok - 1 - key0,
                            &c.poison[k % sched::kMarks], k + 1);
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&c.v_clean[cleaned % DIRTY]);
                    ++cleaned;
                };
#pragma unroll 1
                for (int t0 = 0; t0 < nt; t0 += window) {
                    c.z[kv][lane] = place(t0, id);
                    __syncwarp();
                    if (t0 + window < nt) id = fetch(t0 + window);
                    const int t_end = min(nt, t0 + window);
                    // Dirty tiles one by one, each followed by the cleaning of the one before: that one's copy is landing, and
                    // no copy waits for a stage that only a product of it, or of the tile before it, would free.
#pragma unroll 1
                    for (int ta = t0, t1; ta < t_end; ta = t1) {
                        t1 = ta < dirty ? min(t_end, dirty) : ta + 1;
                        // One lane issues the copies (the choice of it and the return from it cost some 170 cycles).
                        if (ptx::elect_one()) {
                            const int *zt = c.z[kv] + (ta - t0) * tile_pages;
#pragma unroll 1
                            for (int t = ta; t < t1; ++t, zt += tile_pages) {
                                const int x = ring + (kv ? sched::v_place(t, nt, lead) : sched::k_place(t, lead)), st = x % KV_ST;
                                const uint32_t bar = ptx::smem_u32(&c.kv_full[st]), dst = ptx::smem_u32(sKV) + st * TILE;
                                int zp[8];
#pragma unroll
                                for (int u = 0; u < 8; ++u) zp[u] = zt[u];  // (the array behind z is read past a window's end)
                                ok = wait_bar(&c.kv_empty[st], sched::fill_parity(x) ^ 1, err, kErrWaitProducer);
                                if (!ok) break;
                                c.kv_issued[st] = x + 1;
                                ptx::mbar_arrive_expect_tx(&c.kv_full[st], tile_pages * 4096);
#pragma unroll
                                for (int u = 0; u < 5; ++u) {
                                    tma_3d(dst + u * 2048, &tkv, bar, 0, zp[u]);
                                    tma_3d(dst + SUB + u * 2048, &tkv, bar, 64, zp[u]);
                                }
                                if (few) {
#pragma unroll
                                    for (int u = 5; u < 8; ++u) {
                                        tma_3d(dst + u * 2048, &tkv, bar, 0, zp[u]);
                                        tma_3d(dst + SUB + u * 2048, &tkv, bar, 64, zp[u]);
                                    }
                                }
                            }
                        }
                        __syncwarp();
                        if (__any_sync(0xffffffffu, !ok)) break;
                        if (ta > dirty) clean(ta - 1);
                    }
                    if (__any_sync(0xffffffffu, !ok)) break;
                }
                if (dirty < nt && __all_sync(0xffffffffu, ok)) clean(nt - 1);
                if (__any_sync(0xffffffffu, !ok)) break;
                ring += 2 * nt;
            }
        } else if (warp == 1) {
            // ---- tensor-core issuer ----
            constexpr uint32_t idesc_qk = ptx::idesc_bf16_f32(128, TK, false);
            constexpr uint32_t idesc_pv = ptx::idesc_bf16_f32(128, 128, true);
            constexpr uint32_t kHi = 1u << 14 | 2u << 29;  // descriptor bits 32-63: version 1, 128-byte swizzle
            const uint32_t bQ = ptx::smem_u32(sQ) >> 4, bKV = ptx::smem_u32(sKV) >> 4;
            // K-major: rows of 128 bytes, 8-row groups 1024 apart; MN-major (V): 64-dim halves SUB apart, the same groups
            auto kmajor = [](uint32_t at) { return (uint64_t)(kHi | 1024 >> 4) << 32 | (1u << 16 | at); };
            auto mnmajor = [](uint32_t at) { return (uint64_t)(kHi | 1024 >> 4) << 32 | ((uint32_t)(SUB >> 4) << 16 | at); };
            int ring = 0;                // ring items of the items before this one
            uint32_t before0 = 0, before1 = 0;  // products of the items before, a slot
            uint32_t cleaned = 0;               // dirty tiles of the items before
            bool ended = false;
            for (int k = 0;; ++k) {
                bool ok = wait_bar(&c.item_full[k % ITEMS], (k / ITEMS) & 1, err, kErrWaitIssuer);
                if (!__all_sync(0xffffffffu, ok)) break;
                const int ntok = uniform(c.items[k % ITEMS].ntok);
                const int nt = uniform(c.items[k % ITEMS].ke - c.items[k % ITEMS].kb);
                const int dirty = uniform(c.items[k % ITEMS].dirty);
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&c.item_empty[k % ITEMS]);
                if ((ended = ntok == 0)) break;
                const bool wide = ntok > p.tt, few = ntok * p.group <= kFewRows;
                // few: S^T = K Q^T (128 keys x 16 or 32 rows) and O^T = V^T P^T (128 dims x rows, twice)
                const int nrow = ntok * p.group <= 16 ? 16 : 32, np = (ntok * p.group + 7) / 8 * 16;
                const uint32_t idesc_s = ptx::idesc_bf16_f32(128, nrow);
                const uint32_t idesc_o = ptx::idesc_bf16_f32(128, np) | 1u << 15;  // A (V) MN-major
                // Product n's slot is n & 1. S lies beside P, so the next S of a slot is computed as soon as its softmax
                // has taken this one, and waits there for it; only P V waits for P.
                const int count = wide ? 2 * nt : nt;
                // One lane runs the item (choosing it and returning from it cost some 170 cycles); what the MMAs go by was
                // made uniform above, so their descriptors stay in uniform registers.
                if (ptx::elect_one()) {
                    uint32_t st = ring % KV_ST, phase = (ring / KV_ST) & 1;  // the next ring item
                    auto wait = [&](uint32_t bar, uint32_t parity) {
                        ok = wait_bar(bar, parity, err, kErrWaitIssuer);
                        ptx::tc_fence_after();
                        return ok;
                    };
                    // The next tile of the ring: its stage, or -1.
                    auto next_tile = [&]() {
                        const int x = (int)st;
                        const bool got = wait(ptx::smem_u32(&c.kv_full[0]) + 8 * st, phase);
                        if (++st == KV_ST) {
                            st = 0;
                            phase ^= 1;
                        }
                        return got ? x : -1;
                    };
                    auto wait_clean = [&](int t) {
                        const uint32_t n = cleaned + (uint32_t)(t - dirty);
                        return wait(ptx::smem_u32(&c.v_clean[n % DIRTY]), (n / DIRTY) & 1);
                    };
                    const uint32_t s_free = ptx::smem_u32(&c.s_free[0]), p_full = ptx::smem_u32(&c.p_full[0]);
                    wait(ptx::smem_u32(&c.q_full[k & 1]), (k >> 1) & 1);
                    if (wide) {
                        // Both slots of tile t: S of 0, P V of 1 (two tiles back), S of 1, P V of 0 (the tile before).
                        const uint32_t par0 = before0 & 1, par1 = before1 & 1;  // parity of the item's first product
                        int kt = 0, vt = 0;  // stages of the last tiles of K and V
#pragma unroll 1
                        for (int t = 0; ok && t < nt + 2; ++t) {
                            if (t < nt) {
                                if ((kt = next_tile()) < 0) break;
                                if ((t > 0 || before0 > 0) && !wait(s_free, (par0 ^ t ^ 1) & 1)) break;
                                const uint32_t key = bKV + kt * (TILE >> 4);
#pragma unroll
                                for (int kk = 0; kk < 8; ++kk)
                                    ptx::mma_bf16(tmem, kmajor(bQ + (((kk >> 2) * SUB + (kk & 3) * 32) >> 4)),
                                                  kmajor(key + (((kk >> 2) * SUB + (kk & 3) * 32) >> 4)), idesc_qk,
                                                  kk > 0 ? 1u : 0u);
                                ptx::mma_commit(&c.s_full[0]);
                            }
                            if (t >= 2) {
                                if (!wait(p_full + 8, (par1 ^ t) & 1)) break;
                                const uint32_t v = bKV + vt * (TILE >> 4), keep = t > 2 ? 1u : 0u;
#pragma unroll
                                for (int kk = 0; kk < TK / 16; ++kk)
                                    ptx::mma_bf16_ts(tmem + 384, tmem + 256 + P_COL + kk * 8, mnmajor(v + kk * (2048 >> 4)),
                                                     idesc_pv, kk > 0 ? 1u : keep);
                                ptx::mma_commit(&c.o_done[1]);
                                ptx::mma_commit(&c.kv_empty[vt]);
                            }
                            if (t < nt) {
                                if ((t > 0 || before1 > 0) && !wait(s_free + 8, (par1 ^ t ^ 1) & 1)) break;
                                const uint32_t key = bKV + kt * (TILE >> 4);
#pragma unroll
                                for (int kk = 0; kk < 8; ++kk)
                                    ptx::mma_bf16(tmem + 256, kmajor(bQ + ((TILE + (kk >> 2) * SUB + (kk & 3) * 32) >> 4)),
                                                  kmajor(key + (((kk >> 2) * SUB + (kk & 3) * 32) >> 4)), idesc_qk,
                                                  kk > 0 ? 1u : 0u);
                                ptx::mma_commit(&c.s_full[1]);
                                ptx::mma_commit(&c.kv_empty[kt]);
                                if (t == nt - 1) ptx::mma_commit(&c.q_empty[k & 1]);
                            }
                            if (t >= 1 && t <= nt) {
                                if ((vt = next_tile()) < 0) break;
                                // O may be overwritten once the item before has been read out
                                if (t == 1 && k > 0 && !wait(ptx::smem_u32(&c.o_free), (k - 1) & 1)) break;
                                if (!wait(p_full, (par0 ^ t ^ 1) & 1)) break;
                                if (t > dirty && !wait_clean(t - 1)) break;
                                const uint32_t v = bKV + vt * (TILE >> 4), keep = t > 1 ? 1u : 0u;
#pragma unroll
                                for (int kk = 0; kk < TK / 16; ++kk)
                                    ptx::mma_bf16_ts(tmem + 128, tmem + P_COL + kk * 8, mnmajor(v + kk * (2048 >> 4)), idesc_pv,
                                                     kk > 0 ? 1u : keep);
                                ptx::mma_commit(&c.o_done[0]);
                            }
                        }
                    } else {
                        int vt = 0, kt = 0;
#pragma unroll 1
                        for (int m = 0; ok && m < nt + 2; ++m) {
                            const int s = m & 1;
                            const uint32_t tS = tmem + 256 * s, prod = (s ? before1 : before0) + (m >> 1);
                            if (m < nt) {
                                if ((kt = next_tile()) < 0) break;
                                if (prod > 0 && !wait(s_free + 8 * s, (prod - 1) & 1)) break;
                                const uint32_t key = bKV + kt * (TILE >> 4);
                                if (few) {
                                    const uint32_t q = bQ + (k & 1) * (2 * FEW_SUB >> 4);
#pragma unroll
                                    for (int kk = 0; kk < 8; ++kk)
                                        ptx::mma_bf16(tS, kmajor(key + (((kk >> 2) * SUB + (kk & 3) * 32) >> 4)),
                                                      kmajor(q + (((kk >> 2) * FEW_SUB + (kk & 3) * 32) >> 4)), idesc_s,
                                                      kk > 0 ? 1u : 0u);
                                } else {
#pragma unroll
                                    for (int kk = 0; kk < 8; ++kk)
                                        ptx::mma_bf16(tS, kmajor(bQ + (((kk >> 2) * SUB + (kk & 3) * 32) >> 4)),
                                                      kmajor(key + (((kk >> 2) * SUB + (kk & 3) * 32) >> 4)), idesc_qk,
                                                      kk > 0 ? 1u : 0u);
                                }
                                ptx::mma_commit(&c.s_full[s]);
                                ptx::mma_commit(&c.kv_empty[kt]);
                                if (m == nt - 1 && !few) ptx::mma_commit(&c.q_empty[k & 1]);
                            }
                            if (m >= 2) {
                                if ((vt = next_tile()) < 0) break;
                                if (m == 2 && k > 0 && !wait(ptx::smem_u32(&c.o_free), (k - 1) & 1)) break;
                                if (!wait(p_full + 8 * s, (prod - 1) & 1)) break;
                                if (m - 2 >= dirty && !wait_clean(m - 2)) break;
                                const uint32_t v = bKV + vt * (TILE >> 4), keep = m >= 4 ? 1u : 0u;
                                if (few) {
                                    const uint32_t pt = bQ + ((TILE + s * FEW_P) >> 4);
#pragma unroll
                                    for (int kk = 0; kk < 8; ++kk)
                                        ptx::mma_bf16(tS + 128, mnmajor(v + kk * (2048 >> 4)),
                                                      kmajor(pt + (((kk >> 2) * FEW_P_SUB + (kk & 3) * 32) >> 4)), idesc_o,
                                                      kk > 0 ? 1u : keep);
                                } else {
#pragma unroll
                                    for (int kk = 0; kk < TK / 16; ++kk)
                                        ptx::mma_bf16_ts(tS + 128, tS + P_COL + kk * 8, mnmajor(v + kk * (2048 >> 4)),
                                                         idesc_pv, kk > 0 ? 1u : keep);
                                }
                                ptx::mma_commit(&c.o_done[s]);
                                ptx::mma_commit(&c.kv_empty[vt]);
                            }
                        }
                        if (few) ptx::mma_commit(&c.q_empty[k & 1]);  // P lies beside q
                    }
                }
                if (__any_sync(0xffffffffu, !ok)) break;
                ring += 2 * nt;
                before0 += (count + 1) / 2;
                before1 += count / 2;
                cleaned += (uint32_t)max(0, nt - dirty);
            }
            if (!ended && lane == 0) c.gave_up = 1;
            // No MMA may still be writing TMEM when it is freed (this matters on the error path).
            if (ptx::elect_one()) ptx::mma_commit(&c.fin);
            wait_bar(&c.fin, 0, err, kErrWaitIssuer);
        }
    } else {
        // ---- softmax ----
        ptx::setmaxnreg_inc<kRegsSoftmax>();
        const int s = (warp - 4) >> 2;  // slot
        const int quarter = warp & 3;   // TMEM lanes this warp may access
        const int rl = quarter * 32 + lane;
        // this row's token (of the slot) and query head (of the group)
        const int tl = rl * p.inv_group >> 16, hl = rl - tl * p.group;
        const int warp_tl = quarter * 32 * p.inv_group >> 16;  // the warp's first token
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t tS = tmem + 256 * s + lanes;
        const float sc = a.scale_log2;
        uint32_t steps = 0, done[SLOTS] = {};  // products of this slot so far; products of the items before, a slot
        bool ok = true, narrow_before = false;
        for (int k = 0; ok; ++k) {
            if (!wait_bar(&c.item_full[k % ITEMS], (k / ITEMS) & 1, err, kErrWaitSoftmax)) break;
            const Item it = c.items[k % ITEMS];
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&c.item_empty[k % ITEMS]);
            if (it.ntok == 0) break;
            if (it.ntok * p.group <= kFewRows) {
                const RoleState r = {&c, &p, sQ + TILE + s * FEW_P, tmem, s, quarter, lane, cta, k};
                // the sums of p go where a narrow item's O is: both warpgroups have read that out behind this
                if (narrow_before) ptx::named_barrier(1, 256);
                narrow_before = false;
                ok = few_item(r, it, steps, done);
                if (!ok) break;
                continue;
            }
            const bool wide = it.ntok > p.tt;
            narrow_before = !wide;
            const int token = wide ? s * p.tt + tl : tl;  // of the item
            const bool valid = tl < p.tt && token < it.ntok;
            const int warp_token = wide ? s * p.tt + warp_tl : warp_tl;
            const bool active = warp_tl < p.tt && warp_token < it.ntok;  // some row of the warp is real
            const int nt = it.ke - it.kb;
            float m_ref = -INFINITY, l = 0.f;
            bool first = true;
#pragma unroll 1
            for (int j = wide ? 0 : s; j < nt; j += wide ? 1 : 2, ++steps) {
                if (!wait_bar(&c.s_full[s], steps & 1, err, kErrWaitSoftmax)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
                const int key0 = (it.kb + j) * TK;
                float x[TK];
                if (active) {
                    ptx::tmem_ld32(tS, reinterpret_cast<uint32_t *>(x));
                    ptx::tmem_ld32(tS + 32, reinterpret_cast<uint32_t *>(x) + 32);
                    ptx::tmem_ld16(tS + 64, *reinterpret_cast<uint32_t(*)[16]>(x + 64));
                    ptx::tmem_ld_wait();
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&c.s_free[s]);
                float tmax = -INFINITY;
                if (active) {
                    if (key0 + TK - 1 > it.pos0 + warp_token) {
                        const int lim = it.pos0 + token - key0;  // keys 0..lim of the tile are visible
                        const int low = it.pos0 + warp_token - key0;  // keys 0..low are visible to every row of the warp
#pragma unroll
                        for (int b = 0; b < TK; b += 16)
                            if (b + 15 > low) {
#pragma unroll
                                for (int e = b; e < b + 16; ++e) x[e] = e <= lim ? x[e] : -INFINITY;
                            }
                    }
                    float mx[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) mx[u] = fmaxf(x[u], x[u + 8]);
#pragma unroll
                    for (int e = 16; e < TK; e += 16) {
#pragma unroll
                        for (int u = 0; u < 8; ++u) mx[u] = max3(mx[u], x[e + u], x[e + 8 + u]);
                    }
                    tmax = fmaxf(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], max3(mx[5], mx[6], mx[7]))) * sc;
                }
                // The slot's product before has been added to O and has read P: both may be written.
                if (steps > 0 && !wait_bar(&c.o_done[s], (steps - 1) & 1, err, kErrWaitSoftmax)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
                if (active) {
                    bool rescale = false;
                    float alpha = 1.f;
                    if (first) {
                        m_ref = tmax;
                    } else if (valid && tmax > m_ref + kRescaleThreshold) {
                        alpha = ptx::ex2(m_ref - tmax);  // 0 when nothing was visible before
                        m_ref = tmax;
                        rescale = true;
                    }
                    if (__any_sync(0xffffffffu, rescale)) {
                        l *= alpha;
#pragma unroll 1
                        for (int col = 0; col < 128; col += 32) {
                            uint32_t u[32];
                            ptx::tmem_ld32(tS + 128 + col, u);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * alpha);
                            ptx::tmem_st32(tS + 128 + col, u);
                        }
                    }
                    const float nm = m_ref == -INFINITY ? 0.f : -m_ref;  // a row that has seen no key yet: p = 0
                    float la = 0.f, lb = 0.f, lc = 0.f, ld = 0.f;
                    uint32_t pk[TK / 2];
#pragma unroll
                    for (int e = 0; e < TK / 2; ++e) {
                        float u, v;
                        ptx::fma_x2(u, v, x[2 * e], x[2 * e + 1], sc, sc, nm, nm);
                        u = ptx::ex2(u);
                        v = ptx::ex2(v);
                        if (e & 1)
                            add2(lc, ld, u, v);
                        else
                            add2(la, lb, u, v);
                        pk[e] = pack2(u, v);
                    }
                    l += (la + lb) + (lc + ld);
                    ptx::tmem_st32(tS + P_COL, pk);
                    tmem_st8(tS + P_COL + 32, *reinterpret_cast<const float(*)[8]>(pk + 32));
                }
                first = false;
                if (active) ptx::tmem_st_wait();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&c.p_full[s]);
            }
            if (!ok) break;

            // ---- epilogue ----
            const bool used1 = wide || nt > 1;
            done[0] += wide ? nt : (nt + 1) / 2;
            done[1] += wide ? nt : nt / 2;
            auto wait_done = [&](int slot) {
                if (!wait_bar(&c.o_done[slot], (done[slot] - 1) & 1, err, kErrWaitSoftmax)) ok = false;
                ptx::tc_fence_after();
                return ok;
            };
            // this slot's last product first: the other's barrier is then at its own last one's phase
            if ((s == 0 || used1) && !wait_done(s)) break;
            if (!wide && (s == 1 || used1) && !wait_done(1 - s)) break;
            float w[SLOTS] = {1.f, 0.f};  // weights of the two slots' states (narrow)
            if (!wide) {
                // both warpgroups hold the same rows: exchange the states, then each takes half of the dims
                c.ml[s][rl][0] = m_ref;
                c.ml[s][rl][1] = l;
                ptx::named_barrier(1, 256);
                const float m0 = c.ml[0][rl][0], l0 = c.ml[0][rl][1];
                const float m1 = c.ml[1][rl][0], l1 = used1 ? c.ml[1][rl][1] : 0.f;
                m_ref = l0 == 0.f ? m1 : (l1 == 0.f ? m0 : fmaxf(m0, m1));
                w[0] = l0 == 0.f ? 0.f : ptx::ex2(m0 - m_ref);
                w[1] = l1 == 0.f ? 0.f : ptx::ex2(m1 - m_ref);
                l = (l0 == 0.f ? 0.f : w[0] * l0) + (l1 == 0.f ? 0.f : w[1] * l1);
                ptx::named_barrier(1, 256);  // read by both before either may write there again
            }
            const bool poisoned = c.poison[k % sched::kMarks] == k + 1;
            if (active) {
                // o = w[0] O_0 + w[1] O_1 (wide: this slot's O alone), 32 dims at a time
                const uint32_t tO = (wide ? tS : tmem + lanes) + 128;
                const bool two = !wide && used1;
                if (poisoned) {
                    const int lo = max(it.kb * TK, it.pos0 + 1);
                    const int hi = valid ? min(it.pos0 + token, it.ke * TK - 1) : -1;
                    if (wide || nt > s)
                        add_poison(a, it.table, it.kvh, lo, hi, TK, it.kb + (wide ? 0 : s), wide ? 1 : 2, tS + 128);
                    if (!wide) {  // the other warpgroup's warp of these lanes reads this slot's O too
                        ptx::tc_fence_before();
                        ptx::named_barrier(2 + quarter, 64);
                        ptx::tc_fence_after();
                    }
                }
                const int c0 = wide ? 0 : 64 * s, c1 = wide ? 128 : 64 * s + 64;
                const float inv = it.dest < 0 ? 1.f / l : 1.f, w0 = w[0] * inv, w1 = w[1] * inv;
                // Four lanes write 64 contiguous bytes of each of their four rows (a lane's own row alone would be 16 bytes a
                // store: half sectors, which took 11,000 cycles of a partial item against 4,000).
                const size_t part = ((size_t)cta * 2 + (it.dest > 0)) * p.rows_cap;
                if (it.dest >= 0 && valid && c0 == 0)
                    *reinterpret_cast<float2 *>(p.part_ml + (part + token * p.group + hl) * 2) = make_float2(m_ref, l);
                uint8_t *rows[4];
                bool real[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = quarter * 32 + (lane & ~3) + j, tj = r * p.inv_group >> 16, tok = wide ? s * p.tt + tj : tj;
                    const int hj = r - tj * p.group;
                    real[j] = tj < p.tt && tok < it.ntok;
                    rows[j] = it.dest < 0 ? reinterpret_cast<uint8_t *>(a.out + (size_t)(it.tok0 + tok) * a.ld_out +
                                                                        (size_t)(it.kvh * p.group + hj) * kHeadDim)
                                          : reinterpret_cast<uint8_t *>(p.part_o + (part + tok * p.group + hj) * kHeadDim);
                    rows[j] += 16 * (lane & 3);
                }
#pragma unroll 1
                for (int col = c0; col < c1; col += 32) {
                    float o[32];
                    ptx::tmem_ld32(tO + col, reinterpret_cast<uint32_t *>(o));
                    ptx::tmem_ld_wait();
                    if (two) {
                        float o1[32];
                        ptx::tmem_ld32(tO + 256 + col, reinterpret_cast<uint32_t *>(o1));
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = fmaf(o1[e], w1, o[e] * w0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) ptx::fma_x2(o[e], o[e + 1], o[e], o[e + 1], w0, w0, 0.f, 0.f);
                    }
                    uint4 v[4];
                    if (it.dest < 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v[e] = make_uint4(pack2(o[8 * e], o[8 * e + 1]), pack2(o[8 * e + 2], o[8 * e + 3]),
                                              pack2(o[8 * e + 4], o[8 * e + 5]), pack2(o[8 * e + 6], o[8 * e + 7]));
                        quad_transpose(v, lane);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (real[j]) *reinterpret_cast<uint4 *>(rows[j] + col * 2) = v[j];
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint4 *>(o + 16 * h + 4 * e);
                            quad_transpose(v, lane);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (real[j]) *reinterpret_cast<uint4 *>(rows[j] + col * 4 + 64 * h) = v[j];
                        }
                    }
                }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&c.o_free);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (warp == 1) ptx::tmem_dealloc(tmem, 512);
    // Copies in flight must land before the CTA exits. An issuer that got to the end has waited for all of them. Else, since
    // every role has returned, a stage's last copy is the only one of it that can be on its way: the one before was used
    // before the stage was given out again, and nothing refills it now.
    if (tid == 0 && c.gave_up) {
        for (int s = 0; s < KV_ST; ++s)
            if (const int x = c.kv_issued[s]) wait_bar(&c.kv_full[s], sched::fill_parity(x - 1), err, kErrWaitProducer);
        for (int s = 0; s < 2; ++s)
            if (const int k = c.q_issued[s]) wait_bar(&c.q_full[s], (k - 1) >> 1 & 1, err, kErrWaitProducer);
    }
}

// Merges the partial results of the items that a cut passes through: o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i in the
// order of their keys. It is bound by latency, its instructions' fetch included. Block (CTA, part of its record's rows), a
// warp two rows at a time, 4 dims a lane; two parts (a cut or two) are nearly all there is, so the loads of two parts of
// both rows are issued together. A block has 16 rows, which leaves four blocks an SM. (8 chunks of 511 tokens among 56 decodes
// and 26 requests with chunks of up to 250: 61.2 and 19.2 us with the attention; with a block for 32 rows, two an SM, 62.9
// and 20.6; with four blocks a record that loop over its rows, one wave, 63.8 and 23.9; with all records' rows dealt to the
// warps of one wave by a search 63.4 and 20.0, but one row over 900 keys takes 13.1 for 11.5.)
constexpr int kCombineWarps = 8, kCombineAtOnce = 2, kCombineRows = kCombineWarps * kCombineAtOnce;
__global__ void __launch_bounds__(32 * kCombineWarps, 4)
    paged_combine_kernel(const __grid_constant__ Params p) {
    ptx::griddep_wait();
    const int4 rec = *reinterpret_cast<const int4 *>(p.records + blockIdx.x);  // tok0, ntok, kvh, follow
    const int lane = threadIdx.x % 32, n = rec.w + 1, rows = rec.y * p.group;
    // partial i: slot 1 of the record's CTA, then slot 0 of each CTA behind it
    const size_t first = ((size_t)blockIdx.x * 2 + 1) * p.rows_cap, step = (size_t)2 * p.rows_cap;
    const int row0 = blockIdx.y * kCombineRows + threadIdx.x / 32;
    if (row0 >= rows) return;
    float m[kCombineAtOnce], l[kCombineAtOnce];
    float4 acc[kCombineAtOnce];
#pragma unroll
    for (int r = 0; r < kCombineAtOnce; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
        acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 1
    for (int i = 0; i < n; i += 2) {
        float2 ml[2][kCombineAtOnce];
        float4 o[2][kCombineAtOnce];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const size_t part = (i + u ? first + p.rows_cap + (size_t)(i + u - 1) * step : first) + row0;
#pragma unroll
            for (int r = 0; r < kCombineAtOnce; ++r) {
                ml[u][r] = make_float2(-INFINITY, 0.f);
                o[u][r] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i + u < n && row0 + r * kCombineWarps < rows) {
                    const size_t x = part + r * kCombineWarps;
                    ml[u][r] = *reinterpret_cast<const float2 *>(p.part_ml + x * 2);
                    o[u][r] = *reinterpret_cast<const float4 *>(p.part_o + x * kHeadDim + 4 * lane);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < kCombineAtOnce; ++r) {
                if (ml[u][r].y == 0.f) continue;  // the row saw none of this part's keys
                const float m2 = fmaxf(m[r], ml[u][r].x), w = ptx::ex2(ml[u][r].x - m2);
                const float f = l[r] == 0.f ? 0.f : ptx::ex2(m[r] - m2);
                l[r] = l[r] * f + w * ml[u][r].y;
                acc[r].x = acc[r].x * f + w * o[u][r].x;
                acc[r].y = acc[r].y * f + w * o[u][r].y;
                acc[r].z = acc[r].z * f + w * o[u][r].z;
                acc[r].w = acc[r].w * f + w * o[u][r].w;
                m[r] = m2;
            }
    }
#pragma unroll
    for (int r = 0; r < kCombineAtOnce; ++r) {
        const int row = row0 + r * kCombineWarps;
        if (row >= rows) break;
        const float inv = 1.f / l[r];
        const int token = row * p.inv_group >> 16, h = row - token * p.group;
        *reinterpret_cast<uint2 *>(p.a.out + (size_t)(rec.x + token) * p.a.ld_out +
                                   (size_t)(rec.z * p.group + h) * kHeadDim + 4 * lane) =
            make_uint2(pack2(acc[r].x * inv, acc[r].y * inv), pack2(acc[r].z * inv, acc[r].w * inv));
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
    static const EncodeTiledFn fn = [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return (EncodeTiledFn)ptr;
        return (EncodeTiledFn) nullptr;
    }();
    return fn;
}

// bf16 [z][y][128] with the given y and z strides (bytes), boxes of 64 x by x bz, 128-byte swizzle.
bool make_tmap(CUtensorMap *map, const void *ptr, uint64_t y, uint64_t z, uint64_t ystride, uint64_t zstride, uint32_t by,
               uint32_t bz) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {128, y, z}, strides[2] = {ystride, zstride};
    const cuuint32_t box[3] = {64, by, bz}, estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of a partial slot: those of an item, which a call of `tokens` rows bounds too.
int partial_rows(int tokens, int q_heads, int kv_heads) {
    const int group = q_heads / kv_heads, span = sched::make_shape(group).span;
    return (tokens < span ? tokens : span) * group;
}

}  // namespace

uint64_t paged_attention_workspace(int tokens, int q_heads, int kv_heads, int sms) {
    return (uint64_t)sms * (2 * (uint64_t)partial_rows(tokens, q_heads, kv_heads) * (kHeadDim + 2) * sizeof(float) +
                            sizeof(Record));
}

cudaError_t launch_paged_attention(const PagedAttnArgs &a, int sms, cudaStream_t st) {
    Params p;
    p.a = a;
    p.group = a.q_heads / a.kv_heads;
    p.shape = sched::make_shape(p.group);
    p.inv_group = (65535 + p.group) / p.group;
    p.tt = sched::kTileRows / p.group;
    p.rows_cap = partial_rows(a.tokens, a.q_heads, a.kv_heads);
    p.records = reinterpret_cast<Record *>(a.workspace);
    p.part_o = reinterpret_cast<float *>(p.records + sms);
    p.part_ml = p.part_o + (size_t)sms * 2 * p.rows_cap * kHeadDim;
    p.few_tok = kFewRows / p.group > 0 ? kFewRows / p.group : 1;
    CUtensorMap tq, tq_few, tkv;
    const uint64_t qrow = (uint64_t)a.ld_q * 2;
    // a map is made for the boxes that the call can use (each takes the host 0.4 us, a call of one token 11 in all)
    const bool few = p.group <= kFewRows, more = (int64_t)a.tokens * p.group > kFewRows;
    if ((more && !make_tmap(&tq, a.q, a.q_heads, a.tokens, kHeadDim * 2, qrow, p.group, p.tt)) ||
        (few && !make_tmap(&tq_few, a.q, a.q_heads, a.tokens, kHeadDim * 2, qrow, p.group, p.few_tok)) ||
        !make_tmap(&tkv, a.pool, kPageTokens, (uint64_t)a.kv_pages * a.kv_heads * 2, kHeadDim * 2,
                   kPageTokens * kHeadDim * 2, kPageTokens, 1))
        return cudaErrorInvalidValue;
    if (!more) tq = tq_few;
    if (!few) tq_few = tq;
    static SmemOptIn opt;
    if (cudaError_t e = opt.set((const void *)paged_attn_kernel, SMEM_BYTES)) return e;
    cudaError_t e = launch_kernel(paged_attn_kernel, dim3(sms), dim3(kThreads), SMEM_BYTES, st, tq, tq_few, tkv, p);
    if (e != cudaSuccess) return e;
    // The merge launches under the attention kernel's tail; its own wait orders it behind that kernel's writes.
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms, (p.rows_cap + kCombineRows - 1) / kCombineRows);
    cfg.blockDim = dim3(32 * kCombineWarps);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_combine_kernel, p);
}

}  // namespace lrm
