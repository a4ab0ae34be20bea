// paged_sched.h -- how the paged attention's work is counted and cut (host and device: the kernels use it, and it can
// be checked on the CPU).
//
// A request has n new tokens, the last of its kv keys, and `group` query heads a KV head. An item is up to `span`
// consecutive tokens of one request and KV head, all their query heads, and reads the keys that its last token sees in
// tiles: of 128 keys when it has few rows (kFewRows), else of 80. An item counts units of work for its start and end and
// for each tile, as measured (Cost). All units of a call, ordered by (request, KV head, item, key), are cut into `ctas`
// ranges of equal length, one a CTA, so every mixture of lengths is balanced; an item that a cut passes through is merged
// from its CTAs' partial results. (Counting tiles alone left 32 requests of 5 tokens over 100 to 6000 keys at 64 us
// against 43, and 8 chunks of 511 tokens among 56 decodes at 103 against 87.)
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LRM_HD __host__ __device__ __forceinline__
#define LRM_HD_FAR static __host__ __device__ __noinline__  // one copy: instruction space is scarce in the kernel
#else
#define LRM_HD inline
#define LRM_HD_FAR inline
#endif

namespace lrm {
namespace sched {

constexpr int kTileRows = 128;
constexpr int kFewRows = 32, kFewTileKeys = 128, kTileKeys = 80;

// sum over i in [0, n) of floor((a i + b) / m), by Euclid's steps on (a, m); a, b >= 0, m > 0.
LRM_HD_FAR uint64_t floor_sum(uint64_t n, uint32_t m, uint32_t a, uint64_t b) {
    uint64_t sum = 0;
    for (;;) {
        if (n == 0) return sum;
        sum += (n * (n - 1) / 2) * (a / m) + n * (b / m);
        a %= m;
        b %= m;
        const uint64_t y = (uint64_t)a * n + b;
        if (y < m) return sum;
        n = y / m;
        b = y % m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
}

LRM_HD int items_of(int n, int span) { return (n + span - 1) / span; }

struct Shape {
    int group, span;
};
LRM_HD int item_tokens(Shape s, int n, int i) { return n - i * s.span < s.span ? n - i * s.span : s.span; }
LRM_HD int tile_keys(int rows) { return rows <= kFewRows ? kFewTileKeys : kTileKeys; }

// Key tiles of item i.
LRM_HD int item_tiles(Shape s, int n, int kv, int i) {
    const int tokens = item_tokens(s, n, i);
    return (kv - n + i * s.span + tokens - 1) / tile_keys(tokens * s.group) + 1;
}

// An item's units: `own` for its start and end, then `tile` a tile. A unit is about 300 cycles, from a fit over the CTAs of
// forty mixtures: few rows 4,500 + 1,800 a tile, one slot's rows 6,600 + 1,500, two slots' 9,500 + 2,000.
struct Cost {
    int own, tile;
};
LRM_HD Cost item_cost(Shape s, int n, int i) {
    const int tokens = item_tokens(s, n, i);
    return tokens * s.group <= kFewRows ? Cost{15, 6} : (tokens <= s.span / 2 ? Cost{22, 5} : Cost{32, 7});
}
// The first tile that lies behind `units` of an item's units (neighbouring shares round to the same tile).
LRM_HD int tile_at(Cost c, int units) { return units > c.own ? (units - c.own) / c.tile : 0; }

// Units of the items before item i (i <= items - 1, so they are whole spans: more than kFewRows rows) of one head.
LRM_HD uint64_t units_before(Shape s, int n, int kv, int i) {
    if (i == 0) return 0;
    const Cost c = item_cost(s, n, 0);
    return (floor_sum((uint64_t)i, kTileKeys, (uint32_t)s.span, (uint64_t)(kv - n + s.span - 1)) + (uint64_t)i) *
               (uint64_t)c.tile + (uint64_t)i * c.own;
}

// Units of one head.
LRM_HD uint64_t head_units(Shape s, int n, int kv) {
    const int last = items_of(n, s.span) - 1;
    const Cost c = item_cost(s, n, last);
    return units_before(s, n, kv, last) + (uint64_t)(item_tiles(s, n, kv, last) * c.tile + c.own);
}

// The item of a head that holds its unit `off`.
LRM_HD int item_at(Shape s, int n, int kv, uint64_t off) {
    int lo = 0, hi = items_of(n, s.span);  // units_before(lo) <= off < units_before(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (units_before(s, n, kv, mid) <= off)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// CTAs that take part: at least `least` units each (7 or more, so that a share within an item holds a tile), so that
// short work is not cut into pieces that cost more to merge than they save.
LRM_HD int ctas_of(uint64_t units, int ctas, int least) {
    if (units >= (uint64_t)ctas * (uint64_t)least) return ctas;
    const int want = (int)((uint32_t)units / (uint32_t)least);
    return want > 0 ? want : (units > 0 ? 1 : 0);
}

// Where CTA c's range starts. (32-bit arithmetic where it fits: a 64-bit division costs the start of a short call.)
LRM_HD uint64_t cut(uint64_t units, int ctas, int c) {
    if (units < (1u << 20) && ctas <= 4095) return (uint32_t)units * (uint32_t)c / (uint32_t)ctas;
    return units * (uint64_t)c / (uint64_t)ctas;
}

// The CTA whose range holds unit u.
LRM_HD int cta_of(uint64_t units, int ctas, uint64_t u) {
    if (units < (1u << 20) && ctas <= 4095) return (int)((((uint32_t)u + 1) * (uint32_t)ctas - 1) / (uint32_t)units);
    return (int)(((u + 1) * (uint64_t)ctas - 1) / units);
}

LRM_HD uint64_t quotient(uint64_t a, uint64_t b) {
    return (a | b) >> 32 ? a / b : (uint64_t)((uint32_t)a / (uint32_t)b);
}

}  // namespace sched
}  // namespace lrm
