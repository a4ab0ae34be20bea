// paged_sched.h -- how the paged attention's work is counted and cut, and the order of its ring of tiles (host and device:
// the kernels use it, and tests/test_paged_sched.py checks it on the CPU).
//
// A request has n new tokens, the last of its kv keys, and `group` query heads a KV head. An item is up to `span`
// consecutive tokens of one request and KV head, all their query heads, and reads the keys that its last token sees in
// tiles: of 128 keys when it has few rows (kFewRows), else of 80. An item counts units of work for its start and end and
// for each tile, as measured (Cost). All units of a call, ordered by (request, KV head, item, key), are cut into `ctas`
// ranges of equal length, one a CTA, so every mixture of lengths is balanced; an item that a cut passes through is merged
// from its CTAs' partial results. (Counting tiles alone left 32 requests of 5 tokens over 100 to 6000 keys at 64 us
// against 43, and 8 chunks of 511 tokens among 56 decodes at 103 against 87.)
//
// Every CTA computes its range before it can load anything, so this is kept to a few multiplications: an item of a whole
// span counts tile * keys / 80 rather than the tile's cost times its rounded-up tiles, which makes the units of the items
// before one a closed form; divisions are by constants, or by the span with its inverse. (With the exact count, its sum by
// Euclid's steps and divisions, it took 10 us of the 66 of those mixed chunks.)
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LRM_HD __host__ __device__ __forceinline__
#else
#define LRM_HD inline
#endif

namespace lrm {
namespace sched {

constexpr int kTileRows = 128;
constexpr int kFewRows = 32, kFewTileKeys = 128, kTileKeys = 80;

// inv_span = ceil(2^38 / span): x * inv_span >> 38 is x / span for x < 2^30 (span <= 256).
struct Shape {
    int group, span;
    uint64_t inv_span;
};
LRM_HD Shape make_shape(int group) {
    const int span = 2 * (kTileRows / group);
    return Shape{group, span, ((uint64_t(1) << 38) + (uint64_t)span - 1) / (uint64_t)span};
}
LRM_HD int items_of(const Shape &s, int n) { return (int)(((uint64_t)(uint32_t)(n + s.span - 1) * s.inv_span) >> 38); }

// An item's units: `own` for its start and end, then `tile` a tile. A unit is about 300 cycles. Alone, items of few rows
// took 4,000 cycles + 1,400 a tile (with p in one bf16), of one slot's rows 6,700 + 1,400, of two slots' 9,000 + 1,950; where
// the memory's queues are full, as in most mixtures, tiles take longer and part of `own` hides behind them. So the weights are
// from mixtures, and a mixture's best ones are not another's: with kFew 11 + 6, 13 + 6, 15 + 6 and 18 + 7, 8 chunks of 511
// tokens among 56 single ones (8 KV heads) took 63.9, 57.9, 60.1 and 59.3 us, 26 requests with 12 chunks of up to 250 (2 KV
// heads) 19.5, 18.5, 19.6 and 18.3, 15 short requests (8 KV heads) 13.7, 13.1, 13.3 and 13.3; kWide at 40 + 10 with kFew 13 + 5
// left the first at 61 where it was 56.
struct Cost {
    int own, tile;
};
constexpr Cost kFew = {13, 6}, kNarrow = {22, 7}, kWide = {30, 10};
static_assert(kFew.tile != kNarrow.tile && kFew.tile != kWide.tile && kNarrow.tile != kWide.tile, "tile_at goes by them");

// Units of the items before item i of a head: all of them are whole spans, and so of two slots' rows.
LRM_HD uint64_t units_before(const Shape &s, int n, int kv, int i) {
    if (i == 0) return 0;
    const uint64_t keys = (uint64_t)i * (uint64_t)(uint32_t)(kv - n + s.span) + (uint64_t)i * (uint64_t)(i - 1) / 2 * s.span;
    return keys * kWide.tile / kTileKeys + (uint64_t)i * kWide.own;
}

struct Item {
    int tiles, units, own, tile;
};
// Item i of `items`.
LRM_HD Item item_of(const Shape &s, int n, int kv, int i, int items) {
    if (i < items - 1)
        return Item{(int)((uint32_t)(kv - n + (i + 1) * s.span + kTileKeys - 1) / kTileKeys),
                    (int)(units_before(s, n, kv, i + 1) - units_before(s, n, kv, i)), kWide.own, kWide.tile};
    const int tokens = n - i * s.span;
    const bool few = tokens * s.group <= kFewRows, narrow = 2 * tokens <= s.span;
    const Cost c = few ? kFew : (narrow ? kNarrow : kWide);
    const int tiles = few ? (int)((uint32_t)(kv + kFewTileKeys - 1) / kFewTileKeys)
                          : (int)((uint32_t)(kv + kTileKeys - 1) / kTileKeys);
    return Item{tiles, c.own + c.tile * tiles, c.own, c.tile};
}

// The first tile that lies behind `units` of an item's units (neighbouring shares round to the same tile). A whole span's
// units are at most own + tile * tiles, so a unit within it is within its tiles, and `tile` + 1 units on hold one at least.
LRM_HD int tile_at(const Item &t, int units) {
    if (units >= t.units) return t.tiles;
    if (units <= t.own) return 0;
    const uint32_t x = (uint32_t)(units - t.own);
    return (int)(t.tile == kWide.tile ? x / kWide.tile : (t.tile == kFew.tile ? x / kFew.tile : x / kNarrow.tile));
}

// Units of one head.
LRM_HD uint64_t head_units(const Shape &s, int n, int kv) {
    const int last = items_of(s, n) - 1;
    return units_before(s, n, kv, last) + (uint64_t)item_of(s, n, kv, last, last + 1).units;
}

// The item of a head that holds its unit `off`.
LRM_HD int item_at(const Shape &s, int n, int kv, uint64_t off, int items) {
    int lo = 0, hi = items;  // units_before(lo) <= off < units_before(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (units_before(s, n, kv, mid) <= off)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

LRM_HD uint64_t quotient(uint64_t a, uint64_t b) {
    return (a | b) >> 32 ? a / b : (uint64_t)((uint32_t)a / (uint32_t)b);
}

// The share of an item that lies in a range which ends at unit `end` of the item and has `left` units from there back: key
// tiles [kb, ke) (none when it is of the item's own cost alone), from unit `begin` on. dest: -1 the whole item, else which of
// the CTA's two partial results it is, 1 when it has the item's first tile. So a CTA has at most one of each: 1 is its
// range's last item, cut at the range's end, and 0 its first, cut before it.
struct Share {
    int begin, kb, ke, dest;
};
LRM_HD Share share_of(const Item &t, int end, uint64_t left) {
    const int begin = (uint64_t)end > left ? end - (int)left : 0, kb = tile_at(t, begin), ke = tile_at(t, end);
    return Share{begin, kb, ke, kb == 0 && ke == t.tiles ? -1 : (kb == 0 ? 1 : 0)};
}

// The cut of all units: CTA c's range is [begin(c), begin(c + 1)). CTAs that take part have at least `least` units each
// (more than kWide.tile, so that a share within an item holds a tile): short work is not cut into pieces that cost more
// to merge than they save. (One token over 900 keys, 8 KV heads: 10.6 us, with 20 units 12.1; 4 tokens over up to 1700 keys, 4
// KV heads 13.4, 14.7; 26 requests with chunks of up to 250 tokens, 2 KV heads 18.4, 18.8, with 30 20.5. Calls that fill the
// SMs are alike.)
constexpr int kLeastUnits = 12;
static_assert(kLeastUnits > kWide.tile, "a share within an item holds a tile");
struct Cut {
    int ctas;
    uint32_t more;   // the first ranges that are one unit longer
    uint64_t share;
};
LRM_HD Cut make_cut(uint64_t units, int ctas, int least) {
    if (units < (uint64_t)ctas * (uint64_t)least) {
        const int want = (int)((uint32_t)units / (uint32_t)least);
        ctas = want > 0 ? want : (units > 0 ? 1 : 0);
        if (!ctas) return Cut{0, 0, 0};
    }
    const uint64_t share = quotient(units, (uint64_t)ctas);
    return Cut{ctas, (uint32_t)(units - share * (uint64_t)ctas), share};
}
LRM_HD uint64_t begin(const Cut &k, int c) {
    return k.share * (uint64_t)c + ((uint32_t)c < k.more ? (uint32_t)c : k.more);
}
// The CTA whose range holds unit u.
LRM_HD int cta_of(const Cut &k, uint64_t u) {
    const uint64_t longer = (k.share + 1) * k.more;
    return u < longer ? (int)quotient(u, k.share + 1) : (int)(k.more + quotient(u - longer, k.share));
}

// ---- the ring of K and V tiles ----
//
// The ring order of an item's tiles is the order in which the issuer first uses them. In step t it issues S = Q K^T of tile t
// (wide: for both slots) and O += P V of an earlier one. Wide: S of slot 0, P V of slot 1 and tile t - 2, S of slot 1, P V of
// slot 0 and tile t - 1; else tile t is slot t & 1's, and P V is of tile t - 2. So K_t comes before V_{t - lead + 1}, lead
// being 2 (wide) or 3. Ring item x (counted from the CTA's first) is fill x / kRing of stage x % kRing.
constexpr int kRing = 5, kLeadWide = 2, kLead = 3;
LRM_HD int k_place(int t, int lead) { return t + (t >= lead ? t - lead + 1 : 0); }            // of K_t in its item
LRM_HD int v_place(int t, int nt, int lead) { return t + (t + lead < nt ? t + lead : nt); }  // of V_t, nt tiles
// The cleaning of V marks an item (kMarks places, by item) and the item's epilogue reads the mark. While the epilogue of item k
// runs, the P V of item k + 1 waits for it, so the last tile that has been freed is K of k + 1. Of items of one tile (with
// more the ring holds fewer items) that is ring item 2k + 2, its stage's next one is 2k + 2 + kRing, and V of item k + j is
// 2k + 2j + 1: V can be there, and be cleaned, up to (kRing + 1) / 2 items ahead of the mark that is still to be read.
constexpr int kMarks = (kRing + 1) / 2 + 1;

// Waits end after so many polls: 2 s, at 4 us a poll that fails. They are microseconds, but for the scheduler's, which waits
// for a whole item, 0.3 s of the longest that a call can have (2^24 keys). The softmax's warps meet at barriers that have no
// such limit, so they must agree on whether a wait failed: theirs end long after the issuer, which makes at most ten waits
// from one commit to the next of a slot, has either committed or given up for good, so nothing arrives while some have left.
constexpr uint32_t kPolls = 1u << 19, kIssuerWaits = 10, kSoftmaxPolls = 12 * kPolls;
LRM_HD uint32_t fill_parity(int x) { return (uint32_t)(x / kRing) & 1; }

}  // namespace sched
}  // namespace lrm
