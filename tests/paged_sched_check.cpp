// The paged attention's schedule (paged_sched.h) as a host library, for tests/test_paged_sched.py.
#include "../rosylnalive_b200/csrc/paged_sched.h"

#include <map>
#include <random>
#include <tuple>
#include <vector>

using namespace lrm::sched;

namespace {

typedef std::mt19937_64 Rng;
int64_t pick(Rng &r, int64_t lo, int64_t hi) { return lo + (int64_t)(r() % (uint64_t)(hi - lo + 1)); }

struct Request {
    int n, kv;
};

// An item by its definition: its rows' tokens, and the tiles of the keys that its last token sees.
int tiles_of(int group, int n, int kv, int i) {
    const int span = 2 * (128 / group), last = (i + 1) * (int64_t)span < n ? (i + 1) * span : n;
    const int tk = (last - i * span) * group <= 32 ? 128 : 80;
    return (kv - n + last + tk - 1) / tk;
}

}  // namespace

extern "C" {

int ring_stages() { return kRing; }
int lead_of(int wide) { return wide ? kLeadWide : kLead; }
int place_of_k(int t, int lead) { return k_place(t, lead); }
int place_of_v(int t, int nt, int lead) { return v_place(t, nt, lead); }
int marks() { return kMarks; }
int issuer_waits() { return (int)kIssuerWaits; }
int polls(int softmax) { return (int)(softmax ? kSoftmaxPolls : kPolls); }
int parity_of(int x) { return (int)fill_parity(x); }

// One request's items against their definition: 0, or the line that does not hold.
#define HOLDS(x) \
    if (!(x)) return __LINE__
int check_items(uint64_t seed, int group, int n, int kv) {
    Rng r(seed);
    const Shape s = make_shape(group);
    const int span = 2 * (128 / group), items = items_of(s, n);
    HOLDS(s.span == span && items == (int)(((int64_t)n + span - 1) / span));
    const int stride = items > 3000 ? items / 3000 : 1;  // of a very long request some
    for (int i = 0; i < items; i += i + stride < items || i == items - 1 ? stride : items - 1 - i) {
        const uint64_t at = units_before(s, n, kv, i);
        const Item t = item_of(s, n, kv, i, items);
        HOLDS(t.tiles == tiles_of(group, n, kv, i) && t.tiles > 0);
        HOLDS(t.units >= t.own && t.units <= t.own + t.tile * t.tiles);
        HOLDS(at + (uint64_t)t.units == (i + 1 < items ? units_before(s, n, kv, i + 1) : head_units(s, n, kv)));
        HOLDS(item_at(s, n, kv, at, items) == i && item_at(s, n, kv, at + (uint64_t)t.units - 1, items) == i);
        HOLDS(tile_at(t, 0) == 0 && tile_at(t, t.own) == (t.units > t.own ? 0 : t.tiles) && tile_at(t, t.units) == t.tiles);
        HOLDS(tile_at(t, t.units - 1) < t.tiles);  // the last share of an item has a tile
        for (int e = 0; e < 20; ++e) {
            const int a = (int)pick(r, 0, t.units), b = (int)pick(r, a, t.units);
            HOLDS(tile_at(t, a) <= tile_at(t, b) && tile_at(t, a) >= 0);
            HOLDS(a < t.own || b < a + kLeastUnits || tile_at(t, b) > tile_at(t, a));  // and so has one of the least units
        }
    }
    return 0;
}

// A call of random requests, cut for up to `most` CTAs and walked by each as the kernel does: every tile of every item is
// computed once, the partial results are at most one of each kind a CTA, and those of an item are the record's.
int check_call(uint64_t seed, int most) {
    Rng r(seed);
    const int group = (int)(pick(r, 0, 3) ? pick(r, 1, 8) : pick(r, 1, 128)), heads = (int)pick(r, 1, 9);
    const Shape s = make_shape(group);
    std::vector<Request> reqs;
    std::vector<uint64_t> first;
    uint64_t units = 0;
    for (int i = (int)pick(r, 1, 25); i > 0; --i) {
        const int kind = (int)pick(r, 0, 4), n = kind == 0 ? 0 : (int)(kind < 3 ? pick(r, 1, 6) : pick(r, 1, 700));
        reqs.push_back(Request{n, n ? n + (int)(pick(r, 0, 1) ? pick(r, 0, 200) : pick(r, 0, 9000)) : 0});
        first.push_back(units);
        if (n) units += head_units(s, n, reqs.back().kv) * (uint64_t)heads;
    }
    const Cut cut = make_cut(units, (int)pick(r, 1, most), kLeastUnits);
    HOLDS(begin(cut, cut.ctas) == units && (cut.ctas > 0) == (units > 0));
    std::map<std::tuple<int, int, int>, std::vector<int>> seen;  // how often each tile of (request, head, item) was computed
    struct Parts {
        int cta, follow;
    };
    std::map<std::tuple<int, int, int>, Parts> records;
    std::vector<std::tuple<int, int, int>> part[2];
    const std::tuple<int, int, int> none(-1, -1, -1);
    for (int d = 0; d < 2; ++d) part[d].assign(cut.ctas, none);
    for (int c = 0; c < cut.ctas; ++c) {
        const uint64_t u0 = begin(cut, c), u1 = begin(cut, c + 1);
        HOLDS(u1 > u0 && cta_of(cut, u0) == c && cta_of(cut, u1 - 1) == c);
        int q = (int)reqs.size() - 1;
        while (first[q] > u1 - 1 || !reqs[q].n) --q;
        const uint64_t head = head_units(s, reqs[q].n, reqs[q].kv), off = (u1 - 1 - first[q]) % head;
        int h = (int)quotient(u1 - 1 - first[q], head), items = items_of(s, reqs[q].n);
        int i = item_at(s, reqs[q].n, reqs[q].kv, off, items);
        int end = (int)(off - units_before(s, reqs[q].n, reqs[q].kv, i)) + 1;
        for (uint64_t left = u1 - u0;;) {
            const Item t = item_of(s, reqs[q].n, reqs[q].kv, i, items);
            const Share x = share_of(t, end, left);
            HOLDS(x.kb >= 0 && x.kb <= x.ke && x.ke <= t.tiles);
            if (x.ke > x.kb) {
                const auto id = std::make_tuple(q, h, i);
                std::vector<int> &n = seen[id];
                n.resize(t.tiles);
                for (int k = x.kb; k < x.ke; ++k) ++n[k];
                if (x.dest >= 0) {
                    HOLDS(part[x.dest][c] == none);
                    part[x.dest][c] = id;
                }
                if (x.dest == 1) {
                    HOLDS(!records.count(id));
                    records[id] = Parts{c, cta_of(cut, u1 - 1 + (uint64_t)(t.units - end)) - c};
                }
            }
            left -= (uint64_t)(end - x.begin);
            if (left == 0) break;
            if (i > 0) {
                --i;
            } else {
                if (h > 0) {
                    --h;
                } else {
                    do --q;
                    while (!reqs[q].n);
                    h = heads - 1;
                    items = items_of(s, reqs[q].n);
                }
                i = items - 1;
            }
            end = item_of(s, reqs[q].n, reqs[q].kv, i, items).units;
        }
    }
    for (int q = 0; q < (int)reqs.size(); ++q)
        for (int h = 0; h < heads; ++h)
            for (int i = 0; reqs[q].n && i < items_of(s, reqs[q].n); ++i) {
                const std::vector<int> &n = seen[std::make_tuple(q, h, i)];
                HOLDS((int)n.size() == tiles_of(group, reqs[q].n, reqs[q].kv, i));
                for (int x : n) HOLDS(x == 1);
            }
    int parts = 0;
    for (const auto &e : records) {
        HOLDS(part[1][e.second.cta] == e.first && e.second.follow > 0 && e.second.cta + e.second.follow < cut.ctas);
        for (int f = 1; f <= e.second.follow; ++f) HOLDS(part[0][e.second.cta + f] == e.first);
        parts += 1 + e.second.follow;
    }
    for (int d = 0; d < 2; ++d)
        for (const auto &id : part[d]) parts -= id != none;
    HOLDS(parts == 0);
    return 0;
}

}  // extern "C"
