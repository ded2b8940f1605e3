// The plan of an attention call over pages: rows in tiles, tiles' keys in items, items to workgroups.
//
// A sequence's stacked rows (token r / group, head r % group) are cut into tiles of up to paged_wide_rows, each with the
// range of keys that its rows see. Of three ways to give them to the workgroups that are on the GPU at once the one
// whose estimate is least is taken:
//   whole: a tile an item and a workgroup, the longest first;
//   parts: a sequence's tiles cut at the same keys, the sequence with the longest parts first, until the parts fill one or
//     two rounds of workgroups. Tiles over the same keys follow each other, so that they find them in an L2;
//   shares: where most sequences are one tile (single tokens), workgroups take equal shares of all keys, tile after tile,
//     and a share's border cuts a tile.
// Rows that end in parts are joined by a second launch.
// us of both launches, whole / parts / shares: 8192 tokens over 16192 keys (32 heads of 128 over 8) 1515 / - / 1650, 4 x 512
// over 5500 to 9500 275 / 302 / 334, 5 x 301 to 700 over 2000 to 9700 (16 heads of 64 over 8) 139 / 96 / 102, 3 x 500 to 1500
// over 1500 to 5500 with a window of 1024 (4 heads of 256 over 2) 63 / 42 / 49, 64 tokens over 100 to 8000 (32 heads of 128
// over 8) 199 / - / 187. Finer shares gain nothing (2, 3 and 4 times as many: 190, 191 and 192).
#include "paged_plan.hpp"

#include <algorithm>
#include <cstdint>

namespace ge {
namespace {

constexpr int kCus = 256;
// Keys are counted in units of 64. What an item takes besides its keys (its queries, the first keys, its rows' way
// out), the least keys of a part (a token over 512 keys, head dims 256 / 512, us a call: parts of one unit 22.0 / 25.8, of two
// 23.9 / 30.0), and the longest tile that no estimate is made for (over 256 keys whole 22.7 / 31.0, in parts 21.2 / 25.0; over
// 128 20.0 / 24.9 and 20.1 / 24.9).
constexpr int kUnit = 64, kItemUnits = 2, kLeastPart = 1, kWhole = 2;
// Tiles that a plan's estimate follows one by one; more are even enough.
constexpr size_t kManyTiles = 1024;

struct Tile {
    uint32_t seq, row0, n_rows;
    int32_t lo, hi;
    int units() const { return int((uint32_t(hi - lo) + kUnit - 1) / kUnit); }
};

// A sequence's tiles [first, first + n), the longest's units, and the parts they are cut into.
struct Group {
    uint32_t first, n;
    int units;
    int parts;
    int step() const { return std::max(1, (units + parts - 1) / parts); }
};

// The end of items whose units sum up to `load` on the CU that has most of them and are up to `longest`, us. A full CU
// gives each of its workgroups a unit in `full`; one alone takes the part `alone` of that.
float items_us(int head_dim, bool narrow, float load, float longest) {
    const float full = narrow ? (head_dim <= 128 ? 2.8f : 5.6f) : head_dim == 64 ? 3.1f : head_dim == 128 ? 2.0f : head_dim == 256 ? 4.6f : 4.1f;
    const float alone = narrow ? 0.3f : head_dim == 64 ? 0.35f : head_dim == 128 ? 0.6f : head_dim == 256 ? 0.7f : 1.0f;
    return full * std::max(load / float(paged_workgroups(head_dim)), alone * longest);
}

// The joining launch, with its parts' rows written and read.
float join_us(float rows, int kv_heads, int head_dim) { return 5.0f + rows * float(kv_heads) * float(head_dim) * 8 / 8e6f; }

// Where each of `n` counts up to `most` comes when the largest are first, equal ones in order.
template <typename COUNT>
std::vector<uint32_t> largest_first(size_t n, int most, COUNT&& count) {
    std::vector<uint32_t> order(n);
    if (size_t(most) > 16 * n + 4096) {
        for (size_t i = 0; i < n; i++) order[i] = uint32_t(i);
        std::stable_sort(order.begin(), order.end(), [&](uint32_t a, uint32_t b) { return count(a) > count(b); });
        return order;
    }
    std::vector<uint32_t> at(size_t(most) + 2, 0);  // of count c: where those of count most - c begin
    for (size_t i = 0; i < n; i++) at[size_t(most - count(i)) + 1]++;
    for (size_t c = 1; c < at.size(); c++) at[c] += at[c - 1];
    for (size_t i = 0; i < n; i++) order[at[size_t(most - count(i))]++] = uint32_t(i);
    return order;
}

// The units on the CU that has most of them, the tiles taken longest first. Of many a CU, their average and one more.
int64_t heaviest(const std::vector<Tile>& tiles, int longest, int64_t total, int64_t cus) {
    const size_t n = tiles.size();
    if (n <= size_t(cus)) return longest + kItemUnits;
    if (n > 8 * size_t(cus)) return std::max<int64_t>(longest + kItemUnits, total / cus + total / int64_t(n));
    const std::vector<uint32_t> order = largest_first(n, longest, [&](size_t i) { return tiles[i].units(); });
    std::vector<int64_t> load(static_cast<size_t>(cus));
    for (size_t i = 0; i < size_t(cus); i++) load[i] = tiles[order[i]].units() + kItemUnits;
    const auto later = [](int64_t a, int64_t b) { return a > b; };
    std::make_heap(load.begin(), load.end(), later);
    for (size_t i = size_t(cus); i < n; i++) {
        std::pop_heap(load.begin(), load.end(), later);
        load.back() += tiles[order[i]].units() + kItemUnits;
        std::push_heap(load.begin(), load.end(), later);
    }
    return *std::max_element(load.begin(), load.end());
}

PagedItem item_of(const Tile& t, const ge_paged_seq& e, int64_t lo, int64_t hi, uint32_t part) {
    PagedItem i{};
    i.q_token = e.q_start;
    i.row0 = t.row0;
    i.n_rows = t.n_rows;
    i.key0 = e.slot;
    i.k_lo = uint32_t(lo);
    i.k_hi = uint32_t(hi);
    i.shift = int32_t(int64_t(e.kv_len) - int64_t(e.q_len));
    i.part = part;
    i.narrow = t.n_rows <= uint32_t(kCausalNarrowRows);
    return i;
}

int item_units(const PagedItem& i) { return int((i.k_hi - i.k_lo + kUnit - 1) / kUnit); }

void add_join(PagedPlan& p, const Tile& t, const ge_paged_seq& e, size_t first_part, uint32_t splits) {
    CausalJoin j{e.q_start, t.row0, t.n_rows, {}, {}, {}};
    j.part[0] = uint32_t(first_part);
    j.stride[0] = t.n_rows;
    j.splits[0] = splits;
    p.joins.push_back(j);
    p.join_rows = std::max(p.join_rows, int(t.n_rows));
    p.join_parts = std::max(p.join_parts, int(splits));
}

// Raises the parts of the group with the longest ones while the items stay within `most`; returns the longest part.
int cut_groups(std::vector<Group>& groups, int64_t most) {
    int64_t items = 0;
    for (const Group& g : groups) items += g.n;
    const auto shorter = [&](uint32_t a, uint32_t b) { return groups[a].step() < groups[b].step(); };
    std::vector<uint32_t> heap(groups.size());
    for (size_t i = 0; i < heap.size(); i++) heap[i] = uint32_t(i);
    std::make_heap(heap.begin(), heap.end(), shorter);
    for (;;) {
        std::pop_heap(heap.begin(), heap.end(), shorter);
        Group& g = groups[heap.back()];
        if (items + g.n > most || g.step() < 2 * kLeastPart) return g.step();
        items += g.n;
        g.parts++;
        std::push_heap(heap.begin(), heap.end(), shorter);
    }
}

void plan_parts(PagedPlan& p, const std::vector<Group>& groups, const std::vector<Tile>& tiles, const ge_paged_seq* seqs) {
    // where each tile's parts begin among the partial rows, then the items part by part
    std::vector<uint32_t> part(tiles.size());
    std::vector<int> splits(tiles.size());
    for (const Group& g : groups) {
        const int step = g.step();
        for (uint32_t i = g.first; i < g.first + g.n; i++) {
            const Tile& t = tiles[i];
            splits[i] = g.parts == 1 ? 1 : std::max(1, (t.units() + step - 1) / step);
            part[i] = uint32_t(p.part_rows);
            if (splits[i] == 1) continue;
            p.part_rows += size_t(splits[i]) * t.n_rows;
            add_join(p, t, seqs[t.seq], part[i], uint32_t(splits[i]));
        }
    }
    size_t n = 0;
    for (const int x : splits) n += size_t(x);
    std::vector<PagedItem> items;
    items.reserve(n);
    int longest = 0;
    for (const Group& g : groups) {
        const int64_t step = int64_t(g.step()) * kUnit;
        for (int s = 0; s < g.parts; s++)
            for (uint32_t i = g.first; i < g.first + g.n; i++) {
                const Tile& t = tiles[i];
                if (s >= splits[i]) continue;
                const int64_t k = t.lo + s * step;
                items.push_back(item_of(t, seqs[t.seq], k, std::min<int64_t>(t.hi, k + step), splits[i] == 1 ? kDirect : part[i] + uint32_t(s) * t.n_rows));
                longest = std::max(longest, item_units(items.back()));
            }
    }
    p.items.reserve(n);
    for (const uint32_t i : largest_first(n, longest, [&](size_t x) { return item_units(items[x]); })) p.items.push_back(items[i]);
    p.workgroups = p.items.size();
}

void plan_shares(PagedPlan& p, const std::vector<Tile>& tiles, const ge_paged_seq* seqs, int64_t total, int64_t shares) {
    p.items.reserve(size_t(shares) + tiles.size());
    p.joins.reserve(tiles.size());
    std::vector<PagedItem> rest;     // all but the workgroups' first items
    std::vector<size_t> rest_of;     // their workgroups
    rest.reserve(tiles.size());
    rest_of.reserve(tiles.size());
    // units not yet given out, an item more for each border; of the current workgroup's share
    int64_t left = total + (shares - 1) * kItemUnits, room = 0;
    bool open = false;               // the current workgroup has an item
    auto begin = [&] {
        const int64_t groups = shares - int64_t(p.workgroups);
        room = groups > 1 ? (left + groups - 1) / groups : int64_t(1) << 40;
        open = false;
        p.workgroups++;
    };
    for (const Tile& t : tiles) {
        const ge_paged_seq& e = seqs[t.seq];
        const size_t first_part = p.part_rows;
        uint32_t splits = 0;
        int64_t k = t.lo;
        for (bool done = false; !done;) {
            const int64_t units = (t.hi - k + kUnit - 1) / kUnit;
            if (p.workgroups == 0 || (open && room < std::min<int64_t>(units, kLeastPart) + kItemUnits && int64_t(p.workgroups) < shares)) begin();
            int64_t take = std::min(units, std::max<int64_t>(room - kItemUnits, kLeastPart));
            if (units - take < kLeastPart) take = units;
            const int64_t end = std::min<int64_t>(t.hi, k + take * kUnit);
            done = end == t.hi;
            const bool direct = done && splits == 0;
            const PagedItem i = item_of(t, e, k, end, direct ? kDirect : uint32_t(p.part_rows));
            if (!direct) {
                p.part_rows += t.n_rows;
                splits++;
            }
            if (open) {
                rest.push_back(i);
                rest_of.push_back(p.workgroups - 1);
            } else {
                p.items.push_back(i);
                open = true;
            }
            room -= take + kItemUnits;
            left -= take + kItemUnits;
            k = end;
        }
        if (splits) add_join(p, t, e, first_part, splits);
    }
    // the chains: from a workgroup's first item to its others, in order
    std::vector<uint32_t> last(p.workgroups);
    for (size_t w = 0; w < p.workgroups; w++) last[w] = uint32_t(w);
    for (size_t i = 0; i < rest.size(); i++) {
        const uint32_t at = uint32_t(p.items.size());
        p.items[last[rest_of[i]]].next = at;
        last[rest_of[i]] = at;
        p.items.push_back(rest[i]);
    }
}

}  // namespace

PagedPlan plan_paged(const ge_paged_shape& s, const ge_paged_seq* seqs, int n_seqs) {
    PagedPlan p;
    const int group = s.heads / s.kv_heads, wide = paged_wide_rows(s.head_dim);
    std::vector<Tile> tiles;
    std::vector<Group> groups;
    tiles.reserve(size_t(n_seqs) + 64);
    groups.reserve(size_t(n_seqs));
    int64_t total = 0, rows_all = 0, narrow_units = 0;
    int longest = 0;
    for (int q = 0; q < n_seqs; q++) {
        const ge_paged_seq& e = seqs[q];
        const int64_t rows = int64_t(e.q_len) * group, shift = int64_t(e.kv_len) - int64_t(e.q_len);
        if (!rows) continue;
        groups.push_back(Group{uint32_t(tiles.size()), uint32_t((rows + wide - 1) / wide), 0, 1});
        for (int64_t r = 0; r < rows; r += wide) {
            const int64_t n = std::min<int64_t>(wide, rows - r);
            int64_t lo = 0;
            if (s.window) lo = std::max<int64_t>(0, uint32_t(r) / uint32_t(group) + shift - s.window + 1) / kPagedAlign * kPagedAlign;
            int64_t hi = std::min<int64_t>(e.kv_len, uint32_t(r + n - 1) / uint32_t(group) + shift + 1);
            if (hi <= lo) lo = hi = 0;
            tiles.push_back(Tile{uint32_t(q), uint32_t(r), uint32_t(n), int32_t(lo), int32_t(hi)});
            const int units = tiles.back().units();
            total += units + kItemUnits;
            groups.back().units = std::max(groups.back().units, units);
            const bool narrow = n <= kCausalNarrowRows;
            p.kinds |= narrow ? kCausalNarrow : kCausalWide;
            narrow_units += narrow ? units : 0;
            rows_all += n;
        }
        longest = std::max(longest, groups.back().units);
    }
    if (tiles.empty()) return p;

    const int64_t at_once = std::max(1, kCus * paged_workgroups(s.head_dim) / s.kv_heads), cus = std::max(1, kCus / s.kv_heads);
    const int64_t n_tiles = int64_t(tiles.size());
    const float row_avg = float(rows_all) / float(n_tiles);
    auto us = [&](float load, float item) { return items_us(s.head_dim, 2 * narrow_units >= total, load, item); };
    auto joined = [&](int64_t parts) { return join_us(float(parts) * row_avg, s.kv_heads, s.head_dim); };
    int64_t shares = 0, most = 0;  // the way taken: whole where both are 0
    if (longest > kWhole && tiles.size() < std::max(kManyTiles, size_t(at_once))) {
        // Estimates are off by what they leave out: whole single tiles of different lengths leave the memory to the few
        // longest at the end, 10%; shares of wide tiles, over different keys at a time, miss the L2, 15%.
        const bool single = 2 * groups.size() > tiles.size();
        float best = us(float(heaviest(tiles, longest, total, cus)), float(longest + kItemUnits)) * (single ? 1.1f : 1.0f);
        // A row of many parts waits for its join: shares have as many whole units as bring the longest tile to 128 to 255 parts. A
        // token over 30000 keys, head dim 256, in 469, 235 and 118 parts 10.7 + 11.2, 11.0 + 7.4 and 13.4 + 5.4 us, head dim 128
        // 9.3 + 12.3, 8.8 + 8.0 and 9.7 + 5.6; over 16319 keys in 255 and 127 parts (one KV head of 64, 128, 256 and 512) 12.6 and
        // 11.1, 15.6 and 13.1, 16.4 and 16.4, 23.6 and 24.7, over 32000 in 166 and 125 12.3 and 11.8, 15.4 and 14.4, 17.9 and 19.3,
        // 30.2 and 31.7.
        const int64_t n = std::min(at_once, (total - n_tiles * kItemUnits) / std::max(kLeastPart, longest / 128));
        if (n > 1) {
            const float share = float(total) / float(n) + kItemUnits;
            const float t = us(float((n + cus - 1) / cus) * share, share) * (single ? 1.0f : 1.15f) + joined(n + std::min(n, n_tiles));
            if (t < best) {
                best = t;
                shares = n;
            }
        }
        std::vector<Group> cut;
        for (const int64_t fill : {at_once / 2, at_once, 2 * at_once}) {
            if (single || n_tiles >= fill) continue;
            cut = groups;
            const float part = float(cut_groups(cut, fill) + kItemUnits);
            int64_t items = 0, parts = 0;
            for (const Group& g : cut) {
                items += int64_t(g.n) * g.parts;
                parts += g.parts > 1 ? int64_t(g.n) * g.parts : 0;
            }
            // the CU with most has all its parts of an average length and one of the longest
            const float average = float(total + (items - n_tiles) * kItemUnits) / float(items);
            const float t = us(float((items + cus - 1) / cus - 1) * average + part, part) + joined(parts);
            if (parts && t < best) {
                best = t;
                shares = 0;
                most = fill;
            }
        }
    }
    if (shares) {
        plan_shares(p, tiles, seqs, total, shares);
    } else {
        if (most) cut_groups(groups, most);
        plan_parts(p, groups, tiles, seqs);
    }
    return p;
}

}  // namespace ge
