// Host side of an attention plan: the cut of its row blocks into parts for the card's workgroups.  No device
// code; a step's plan is made once per step and has to cost less than a layer's launches.
#include <algorithm>
#include <exception>
#include <functional>
#include <map>
#include <queue>
#include <vector>

#include "common.h"

namespace rch {

namespace {

constexpr int kXcds = 8;
// Fewest key tiles of a part (of 64 keys), and about the most parts of an item within an XCD.  Single tokens of 8
// short sequences (37 to 1000 tokens) take 13.1 / 14.3 / 21.5 us with parts of at least 2 / 3 / 4 tiles, of 16
// sequences of 2000 tokens 23.9 / 19.8 us with 2 / 3; of 2 of 16000 tokens 31.7 us with up to 64 parts, 23.1 with 32
// (their merge grows).
constexpr int64_t kShortestPart = 3, kMostParts = 32;
// Of waves of single tokens over codes (8 of 37 to 1000 tokens: 14.6 / 15.0 / 16.7 us with parts of at least 1 / 2 / 3), which
// fill the card by parts alone: an item in up to half of an XCD's places (one sequence of 65536 tokens,
// 8 key heads of 256 int8 channels: 98 us, and 176 with parts of at least 3 tiles and at most 32 of them).
constexpr int64_t kShortestWave = 1;
struct Rule {
    int64_t fewest, most;  // tiles of a part, parts of an item within an XCD
};

struct Piece {
    int64_t item, first, last;  // item: rank within the XCD
};

typedef std::priority_queue<int64_t, std::vector<int64_t>, std::greater<int64_t>> Loads;

// Cuts items (longest first) so that `resident` workgroups end by `limit`: what an item has beyond `limit` goes to
// workgroups of its own, the rest to the least loaded one, cut at the room there is.  False if they cannot.
bool ending_by(const std::vector<int64_t>& costs, int64_t resident, int64_t overhead, int64_t fewest, int64_t limit, std::vector<Piece>& pieces) {
    const int64_t room_of_one = limit - overhead;
    struct Rest {
        int64_t cost, item, at;
    };
    std::vector<Rest> rest;
    pieces.clear();
    int64_t busy = 0;
    for (size_t i = 0; i < costs.size(); ++i) {
        int64_t at = 0, cost = costs[i];
        const int64_t item = static_cast<int64_t>(i);
        while (cost - at > room_of_one) {
            // A rest too short for a part takes some of the last full one.
            const int64_t left = cost - at - room_of_one, end = at + room_of_one - (left < fewest ? fewest - left : 0);
            pieces.push_back({item, at, end});
            at = end;
            ++busy;
        }
        rest.push_back({cost - at, item, at});
    }
    if (busy >= resident) return false;
    std::stable_sort(rest.begin(), rest.end(), [](const Rest& a, const Rest& b) { return a.cost > b.cost; });
    Loads loads(std::greater<int64_t>(), std::vector<int64_t>(static_cast<size_t>(resident - busy), 0));
    for (Rest& r : rest) {
        int64_t left = r.cost, at = r.at;
        do {
            const int64_t load = loads.top(), room = room_of_one - load;
            int64_t piece = left;
            if (left > room) {
                if (room < fewest) return false;
                piece = left - room >= fewest ? room : left - fewest;
                if (piece < 1) return false;
            }
            loads.pop();
            loads.push(load + piece + overhead);
            pieces.push_back({r.item, at, at + piece});
            at += piece;
            left -= piece;
        } while (left > 0);
    }
    return true;
}

// Cuts items (longest first) so that `resident` workgroups that take parts in order, longest first, end together as
// early as they can.
void cut(const std::vector<int64_t>& costs, int64_t resident, int64_t overhead, const Rule& rule, std::vector<Piece>& pieces) {
    const int64_t n = static_cast<int64_t>(costs.size()), longest = costs[0], fewest = rule.fewest;
    pieces.clear();
    auto whole = [&]() {
        pieces.clear();
        for (int64_t i = 0; i < n; ++i) pieces.push_back({i, 0, costs[static_cast<size_t>(i)]});
    };
    if (longest < 2 * fewest || n > 4 * resident) return whole();
    int64_t total = 0, uncut = longest + overhead;
    for (const int64_t cost : costs) total += cost;
    if (n > resident) {
        Loads loads(std::greater<int64_t>(), std::vector<int64_t>(static_cast<size_t>(resident), 0));
        uncut = 0;
        for (const int64_t cost : costs) {
            const int64_t load = loads.top() + cost + overhead;
            loads.pop();
            loads.push(load);
            uncut = std::max(uncut, load);
        }
    }
    const int64_t shortest = std::max(fewest, (longest + rule.most - 1) / rule.most);
    int64_t low = std::max((total + n * overhead) / resident, shortest + overhead), high = uncut;
    std::vector<Piece> found;
    while (50 * low < 49 * high) {  // the earliest end that parts reach, within a fiftieth
        const int64_t middle = (low + high) / 2;
        if (ending_by(costs, resident, overhead, fewest, middle, found)) {
            high = middle;
            pieces.swap(found);
        } else {
            low = middle + 1;
        }
    }
    if (pieces.empty() || 20 * high > 19 * uncut) whole();  // joining the parts would cost what little they save
}

int share_out(const int64_t* tiles, const int64_t* owner, int64_t n, int64_t resident, int64_t overhead, int64_t* parts,
              int64_t capacity, int64_t* count) {
    const int64_t places = std::max<int64_t>(1, resident / kXcds);
    const bool waves = overhead >= RCH_SHARE_WAVES;
    const Rule rule = waves ? Rule{kShortestWave, std::max<int64_t>(1, places / 2)} : Rule{kShortestPart, kMostParts};
    const int64_t fewest = rule.fewest;
    overhead -= waves ? RCH_SHARE_WAVES : 0;
    std::vector<int64_t> order(static_cast<size_t>(n)), starts(order.size());
    for (int64_t i = 0; i < n; ++i) order[static_cast<size_t>(i)] = i;
    std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return owner[a] < owner[b]; });
    // Every block takes room on this line, so that one without keys lies in one XCD's share too.
    const int64_t least = std::max<int64_t>(overhead, 1);
    int64_t work = 0;
    for (size_t i = 0; i < order.size(); ++i) {
        starts[i] = work;
        work += tiles[order[i]] + least;
    }
    struct Part {
        int64_t item, first, last, xcd;
    };
    std::vector<Part> out;
    std::map<std::vector<int64_t>, std::vector<Piece>> known;  // XCDs with the same costs are cut alike
    // A border within an item: too short a piece joins the neighbour's.
    auto border = [&](int64_t at, int64_t limit) {
        at = std::min(std::max<int64_t>(at, 0), limit);
        if (at < limit && at < fewest) return int64_t{0};
        return limit - at < fewest ? limit : at;
    };
    struct Inside {
        int64_t cost, item, low;
    };
    size_t from = 0;
    for (int64_t xcd = 0; xcd < kXcds; ++xcd) {
        const int64_t begin = xcd * work / kXcds, end = (xcd + 1) * work / kXcds;
        std::vector<Inside> inside;
        while (from < order.size() && starts[from] + tiles[order[from]] + least <= begin) ++from;
        for (size_t i = from; i < order.size() && starts[i] < end; ++i) {
            const int64_t limit = tiles[order[i]], low = border(begin - starts[i], limit), high = border(end - starts[i], limit);
            // An item without keys is a part of its own where it begins.
            if (high > low || (limit == 0 && starts[i] >= begin)) inside.push_back({high - low, order[i], low});
        }
        if (inside.empty()) continue;
        std::stable_sort(inside.begin(), inside.end(), [](const Inside& a, const Inside& b) { return a.cost > b.cost; });
        std::vector<int64_t> costs;
        for (const Inside& i : inside) costs.push_back(i.cost);
        auto made = known.find(costs);
        if (made == known.end()) {
            std::vector<Piece> pieces;
            cut(costs, places, overhead, rule, pieces);
            made = known.emplace(std::move(costs), std::move(pieces)).first;
        }
        for (const Piece& p : made->second) {
            const Inside& i = inside[static_cast<size_t>(p.item)];
            out.push_back({i.item, i.low + p.first, i.low + p.last, xcd});
        }
    }
    std::sort(out.begin(), out.end(), [](const Part& a, const Part& b) { return a.item != b.item ? a.item < b.item : a.first < b.first; });
    if (static_cast<int64_t>(out.size()) > capacity) return fail(RCH_E_CONFIG, "rch_attend_share: %zu parts do not fit", out.size());
    for (size_t i = 0; i < out.size(); ++i) {
        parts[4 * i] = out[i].item;
        parts[4 * i + 1] = out[i].first;
        parts[4 * i + 2] = out[i].last;
        parts[4 * i + 3] = out[i].xcd;
    }
    *count = static_cast<int64_t>(out.size());
    return RCH_OK;
}

}  // namespace

}  // namespace rch

extern "C" {

int rch_attend_share(const int64_t* tiles, const int64_t* owner, int64_t n, int64_t resident, int64_t overhead, int64_t* parts,
                     int64_t capacity, int64_t* count) {
    using namespace rch;
    if (!tiles || !owner || !parts || !count || n < 0 || resident < 1 || overhead < 0 || capacity < 0)
        return fail(RCH_E_CONFIG, "rch_attend_share: invalid arguments");
    for (int64_t i = 0; i < n; ++i)
        if (tiles[i] < 0 || tiles[i] > (int64_t{1} << 31)) return fail(RCH_E_CONFIG, "rch_attend_share: invalid tile count");
    try {
        return share_out(tiles, owner, n, resident, overhead, parts, capacity, count);
    } catch (const std::exception& e) {
        return fail(RCH_E_LAUNCH, "rch_attend_share: %s", e.what());
    }
}

}  // extern "C"
