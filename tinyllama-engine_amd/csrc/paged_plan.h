// Host side of paged attention: which work items a call's sequences become.
#pragma once

#include <algorithm>
#include <cstdlib>

#include "paged.h"

namespace tla {

// The smallest part length from `least` to `most` tiles with which the units
// (items_at(length) work items) are at most `slots`, as many as run at once;
// `most` if there are more even so.
template <class F>
inline int part_tiles(int least, int most, long long slots, F&& items_at)
{
    int lo = least, hi = std::max(least, most);
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (items_at(mid) <= slots)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

// Parts of at least one tile per wave, such that the launch is one round of
// four workgroups per CU if it can be.
inline void plan_stream(int n_seq, int n_head_kv, int gqa, int n_cu, PagedPlan* p)
{
    PagedBatch& b = p->batch;
    int tiles[kMaxSeqPerLaunch], most = 0;
    for (int s = 0; s < n_seq; ++s) {
        const int n_tok = b.tok[s + 1] - b.tok[s];
        tiles[s] = n_tok > 0 && n_tok * gqa <= kStreamRows ? (b.pos[s] + n_tok + kStreamTile - 1) / kStreamTile : 0;
        most = std::max(most, tiles[s]);
    }
    const char* sl = getenv("SL"); const int slots = sl ? atoi(sl) : 4;
    const int least = std::max(getenv("LE") ? atoi(getenv("LE")) : 4, (most + kMaxStreamParts - 1) / kMaxStreamParts);
    const int part = part_tiles(least, most, (long long)slots * n_cu, [&](int len) {
        long long n = 0;
        for (int s = 0; s < n_seq; ++s) n += (tiles[s] + len - 1) / len;
        return n * n_head_kv;
    });
    p->shared = false;
    long long at = 0;
    for (int s = 0; s < n_seq; ++s) {
        b.first[s] = static_cast<int>(at);
        b.set_id(s, s);
        const int n = (tiles[s] + part - 1) / part;
        p->shared |= n > 1;
        at += static_cast<long long>(n) * n_head_kv;
    }
    b.first[n_seq] = p->n_items = static_cast<int>(at);
}

// Parts of the keys by estimated time, in tile steps: one round of workgroups
// takes the longest part, several their even share and half a part for the
// uneven end; a part costs about three steps of its own (its queries, its first
// tile, handing over its state).
inline void plan_chunk(int n_seq, int n_head_kv, int gqa, int n_cu, int type, PagedPlan* p)
{
    PagedBatch& b = p->batch;
    const int keys = chunk_tile(type);
    const double slots = 3.0 * n_cu;
    int last[kMaxSeqPerLaunch], most = 0;  // tiles of a sequence's last row tile
    long long units[kMaxSeqPerLaunch], all = 0;
    double total = 0;
    const auto first_of = [&](int s) { return b.pos[s] / keys + 1; };
    for (int s = 0; s < n_seq; ++s) {
        const int n_tok = b.tok[s + 1] - b.tok[s];
        const long long rows = static_cast<long long>(n_tok) * gqa;
        last[s] = rows > kStreamRows ? (b.pos[s] + n_tok - 1) / keys + 1 : 0;
        units[s] = last[s] ? (rows + kChunkRows - 1) / kChunkRows * n_head_kv : 0;
        all += units[s];
        total += 0.5 * units[s] * (first_of(s) + last[s]);
        most = std::max(most, last[s]);
    }
    p->split_tiles = std::max(most, 1);
    p->n_items = 0;
    p->shared = false;
    if (!most) return;
    double best = 0;
    for (const int parts : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64}) {
        const int len = (most + parts - 1) / parts;
        if (parts > 1 && (len < 4 || all > 4 * slots)) break;
        double items = 0;
        for (int s = 0; s < n_seq; ++s) {
            const int lo = (first_of(s) + len - 1) / len, hi = (last[s] + len - 1) / len;
            items += units[s] * (lo == hi ? hi : std::max(1.0, 0.5 * (first_of(s) + last[s]) / len + 0.5));
        }
        const double steps = (items <= slots ? len : std::max<double>(len, total / slots + 0.5 * len)) +
                             3 * std::max(1.0, items / slots) + (parts > 1 ? 0.3 * parts : 0);
        if (parts == 1 || steps < best) {
            best = steps;
            p->split_tiles = len;
        }
    }
    long long at = 0;
    for (int s = 0; s < n_seq; ++s) {
        b.first[s] = static_cast<int>(at);
        b.set_id(s, s);
        const int n = (last[s] + p->split_tiles - 1) / p->split_tiles;
        p->shared |= n > 1;
        at += n * units[s];
    }
    b.first[n_seq] = p->n_items = static_cast<int>(at);
}

}  // namespace tla
