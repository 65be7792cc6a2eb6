// Host side of paged attention: which work items a call's sequences become.
#pragma once

#include <algorithm>

#include "paged.h"

namespace tla {

// Hands out the work items, tiles[s] key tiles in parts of at most p->split_tiles
// times units(s) for sequence s: the longest sequences first, so that the last
// items to start are short ones and those that share rows come before all others.
template <class F>
inline void rank_items(int n_seq, const int* tiles, F&& units, PagedPlan* p)
{
    PagedBatch& b = p->batch;
    long long order[kMaxSeqPerLaunch];  // descending tiles, then ascending sequence
    for (int s = 0; s < n_seq; ++s) order[s] = -(static_cast<long long>(tiles[s]) << 8) + s;
    if (!std::is_sorted(order, order + n_seq)) std::sort(order, order + n_seq);
    long long at = 0;
    p->n_shared = 0;
    for (int r = 0; r < n_seq; ++r) {
        const int s = static_cast<int>(order[r] & 255);
        b.first[r] = static_cast<int>(std::min<long long>(at, kMaxPagedItems));
        b.set_id(r, s);
        const int n = (tiles[s] + p->split_tiles - 1) / p->split_tiles;
        at += n * static_cast<long long>(units(s));
        if (n > 1) p->n_shared = static_cast<int>(std::min<long long>(at, kMaxPagedItems));
    }
    b.first[n_seq] = p->n_items = static_cast<int>(std::min<long long>(at, kMaxPagedItems));
}

// Parts of the keys by estimated time in us, fitted to launches of 1 to 200
// sequences of 128 to 16384 positions, 32 / 4 heads (F16, one sequence of 16384
// positions in 16 / 32 / 64 / 128 parts 15.5 / 14.1 / 17.1 / 26.6 us; 64 of 1100
// whole / in halves 15.9 / 18.6; 64 of 255 to 2047 whole / by 32 / 21 / 16 tiles
// 24.3 / 21.4 / 20.9 / 20.8; F32, 8 of 16384 in 6 / 8 / 16 / 32 parts 59.9 / 55.6 /
// 56.9 / 59.8): all tiles at the rate of memory, less with fewer work items than
// CUs, or the longest part's steps of a wave if that is longer; an uneven end, the
// less the more items a CU has; handing over, and adding one part after the other;
// each further round of four workgroups per CU (96 of 125 to 1000 in 1080 / 700
// items 21.1 / 17.2).
inline void plan_stream(int n_seq, int n_head_kv, int gqa, int n_cu, int type, int rows, PagedPlan* p)
{
    PagedBatch& b = p->batch;
    const double memory = (type == kKvF32 ? 2.6e-3 : 1.3e-3) * 256 / n_cu, compute = (type == kKvF32 ? 1.65e-3 : 0.85e-3) * 256 / n_cu;
    const double step = type == kKvF32 ? 0.4 : 0.19;
    int tiles[kMaxSeqPerLaunch], units[kMaxSeqPerLaunch], most = 0;
    double total = 0, distinct = 0;  // tiles of all units, and without those read again
    for (int s = 0; s < n_seq; ++s) {
        const int n_tok = b.tok[s + 1] - b.tok[s];
        tiles[s] = n_tok > 0 && n_tok <= rows / gqa ? (b.pos[s] + n_tok + kStreamTile - 1) / kStreamTile : 0;
        units[s] = tiles[s] ? stream_units(n_tok * gqa, n_head_kv) : 0;
        most = std::max(most, tiles[s]);
        // a unit's tiles end with its last row's position
        total += 0.5 * units[s] * (tiles[s] + b.pos[s] / kStreamTile + (tiles[s] ? 1 : 0));
        distinct += static_cast<double>(tiles[s]) * n_head_kv;
    }
    p->n_items = p->n_shared = 0;
    p->us = 0;
    if (!most) return;
    p->split_tiles = most;
    double best = 0;
    int worse = 0;
    for (const int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128}) {
        static_assert(kMaxStreamParts == 128);
        const int len = (most + parts - 1) / parts;
        if (parts > 1 && (len < 4 || worse > 3)) break;  // a tile for each wave
        long long items = 0;
        for (int s = 0; s < n_seq; ++s) items += static_cast<long long>((tiles[s] + len - 1) / len) * units[s];
        const double per_item = static_cast<double>(n_cu) / items;  // CUs
        const double us = std::max(std::max(distinct * memory, total * compute) * std::max(1.0, per_item), len * step) +
                          (total < 0.8 * len * items ? 0.14 * len * std::min(1.0, per_item) : 0) +
                          (parts > 1 ? 2.2 + 0.15 * parts : 0) + 3.0 * ((items - 1) / (4 * n_cu));
        if (parts == 1 || us < best) {
            best = us;
            p->split_tiles = len;
            worse = 0;
        } else {
            ++worse;
        }
    }
    p->us = 3 + best;
    rank_items(n_seq, tiles, [&](int s) { return units[s]; }, p);
}

// Parts of the keys by estimated time in us, fitted to 33 calls of 1 to 16 chunks of
// 128 to 4096 tokens over 0 to 8000 positions, in 1 to 12 parts (to 12%): a CU takes
// 0.76 / 0.92 / 1.15 64-key tiles of F16 a us with one, two and three workgroups (1.3
// times the time for one of BF16 or 32 keys of F32), the longest part alone 1.3 us for
// each of its tiles; a third of the longest part for the uneven end, twice that in
// several rounds; 8 us for a workgroup's start and end, and for handing over 0.75 us
// a part and 1.65 us for each work item of a CU.  (F16, 512 tokens after 8000 in 1 /
// 2 / 4 / 6 / 12 parts 191 / 112 / 87.7 / 85.3 / 98.6 us, 4 x 1500 after none in 1 / 2 / 3 / 6
// 106 / 104 / 117 / 142; BF16, 8 kv heads, 2 x 900 after 300 in 1 / 2 / 3 / 8 55.7 / 48.8 /
// 53.3 / 58.2.)
inline void plan_chunk(int n_seq, int n_head_kv, int gqa, int n_cu, int type, int stream_rows, PagedPlan* p)
{
    PagedBatch& b = p->batch;
    const int keys = chunk_tile(type);
    const double unit = type == kKvF16 ? 1.0 : type == kKvBF16 ? 1.33 : 1.3;
    int last[kMaxSeqPerLaunch], most = 0;  // tiles of a sequence's last row tile
    long long units[kMaxSeqPerLaunch];
    double total = 0;
    const auto first_of = [&](int s) { return b.pos[s] / keys + 1; };
    for (int s = 0; s < n_seq; ++s) {
        const int n_tok = b.tok[s + 1] - b.tok[s];
        const long long rows = static_cast<long long>(n_tok) * gqa;
        last[s] = rows > stream_rows ? (b.pos[s] + n_tok - 1) / keys + 1 : 0;
        units[s] = last[s] ? (rows + kChunkRows - 1) / kChunkRows * n_head_kv : 0;
        total += 0.5 * units[s] * (first_of(s) + last[s]);
        most = std::max(most, last[s]);
    }
    p->split_tiles = std::max(most, 1);
    p->n_items = p->n_shared = 0;
    p->us = 0;
    if (!most) return;
    double best = 0;
    int worse = 0;
    for (const int parts : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64}) {
        const int len = (most + parts - 1) / parts;
        if (parts > 1 && (len < 2 || worse > 3)) break;
        double items = 0;  // with any work
        for (int s = 0; s < n_seq; ++s) {
            const int lo = (first_of(s) + len - 1) / len, hi = (last[s] + len - 1) / len;
            items += units[s] * (lo == hi ? hi : std::max(1.0, 0.5 * (first_of(s) + last[s]) / len + 0.5));
        }
        const double per_cu = items / n_cu;
        const double rate = per_cu <= 1 ? 0.76 * per_cu : per_cu <= 2 ? 0.76 + 0.16 * (per_cu - 1) : std::min(1.15, 0.92 + 0.23 * (per_cu - 2));
        const double us = unit * (std::max(total / (n_cu * rate), 1.3 * len) + (per_cu > 3 ? 0.6 : 0.3) * len) +
                          (parts > 1 ? 0.5 + 0.75 * std::min(parts, (most + len - 1) / len) + 1.65 * per_cu : 0);
        if (parts == 1 || us < best) {
            best = us;
            p->split_tiles = len;
            worse = 0;
        } else {
            ++worse;
        }
    }
    p->us = 8 + best;
    rank_items(n_seq, last, [&](int s) { return units[s]; }, p);
}

// Both kinds in one launch start and end side by side.
inline double launch_us(const PagedPlan& chunks, const PagedPlan& streams)
{
    return chunks.us + streams.us - (chunks.n_items && streams.n_items ? 8 : 0);
}

// Both kinds of a call's work; positions and tokens set in chunks->batch.
inline void plan_attention(int n_seq, int n_head_kv, int gqa, int n_cu, int type, PagedPlan* chunks, PagedPlan* streams)
{
    streams->batch = chunks->batch;
    plan_chunk(n_seq, n_head_kv, gqa, n_cu, type, kStreamRows, chunks);
    plan_stream(n_seq, n_head_kv, gqa, n_cu, type, kStreamRows, streams);
    if (!chunks->n_items) return;
    PagedPlan c{}, s{};
    c.batch = s.batch = chunks->batch;
    plan_stream(n_seq, n_head_kv, gqa, n_cu, type, kStreamRowsMost, &s);
    const double us = launch_us(*chunks, *streams);
    if (s.us >= us) return;
    plan_chunk(n_seq, n_head_kv, gqa, n_cu, type, kStreamRowsMost, &c);
    if (launch_us(c, s) >= us) return;
    *chunks = c;
    *streams = s;
}

}  // namespace tla
