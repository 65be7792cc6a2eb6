// Plans of paged attention on the CPU: every query row of every sequence is
// served by exactly one kernel, every key tile by exactly one work item of its
// rows, as the kernels take the items apart.
#include <cstdio>
#include <cstdlib>
#include <memory>
#include <random>
#include <vector>

#include "paged_plan.h"

using namespace tla;

#define CHECK(x)                                                          \
    do {                                                                  \
        if (!(x)) {                                                       \
            std::printf("line %d: %s fails (case %d)\n", __LINE__, #x, n_case); \
            std::exit(1);                                                 \
        }                                                                 \
    } while (0)

int main()
{
    std::mt19937 rng(1);
    const auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); };
    for (int n_case = 0; n_case < 3000; ++n_case) {
        const int n_seq = n_case % 5 == 0 ? 1 : pick(1, n_case % 7 == 0 ? 256 : 12);
        const int gqa = pick(1, 16), hkv = pick(1, 8), n_cu = n_case % 11 == 0 ? 8 : 256;
        const int type = n_case % 3 == 0 ? kKvF32 : n_case % 3 == 1 ? kKvF16 : kKvBF16;
        auto plan = std::make_unique<PagedPlan>();
        PagedBatch& b = plan->batch;
        int t = 0;
        for (int s = 0; s < n_seq; ++s) {
            b.pos[s] = pick(0, 3) ? pick(0, 1 << pick(0, 14)) : 0;
            b.tok[s] = t;
            t += pick(0, 3) == 0 ? 0 : pick(0, 2) ? 1 : pick(1, 1 << pick(0, 11));
        }
        b.tok[n_seq] = t;
        std::vector<int> served(n_seq, 0);
        auto streams = std::make_unique<PagedPlan>();
        plan_attention(n_seq, hkv, gqa, n_cu, type, plan.get(), streams.get());
        for (const bool chunk : {true, false}) {
            if (!chunk) std::swap(*plan, *streams);
            if (plan->n_items == 0) continue;
            CHECK(plan->n_items == b.first[n_seq] && b.first[0] == 0);
            int shared = 0;
            std::vector<int> ids(n_seq, 0);
            for (int r = 0; r < n_seq; ++r) {
                const int s = b.id(r), items = b.first[r + 1] - b.first[r];
                CHECK(items >= 0 && ++ids[s] == 1);
                const int n_tok = b.tok[s + 1] - b.tok[s], len = b.pos[s] + n_tok, rows = n_tok * gqa;
                if (!items) continue;
                ++served[s];
                CHECK(items % hkv == 0);
                if (!chunk) {
                    const int n_unit = stream_units(rows, hkv);
                    CHECK(items % n_unit == 0);
                    CHECK(rows >= 1 && rows <= kStreamRowsMost);
                    const int n_split = items / n_unit, n_tiles = (len + kStreamTile - 1) / kStreamTile;
                    for (int row0 = 0; row0 < rows; row0 += 16) {  // each unit's tiles in equal parts
                        const int n = (b.pos[s] + (std::min(row0 + 16, rows) - 1) / gqa) / kStreamTile + 1;
                        CHECK(n >= 1 && n <= n_tiles && static_cast<long long>((n + n_split - 1) / n_split) * n_split >= n);
                    }
                    const int per = (n_tiles + n_split - 1) / n_split;
                    if (n_split > 1) shared = b.first[r + 1];
                    CHECK(n_split == 1 || per >= 2);
                    CHECK(n_split <= kMaxStreamParts);
                } else {
                    CHECK(rows > kStreamRows);
                    const int n_rt = (rows + kChunkRows - 1) / kChunkRows;
                    CHECK(items % (n_rt * hkv) == 0);
                    const int splits = items / (n_rt * hkv), keys = chunk_tile(type);
                    for (int rt = 0; rt < n_rt; rt += 1 + n_rt / 7) {
                        const int last_row = std::min((rt + 1) * kChunkRows, rows) - 1;
                        const int n_tiles = (b.pos[s] + last_row / gqa) / keys + 1;
                        const int n_split = (n_tiles + plan->split_tiles - 1) / plan->split_tiles;
                        CHECK(n_split >= 1 && n_split <= splits);
                        if (n_split > 1) shared = b.first[r + 1];
                    }
                }
            }
            CHECK(plan->n_shared >= shared && plan->n_shared <= plan->n_items);
        }
        for (int s = 0; s < n_seq; ++s) CHECK(served[s] == (b.tok[s + 1] > b.tok[s] ? 1 : 0));
    }
    // One sequence of 4096 rows in each of 64 kv heads after millions of positions,
    // beside short ones: the parts' states stay within the 32 bits that address them
    // (so many units are more work items than further parts would be worth).
    for (int n_case = 4000; n_case < 4200; ++n_case) {
        const int n_seq = pick(1, 64), hkv = 64;
        auto plan = std::make_unique<PagedPlan>();
        PagedBatch& b = plan->batch;
        for (int s = 0; s < n_seq; ++s) {
            b.pos[s] = s == 0 ? pick(1 << 20, 1 << 27) : pick(0, 1000);
            b.tok[s + 1] = b.tok[s] + (s == 0 ? 4096 : pick(1, 4096));
        }
        plan_stream(n_seq, hkv, 1, 256, kKvF16, kStreamRowsMost, plan.get());
        for (int r = 0; r < n_seq; ++r) {
            const int s = b.id(r), n = b.first[r + 1] - b.first[r];
            const int units = stream_units(b.tok[s + 1] - b.tok[s], hkv);
            CHECK(n % units == 0 && (n == units || static_cast<long long>(n) * kStreamStateBytes < 1ll << 32));
        }
    }
    // More items than a launch takes are told apart from any that it does.
    {
        const int n_case = 5000, n_seq = 256;
        auto plan = std::make_unique<PagedPlan>();
        for (int s = 0; s < n_seq; ++s) plan->batch.tok[s + 1] = plan->batch.tok[s] + (1 << 16);
        plan_chunk(n_seq, 1024, 16, 256, kKvF16, kStreamRows, plan.get());
        CHECK(plan->n_items == kMaxPagedItems);
    }
    std::printf("plans hold\n");
    return 0;
}
