// Paged KV cache: launches of paged.hip.
#pragma once

#include "tla_internal.h"

namespace tla {

enum KvType { kKvF32 = 0, kKvF16 = 1, kKvBF16 = 30 };  // the ggml_type ids of the elements

// One layer of a paged cache.  Position p of sequence s is row p % page_size
// of page table[s * table_stride + p / page_size]; an entry outside
// [0, n_pages) is an absent page: nothing is written to it, and its positions
// are not attended to.
struct PagedPool {
    void* k;               // page 0 of the layer
    void* v;
    const int* table;
    long long page_stride;  // elements
    int table_stride;
    int n_pages;
    int page_shift;        // page_size = 1 << page_shift
    int type;              // KvType
};

// The sequences of one launch, in the kernel arguments: sequence s holds
// pos[s] positions before the call, its new tokens are rows tok[s] ..
// tok[s + 1] - 1 of the packed inputs.  Work items are handed out by rank:
// rank r is sequence id(r), its items first[r] .. first[r + 1] - 1 (none for a
// sequence that this launch does not serve).  The ids are bytes of whole words:
// from an array of bytes next to arrays of words the compiler made scalar word
// loads whose base address is not a multiple of 4, which the hardware rounds
// down (ROCm 7.2).
template <int kMaxSeq>
struct PagedSeqs {
    int pos[kMaxSeq];
    int tok[kMaxSeq + 1];
    int first[kMaxSeq + 1];
    unsigned ids[kMaxSeq / 4];
    __host__ __device__ int id(int rank) const { return (int)(ids[rank >> 2] >> (8 * (rank & 3)) & 255); }
    void set_id(int rank, int s)
    {
        ids[rank >> 2] = (ids[rank >> 2] & ~(255u << (8 * (rank & 3)))) | (unsigned)s << (8 * (rank & 3));
    }
};
static_assert(kMaxSeqPerLaunch <= 256, "PagedSeqs::ids");
typedef PagedSeqs<kMaxSeqPerLaunch> PagedBatch;

struct PagedAppendParams {
    PagedPool pool;
    const float* k;  // [total tokens][n_head_kv][64]
    const float* v;
    const float2* rope;
    int n_seq;
    int n_head_kv;
    int n_items;
    int rotate;
};
hipError_t launch_paged_append(const PagedAppendParams& p, const PagedBatch& b, hipStream_t s);

// Words from one arrival counter to the next.  Device-scope atomics on one line of
// memory take about 0.11 us each, one after the other: next to each other, the
// counters of 1024 work items kept a launch of 8 x 16384 positions to 110 us.
constexpr int kCounterStride = 64;

// The work items of one kind of a call, and the workspace of its own that they
// share rows through.
struct PagedWork {
    float* part;     // softmax states of the items that share rows, by item
    int* counters;   // and their arrivals, by the rows' first item, kCounterStride apart; zero
                     // between launches
    int n_items;     // 0: none of the kind in the call
    int split_tiles; // chunks: key tiles per item at most
};

struct PagedAttentionParams {
    PagedPool pool;
    const float* q;  // [total tokens][n_head][64]
    float* out;
    const float2* rope;
    PagedWork chunk, stream;
    int n_seq;
    int n_head;
    int n_head_kv;
    int gqa;
    int rotate;
    float scale_log2;
};

// How one call's sequences are served: those of at most `rows` query rows per kv
// head stream their keys and values past 16 rows held in registers
// (paged_stream_kernel; further rows read them again, from the L2), longer chunks
// go through LDS tiles (paged_chunk_kernel), which need a third of the time for each
// product but more before the first and after the last.  Up to kStreamRows rows
// streaming was faster throughout (F16, 4 kv heads, 64 rows over 500 / 4000 / 16000
// positions 7.3 / 9.5 / 15.6 us against 11.9 / 22.3 / 37.9; 16 sequences of 1500 16.9
// against 20.2); up to kStreamRowsMost the plans' estimates decide (128 rows: 8.0 /
// 10.2 / 22.0 against 13.3 / 22.9 / 38.6; 16 of 1500 23.7 against 21.9; a prompt of
// 512 tokens, 4096 rows, 16.1 either way, over F32 22.1 against 23.5).
constexpr int kStreamRows = 64;
constexpr int kStreamRowsMost = 4096;
// Units of 16 rows of one kv head that a streamed sequence of `rows` rows has.
__host__ __device__ constexpr int stream_units(int rows, int n_head_kv) { return (rows + 15) / 16 * n_head_kv; }
constexpr int kStreamTile = 32;  // keys per tile of one wave
constexpr int kMaxStreamParts = 128;  // work items that share a row
constexpr int kChunkRows = 128;  // query rows of a workgroup
struct PagedPlan {
    PagedBatch batch;  // pos and tok set by the caller
    int n_items;       // 0: no such sequence in the call
    int split_tiles;
    double us;         // its estimated time
    int n_shared;      // the items before this one may share rows with others
};
constexpr int kMaxPagedItems = (1 << 24) - 1;  // a launch's threads, 256 to an item, are counted in 32 bits; a
                                               // plan of that many or more says this
// Bytes of one work item's softmax state.
constexpr int kStreamStateBytes = 64 * 18 * 4;
constexpr int kChunkStateBytes = 4 * 64 * 34 * 4;
// Keys per tile of paged_chunk_kernel.
constexpr int chunk_tile(int type) { return type == kKvF32 ? 32 : 64; }
hipError_t launch_paged_stream(const PagedAttentionParams& p, const PagedBatch& b, hipStream_t s);
hipError_t launch_paged_chunk(const PagedAttentionParams& p, const PagedBatch& b, hipStream_t s);
// Both kinds at once: pages of at least 16 positions, and no more sequences than
// two kinds' argument blocks hold in 4 KiB.
constexpr int kMaxMixedSeqs = 64;
hipError_t launch_paged_mixed(const PagedAttentionParams& p, const PagedBatch& chunks, const PagedBatch& streams, hipStream_t s);

hipError_t load_paged_code();

}  // namespace tla
