// Paged KV cache for gfx950: append of new keys (rotated) and values, and
// attention of new tokens over their sequences' pages.
#include "paged.h"
#include "rope_math.h"

namespace tla {
namespace {

constexpr int kWave = 64;

// Elements of the pages: 4 at a time, as floats.
template <int kType>
struct Elem;
template <>
struct Elem<kKvF32> {
    typedef float T;
};
template <>
struct Elem<kKvF16> {
    typedef _Float16 T;
};
template <>
struct Elem<kKvBF16> {
    typedef __bf16 T;
};
template <class T>
struct alignas(4 * sizeof(T)) Four {
    T x[4];
};
template <class T>
__device__ __forceinline__ float4 widen(Four<T> f)
{
    return make_float4((float)f.x[0], (float)f.x[1], (float)f.x[2], (float)f.x[3]);
}
template <class T>
__device__ __forceinline__ Four<T> narrow(float4 f)  // to nearest, ties to even
{
    return Four<T>{{(T)f.x, (T)f.y, (T)f.z, (T)f.w}};
}

// The rank whose work items hold `item` (uniform over the wave): the last of
// those whose first item is at or below it.  One load per 64
// sequences, all in flight together; a search by halves would wait for each of
// its loads in turn.
template <int kMaxSeq>
__device__ __forceinline__ int rank_of(const PagedSeqs<kMaxSeq>& b, int n_seq, int item)
{
    const int lane = threadIdx.x & (kWave - 1);
    int i = -1;
#pragma unroll
    for (int j = 0; j < (kMaxSeq + kWave - 1) / kWave; ++j) {
        const int at = j * kWave + lane;
        const bool below = at < n_seq && b.first[at < n_seq ? at : 0] <= item;
        i += __popcll(__ballot(below));
    }
    return i;
}

// Row (page and row in the page, as an element offset into the pool) of
// position pos of the sequence at table row `table`; -1: an absent page.
__device__ __forceinline__ long long row_of(const PagedPool& c, const int* table, int pos, int kv_dim)
{
    const int page = table[pos >> c.page_shift];
    if ((unsigned)page >= (unsigned)c.n_pages) return -1;
    return (long long)page * c.page_stride + (long long)(pos & ((1 << c.page_shift) - 1)) * kv_dim;
}

// One wave per token: its k and v rows in pieces of 4 floats, lanes over both.
template <int kType, int kMaxSeq>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p, const PagedSeqs<kMaxSeq> b)
{
    typedef typename Elem<kType>::T T;
    const int item = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (item >= p.n_items) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int rank = rank_of(b, p.n_seq, item), i = b.id(rank);
    const int t = item - b.first[rank], pos = b.pos[i] + t;
    const int kv_dim = p.n_head_kv * kHeadDim, n4 = kv_dim / 4;
    const long long row = row_of(p.pool, p.pool.table + (long long)i * p.pool.table_stride, pos, kv_dim);
    if (row < 0) return;
    const long long src = (long long)(b.tok[i] + t) * kv_dim;
    for (int c = lane; c < 2 * n4; c += kWave) {
        const bool is_v = c >= n4;
        const int j = 4 * (is_v ? c - n4 : c);
        float4 x = ldg4((is_v ? p.v : p.k) + src + j);
        if (p.rotate && !is_v)
            x = rotate4(x, ldg4(reinterpret_cast<const float*>(p.rope + (long long)pos * kPairs) + j % kHeadDim));
        *reinterpret_cast<Four<T>*>(static_cast<T*>(is_v ? p.pool.v : p.pool.k) + row + j) = narrow<T>(x);
    }
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

__device__ __forceinline__ float lane_of(float v, int lane)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// One output row by one wave in plain fp32: scores of 64 keys at a time, one
// key per lane, running max and sum, then the lanes as dimensions for P.V.  A
// key that is not seen (later than qpos, or in an absent page) is not
// touched.  x: dimension `lane` of q, rotated and scaled.
template <int kType>
__device__ float plain_row(const PagedPool& c, const int* table, int kv_dim, int head_off, int qpos, float x)
{
    typedef typename Elem<kType>::T T;
    const int lane = threadIdx.x & (kWave - 1);
    const T* const kp = static_cast<const T*>(c.k) + head_off;
    const T* const vp = static_cast<const T*>(c.v) + head_off;
    float m_run = -INFINITY, l_run = 0.f, acc = 0.f;
    for (int k0 = 0; k0 <= qpos; k0 += kWave) {
        const long long row = k0 + lane <= qpos ? row_of(c, table, k0 + lane, kv_dim) : -1;
        float s = 0.f;
        if (row >= 0) {
#pragma unroll
            for (int d = 0; d < kHeadDim; d += 4) {
                const float4 k4 = widen(*reinterpret_cast<const Four<T>*>(kp + row + d));
                s = fmaf(lane_of(x, d), k4.x, s);
                s = fmaf(lane_of(x, d + 1), k4.y, s);
                s = fmaf(lane_of(x, d + 2), k4.z, s);
                s = fmaf(lane_of(x, d + 3), k4.w, s);
            }
        }
        unsigned long long seen = __ballot(row >= 0);
        const float m_new = fmaxf(m_run, wave_max(row >= 0 ? s : -INFINITY));
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
        const float w = row >= 0 ? __builtin_amdgcn_exp2f(s - m_use) : 0.f;
        m_run = m_new;
        l_run = l_run * alpha + wave_sum(w);
        acc *= alpha;
        while (seen) {
            const int j = __builtin_ctzll(seen);
            seen &= seen - 1;
            const unsigned lo = __builtin_amdgcn_readlane((int)(row & 0xffffffff), j);
            const unsigned hi = __builtin_amdgcn_readlane((int)(row >> 32), j);
            acc = fmaf(lane_of(w, j), (float)vp[(long long)((unsigned long long)hi << 32 | lo) + lane], acc);
        }
    }
    return l_run == 0.f ? 0.f : acc / l_run;  // no key seen: zeros
}

// Dimension `lane` of the q row at q, rotated (cs: its position's cos and
// sin) and scaled.
__device__ __forceinline__ float q_lane(const float* q, const float2* cs, int rotate, float scale)
{
    const int lane = threadIdx.x & (kWave - 1);
    float x = q[lane];
    if (rotate) {
        const float other = q[lane ^ 1];
        const float2 r = cs[lane >> 1];
        x = lane & 1 ? rot_hi(other, x, r.x, r.y) : rot_lo(x, other, r.x, r.y);
    }
    return x * scale;
}

// One wave per (token, head).
template <int kType, int kMaxSeq>
__global__ __launch_bounds__(256) void paged_attention_kernel(const PagedAttentionParams p, const PagedSeqs<kMaxSeq> b)
{
    const int item = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (item >= p.n_items) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int rank = rank_of(b, p.n_seq, item), i = b.id(rank);
    const int t = (item - b.first[rank]) / p.n_head, h = (item - b.first[rank]) % p.n_head;
    const int qpos = b.pos[i] + t;
    const long long row = ((long long)(b.tok[i] + t) * p.n_head + h) * kHeadDim;
    const float x = q_lane(p.q + row, p.rope + (long long)qpos * kPairs, p.rotate, p.scale_log2);
    p.out[row + lane] = plain_row<kType>(p.pool, p.pool.table + (long long)i * p.pool.table_stride,
                                         p.n_head_kv * kHeadDim, h / p.gqa * kHeadDim, qpos, x);
}

// f(batch) with the kernel argument block of the smallest size that holds n
// sequences: a launch of one or a few does not pay for 3 KiB of arguments.
template <int kMaxSeq>
PagedSeqs<kMaxSeq> fewer(const PagedBatch& b, int n)
{
    PagedSeqs<kMaxSeq> f{};
    for (int i = 0; i < n; ++i) {
        f.pos[i] = b.pos[i];
        f.set_id(i, b.id(i));
    }
    for (int i = 0; i <= n; ++i) {
        f.tok[i] = b.tok[i];
        f.first[i] = b.first[i];
    }
    return f;
}
template <class F>
hipError_t with_batch(const PagedBatch& b, int n, F&& f)
{
    if (n <= 8)
        f(fewer<8>(b, n));
    else if (n <= 64)
        f(fewer<64>(b, n));
    else
        f(b);
    return hipGetLastError();
}
template <class F>
hipError_t with_type(int type, F&& f)
{
    if (type == kKvF32) return f(std::integral_constant<int, kKvF32>{});
    if (type == kKvF16) return f(std::integral_constant<int, kKvF16>{});
    if (type == kKvBF16) return f(std::integral_constant<int, kKvBF16>{});
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t load_paged_code()
{
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&paged_append_kernel<kKvF32, 8>));
}

hipError_t launch_paged_append(const PagedAppendParams& p, const PagedBatch& b, hipStream_t s)
{
    return with_type(p.pool.type, [&](auto type) {
        return with_batch(b, p.n_seq, [&](const auto& seqs) {
            constexpr int kMax = sizeof(seqs.pos) / sizeof(int);
            hipLaunchKernelGGL((paged_append_kernel<type.value, kMax>), dim3((p.n_items + 3) / 4), dim3(256), 0, s, p,
                               seqs);
        });
    });
}

hipError_t launch_paged_attention(const PagedAttentionParams& p, const PagedBatch& b, hipStream_t s)
{
    return with_type(p.pool.type, [&](auto type) {
        return with_batch(b, p.n_seq, [&](const auto& seqs) {
            constexpr int kMax = sizeof(seqs.pos) / sizeof(int);
            hipLaunchKernelGGL((paged_attention_kernel<type.value, kMax>), dim3((p.n_items + 3) / 4), dim3(256), 0, s,
                               p, seqs);
        });
    });
}

}  // namespace tla
