// Rules on a batch of logits: penalties for tokens of the history, biases, a
// mask of allowed tokens, and the best token that is left.
#include <type_traits>

#include "lane_math.h"
#include "logits.h"

namespace tla {
namespace {

// Four logits; a row of an odd vocabulary starts at any multiple of 4 bytes.
typedef float floatx4 __attribute__((ext_vector_type(4), aligned(4)));

// Keys that order by value, then lower index first; 0 is below all of them.
__device__ __forceinline__ unsigned long long best_key(float v, int j)
{
    unsigned u = __builtin_bit_cast(unsigned, v == 0.f ? 0.f : v);  // -0 ties with +0
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (unsigned long long)u << 32 | (0xffffffffu - (unsigned)j);
}

template <int kCtrl>
__device__ __forceinline__ int dpp(int x)
{
    return __builtin_amdgcn_mov_dpp(x, kCtrl, 0xf, 0xf, true);
}

// The largest x of the wave, in every lane, never a NaN: within quads, the
// halves of rows of 16 and rows by lane permutations, then the rows.
__device__ __forceinline__ float wave_max(float x)
{
    const auto step = [&](auto ctrl) {
        x = fmaxf(x, __builtin_bit_cast(float, dpp<ctrl.value>(__builtin_bit_cast(int, x))));
    };
    step(std::integral_constant<int, 0xb1>{});   // quad_perm 1 0 3 2
    step(std::integral_constant<int, 0x4e>{});   // quad_perm 2 3 0 1
    step(std::integral_constant<int, 0x141>{});  // row_half_mirror
    step(std::integral_constant<int, 0x140>{});  // row_mirror
    return max_xor32(max_xor16(x));
}

__device__ __forceinline__ unsigned long long wave_best(unsigned long long k)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const unsigned long long o = __shfl_xor(k, m);
        k = o > k ? o : k;
    }
    return k;
}

// A logit under its row's rules.  Each operation is rounded on its own.
__device__ __forceinline__ float ruled(float x, int count, float rep, float pres, float freq)
{
#pragma clang fp contract(off)
    if (count > 0) {
        x = x > 0.f ? x / rep : x * rep;
        x = x - ((float)count * freq + pres);
    }
    return x;
}

// One workgroup per slice of 4 kPer x kThreads logits of a row.  The counts of the
// history's tokens in the slice and the places of its last biases are gathered in
// LDS, a word of each per logit: every workgroup of a row reads the row's lists
// (integer atomics, whose order does not show).  The logits and the first parts of
// the lists, the biases' values too, are requested before anything is waited for.
//
// Bound by memory: 8 bytes per logit.  200 x 100003 logits with all rules 42.3 us
// and without any 31.2, a copy of them 31.4; the rest are the lists (about 4 us the
// history, 3 the biases, 2 the mask: loads, LDS atomics, a barrier) and the rows'
// hand-over.  64 x 32000 8.4 us, a copy 3.9: the same chain, once.  (One array for
// both lists, one after the other, and the values loaded when their places are known:
// 43.9 and 8.8 us.)  The hand-over passes no release or acquire: at device scope
// those write back and drop the XCD's L2, in every workgroup (61 us became 247).
template <int kThreads, int kPer>
__global__ __launch_bounds__(kThreads) void logits_kernel(const LogitsParams p)
{
    constexpr int kSlice = 4 * kPer * kThreads;
    __shared__ int4 s_count4[kPer * kThreads];  // how often the history holds each logit's token
    __shared__ int4 s_place4[kPer * kThreads];  // 1 + the place of its last bias, 0: none
    __shared__ unsigned long long s_best[kThreads / 64];
    __shared__ float s_value[kThreads];  // the first biases
    const int tid = threadIdx.x;
    const int row = blockIdx.x / p.n_slices, slice = blockIdx.x % p.n_slices;
    const int j0 = slice * kSlice, n = min(kSlice, p.n_vocab - j0);
    const tla_logit_rules& r = p.rules;
    const float* const x = p.x + (long long)row * p.n_vocab + j0;
    float* const out = p.out + (long long)row * p.n_vocab + j0;

    // Piece i of the thread: logits 4 (tid + kThreads i) .. + 3 of the slice.
    floatx4 v[kPer];
    unsigned mask[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = 4 * (tid + kThreads * i);
        if (j + 3 < n)
            v[i] = *reinterpret_cast<const floatx4*>(x + j);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = j + e < n ? x[j + e] : -INFINITY;
        mask[i] = r.mask_dev && j < n ? r.mask_dev[(long long)row * r.mask_stride + (j0 + j) / 32] >> ((j0 + j) & 31) : 15u;
    }
    const int* const h = r.history_dev + (long long)row * r.history_stride;
    const int* const t = r.bias_token_dev + (long long)row * r.bias_stride;
    int h_len = 0, b_len = 0, h0 = -1, h1 = -1, t0 = -1;
    float rep = 1.f, pres = 0.f, freq = 0.f, b0 = 0.f;
    if (r.history_dev) {
        if (tid < r.history_stride) h0 = h[tid];
        if (tid + kThreads < r.history_stride) h1 = h[tid + kThreads];
        h_len = min(max(r.history_len_dev[row], 0), r.history_stride);
        rep = r.penalties_dev[3 * (long long)row];
        pres = r.penalties_dev[3 * (long long)row + 1];
        freq = r.penalties_dev[3 * (long long)row + 2];
    }
    if (r.bias_token_dev) {
        if (tid < r.bias_stride) {
            t0 = t[tid];
            b0 = r.bias_value_dev[(long long)row * r.bias_stride + tid];
        }
        b_len = min(max(r.bias_len_dev[row], 0), r.bias_stride);
    }
    if (r.history_dev || r.bias_token_dev) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s_count4[tid + kThreads * i] = make_int4(0, 0, 0, 0);
            s_place4[tid + kThreads * i] = make_int4(0, 0, 0, 0);
        }
        s_value[tid] = b0;
        __syncthreads();
        if (r.history_dev) {
            const auto add = [&](int token) {
                const unsigned j = (unsigned)token - (unsigned)j0;
                if (j < (unsigned)n) atomicAdd(&reinterpret_cast<int*>(s_count4)[j], 1);
            };
            if (tid < h_len) add(h0);
            if (tid + kThreads < h_len) add(h1);
            for (int i = tid + 2 * kThreads; i < h_len; i += 4 * kThreads) {  // four loads in flight
                int k[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) k[u] = i + u * kThreads < h_len ? h[i + u * kThreads] : -1;
#pragma unroll
                for (int u = 0; u < 4; ++u) add(k[u]);
            }
        }
        if (r.bias_token_dev)
            for (int i = tid; i < b_len; i += kThreads) {
                const unsigned j = (unsigned)(i == tid ? t0 : t[i]) - (unsigned)j0;
                if (j < (unsigned)n) atomicMax(&reinterpret_cast<int*>(s_place4)[j], i + 1);
            }
        __syncthreads();
        const float* const value = r.bias_value_dev + (long long)row * r.bias_stride - 1;
        const auto bias = [&](int place) { return place <= kThreads ? s_value[place - 1] : value[place]; };
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int4 c = s_count4[tid + kThreads * i];
            if (c.x | c.y | c.z | c.w) {
                v[i][0] = ruled(v[i][0], c.x, rep, pres, freq);
                v[i][1] = ruled(v[i][1], c.y, rep, pres, freq);
                v[i][2] = ruled(v[i][2], c.z, rep, pres, freq);
                v[i][3] = ruled(v[i][3], c.w, rep, pres, freq);
            }
            const int4 b = s_place4[tid + kThreads * i];
            if (b.x | b.y | b.z | b.w) {
                if (b.x) v[i][0] += bias(b.x);
                if (b.y) v[i][1] += bias(b.y);
                if (b.z) v[i][2] += bias(b.z);
                if (b.w) v[i][3] += bias(b.w);
            }
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!(mask[i] >> e & 1)) v[i][e] = -INFINITY;
            top = fmaxf(top, v[i][e]);  // past the slice's end: -inf
        }
    const auto store = [&] {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int j = 4 * (tid + kThreads * i);
            if (j + 3 < n)
                *reinterpret_cast<floatx4*>(out + j) = v[i];
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j + e < n) out[j + e] = v[i][e];
        }
    };
    // The first wave hands in the workgroup's best before it stores its logits:
    // its wait below would otherwise cover them.
    if (tid >= 64 || !p.tokens) store();
    if (!p.tokens) return;
    // The first of the wave's largest: its lanes that hold it look for it.
    const float most = wave_max(top);
    int at = 0x7fffffff;
    if (top == most && most > -INFINITY) {
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i)
#pragma unroll
            for (int e = 3; e >= 0; --e) at = v[i][e] == most ? 4 * (tid + kThreads * i) + e : at;
    }
    unsigned long long best = 0;
    for (unsigned long long who = __ballot(at != 0x7fffffff); who; who &= who - 1)
        best = max(best, best_key(most, j0 + __builtin_amdgcn_readlane(at, __builtin_ctzll(who))));
    if ((tid & 63) == 0) s_best[tid >> 6] = best;
    __syncthreads();
    if (tid >= 64) return;
    best = tid < kThreads / 64 ? s_best[tid] : 0;
    best = wave_best(best);
    if (p.n_slices > 1) {
        // The row's last workgroup to arrive reads all of its slots: a place's
        // key may still be on its way when its arrival has been counted, so the
        // reader waits until it is there (its store was issued before the count),
        // and leaves the slot empty.  1: a key that no logit has.
        int last = 0;
        if (tid == 0) {
            __hip_atomic_store(&p.best[(long long)row * p.n_slices + slice], best ? best : 1ull, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            last = __hip_atomic_fetch_add(&p.counters[(long long)row * kRowCounterStride], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.n_slices - 1;
        }
        store();
        if (!__builtin_amdgcn_readfirstlane(last)) return;
        best = 0;
        for (int i = tid; i < p.n_slices; i += 64) {
            unsigned long long* const slot = &p.best[(long long)row * p.n_slices + i];
            unsigned long long k;
            do k = __hip_atomic_load(slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            while (k == 0);
            __hip_atomic_store(slot, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            best = max(best, k);
        }
        best = wave_best(best);
        if (tid == 0) __hip_atomic_store(&p.counters[(long long)row * kRowCounterStride], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
        store();
    }
    if (tid == 0) p.tokens[row] = best > 1 ? (int)(0xffffffffu - (unsigned)best) : -1;
}

}  // namespace

// Few logits: short slices, so that more CUs share the row (1 x 32000 logits,
// 500 tokens of history, slices of 2048 / 4096 / 8192: 4.9 / 5.3 / 5.4 us).  Up to
// about one workgroup per CU slices of 4096 (32 x 32000 9.2 / 7.35 / 7.6 us: each
// workgroup of a row reads its lists again).  Beyond, 8192 (64 x 131072 46 /
// 30.4 / 21.2 us).
int logits_slice(int n_seq, int n_vocab, int n_cu)
{
    const long long n = static_cast<long long>(n_seq) * n_vocab;
    return n <= 512ll * n_cu ? 2048 : n <= 4096ll * n_cu ? 4096 : 8192;
}

hipError_t load_logits_code()
{
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&logits_kernel<512, 1>));
}

hipError_t launch_logits_process(const LogitsParams& p, int n_seq, hipStream_t s)
{
    const dim3 grid((unsigned)(n_seq * p.n_slices));
    if (p.slice == 2048)
        hipLaunchKernelGGL((logits_kernel<512, 1>), grid, dim3(512), 0, s, p);
    else if (p.slice == 4096)
        hipLaunchKernelGGL((logits_kernel<1024, 1>), grid, dim3(1024), 0, s, p);
    else
        hipLaunchKernelGGL((logits_kernel<1024, 2>), grid, dim3(1024), 0, s, p);
    return hipGetLastError();
}

}  // namespace tla
