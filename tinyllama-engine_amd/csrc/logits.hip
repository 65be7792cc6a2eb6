// Rules on a batch of logits: penalties for tokens of the history, biases, a
// mask of allowed tokens, and the best token that is left.
#include "logits.h"

namespace tla {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;  // logits per workgroup

// Keys that order by value, then lower index first; 0 is below all of them.
__device__ __forceinline__ unsigned long long best_key(float v, int j)
{
    unsigned u = __builtin_bit_cast(unsigned, v == 0.f ? 0.f : v);  // -0 ties with +0
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (unsigned long long)u << 32 | (0xffffffffu - (unsigned)j);
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

// One workgroup per slice of a row.  The slice's counts of the history's
// tokens and the places of its last biases are gathered in LDS: every
// workgroup of a row reads the row's history (integer atomics, whose order
// does not show).
__global__ __launch_bounds__(kThreads) void logits_kernel(const LogitsParams p)
{
    __shared__ int s_count[kSlice];
    __shared__ int s_bias[kSlice];  // 1 + the place of the last bias of the token, 0: none
    __shared__ unsigned long long s_best[kThreads / 64];
    __shared__ int s_last;
    const int row = blockIdx.x / p.n_slices, slice = blockIdx.x % p.n_slices;
    const int j0 = slice * kSlice, n = min(kSlice, p.n_vocab - j0);
    const tla_logit_rules& r = p.rules;
    for (int j = threadIdx.x; j < n; j += kThreads) {
        s_count[j] = 0;
        s_bias[j] = 0;
    }
    __syncthreads();
    float rep = 1.f, pres = 0.f, freq = 0.f;
    if (r.history_dev) {
        const int len = min(max(r.history_len_dev[row], 0), r.history_stride);
        const int* const h = r.history_dev + (long long)row * r.history_stride;
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const unsigned j = (unsigned)(h[i] - j0);
            if (h[i] >= j0 && j < (unsigned)n) atomicAdd(&s_count[j], 1);
        }
        rep = r.penalties_dev[3 * (long long)row];
        pres = r.penalties_dev[3 * (long long)row + 1];
        freq = r.penalties_dev[3 * (long long)row + 2];
    }
    if (r.bias_token_dev) {
        const int len = min(max(r.bias_len_dev[row], 0), r.bias_stride);
        const int* const t = r.bias_token_dev + (long long)row * r.bias_stride;
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const unsigned j = (unsigned)(t[i] - j0);
            if (t[i] >= j0 && j < (unsigned)n) atomicMax(&s_bias[j], i + 1);
        }
    }
    __syncthreads();
    const float* const x = p.x + (long long)row * p.n_vocab + j0;
    float* const out = p.out + (long long)row * p.n_vocab + j0;
    unsigned long long best = 0;
    for (int j = threadIdx.x; j < n; j += kThreads) {
        float v = ruled(x[j], s_count[j], rep, pres, freq);
        if (s_bias[j]) v += r.bias_value_dev[(long long)row * r.bias_stride + s_bias[j] - 1];
        if (r.mask_dev && !(r.mask_dev[(long long)row * r.mask_stride + (j0 + j) / 32] >> ((j0 + j) & 31) & 1))
            v = -INFINITY;
        out[j] = v;
        if (v > -INFINITY) best = max(best, best_key(v, j0 + j));  // not a NaN
    }
    if (!p.tokens) return;
    best = wave_best(best);
    if ((threadIdx.x & 63) == 0) s_best[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 64; ++w) best = max(best, s_best[w]);
        __hip_atomic_store(&p.best[(long long)row * p.n_slices + slice], best, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
        s_last = __hip_atomic_fetch_add(&p.counters[row], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
                 p.n_slices - 1;
    }
    __syncthreads();
    if (!s_last || threadIdx.x >= 64) return;
    best = 0;
    for (int i = threadIdx.x; i < p.n_slices; i += 64)
        best = max(best, __hip_atomic_load(&p.best[(long long)row * p.n_slices + i], __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT));
    best = wave_best(best);
    if (threadIdx.x == 0) {
        p.tokens[row] = best ? (int)(0xffffffffu - (unsigned)best) : -1;
        __hip_atomic_store(&p.counters[row], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

}  // namespace

int logits_slices(int n_vocab)
{
    return (n_vocab + kSlice - 1) / kSlice;
}

hipError_t load_logits_code()
{
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&logits_kernel));
}

hipError_t launch_logits_process(const LogitsParams& p, int n_seq, hipStream_t s)
{
    hipLaunchKernelGGL(logits_kernel, dim3((unsigned)(n_seq * p.n_slices)), dim3(kThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace tla
