// Paged KV cache for gfx950: append of new keys (rotated) and values, and
// attention of new tokens over their sequences' pages.
//
// Row r, a (token, head) pair with query q (rotated at its position p_r), over the
// seen keys j <= p_r of its kv head (those in pages that are there):
//     s_j = q . K_j / 8,  out = sum_j 2^(s_j log2 e - m) V_j / sum_j 2^(s_j log2 e - m).
// One pass: m is a running maximum, and a part of the keys is the state (m, l, O);
// two parts make one, O = O_a 2^(m_a - m) + O_b 2^(m_b - m) and l likewise.  All states
// and sums are fp32.  A row that sees nothing has l = 0 and is 0.
//
// Single tokens are bound by memory (each key and value read once), chunks by the
// matrix cores and the vector operations between their products: two kernels, and a
// third that runs items of both.
#include "bf16_split.h"
#include "lane_math.h"
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
__device__ __forceinline__ long long row_in(const PagedPool& c, int page, int pos, int kv_dim)
{
    if ((unsigned)page >= (unsigned)c.n_pages) return -1;
    return (long long)page * c.page_stride + (long long)(pos & ((1 << c.page_shift) - 1)) * kv_dim;
}
__device__ __forceinline__ long long row_of(const PagedPool& c, const int* table, int pos, int kv_dim)
{
    return row_in(c, table[pos >> c.page_shift], pos, kv_dim);
}

// One wave per token: its k and v rows in pieces of 4 floats, lanes over both.  k is
// rotated with the operations of tla_rope, each rounded on its own: F32 pages hold its
// bits, F16 and BF16 ones those rounded once, to nearest.  Bound by memory where
// there are many tokens (BF16, 16 x 2048 tokens of 4 kv heads 21.3 us, 4.7 TB/s of the
// 100.7 MB read and written; a copy reaches 5.05), by the launch where there are few (64
// tokens 4.4 us a call, 3.8 in the kernel).
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

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kRawBufferWord3 = 0x00020000;  // untyped 32-bit buffer (gfx9 family)
constexpr int kDeviceScope = 16;             // cache-policy bit SC1: device scope
constexpr float kRescaleSlack = 8.f;         // log2 units a running max may lag behind

// Products with fp32 accuracy on the 16-bit matrix cores.  A key or value of
// the cache is exact in its own type; an fp32 operand (a query, a
// probability) is a sum of pieces of that type, and every product of two
// 16-bit numbers is exact in the fp32 accumulator.
//   F16: two pieces, 22 bits: to 2^-22 of the operand, or to 2^-25 (half the
//   smallest step of an F16) where that is more.  Query rows are brought to
//   2^13 .. 2^14 by a power of two first, probabilities carry a factor of 2^6,
//   so that the latter is below 2^-38 of the row's largest.
//   BF16: three pieces, all 24 bits, in fp32's own range.
//   F32: the cache's elements are three BF16 pieces as well: the six products of
//   pieces down to 2^-16 (the three left out are below 2^-24).
template <int kType>
struct Pieces;
template <>
struct Pieces<kKvF16> {
    typedef f16x8 Frag;
    static constexpr int kN = 2;
    static constexpr float kShift = 6.f;
    static constexpr bool kScaled = true;
    static __device__ __forceinline__ void split(floatx8 v, Frag (&o)[kN])
    {
        o[0] = __builtin_convertvector(v, f16x8);
        // v - o[0], exact, by the mixed fma, which reads either half of a word as
        // an F16: half the operations of widening and subtracting.
        const uintx4 w = __builtin_bit_cast(uintx4, o[0]);
        floatx8 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(w[i]), "v"(v[2 * i]));
            asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(hi) : "v"(w[i]), "v"(v[2 * i + 1]));
            r[2 * i] = lo;
            r[2 * i + 1] = hi;
        }
        o[1] = __builtin_convertvector(r, f16x8);
    }
    static __device__ __forceinline__ floatx4 mfma16(Frag a, Frag b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx16 mfma32(Frag a, Frag b, floatx16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Pieces<kKvBF16> {
    typedef bf16x8 Frag;
    static constexpr int kN = 3;
    static constexpr float kShift = 0.f;
    static constexpr bool kScaled = false;
    static __device__ __forceinline__ void split(floatx8 v, Frag (&o)[kN]) { split3x8(v, o[0], o[1], o[2]); }
    static __device__ __forceinline__ floatx4 mfma16(Frag a, Frag b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx16 mfma32(Frag a, Frag b, floatx16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Pieces<kKvF32> : Pieces<kKvBF16> {};

// The power of two that brings a row whose largest magnitude is `top` to
// 2^13 .. 2^14, and its inverse.  Rows of zeros, and of numbers so small or
// large that the factor would leave the fp32 range, get the nearest one that
// does not.
__device__ __forceinline__ void row_scale(float top, float& up, float& down)
{
    const int e = (int)(__builtin_bit_cast(unsigned, top) >> 23 & 255) - 127;
    const int s = min(max(13 - e, -100), 100);
    up = __builtin_bit_cast(float, (unsigned)(127 + s) << 23);
    down = __builtin_bit_cast(float, (unsigned)(127 - s) << 23);
}

// The rotation of rotate4 with fused multiply-adds, for operands that are not
// stored (q).
__device__ __forceinline__ float4 rotate4_fma(float4 x, float4 cs)
{
    return make_float4(__builtin_fmaf(x.x, cs.x, -(x.y * cs.y)), __builtin_fmaf(x.x, cs.y, x.y * cs.x),
                       __builtin_fmaf(x.z, cs.z, -(x.w * cs.w)), __builtin_fmaf(x.z, cs.w, x.w * cs.z));
}

// kN pieces of four dimensions of a query row, dim(i) .., scaled and, if asked,
// rotated.  All loads are issued before any is used, the (cos, sin) also where they
// are not needed: with a branch for them each piece waits for its loads in turn
// (16 times 0.6 us in a chunk's workgroup).
template <int kN, class F>
__device__ __forceinline__ void load_q(const float* q, const float* cs, F&& dim, int rotate, float scale, floatx4 (&x)[kN])
{
    float4 v[kN], r[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        v[i] = ldg4(q + dim(i));
        r[i] = ldg4(cs + dim(i));
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        const float4 s = make_float4(v[i].x * scale, v[i].y * scale, v[i].z * scale, v[i].w * scale);
        const float4 t = rotate4_fma(s, r[i]);
        x[i] = rotate ? floatx4{t.x, t.y, t.z, t.w} : floatx4{s.x, s.y, s.z, s.w};
    }
}

__device__ __forceinline__ bool not_finite(float x)
{
    return !(__builtin_fabsf(x) <= 3.4028234663852886e38f);
}

// A word of a page table at a place that is the same for the whole wave, by a
// scalar load.  (Next to loads into LDS the compiler takes the table for memory
// that they may change, reads it through the vector cache, and waits for them.)
__device__ __forceinline__ int page_at(const int* table, int at)
{
    typedef const int __attribute__((address_space(4))) * Constant;
    return ((Constant)(uintptr_t)table)[at];
}

// Up to 16 rows of 64 elements of one kv head from one page, as a buffer
// whose range ends with them: loads past the last row, and all of an absent
// page's, give zeros without touching memory.
struct Rows {
    const char* base;
    unsigned bytes;  // 0: absent
};
__device__ __forceinline__ auto rsrc_of(const Rows& r)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(r.base), 0, r.bytes, kRawBufferWord3);
}

// Counts this workgroup in after its device-scope stores are acknowledged;
// true for the last of n, which also returns the counter to zero.  All
// threads of the workgroup call it.
__device__ __forceinline__ bool last_to_arrive(int* counter, int n, int& s_last)
{
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
    __syncthreads();
    const bool last = s_last;
    if (last && threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return last;
}

// A wave's operands of one 32-key tile, as the 16x16 MFMAs read them, and the
// two products.  Lane l = 16 g + c.  Keys: K operand row c of half hf is key
// 16 hf + c, so that score register r of lane (g, c) is key 16 hf + 4 g + r
// for query row c.  The same registers are the B operand (P^T) of the P.V
// product if V's k index 8 g + e is key 4 g + e (e < 4) or 16 + 4 g + e - 4.
// V operand row c of dt holds dimension 4 c + dt, so that O register r of dt
// is dimension 16 g + 4 r + dt of query row c.
template <int kType>
struct StreamTile {
    typedef Pieces<kType> P;
    typedef typename P::Frag Frag;
    // k step ks: dimensions 32 ks + 8 g .. + 7, so that one load instruction
    // takes 64 consecutive bytes of each row
    uintx4 k[2][2];
    uintx2 v[8];
    struct Query {
        Frag f[2][P::kN];
        float down;
    };
    // x[i] of Query::query: dimensions q_dim(i, g) .. + 3
    static __device__ __forceinline__ int q_dim(int i, int g) { return 32 * (i >> 1) + 8 * g + 4 * (i & 1); }
    template <class L>  // load16(o): 16 bytes at byte o + 16 g of row c
    __device__ __forceinline__ void load_k(int hf, L&& load16)
    {
        k[hf][0] = load16(0);
        k[hf][1] = load16(64);
    }
    template <class L>
    __device__ __forceinline__ void load_v(int hf, int r, L&& load8)
    {
        v[4 * hf + r] = load8();
    }
    static __device__ __forceinline__ void query(const floatx4 (&x)[4], Query& q)
    {
        float up = 1.f;
        q.down = 1.f;
        if constexpr (P::kScaled) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, __builtin_fabsf(x[i][e]));
            row_scale(max_xor32(max_xor16(top)), up, q.down);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            floatx8 v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = x[2 * ks + (e >> 2)][e & 3] * up;
            P::split(v, q.f[ks]);
        }
    }
    __device__ __forceinline__ floatx4 scores(int hf, const Query& q) const
    {
        floatx4 s = {};
#pragma unroll
        for (int i = P::kN - 1; i >= 0; --i)  // small ones first
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) s = P::mfma16(__builtin_bit_cast(Frag, k[hf][ks]), q.f[ks][i], s);
        return s;
    }
    __device__ __forceinline__ void accumulate(const floatx4 (&p)[2], floatx4 (&o)[4]) const
    {
        Frag f[P::kN];
        P::split(floatx8{p[0][0], p[0][1], p[0][2], p[0][3], p[1][0], p[1][1], p[1][2], p[1][3]}, f);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
            uintx4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = __builtin_amdgcn_perm(v[2 * i + 1][dt >> 1], v[2 * i][dt >> 1], dt & 1 ? 0x07060302 : 0x05040100);
            const Frag a = __builtin_bit_cast(Frag, w);
#pragma unroll
            for (int i = P::kN - 1; i >= 0; --i) o[dt] = P::mfma16(a, f[i], o[dt]);
        }
    }
};
// fp32 elements: the fp32 MFMA, exact products at the rate that one pass over
// the keys needs.  Its k step 4 i + e takes dimension 16 i + 4 g + e.
template <>
struct StreamTile<kKvF32> {
    floatx4 k[2][4];
    floatx4 v[8];
    struct Query {
        floatx4 x[4];
        float down;
    };
    static __device__ __forceinline__ int q_dim(int i, int g) { return 16 * i + 4 * g; }
    template <class L>
    __device__ __forceinline__ void load_k(int hf, L&& load16)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) k[hf][i] = __builtin_bit_cast(floatx4, load16(64 * i));
    }
    template <class L>
    __device__ __forceinline__ void load_v(int hf, int r, L&& load16)
    {
        v[4 * hf + r] = __builtin_bit_cast(floatx4, load16());
    }
    static __device__ __forceinline__ void query(const floatx4 (&x)[4], Query& q)
    {
        q.down = 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) q.x[i] = x[i];
    }
    __device__ __forceinline__ floatx4 scores(int hf, const Query& q) const
    {
        floatx4 s = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[hf][i][e], q.x[i][e], s, 0, 0, 0);
        return s;
    }
    __device__ __forceinline__ void accumulate(const floatx4 (&p)[2], floatx4 (&o)[4]) const
    {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j][dt], p[j >> 2][j & 3], o[dt], 0, 0, 0);
    }
};

// Rows of one sequence and kv head: 16 (token, head) pairs, row i being token
// i / gqa, head i % gqa of the kv head.  One work item is an equal part of
// the unit's 32-key tiles, its four waves taking every fourth tile each, with
// no word to each other until the end: then the waves' states meet in LDS,
// and the items of one unit in the workspace, where the last to arrive adds
// them in order.  A wave holds one tile: its keys' registers take the next
// tile's as soon as the scores are formed, its values' after P.V.  The other
// waves of the SIMD cover the wait.
//
// Bound by memory: 64 sequences of 256 to 2047 F16 positions 19.0 us, 4.0 TB/s of
// their 76.6 MB, of which about 4 us are the launch, the table and the query on their
// way first and the parts' meeting last; 8 x 16384 F32 52.7 us, 5.1 TB/s, the rate of a
// copy.  Four waves to a workgroup and one kv head: eight and sixteen waves, two and
// four heads were slower or the same.  Parts are added by the last to arrive (a
// second launch for it costs 3 us and more); their states go past the L2 to device
// scope word by word, as a release and an acquire would write back and drop it (the
// merge by plain loads after an acquire: 28 us for 20.7).
// kSmall: pages of fewer than 16 positions: each lane looks up one row of the
// next tile, and the lanes that load it ask that lane (BF16, pages of 8, 2
// sequences of 15318: 17.0 us; 29 with ten look-ups by each lane as a tile's
// loads begin); else each half of a tile lies in one page, looked up by the wave.
struct StreamShared {
    floatx4 o[4][4][kWave];  // [wave][r][lane]
    float2 ml[4][kWave];
    int bad[16];
    int last;
};
template <int kType, bool kSmall, int kMaxSeq>
__device__ __forceinline__ void stream_item(const PagedAttentionParams& p, const PagedWork& work, const PagedSeqs<kMaxSeq>& b,
                                            const int item, StreamShared& sh)
{
    typedef typename Elem<kType>::T T;
    typedef StreamTile<kType> Tile;
    auto& s_o = sh.o;
    auto& s_ml = sh.ml;
    auto& s_bad = sh.bad;
    auto& s_last = sh.last;
    const int rank = rank_of(b, p.n_seq, item), seq = b.id(rank);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & (kWave - 1);
    const int pos = b.pos[seq], n_tok = b.tok[seq + 1] - b.tok[seq], len = pos + n_tok;
    const int n_unit = stream_units(n_tok * p.gqa, p.n_head_kv), local = item - b.first[rank];
    const int unit = local % n_unit, split = local / n_unit, n_split = (b.first[rank + 1] - b.first[rank]) / n_unit;
    const int kvh = unit % p.n_head_kv, row0 = 16 * (unit / p.n_head_kv), n_rows = min(16, n_tok * p.gqa - row0);
    const int n_tiles = (pos + (row0 + n_rows - 1) / p.gqa) / kStreamTile + 1;  // up to its last row's position
    const int c = lane & 15, g = lane >> 4;
    const int* const table = p.pool.table + (long long)seq * p.pool.table_stride;
    const int kv_dim = p.n_head_kv * kHeadDim, head_off = kvh * kHeadDim;

    // The row's query.  Rows past the last repeat it (their results are not stored).
    const int row = row0 + min(c, n_rows - 1), t = row / p.gqa, qpos = pos + t;
    const long long q_at = ((long long)(b.tok[seq] + t) * p.n_head + kvh * p.gqa + row - t * p.gqa) * kHeadDim;
    const float* const cs = reinterpret_cast<const float*>(p.rope + (long long)qpos * kPairs);
    if (threadIdx.x < 16) s_bad[threadIdx.x] = 0;

    // The tile's operands, and which of its keys are there: kSmall: bit 4 hf + r
    // of mask, the lane's key 4 g + r of half hf; else the halves' pages.
    Tile kv;
    struct There {
        unsigned mask;
        bool half[2];
    } there = {}, next = {};
    int page[2] = {};
    long long my_row = -1;  // kSmall: of the tile's key lane % 32, from the page in page[0]
    const auto look_up = [&](int tile) {
        if constexpr (kSmall) {
            page[0] = table[min(tile * kStreamTile + (lane & 31), len - 1) >> p.pool.page_shift];
        } else {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) page[hf] = page_at(table, min(tile * kStreamTile + 16 * hf, len - 1) >> p.pool.page_shift);
        }
    };
    const unsigned row_bytes = kv_dim * sizeof(T);
    const auto rows_of = [&](const void* pool, int tile, int hf) {  // of the page looked up last
        const int key = tile * kStreamTile + 16 * hf;
        const bool seen = key < len && (unsigned)page[hf] < (unsigned)p.pool.n_pages;
        next.half[hf] = seen;
        const long long at = (long long)page[hf] * p.pool.page_stride +
                             (long long)(key & ((1 << p.pool.page_shift) - 1)) * kv_dim + head_off;
        return rsrc_of({reinterpret_cast<const char*>(static_cast<const T*>(pool) + (seen ? at : 0)),
                        seen ? (min(16, len - key) - 1) * row_bytes + kHeadDim * (unsigned)sizeof(T) : 0});
    };
    const auto row_of_lane = [&](int from) {
        const unsigned lo = __shfl((int)(my_row & 0xffffffff), from), hi = __shfl((int)(my_row >> 32), from);
        return (long long)((unsigned long long)hi << 32 | lo);
    };
    const auto load_k = [&](int tile) {
        if constexpr (kSmall) {
            const int key = tile * kStreamTile + (lane & 31);
            my_row = key < len ? row_in(p.pool, page[0], key, kv_dim) : -1;
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if constexpr (kSmall) {
                const long long at = row_of_lane(16 * hf + c);
                const char* const from =
                    reinterpret_cast<const char*>(static_cast<const T*>(p.pool.k) + at + head_off) + 16 * g;
                kv.load_k(hf, [&](int o) { return at >= 0 ? *reinterpret_cast<const uintx4*>(from + o) : uintx4{}; });
            } else {
                const auto rs = rows_of(p.pool.k, tile, hf);
                kv.load_k(hf, [&](int o) {
                    return __builtin_amdgcn_raw_buffer_load_b128(rs, c * row_bytes + 16 * g + o, 0, 0);
                });
            }
        }
    };
    const auto load_v = [&](int tile) {
        typedef std::conditional_t<kType == kKvF32, uintx4, uintx2> V;
        next.mask = 0;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if constexpr (kSmall) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const long long at = row_of_lane(16 * hf + 4 * g + r);
                    const T* const from = static_cast<const T*>(p.pool.v) + at + head_off + 4 * c;
                    kv.load_v(hf, r, [&] { return at >= 0 ? *reinterpret_cast<const V*>(from) : V{}; });
                    next.mask |= at >= 0 ? 1u << (4 * hf + r) : 0u;
                }
            } else {
                const auto rs = rows_of(p.pool.v, tile, hf);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    kv.load_v(hf, r, [&] {
                        if constexpr (kType == kKvF32)
                            return __builtin_amdgcn_raw_buffer_load_b128(rs, (4 * g + r) * row_bytes + 16 * c, 0, 0);
                        else
                            return __builtin_amdgcn_raw_buffer_load_b64(rs, (4 * g + r) * row_bytes + 8 * c, 0, 0);
                    });
            }
        }
    };

    const int per = (n_tiles + n_split - 1) / n_split;  // the unit's tiles in equal parts
    int tile = split * per + wave;
    const int tile_end = min((split + 1) * per, n_tiles);
    if (tile < tile_end) {  // first the keys, on whose way the query is rotated
        look_up(tile);
        load_k(tile);
        load_v(tile);
        look_up(min(tile + 4, n_tiles - 1));
    }
    typename Tile::Query q;
    {
        floatx4 x[4];
        load_q(p.q + q_at, cs, [&](int i) { return Tile::q_dim(i, g); }, p.rotate, p.scale_log2, x);
        Tile::query(x, q);
    }
    floatx4 o[4] = {};
    float m_run = -INFINITY, l_run = 0.f;
    constexpr float kShift = Pieces<kType>::kShift;
    for (; tile < tile_end; tile += 4) {
        const bool more = tile + 4 < tile_end;
        there = next;
        floatx4 s[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) s[hf] = kv.scores(hf, q);
        if (more) load_k(tile + 4);  // into the registers just read
        const int key = tile * kStreamTile + 4 * g;
        if (kSmall || (tile + 1) * kStreamTile > pos + row0 / p.gqa + 1 || !there.half[0] || !there.half[1]) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool seen = kSmall ? (there.mask >> (4 * hf + r) & 1) != 0 : there.half[hf];
                    s[hf][r] = seen && key + 16 * hf + r <= qpos ? s[hf][r] : -INFINITY;
                }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_xor32(max_xor16(mx)) * q.down;
        // The running max moves only when a row's exceeds it by more than the
        // slack: most tiles do not rescale O.  A row that has seen nothing
        // keeps -inf; its probabilities are 0.
        if (__any(mx > m_run + kRescaleSlack)) {
            const float m_new = fmaxf(m_run, mx);
            const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
        }
        const float m_use = m_run == -INFINITY ? 0.f : m_run - kShift;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[hf][r] = __builtin_amdgcn_exp2f(fmaf(s[hf][r], q.down, -m_use));
                l_run += s[hf][r];
            }
        kv.accumulate(s, o);
        if (more) {
            load_v(tile + 4);
            look_up(min(tile + 8, n_tiles - 1));
        }
    }
    l_run = sum_xor32(sum_xor16(l_run));  // the lane groups summed different keys

    // The waves' states meet: wave w goes on with dimensions 16 g + 4 w .. + 3.
#pragma unroll
    for (int r = 0; r < 4; ++r) s_o[wave][r][lane] = floatx4{o[0][r], o[1][r], o[2][r], o[3][r]};
    s_ml[wave][lane] = make_float2(m_run, l_run);
    __syncthreads();
    const auto weight = [](float m, float m_new) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new); };
    const bool real = c < n_rows;
    floatx4 acc = {};
    m_run = fmaxf(fmaxf(s_ml[0][lane].x, s_ml[1][lane].x), fmaxf(s_ml[2][lane].x, s_ml[3][lane].x));
    l_run = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = weight(s_ml[w][lane].x, m_run);
        l_run = fmaf(s_ml[w][lane].y, f, l_run);
        acc += s_o[w][wave][lane] * f;
    }
    if (n_split > 1) {
        // Parts in order.  A CU's device-scope loads bring about 14 GB/s here: only
        // real rows' are made, and each max and sum is read by one lane, into the
        // LDS that the waves' states leave.
        const unsigned stride = n_unit * kStreamStateBytes;  // from part to part
        const auto rs = __builtin_amdgcn_make_buffer_rsrc(work.part + (long long)(b.first[rank] + unit) * (kStreamStateBytes / 4), 0,
                                                          n_split * stride, kRawBufferWord3);
        const unsigned o_at = 1024 * wave + 16 * lane, ml_at = 4096;
        if (real) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, acc), rs, o_at, split * stride, kDeviceScope);
            if (wave == 0 && g == 0)
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uintx2, make_float2(m_run, l_run)), rs, ml_at + 8 * c,
                                                      split * stride, kDeviceScope);
        }
        if (!last_to_arrive(work.counters + (long long)(b.first[rank] + unit) * kCounterStride, n_split, s_last)) return;
        float2* const s_part = reinterpret_cast<float2*>(s_o);  // [n_split][16]
        static_assert(sizeof(s_o) >= kMaxStreamParts * 16 * sizeof(float2), "the parts' max and sum");
        for (int i = threadIdx.x; i < 16 * n_split; i += 256)
            if ((i & 15) < n_rows)
                s_part[i] = __builtin_bit_cast(
                    float2, __builtin_amdgcn_raw_buffer_load_b64(rs, (i >> 4) * stride + ml_at + 8 * (i & 15), 0, kDeviceScope));
        __syncthreads();
        acc = floatx4{};
        if (real) {
            m_run = -INFINITY;
            for (int s = 0; s < n_split; ++s) m_run = fmaxf(m_run, s_part[16 * s + c].x);
            l_run = 0.f;
            constexpr int kBatch = 8;
#pragma unroll 1
            for (int s0 = 0; s0 < n_split; s0 += kBatch) {
                floatx4 x[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j)
                    if (s0 + j < n_split)
                        x[j] = __builtin_bit_cast(
                            floatx4, __builtin_amdgcn_raw_buffer_load_b128(rs, o_at, (s0 + j) * stride, kDeviceScope));
#pragma unroll
                for (int j = 0; j < kBatch; ++j)
                    if (s0 + j < n_split) {
                        const float2 ml = s_part[16 * (s0 + j) + c];
                        const float f = weight(ml.x, m_run);
                        l_run = fmaf(ml.y, f, l_run);
                        acc += x[j] * f;
                    }
            }
        }
    }
    acc *= l_run == 0.f ? 0.f : 1.f / l_run;
    if (real && (not_finite(l_run) || not_finite(acc[0]) || not_finite(acc[1]) || not_finite(acc[2]) || not_finite(acc[3])))
        s_bad[c] = 1;
    __syncthreads();  // the row as a whole: its query may lie where its output goes
    if (real && !s_bad[c]) stg4(p.out + q_at + 16 * g + 4 * wave, make_float4(acc[0], acc[1], acc[2], acc[3]));
    // Rows that met something infinite or NaN, seen or not, once more in plain fp32.
    for (int i = wave; i < n_rows; i += 4) {
        if (!s_bad[i]) continue;
        const int ti = (row0 + i) / p.gqa;
        const long long at = ((long long)(b.tok[seq] + ti) * p.n_head + kvh * p.gqa + row0 + i - ti * p.gqa) * kHeadDim;
        const float x = q_lane(p.q + at, p.rope + (long long)(pos + ti) * kPairs, p.rotate, p.scale_log2);
        p.out[at + lane] = plain_row<kType>(p.pool, table, kv_dim, head_off, pos + ti, x);
    }
}

// ---- chunks --------------------------------------------------------------------------

// 32 keys and values in LDS, as the 32x32 MFMA operands are read.  Score register
// r of lane (half, col) is key 16 (r / 8) + 8 half + r % 8 for query col, if row
// i of the K operand is key kperm(i) (bits 2 and 3 swapped); the same registers
// are the B operand (P^T) of P.V, whose k step s, element e of half is key 16 s +
// 8 half + e.
constexpr int kPlane = 32 * kHeadDim * 2;  // bytes of 32 rows of 16-bit elements

__device__ __forceinline__ int kperm(int i)
{
    return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1);
}

// 16-bit elements: K, then V, as rows of 128 bytes whose 16-byte chunks are
// permuted, chunk c of key i at place c ^ chunk_swap(i), so that both kinds of
// read take each bank once.  V's operand, eight keys of one dimension, is read
// through the LDS transpose: of the 16 lanes of a group, lane 4 j + m gives the
// address of dimensions 4 m .. of key j, and lane i receives dimension i of keys
// 0 .. 3.  O register r of dt is dimension 32 dt + 8 (r / 4) + 4 half + r % 4.
__device__ __forceinline__ int chunk_swap(int key)
{
    return key >> 1 & 7;
}

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t* lds_short4;

template <int kType>
struct ChunkTile {
    typedef Pieces<kType> P;
    typedef typename P::Frag Frag;
    static constexpr int kKeys = chunk_tile(kType);
    static constexpr int kSub = kKeys / 32;  // per tile
    static constexpr int kBytes = 2 * kPlane;
    static __device__ __forceinline__ int dim_of(int dt, int r, int half) { return 32 * dt + 8 * (r >> 2) + 4 * half + (r & 3); }
    // The byte of this lane's pieces: K at k step 0, V at k step 0, dt 0, keys 0 .. 3.
    static __device__ __forceinline__ int k_at(int lane)
    {
        const int key = kperm(lane & 31);
        return 128 * key + 16 * ((lane >> 5) ^ chunk_swap(key));
    }
    static __device__ __forceinline__ int v_at(int lane)
    {
        const int key = 8 * (lane >> 5) + (lane >> 2 & 3), chunk = 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
        return kPlane + 128 * key + 16 * (chunk ^ chunk_swap(key)) + 8 * (lane & 1);
    }
    static __device__ __forceinline__ floatx16 scores(const unsigned char* at, const Frag (&q)[4][P::kN], int k_at)
    {
        floatx16 s = {};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const Frag a = *reinterpret_cast<const Frag*>(at + (k_at ^ 32 * ks));
#pragma unroll
            for (int i = P::kN - 1; i >= 0; --i) s = P::mfma32(a, q[ks][i], s);
        }
        return s;
    }
    static __device__ __forceinline__ void accumulate(const floatx16& s, const unsigned char* at, int v_at, floatx16 (&o)[2])
    {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            floatx8 pv;
#pragma unroll
            for (int e = 0; e < 8; ++e) pv[e] = s[8 * ks + e];
            Frag f[P::kN];
            P::split(pv, f);
#pragma unroll
            for (int dt = 0; dt < 2; ++dt) {
                struct {
                    short4_t x[2];
                } w;
#pragma unroll
                for (int h = 0; h < 2; ++h)  // keys 4 h .. + 3: chunk_swap is 2 h further
                    w.x[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_short4)(at + (v_at ^ 32 * h ^ 64 * dt) + 512 * h + 2048 * ks));
                const Frag a = __builtin_bit_cast(Frag, w);
#pragma unroll
                for (int i = P::kN - 1; i >= 0; --i) o[dt] = P::mfma32(a, f[i], o[dt]);
            }
        }
    }
};

// F32 elements, split into three planes each when a tile arrives.
//   K plane: byte 512 c + 16 (kperm(i) ^ c) = dimensions 8 c .. + 7 of key i (c spreads
//     the eight pieces of a row that one load brings over the banks).
//   V plane: byte 2048 dt + 1024 s + 512 h + 16 i = keys 16 s + 8 h .. + 7 of dimension 2 i + dt.
template <>
struct ChunkTile<kKvF32> {
    typedef Pieces<kKvF32> P;
    typedef P::Frag Frag;
    static constexpr int kKeys = chunk_tile(kKvF32);
    static constexpr int kSub = kKeys / 32;
    static constexpr int kBytes = 6 * kPlane;
    static __device__ __forceinline__ int dim_of(int dt, int r, int half) { return 16 * (r >> 2) + 8 * half + 2 * (r & 3) + dt; }
    static __device__ __forceinline__ int k_at(int lane) { return lane; }
    static __device__ __forceinline__ int v_at(int lane) { return 3 * kPlane + 16 * lane; }
    // One thread's share of 32 keys: dimensions 8 kc .. of key kk, dimensions
    // 2 vi, 2 vi + 1 of keys 4 vg ..
    static __device__ __forceinline__ void store(const floatx8& k, const floatx2 (&v)[4], unsigned char* at, int kk, int kc,
                                                 int vi, int vg)
    {
        Frag f[3];
        P::split(k, f);
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<Frag*>(at + i * kPlane + 512 * kc + 16 * (kperm(kk) ^ kc)) = f[i];
        floatx8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v[e & 3][e >> 2];
        P::split(x, f);  // dt 0, then dt 1
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uintx4 w = __builtin_bit_cast(uintx4, f[i]);
            unsigned char* const va = at + (3 + i) * kPlane + 1024 * (vg >> 2) + 512 * (vg >> 1 & 1) + 16 * vi + 8 * (vg & 1);
            *reinterpret_cast<uintx2*>(va) = uintx2{w[0], w[1]};
            *reinterpret_cast<uintx2*>(va + 2048) = uintx2{w[2], w[3]};
        }
    }
    // The six products of pieces, small ones first.
    static __device__ __forceinline__ floatx16 products(const Frag (&a)[3], const Frag (&b)[3], floatx16 c)
    {
        c = P::mfma32(a[2], b[0], c);
        c = P::mfma32(a[1], b[1], c);
        c = P::mfma32(a[0], b[2], c);
        c = P::mfma32(a[1], b[0], c);
        c = P::mfma32(a[0], b[1], c);
        c = P::mfma32(a[0], b[0], c);
        return c;
    }
    static __device__ __forceinline__ floatx16 scores(const unsigned char* at, const Frag (&q)[4][3], int lane)
    {
        floatx16 s = {};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int c = 2 * ks + (lane >> 5);
            Frag a[3];
#pragma unroll
            for (int i = 0; i < 3; ++i)
                a[i] = *reinterpret_cast<const Frag*>(at + i * kPlane + 512 * c + 16 * ((lane & 31) ^ c));
            s = products(a, q[ks], s);
        }
        return s;
    }
    static __device__ __forceinline__ void accumulate(const floatx16& s, const unsigned char* at, int v_at, floatx16 (&o)[2])
    {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            floatx8 pv;
#pragma unroll
            for (int e = 0; e < 8; ++e) pv[e] = s[8 * ks + e];
            Frag f[3];
            P::split(pv, f);
#pragma unroll
            for (int dt = 0; dt < 2; ++dt) {
                Frag a[3];
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    a[i] = *reinterpret_cast<const Frag*>(at + i * kPlane + 2048 * dt + 1024 * ks + v_at);
                o[dt] = products(a, f, o[dt]);
            }
        }
    }
};

// Rows of one sequence and kv head, 128 of them: (token, head) pairs in order,
// 32 to a wave.  A work item is such a tile of rows over a range of key tiles;
// its waves share the tiles in LDS, double-buffered: the next one's rows are on
// their way while the waves compute, directly into LDS (16-bit elements of large
// pages) or in registers.
//
// Bound by issue: per 32 x 32 tile of F16 scores 16 matrix instructions of 32 cycles
// stand beside about 90 vector ones of 4 (the 16 exponentials of 16), and a SIMD
// overlaps the two in part only: in a chunk of 512 tokens after 8000 (82.7 us, 838
// TFLOP/s of F16 pieces; a large F16 matrix product reaches 1270) the matrix cores are
// busy 41 % of the cycles and the vector units 46 %.  F32, a prompt of 2048: 111 us, 926
// TFLOP/s of BF16 pieces, 44 % and 44 %.  128 rows to a workgroup: 3 of them fit a CU,
// and their 12 waves share 64 keys' reads.  The maximum is formed in few tiles only
// (below).
// kSmall: pages of fewer than 8 positions, whose rows are looked up by each
// lane; else the eight rows that a wave loads lie in one page.
template <int kType>
struct ChunkShared {
    alignas(16) unsigned char kv[2][ChunkTile<kType>::kSub][ChunkTile<kType>::kBytes];
    unsigned there[2][ChunkTile<kType>::kSub];  // bit i: key i of the 32 is there
    int last;
};
template <int kType, bool kSmall, int kMaxSeq>
__device__ __forceinline__ void chunk_item(const PagedAttentionParams& p, const PagedWork& work, const PagedSeqs<kMaxSeq>& b,
                                           const int item, ChunkShared<kType>& sh)
{
    typedef typename Elem<kType>::T T;
    typedef ChunkTile<kType> Tile;
    typedef Pieces<kType> P;
    typedef typename P::Frag Frag;
    constexpr int kKeys = Tile::kKeys, kSub = Tile::kSub;
    auto& s_kv = sh.kv;
    auto& s_there = sh.there;
    auto& s_last = sh.last;
    const int rank = rank_of(b, p.n_seq, item), seq = b.id(rank);
    const int pos = b.pos[seq], n_tok = b.tok[seq + 1] - b.tok[seq], len = pos + n_tok;
    const int n_rows = n_tok * p.gqa, n_rt = (n_rows + kChunkRows - 1) / kChunkRows;
    // Row tiles last first (they see most keys); the items of one tile next to
    // each other, so that with a multiple of 8 of them, or a divisor, the row
    // tiles that read one range of keys of one head run on the same XCDs.  Where
    // the tiles of a prompt see very different numbers of keys, those XCDs would
    // have very different numbers of items with any work (a 2048-token prompt in
    // two parts 66 us): there each row tile starts one place further.
    const int local = item - b.first[rank];
    const int n_combo = (b.first[rank + 1] - b.first[rank]) / n_rt;
    const int rt_rank = local / n_combo, rt = n_rt - 1 - rt_rank;
    const int combo = (local - rt_rank * n_combo + (pos < 4 * n_tok ? rt_rank : 0)) % n_combo;
    const int kvh = combo % p.n_head_kv, split = combo / p.n_head_kv;
    const int row0 = rt * kChunkRows, last_row = min(row0 + kChunkRows, n_rows) - 1;
    const int last_key = pos + last_row / p.gqa;
    const int n_tiles = last_key / kKeys + 1;
    const int n_split = (n_tiles + work.split_tiles - 1) / work.split_tiles;
    if (split >= n_split) return;  // the whole workgroup
    const int tile0 = split * work.split_tiles, tile_end = min(tile0 + work.split_tiles, n_tiles);

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & (kWave - 1);
    const int col = lane & 31, half = lane >> 5;
    const int* const table = p.pool.table + (long long)seq * p.pool.table_stride;
    const int kv_dim = p.n_head_kv * kHeadDim, head_off = kvh * kHeadDim;
    // This thread's piece of 32 keys.  F32: eight dimensions of key kk, and two of
    // four keys' values; else 16 bytes of key kk and of its values: chunk kc's place.
    constexpr bool kF32 = kType == kKvF32, kDirect = !kF32 && !kSmall;
    const int kk = threadIdx.x >> 3, kc = threadIdx.x & 7;
    const int vg = threadIdx.x >> 5, vi = threadIdx.x & 31;
    const int chunk = kF32 ? kc : kc ^ chunk_swap(kk);
    typedef std::conditional_t<kF32, floatx8, uintx4> KRaw;
    KRaw k_raw[kSub];
    uintx4 w_raw[kSub];       // values: 16-bit
    floatx2 v_raw[kSub][4];   // F32
    unsigned there[kSub];     // the wave's eight rows
    int page[kSub], v_page[kSub][4];  // kSmall: of the thread's key, and (F32) of its four keys' values
    const unsigned row_bytes = kv_dim * sizeof(T);
    const unsigned k_off = (kk & 7) * row_bytes + 8 * chunk * sizeof(T), v_off = 4 * (vg & 1) * row_bytes + 2 * vi * sizeof(T);
    const auto look_up = [&](int tile) {
        if constexpr (kSmall) {
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const int key = tile * kKeys + 32 * u;
                page[u] = table[min(key + kk, len - 1) >> p.pool.page_shift];
                if constexpr (kF32)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v_page[u][e] = table[min(key + 4 * vg + e, len - 1) >> p.pool.page_shift];
            }
        } else {
#pragma unroll
            for (int u = 0; u < kSub; ++u) page[u] = page_at(table, min(tile * kKeys + 32 * u + 8 * wave, len - 1) >> p.pool.page_shift);
        }
    };
    // Requests a tile's rows: into registers, or (kDirect) into LDS buffer buf.
    const auto load = [&](int tile, int buf) {
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            const int key = tile * kKeys + 32 * u + 8 * wave;  // the wave's first
            if constexpr (kSmall) {
                const auto at = [&](int j, int id) { return j < len ? row_in(p.pool, id, j, kv_dim) : -1; };
                const long long kr = at(tile * kKeys + 32 * u + kk, page[u]);
                const long long k_el = kr + head_off + 8 * chunk;
                k_raw[u] = kr >= 0 ? *reinterpret_cast<const KRaw*>(static_cast<const T*>(p.pool.k) + k_el) : KRaw{};
                if constexpr (kF32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const long long vr = at(tile * kKeys + 32 * u + 4 * vg + e, v_page[u][e]);
                        const T* const va = static_cast<const T*>(p.pool.v) + vr + head_off + 2 * vi;
                        v_raw[u][e] = vr >= 0 ? *reinterpret_cast<const floatx2*>(va) : floatx2{};
                    }
                } else {
                    w_raw[u] = kr >= 0 ? *reinterpret_cast<const uintx4*>(static_cast<const T*>(p.pool.v) + k_el) : uintx4{};
                }
                const unsigned long long m = __ballot(kr >= 0);  // eight lanes to a key
                there[u] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) there[u] |= (unsigned)(m >> (8 * i) & 1) << i;
            } else {
                const bool seen = key < len && (unsigned)page[u] < (unsigned)p.pool.n_pages;
                const long long at = seen ? (long long)page[u] * p.pool.page_stride +
                                                (long long)(key & ((1 << p.pool.page_shift) - 1)) * kv_dim + head_off
                                          : 0;
                const unsigned bytes = seen ? (min(8, len - key) - 1) * row_bytes + kHeadDim * (unsigned)sizeof(T) : 0;
                const auto rk = rsrc_of({reinterpret_cast<const char*>(static_cast<const T*>(p.pool.k) + at), bytes});
                const auto rv = rsrc_of({reinterpret_cast<const char*>(static_cast<const T*>(p.pool.v) + at), bytes});
                if constexpr (kF32) {
                    const floatx4 x = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off, 0, 0));
                    const floatx4 y = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 16, 0, 0));
                    k_raw[u] = floatx8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v_raw[u][e] = __builtin_bit_cast(floatx2, __builtin_amdgcn_raw_buffer_load_b64(rv, v_off + e * row_bytes, 0, 0));
                } else {  // lane l's 16 bytes land at byte 16 l of the wave's KiB
                    unsigned char* const to = s_kv[buf][u] + 1024 * wave;
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr)to, 16, k_off, 0, 0, 0);
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr)(to + kPlane), 16, k_off, 0, 0, 0);
                }
                there[u] = seen ? 255 : 0;
            }
            if constexpr (kDirect)
                if (lane == 0) reinterpret_cast<unsigned char*>(&s_there[buf][u])[wave] = (unsigned char)there[u];
        }
    };
    // Puts the tile requested last into LDS buffer buf, or waits until it is there.
    const auto store = [&](int buf) {
        if constexpr (kDirect) {
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0)
        } else {
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                if constexpr (kF32) {
                    Tile::store(k_raw[u], v_raw[u], s_kv[buf][u], kk, kc, vi, vg);
                } else {
                    unsigned char* const to = s_kv[buf][u] + 128 * kk + 16 * kc;
                    *reinterpret_cast<uintx4*>(to) = k_raw[u];
                    *reinterpret_cast<uintx4*>(to + kPlane) = w_raw[u];
                }
                if (lane == 0) reinterpret_cast<unsigned char*>(&s_there[buf][u])[wave] = (unsigned char)there[u];
            }
        }
    };
    const int k_at = Tile::k_at(lane), v_at = Tile::v_at(lane);

    look_up(tile0);
    load(tile0, 0);
    look_up(min(tile0 + 1, n_tiles - 1));

    // The row's query: lane (half, col) holds dimensions 16 s + 8 half .. + 7 for k step s.
    const int row = min(row0 + 32 * wave + col, n_rows - 1), t = row / p.gqa, qpos = pos + t;
    const long long q_at = ((long long)(b.tok[seq] + t) * p.n_head + kvh * p.gqa + row - t * p.gqa) * kHeadDim;
    const bool real = row0 + 32 * wave + col < n_rows;
    Frag q[4][P::kN];
    float down = 1.f;
    {
        const float* const cs = reinterpret_cast<const float*>(p.rope + (long long)qpos * kPairs);
        floatx4 x[8];
        load_q(p.q + q_at, cs, [&](int i) { return 16 * (i >> 1) + 8 * half + 4 * (i & 1); }, p.rotate, p.scale_log2, x);
        float up = 1.f;
        if constexpr (P::kScaled) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, __builtin_fabsf(x[i][e]));
            row_scale(max_xor32(top), up, down);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            floatx8 v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = x[2 * s + (e >> 2)][e & 3] * up;
            P::split(v, q[s]);
        }
    }
    // Keys that some row of the wave sees, and those that all of them do.
    const int wave_row = row0 + 32 * wave;
    const int wave_last = wave_row < n_rows ? pos + min(wave_row + 31, n_rows - 1) / p.gqa : -1;
    const int wave_first = pos + min(wave_row, n_rows - 1) / p.gqa;

    store(0);
    __syncthreads();
    floatx16 o[2] = {};
    // Probabilities are 2^(s + off), off = kShift - m_run.  m_run is a row's largest
    // score of some tile, -inf before its first key; it is looked for again when
    // the sum of a lane's 16 probabilities passes kLimit: most tiles form no
    // maximum and do not rescale O.  The scores are then formed once more (kAgain):
    // 16 registers fewer are live.  Not for F32, whose products are 3 to 6 times as
    // many.  F16: a sum of 2^14 keeps every probability below F16's largest, and one
    // at the maximum found last is 2^6; BF16 pieces need no such care, and 2^8 keeps
    // the sums of many tiles far from fp32's end.
    float m_run = -INFINITY, l_run = 0.f, off = 0.f;
    constexpr float kShift = P::kShift;
    constexpr bool kAgain = kType != kKvF32;
    constexpr float kLimit = kType == kKvF16 ? 16384.f : 256.f;
    for (int tile = tile0; tile < tile_end; ++tile) {
        const int buf = (tile - tile0) & 1;
        if (tile + 1 < tile_end) {
            load(tile + 1, buf ^ 1);  // read before the barrier that ended the last step
            look_up(min(tile + 2, n_tiles - 1));
        }
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            const int key = tile * kKeys + 32 * u;
            const unsigned seen = __builtin_amdgcn_readfirstlane(s_there[buf][u]);
            if (key > wave_last || seen == 0) continue;  // uniform over the wave
            const auto scores = [&] {
                floatx16 s = Tile::scores(s_kv[buf][u], q, k_at);
                if (key + 31 > wave_first || seen != ~0u) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = 16 * (r >> 3) + 8 * half + (r & 7);
                        s[r] = key + j <= qpos && (seen >> j & 1) ? s[r] : -INFINITY;
                    }
                }
                return s;
            };
            float sum;
            const auto weights = [&](floatx16 s) {
                sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = __builtin_amdgcn_exp2f(P::kScaled ? fmaf(s[r], down, off) : s[r] + off);
                    sum += s[r];
                }
                return s;
            };
            const floatx16 first = scores();
            floatx16 e = weights(first);
            if (__any(m_run == -INFINITY || sum > kLimit)) {
                floatx16 s;
                if constexpr (kAgain)
                    s = scores();
                else
                    s = first;
                float mx = s[0];
#pragma unroll
                for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
                const float m_new = fmaxf(m_run, max_xor32(mx) * down);
                // a row that has seen nothing yet keeps its offset of 0
                off = m_new == -INFINITY ? 0.f : kShift - m_new;
                const float alpha = m_run == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
                o[0] *= alpha;
                o[1] *= alpha;
                e = weights(s);
            }
            l_run += sum;
            // P.V before the SIMD's other waves' vector operations (F16, 4 x 1500 tokens
            // 103.9 -> 99.8 us, F32 512 after 8000 192 -> 185; raised for the scores too,
            // or for the vector operations instead, neither gained).
            __builtin_amdgcn_s_setprio(1);
            Tile::accumulate(e, s_kv[buf][u], v_at, o);
            __builtin_amdgcn_s_setprio(0);
        }
        if (tile + 1 < tile_end) store(buf ^ 1);
        __syncthreads();
    }
    l_run = sum_xor32(l_run);

    if (n_split > 1) {
        const auto part_of = [&](int s) {
            const long long i = b.first[rank] + (long long)(n_rt - 1 - rt) * n_combo + s * p.n_head_kv + kvh;
            return __builtin_amdgcn_make_buffer_rsrc(work.part + i * (kChunkStateBytes / 4) + wave * (64 * 34), 0, 64 * 34 * 4, kRawBufferWord3);
        };
        const auto mine = part_of(split);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            floatx4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[i >> 2][4 * (i & 3) + e];
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, x), mine, 1024 * i + 16 * lane, 0, kDeviceScope);
        }
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uintx2, make_float2(m_run, l_run)), mine, 8192 + 8 * lane, 0, kDeviceScope);
        if (!last_to_arrive(work.counters + (long long)(b.first[rank] + (n_rt - 1 - rt) * n_combo + kvh) * kCounterStride, n_split, s_last)) return;
        m_run = -INFINITY;
        l_run = 0.f;
        o[0] = o[1] = floatx16{};
        for (int i = 0; i < n_split; ++i) {
            const auto rs = part_of(i);
            floatx4 x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rs, 1024 * j + 16 * lane, 0, kDeviceScope));
            const float2 ml = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rs, 8192 + 8 * lane, 0, kDeviceScope));
            const float m_new = fmaxf(m_run, ml.x);
            const float fa = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
            const float fb = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m_new);
            m_run = m_new;
            l_run = l_run * fa + ml.y * fb;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                o[0][e] = o[0][e] * fa + x[e >> 2][e & 3] * fb;
                o[1][e] = o[1][e] * fa + x[4 + (e >> 2)][e & 3] * fb;
            }
        }
    }
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
    bool bad = not_finite(l_run);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) {
        o[dt] *= inv;
#pragma unroll
        for (int e = 0; e < 16; ++e) bad |= not_finite(o[dt][e]);
    }
    // The row as a whole: its query may lie where its output goes.
    const unsigned long long bads = __ballot(real && bad);
    const unsigned bad_rows = (unsigned)bads | (unsigned)(bads >> 32);
    if (real && !(bad_rows >> col & 1)) {
        float* const orow = p.out + q_at;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            if constexpr (kF32) {  // two dt side by side
                float* const to = orow + Tile::dim_of(0, 4 * a, half);
                stg4(to, make_float4(o[0][4 * a], o[1][4 * a], o[0][4 * a + 1], o[1][4 * a + 1]));
                stg4(to + 4, make_float4(o[0][4 * a + 2], o[1][4 * a + 2], o[0][4 * a + 3], o[1][4 * a + 3]));
            } else {
#pragma unroll
                for (int dt = 0; dt < 2; ++dt)
                    stg4(orow + Tile::dim_of(dt, 4 * a, half),
                         make_float4(o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]));
            }
        }
    }
    // Rows that met something infinite or NaN, seen or not, once more in plain fp32.
    for (unsigned rows = bad_rows; rows; rows &= rows - 1) {
        const int i = wave_row + __builtin_ctz(rows), ti = i / p.gqa;
        const long long at = ((long long)(b.tok[seq] + ti) * p.n_head + kvh * p.gqa + i - ti * p.gqa) * kHeadDim;
        const float x = q_lane(p.q + at, p.rope + (long long)(pos + ti) * kPairs, p.rotate, p.scale_log2);
        p.out[at + lane] = plain_row<kType>(p.pool, table, kv_dim, head_off, pos + ti, x);
    }
}

template <int kType, bool kSmall, int kMaxSeq>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4, 4))) void paged_stream_kernel(const PagedAttentionParams p,
                                                                                                     const PagedSeqs<kMaxSeq> b)
{
    __shared__ StreamShared sh;
    stream_item<kType, kSmall>(p, p.stream, b, blockIdx.x, sh);
}

template <int kType, bool kSmall, int kMaxSeq>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3, 3))) void paged_chunk_kernel(const PagedAttentionParams p,
                                                                                                    const PagedSeqs<kMaxSeq> b)
{
    __shared__ ChunkShared<kType> sh;
    chunk_item<kType, kSmall>(p, p.chunk, b, blockIdx.x, sh);
}

// Chunks and single tokens in one launch, the chunks' items first: either kind
// alone seldom fills the GPU to its end (BF16, 32 sequences of up to 2047 positions, one
// with 333 new tokens: 33.0 us in two launches, 26.3 in one).
template <int kType, int kMaxSeq>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3, 3))) void paged_mixed_kernel(
    const PagedAttentionParams p, const PagedSeqs<kMaxSeq> chunks, const PagedSeqs<kMaxSeq> streams)
{
    __shared__ union {
        ChunkShared<kType> c;
        StreamShared s;
    } sh;
    const int item = blockIdx.x;
    if (item < p.chunk.n_items)
        chunk_item<kType, false>(p, p.chunk, chunks, item, sh.c);
    else
        stream_item<kType, false>(p, p.stream, streams, item - p.chunk.n_items, sh.s);
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

hipError_t launch_paged_stream(const PagedAttentionParams& p, const PagedBatch& b, hipStream_t s)
{
    return with_type(p.pool.type, [&](auto type) {
        return with_batch(b, p.n_seq, [&](const auto& seqs) {
            constexpr int kMax = sizeof(seqs.pos) / sizeof(int);
            const dim3 grid(p.stream.n_items);
            if (p.pool.page_shift < 4)
                hipLaunchKernelGGL((paged_stream_kernel<type.value, true, kMax>), grid, dim3(256), 0, s, p, seqs);
            else
                hipLaunchKernelGGL((paged_stream_kernel<type.value, false, kMax>), grid, dim3(256), 0, s, p, seqs);
        });
    });
}

hipError_t launch_paged_chunk(const PagedAttentionParams& p, const PagedBatch& b, hipStream_t s)
{
    return with_type(p.pool.type, [&](auto type) {
        return with_batch(b, p.n_seq, [&](const auto& seqs) {
            constexpr int kMax = sizeof(seqs.pos) / sizeof(int);
            const dim3 grid(p.chunk.n_items);
            if (p.pool.page_shift < 3)
                hipLaunchKernelGGL((paged_chunk_kernel<type.value, true, kMax>), grid, dim3(256), 0, s, p, seqs);
            else
                hipLaunchKernelGGL((paged_chunk_kernel<type.value, false, kMax>), grid, dim3(256), 0, s, p, seqs);
        });
    });
}

hipError_t launch_paged_mixed(const PagedAttentionParams& p, const PagedBatch& chunks, const PagedBatch& streams, hipStream_t s)
{
    if (p.pool.page_shift < 4 || p.n_seq > kMaxMixedSeqs) return hipErrorInvalidValue;
    const dim3 grid(p.chunk.n_items + p.stream.n_items);
    return with_type(p.pool.type, [&](auto type) {
        if (p.n_seq <= 8)
            hipLaunchKernelGGL((paged_mixed_kernel<type.value, 8>), grid, dim3(256), 0, s, p, fewer<8>(chunks, p.n_seq),
                               fewer<8>(streams, p.n_seq));
        else
            hipLaunchKernelGGL((paged_mixed_kernel<type.value, kMaxMixedSeqs>), grid, dim3(256), 0, s, p,
                               fewer<kMaxMixedSeqs>(chunks, p.n_seq), fewer<kMaxMixedSeqs>(streams, p.n_seq));
        return hipGetLastError();
    });
}

}  // namespace tla
