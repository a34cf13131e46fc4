// Device parts that the paged caches' kernels share, whatever their codes: rotation
// pairs, fp16 pairs, parts of a tile passed between workgroups and merged.
#pragma once

#include "../../include/jev.h"
#include "jev_dev.h"

namespace jev {

template <typename T>
T *layer_of(const Pages &p, T *base, int layer, size_t per_block) { return base + layer * p.n_blocks() * per_block; }

// The plan on the device may be a replayed graph's, and larger than the one that
// this call's grid and its caller's arrays were made for.  Then the call does
// nothing, and the plan's status says so.
template <typename View>
__device__ __forceinline__ bool outgrown(const View &p, const PagesPlanHead &h)
{
    if (h.n_tokens <= p.n_tokens && h.n_requests <= p.n_requests && (p.wide || h.n_wide == 0)) return false;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.head->status = JEV_ESTATE;
    return true;
}

__device__ __forceinline__ int div_up(int a, int b) { return (a + b - 1) / b; }

// The eight (HD 128) or four (HD 64) elements of a head's row that thread j of
// its sixteen holds: NP rotation pairs (p, i.e. their two elements), consecutive
// pairs; past the rotated part of the head a pair is two neighbours.
template <int HD>
struct RowPairs {
    static constexpr int NP = HD / 32;
    int e0[NP], e1[NP];
    template <typename View>
    __device__ __forceinline__ RowPairs(const View &p, int j)
    {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int q = NP * j + i;
            const bool half = p.rope_half && q < p.half;
            e0[i] = half ? q : 2 * q;
            e1[i] = half ? q + p.half : 2 * q + 1;
        }
    }
};

template <int HD, bool VEC>
__device__ __forceinline__ void load_pairs(const RowPairs<HD> &e, const float *x, float2 (&v)[HD / 32])
{
    constexpr int NP = HD / 32;
    if constexpr (VEC) {
        // the pairs are either neighbours throughout or two runs of NP floats
        float r[2 * NP];
        const bool split = e.e1[0] != e.e0[0] + 1;
        const float *b = x + (split ? e.e1[0] : e.e0[0] + NP);
        if constexpr (NP == 4) {
            const float4 lo = *(const float4 *)(x + e.e0[0]), hi = *(const float4 *)b;
            r[0] = lo.x, r[1] = lo.y, r[2] = lo.z, r[3] = lo.w, r[4] = hi.x, r[5] = hi.y, r[6] = hi.z, r[7] = hi.w;
        } else {
            const float2 lo = *(const float2 *)(x + e.e0[0]), hi = *(const float2 *)b;
            r[0] = lo.x, r[1] = lo.y, r[2] = hi.x, r[3] = hi.y;
        }
#pragma unroll
        for (int i = 0; i < NP; i++) v[i] = split ? make_float2(r[i], r[NP + i]) : make_float2(r[2 * i], r[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < NP; i++) v[i] = make_float2(x[e.e0[i]], x[e.e1[i]]);
    }
}

template <int HD, bool VEC>
__device__ __forceinline__ void store_pairs(const RowPairs<HD> &e, float *x, const float2 (&v)[HD / 32])
{
    constexpr int NP = HD / 32;
    if constexpr (VEC) {
        float r[2 * NP];
        const bool split = e.e1[0] != e.e0[0] + 1;
#pragma unroll
        for (int i = 0; i < 2 * NP; i++) {
            const float near = i & 1 ? v[i / 2].y : v[i / 2].x, apart = i < NP ? v[i % NP].x : v[i % NP].y;
            r[i] = split ? apart : near;
        }
        float *b = x + (split ? e.e1[0] : e.e0[0] + NP);
        if constexpr (NP == 4) {
            *(float4 *)(x + e.e0[0]) = make_float4(r[0], r[1], r[2], r[3]);
            *(float4 *)b = make_float4(r[4], r[5], r[6], r[7]);
        } else {
            *(float2 *)(x + e.e0[0]) = make_float2(r[0], r[1]);
            *(float2 *)b = make_float2(r[2], r[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            x[e.e0[i]] = v[i].x;
            x[e.e1[i]] = v[i].y;
        }
    }
}

// split2_rtz with the remainders as mixed-precision multiply-adds: four
// instructions for the two values instead of six (the compiler converts first).
__device__ __forceinline__ void split2_mix(float x0, float x1, uint32_t &hi, uint32_t &lo)
{
    float r0, r1;
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(hi), "v"(x1));
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r0, r1));
}


// Outputs held times 2^(9 - e), weights relative to 2^m and their sum l: a row's mean of
// its values is (o * f1) * f2.  In two steps, 2^(e - 9 - m) itself may be outside fp32's
// range.  Means are also what parts of a row pass on: weighted sums of values that fp32
// holds may be past it.  A part that sees no key (l = 0) has a mean of zeros; a row that
// has no weight in any part, all its scores past fp32's range, is NaN.
struct MeanScale {
    float f1, f2;
    __device__ __forceinline__ MeanScale(float e, float m, float l)
        : f1(e == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(0.5f * (e - 9.f - m))), f2(l == 0.f ? 0.f : f1 / l) {}
};

// Partial results pass between workgroups inside a launch, which may run on
// different dies with an L2 each: they are stored and read as agent-scope atomics
// (written through, and read past, caches that other dies do not see), two floats
// at a time.  A fence would write back the whole L2 of the die for every part
// (measured: 64 rows of up to 12000 keys 1090 us instead of 104, a launch at a time).
__device__ __forceinline__ void store_shared(float *p, float x, float y)
{
    __hip_atomic_store((uint64_t *)p, (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_shared(const float *p)
{
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// True in the workgroup that is the last of `parts` to come here; its ticket is
// left at zero for the next call.  Every thread's store_shared()s are complete
// (acknowledged by memory) before its workgroup's arrival is counted, so the last
// one's load_shared()s, issued after it has read the count, find them.
__device__ __forceinline__ bool arrives_last(int32_t *ticket, int parts, int &shared)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const int before = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        shared = before == parts - 1;
        if (shared) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return shared;
}

// One row's parts (part k at at(k): HD means, maximum, sum) merged in their order by
// sixteen threads.
template <int HD, typename At>
__device__ __forceinline__ void merge_parts(At at, int n_parts, float *dst, int j)
{
    constexpr int N = HD / 16;
    float m = -INFINITY, l = 0.f;
    auto join = [&](float mk, float lk) {
        const float mn = fmaxf(m, mk), mu = mn == -INFINITY ? 0.f : mn;
        l = l * exp2f(m - mu) + lk * exp2f(mk - mu);
        m = mn;
    };
    for (int k = j; k < n_parts; k += 16) {
        const float2 ml = load_shared(at(k) + HD);
        join(ml.x, ml.y);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) join(__shfl_xor(m, o, 64), __shfl_xor(l, o, 64));
    if (m == -INFINITY) m = 0.f;
    const float inv = 1.f / l;
    float x[N] = {};
#pragma unroll 4
    for (int k = 0; k < n_parts; k++) {
        const float *src = at(k);
        const float2 ml = load_shared(src + HD);
        const float f = ml.y * exp2f(ml.x - m) * inv;
#pragma unroll
        for (int i = 0; i < N; i += 2) { // (a row's sixteen threads side by side)
            const float2 y = load_shared(src + 16 * i + 2 * j);
            x[i] += y.x * f;
            x[i + 1] += y.y * f;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        dst[16 * i + 2 * j] = x[i];
        dst[16 * i + 2 * j + 1] = x[i + 1];
    }
}

typedef float floatx16 __attribute__((ext_vector_type(16)));

// A wide tile's end: its outputs, or its part and, from its last part, theirs.
template <int HD, typename View, typename Lds>
__device__ __forceinline__ void wide_result(const View &p, Lds &lds, int item, int h,
                                            const floatx16 (&o)[HD / 32], const MeanScale &mean, float m, float l)
{
    constexpr int ND = HD / 32, LD = HD + 4, kMost = 8;
    // read again: nothing of them takes registers during the products
    asm volatile("" : "+s"(item));
    const PagesItem it = p.wide_item[item], &r = it;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5, n = lane & 31, wrow = 32 * (tid >> 6) + n;
    const int n_rows = it.row1 - it.row0; // of the tile
    auto out_of = [&](int c) { // the tile's row c
        const int row = it.row0 + c;
        return p.out + ((size_t)(r.start + row / p.group) * p.n_heads + h * p.group + row % p.group) * HD;
    };
    if (it.part < 0) {
        if (wrow >= n_rows) return;
        float *dst = out_of(wrow);
        const float f2 = mean.f1 / l;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) dst[32 * d + 8 * (i >> 2) + 4 * hh + (i & 3)] = o[d][i] * mean.f1 * f2;
        return;
    }
    // through LDS, where the fragments were: whole runs of a row to a store
    float *rows = lds.rows, *mine = rows + wrow * LD;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *(floatx4 *)(mine + 32 * d + 8 * i + 4 * hh) =
                floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * mean.f1 * mean.f2;
    if (hh == 0) *(float2 *)(mine + HD) = make_float2(m, l);
    __syncthreads();
    float *part = p.wide_part + ((size_t)it.part * p.n_kv + h) * kPagesWideRows * LD;
    for (int i = 2 * tid; i < n_rows * LD; i += 512)
        if (i % LD < HD + 2) store_shared(part + i, rows[i], rows[i + 1]);
    const int part0 = it.part - (it.part - r.part0) % r.n_parts; // of this tile
    if (!arrives_last(p.wide_tickets + (size_t)part0 * p.n_kv + h, r.n_parts, lds.last)) return;
    if (r.n_parts > kMost) {
        for (int c = tid >> 4; c < n_rows; c += 16)
            merge_parts<HD>([&](int k) { return p.wide_part + (((size_t)(part0 + k) * p.n_kv + h) * kPagesWideRows + c) * LD; }, r.n_parts,
                            out_of(c), tid & 15);
        return;
    }
    // few parts: every row's factors first, then no sum waits for them
    const float *at = p.wide_part + ((size_t)part0 * p.n_kv + h) * kPagesWideRows * LD;
    const size_t step = (size_t)p.n_kv * kPagesWideRows * LD;
    if (tid < n_rows) {
        float2 ml[kMost];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < kMost; k++)
            if (k < r.n_parts) ml[k] = load_shared(at + k * step + tid * LD + HD);
#pragma unroll
        for (int k = 0; k < kMost; k++)
            if (k < r.n_parts) top = fmaxf(top, ml[k].x);
        if (top == -INFINITY) top = 0.f;
#pragma unroll
        for (int k = 0; k < kMost; k++)
            if (k < r.n_parts) sum += ml[k].y * exp2f(ml[k].x - top);
#pragma unroll
        for (int k = 0; k < kMost; k++)
            if (k < r.n_parts) lds.factor[k][tid] = ml[k].y * exp2f(ml[k].x - top) / sum;
    }
    __syncthreads();
    constexpr int TH = HD / 2, RT = 256 / TH; // threads of a row, rows at once
    const int j = 2 * (tid % TH);
#pragma unroll 4
    for (int c = tid / TH; c < n_rows; c += RT) {
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int k = 0; k < kMost; k++)
            if (k < r.n_parts) {
                const float2 v = load_shared(at + k * step + c * LD + j);
                x += v.x * lds.factor[k][c];
                y += v.y * lds.factor[k][c];
            }
        float *dst = out_of(c) + j;
        dst[0] = x;
        dst[1] = y;
    }
}

} // namespace jev
