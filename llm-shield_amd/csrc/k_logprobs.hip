// Log probabilities of rows of logits: of given tokens, of the most probable ones, and a
// row's entropy, from one pass over it.
#include <algorithm>
#include <cmath>

#include "jev_pages_dev.h"

namespace jev {

namespace {

constexpr int kTile = 32;                           // logits a lane holds at a time
constexpr int kKeys = kLogprobsTop * (kTile + 1);   // the most that a wave's list can hold between two cuts

struct LogprobsView {
    const float *logits;
    int64_t ld;
    const int32_t *given;
    float *logp, *entropy, *top_logp;
    int32_t *top;
    LogprobsPart *part;
    int32_t *tickets;
    int vocab, n_given, n_top, parts, chunk; // a row's parts, of `chunk` logits each
    float temperature, c;                    // c = log2(e) / temperature
};

typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));

// A logit's place among the others: NaN first, then by value (+0 above -0), the lower index
// first.  Distinct logits have distinct keys.
__device__ __forceinline__ uint64_t key_of(float x, int index)
{
    const uint32_t b = __float_as_uint(x), up = x != x ? ~0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return (uint64_t)up << 32 | (uint32_t)~index;
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }
// The value that a key stands for, as a bound: NaN for NaN.
__device__ __forceinline__ float value_of(uint64_t key)
{
    const uint32_t up = (uint32_t)(key >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

__device__ __forceinline__ uint64_t lane_key(uint64_t key, int lane)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, lane);
}

// What the wave's lanes have put into LDS so far is there.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wave's largest keys: `n` of them in LDS, more than k only between a push and its cut.
// Every key that is not there is below `least`, once there are k.
struct Best {
    uint64_t *keys, least = 0;
    float bound = -INFINITY; // value_of(least): what is below it need not be looked at
    int n = 0, k;
    __device__ __forceinline__ Best(uint64_t *lds, int k) : keys(lds), k(k) {}

    __device__ __forceinline__ void push(bool mine, uint64_t key)
    {
        const uint64_t m = __ballot(mine);
        if (mine) keys[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u))] = key;
        n += __popcll(m);
    }
    // Lanes' largest keys `top` are of k lanes or more: the k-th of them bounds the k-th of all.
    __device__ __forceinline__ void raise(uint64_t top)
    {
        int above = 0;
        for (int i = 0; i < 64; i++) above += lane_key(top, i) > top ? 1 : 0;
        const uint64_t at = __ballot(above == k - 1);
        if (at == 0) return; // fewer lanes have one
        const uint64_t t = lane_key(top, __ffsll((unsigned long long)at) - 1);
        if (t <= least) return;
        least = t;
        bound = value_of(t);
    }
    // Cuts the list to its k largest (not in order).
    __device__ __forceinline__ void cut()
    {
        if (n <= k) return;
        const int lane = threadIdx.x & 63;
        wave_sync();
        uint64_t t = 0; // the k-th largest, bit by bit: the greatest t with k keys at or above it
        for (int bit = 63; bit >= 0; bit--) {
            const uint64_t trial = t | 1ull << bit;
            int at = 0;
            for (int i = 0; i < n; i += 64) at += __popcll(__ballot(i + lane < n && keys[i + lane] >= trial));
            if (at >= k) t = trial;
        }
        const int all = n;
        n = 0;
        for (int i = 0; i < all; i += 64) { // (to places at or before those that are read)
            const uint64_t key = i + lane < all ? keys[i + lane] : 0;
            wave_sync();
            push(i + lane < all && key >= t, key);
            wave_sync();
        }
        least = t;
        bound = value_of(t);
    }
    // The list, at most 64 long, in order.
    __device__ __forceinline__ void sort()
    {
        const int lane = threadIdx.x & 63;
        wave_sync();
        const uint64_t key = lane < n ? keys[lane] : 0;
        int above = 0;
        for (int i = 0; i < n; i++) above += keys[i] > key ? 1 : 0;
        wave_sync();
        if (lane < n) keys[above] = key;
        wave_sync();
    }
};

// A softmax's statistics: the largest logit m, s = sum exp2((x - m) c) over all logits but
// one that is m (next to a certain token everything lies in them), and t = the same sum
// times (x - m) c.  What is added up over a row is in 64 bits.
struct Stats {
    float m;
    double s, t;
    static __device__ __forceinline__ Stats none() { return {-INFINITY, 0.0, 0.0}; }
    // to a larger maximum, which is not among what has been added up; without a logit above
    // -inf the sums are zero (or NaN)
    __device__ __forceinline__ void rescale(float to, float c)
    {
        const float d = fmaxf((m - to) * c, -1e4f);
        const double f = (double)__builtin_amdgcn_exp2f(d), all = s + (m > -INFINITY ? 1.0 : 0.0);
        t = f * (t + (double)d * all);
        s = f * all;
        m = to;
    }
    __device__ __forceinline__ void join(Stats o, float c)
    {
        const float to = fmaxf(m, o.m);
        if (m == o.m) s += to > -INFINITY ? 1.0 : 0.0;
        else if (m != to) rescale(to, c);
        else o.rescale(to, c);
        s += o.s;
        t += o.t;
    }
};
__device__ __forceinline__ Stats across(const Stats &a, int o)
{
    Stats b;
    b.m = __shfl_xor(a.m, o, 64);
    b.s = __shfl_xor(a.s, o, 64);
    b.t = __shfl_xor(a.t, o, 64);
    return b;
}

__device__ __forceinline__ void store_shared64(void *p, uint64_t x)
{
    __hip_atomic_store((uint64_t *)p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t load_shared64(const void *p)
{
    return __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

} // namespace

// A workgroup per row and part of it.  A lane holds 32 logits at a time: their maximum
// (which moves the running sums only where it rises), the exponentials, and, where one of
// them passes the wave's k-th largest so far, their places in its list.  A wave's list is
// its own, so nothing waits inside the pass.  The last part of a row to arrive merges all
// of them.  Bounded by HBM: each logit is read once.
template <bool TOP>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobsView p)
{
    __shared__ uint64_t keys[4][TOP ? kKeys : 1];
    __shared__ Stats stats[4];
    __shared__ int count[4], last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const float *x0 = p.logits + row * p.ld;

    Stats st = Stats::none();
    Best best(keys[wave], p.n_top);
    const int w0 = part * p.chunk + wave * (p.chunk / 4), w1 = min(p.vocab, w0 + p.chunk / 4);
    for (int base = w0; base < w1; base += 64 * kTile) {
        float x[kTile];
        if (base + 64 * kTile <= w1) {
#pragma unroll
            for (int i = 0; i < kTile / 4; i++) *(floatx4u *)&x[4 * i] = *(const floatx4u *)(x0 + base + 256 * i + 4 * lane);
        } else { // places past the end: -inf, and in no list
#pragma unroll
            for (int i = 0; i < kTile; i++) {
                const int at = base + 256 * (i >> 2) + 4 * lane + (i & 3);
                x[i] = at < w1 ? x0[at] : -INFINITY;
            }
        }
        float m = x[0];
#pragma unroll
        for (int i = 1; i < kTile; i++) m = fmaxf(m, x[i]); // (NaN only where all are)
        double own = 0.0; // a new maximum is counted among the logits and is not in the sum
        if (m > st.m) {
            st.rescale(m, p.c);
            own = 1.0;
        }
        const float mu = st.m == -INFINITY ? 0.f : st.m;
        float s = 0.f, t = 0.f;
        int ones = 0;
#pragma unroll
        for (int i = 0; i < kTile; i++) {
            const float d = (x[i] - mu) * p.c, e = __builtin_amdgcn_exp2f(d);
            const bool one = x[i] == mu;
            ones += one ? 1 : 0;
            s += one ? 0.f : e;
            t = fmaf(e, fmaxf(d, -1e4f), t); // (0 times -inf is 0 here)
        }
        st.s += (double)s + ((double)ones - own);
        st.t += (double)t;
        if constexpr (TOP) {
            // a lane is looked at where its largest is not below the bound, or it has a NaN
            const bool look = !(m < best.bound) || s != s;
            const uint64_t lanes = __ballot(look);
            if (lanes) {
                auto key = [&](int i) {
                    const int at = base + 256 * (i >> 2) + 4 * lane + (i & 3);
                    return look && at < w1 ? key_of(x[i], at) : 0;
                };
                if (__popcll(lanes) > p.n_top) {
                    uint64_t top = 0;
#pragma unroll
                    for (int i = 0; i < kTile; i++) {
                        const uint64_t k = key(i);
                        if (k > top) top = k;
                    }
                    best.raise(top);
                }
#pragma unroll
                for (int i = 0; i < kTile; i++) {
                    if (!__any(look && !(x[i] < best.bound))) continue;
                    const uint64_t k = key(i);
                    best.push(k != 0 && k >= best.least, k);
                }
                best.cut();
            }
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) st.join(across(st, o), p.c);
    if (lane == 0) {
        stats[wave] = st;
        count[wave] = best.n;
    }
    __syncthreads();

    // the workgroup's, in its first wave
    Best all(keys[0], p.n_top);
    if (wave == 0) {
        st = stats[0];
        for (int w = 1; w < 4; w++) st.join(stats[w], p.c);
        if constexpr (TOP) {
            all.n = count[0];
            for (int w = 1; w < 4; w++) {
                const int n = count[w];
                const uint64_t key = lane < n ? keys[w][lane] : 0; // (at most k, which is at most 32)
                all.push(lane < n, key);
            }
            all.cut();
            all.sort();
        }
    }
    if (p.parts > 1) {
        LogprobsPart *mine = p.part + blockIdx.x;
        if (wave == 0) {
            if (lane == 0) {
                store_shared64(&mine->s, __builtin_bit_cast(uint64_t, st.s));
                store_shared64(&mine->t, __builtin_bit_cast(uint64_t, st.t));
                store_shared64(&mine->m, (uint64_t)__float_as_uint(st.m));
            }
            if constexpr (TOP)
                if (lane < p.n_top) store_shared64(&mine->key[lane], lane < all.n ? keys[0][lane] : 0);
        }
        if (!arrives_last(p.tickets + row, p.parts, last)) return;
        if (wave == 0) { // a lane to a part
            const LogprobsPart *from = p.part + (size_t)row * p.parts + min(lane, p.parts - 1);
            st = Stats::none();
            if (lane < p.parts) {
                st.m = __uint_as_float((uint32_t)load_shared64(&from->m));
                st.s = __builtin_bit_cast(double, load_shared64(&from->s));
                st.t = __builtin_bit_cast(double, load_shared64(&from->t));
            }
            if constexpr (TOP) {
                all = Best(keys[0], p.n_top);
                const uint64_t top = lane < p.parts ? load_shared64(&from->key[0]) : 0;
                if (p.parts > p.n_top) all.raise(top);
                for (int i = 0; i < p.n_top; i++) {
                    const uint64_t key = i == 0 ? top : lane < p.parts ? load_shared64(&from->key[i]) : 0;
                    const bool take = key != 0 && key >= all.least;
                    if (!__any(take)) break; // lists are in order
                    all.push(take, key);
                }
                all.cut();
                all.sort();
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) st.join(across(st, o), p.c);
        }
    }
    if (wave == 0 && lane == 0) stats[0] = st;
    __syncthreads();

    // logp(x) = (x - m) / T - log(1 + s);  H = log(1 + s) - (sum e (x - m) / T) / (1 + s)
    const Stats r = stats[0];
    const double log_s = fabsf(r.m) < INFINITY ? log1p(r.s) : NAN;
    auto logp = [&](float x) { return (float)(((double)x - (double)r.m) / (double)p.temperature - log_s); };
    for (int i = tid; i < p.n_given; i += 256) {
        const int id = p.given[(size_t)row * p.n_given + i];
        p.logp[(size_t)row * p.n_given + i] = id >= 0 && id < p.vocab ? logp(x0[id]) : NAN;
    }
    if (tid == 0 && p.entropy) p.entropy[row] = (float)(log_s - 0.69314718055994530942 * r.t / (1.0 + r.s));
    if constexpr (TOP)
        if (tid < p.n_top) {
            const int id = index_of(keys[0][tid]);
            if (p.top) p.top[(size_t)row * p.n_top + tid] = id;
            if (p.top_logp) p.top_logp[(size_t)row * p.n_top + tid] = logp(x0[id]);
        }
}

// Parts of a row: enough workgroups for the whole GPU, of no less than 4096 logits each, a
// lane of the merging wave to a part.
int logprobs_parts(int rows, int vocab)
{
    return std::max(1, std::min({kLogprobsParts / std::max(rows, 1), (vocab + 4095) / 4096, 64}));
}

hipError_t launch_logprobs(const LogprobsArgs &a, hipStream_t s)
{
    if (a.rows <= 0) return hipSuccess;
    const int parts = logprobs_parts(a.rows, a.vocab);
    const int chunk = ((a.vocab + parts - 1) / parts + 1023) & ~1023;
    const LogprobsView v = {a.logits, a.ld, a.given, a.logp, a.entropy, a.top_logp, a.top, a.part, a.tickets, a.vocab, a.n_given, a.n_top,
                            parts, chunk, a.temperature, (float)(1.4426950408889634074 / (double)a.temperature)};
    const dim3 grid((unsigned)a.rows * parts);
    if (a.n_top > 0) hipLaunchKernelGGL(logprobs_kernel<true>, grid, dim3(256), 0, s, v);
    else hipLaunchKernelGGL(logprobs_kernel<false>, grid, dim3(256), 0, s, v);
    return hipGetLastError();
}

} // namespace jev
