// Log probabilities of rows of logits: of given tokens, of the most probable ones, and a
// row's entropy, from one pass over it.
#include <algorithm>
#include <cmath>

#include "jev_pages_dev.h"

namespace jev {

namespace {

constexpr int kTile = 32;                           // logits a lane holds at a time
constexpr int kRoom = kLogprobsTop * (kTile + 1);   // the most that a wave's list can hold between two cuts
constexpr int kKeys = kRoom + 8;                    // and zeros behind them

struct LogprobsView {
    const float *logits;
    int64_t ld;
    const int32_t *given;
    float *logp, *entropy, *top_logp;
    int32_t *top;
    LogprobsPart *part;
    int32_t *tickets;
    int vocab, n_given, n_top, parts, chunk; // a row's parts, of `chunk` logits each
    float c;                                 // log2(e) / temperature
    double inverse;                          // 1 / temperature
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

// x of the lane that is `TO - 0x120` before in its row of sixteen, round it.
template <int TO>
__device__ __forceinline__ int turned(int x) { return __builtin_amdgcn_update_dpp(x, x, TO, 0xf, 0xf, false); }
// f over the wave's lanes: within their rows, then between these.
template <typename T, typename F>
__device__ __forceinline__ T over_wave(T x, F f)
{
    constexpr int W = sizeof(T) / 4;
    struct Words {
        int w[W];
    };
    auto moved = [](T y, auto move) {
        Words a = __builtin_bit_cast(Words, y);
#pragma unroll
        for (int i = 0; i < W; i++) a.w[i] = move(a.w[i]);
        return __builtin_bit_cast(T, a);
    };
    x = f(x, moved(x, [](int b) { return turned<0x121>(b); }));
    x = f(x, moved(x, [](int b) { return turned<0x122>(b); }));
    x = f(x, moved(x, [](int b) { return turned<0x124>(b); }));
    x = f(x, moved(x, [](int b) { return turned<0x128>(b); }));
    auto of = [&](int lane) { return moved(x, [&](int b) { return __builtin_amdgcn_readlane(b, lane); }); };
    return f(f(of(0), of(16)), f(of(32), of(48)));
}
// What the wave's lanes have put into LDS so far is there.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// How many of n numbers in LDS, with eight zeros behind them, are larger than x.
template <typename T>
__device__ __forceinline__ int count_above(const T *from, int n, T x)
{
    int above = 0;
#pragma unroll 1 // (their registers)
    for (int i = 0; i < n; i += 8) {
        T y[8];
#pragma unroll
        for (int u = 0; u < 8; u++) y[u] = from[i + u];
#pragma unroll
        for (int u = 0; u < 8; u++) above += y[u] > x ? 1 : 0;
    }
    return above;
}

// A number that `rank` of the lanes' numbers, or more, are not below; 0 where fewer are more
// than 0.  The rank-th largest itself or (few wanted, some equal) a larger one; past three its
// upper half.
__device__ __forceinline__ uint32_t rank_of(uint32_t up, int rank)
{
    auto larger = [](uint32_t a, uint32_t b) { return max(a, b); };
    if (rank <= 3) { // one after the other: 300 cycles each
        uint32_t most = 0;
        for (int n = 0; n < rank;) {
            most = over_wave(up, larger);
            if (most == 0) return 0;
            n += __popcll(__ballot(up == most));
            up = up == most ? 0 : up;
        }
        return most;
    }
    uint32_t t = 0;
#pragma unroll 4
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t trial = t | 1u << bit;
        if (__popcll(__ballot(up >= trial)) >= rank) t = trial;
    }
    return t;
}

// A wave's largest keys: `n` of them in LDS, in order except between a push and its cut,
// when there may be more than k.  Every key that is not there is below `least`, once
// there are k.
struct Best {
    uint64_t *keys, least = 0;
    float bound = -INFINITY; // the value of `least`: what is below it need not be looked at
    int n = 0, k;
    __device__ __forceinline__ Best(uint64_t *lds, int k) : keys(lds), k(k) {}

    __device__ __forceinline__ void push(bool mine, uint64_t key)
    {
        const uint64_t m = __ballot(mine);
        if (mine) keys[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u))] = key;
        n += __popcll(m);
    }
    __device__ __forceinline__ void at_least(uint64_t key)
    {
        if (key <= least) return;
        least = key;
        bound = value_of(key);
    }
    // Where more than k lanes have a candidate, the k-th largest of the lanes' own largest
    // bounds the k-th of all.  `up`: its order as 32 bits, 0 without one.  False where that
    // leaves more than k lanes: equal logits.
    __device__ __forceinline__ bool raise(uint32_t up)
    {
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < 64; i++) above += (uint32_t)__builtin_amdgcn_readlane((int)up, i) > up ? 1 : 0;
        const uint64_t at = __ballot(up != 0 && above < k);
        if (__popcll(at) > k) return false;
        const uint64_t kth = __ballot(up != 0 && above == k - 1);
        if (kth) at_least((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)up, __ffsll((unsigned long long)kth) - 1) << 32);
        return true;
    }
    // The same for whole keys, which are distinct.
    __device__ __forceinline__ void raise_keys(uint64_t top)
    {
        int above = 0;
        for (int i = 0; i < 64; i++) above += lane_key(top, i) > top ? 1 : 0;
        const uint64_t kth = __ballot(top != 0 && above == k - 1);
        if (kth) at_least(lane_key(top, __ffsll((unsigned long long)kth) - 1));
    }
    // Cuts the list to its k largest, in order.
    __device__ __forceinline__ void cut()
    {
        const int lane = threadIdx.x & 63;
        wave_sync();
        if (n > 128) { // the k-th largest, bit by bit: the greatest t with k keys at or above it
            constexpr int C = (kRoom + 63) / 64;
            uint64_t mine[C], t = 0;
#pragma unroll
            for (int i = 0; i < C; i++) mine[i] = 64 * i + lane < n ? keys[64 * i + lane] : 0;
            for (int bit = 63; bit >= 0; bit--) {
                const uint64_t trial = t | 1ull << bit;
                int at = 0;
#pragma unroll
                for (int i = 0; i < C; i++)
                    if (64 * i < n) at += __popcll(__ballot(mine[i] >= trial));
                if (at >= k) t = trial;
            }
            wave_sync();
            n = 0;
#pragma unroll
            for (int i = 0; i < C; i++) push(mine[i] >= t && mine[i] != 0, mine[i]);
            wave_sync();
        }
        if (lane < 8) keys[n + lane] = 0;
        wave_sync();
        uint64_t key[2];
        int above[2] = {0, 0};
        key[0] = lane < n ? keys[lane] : 0;
        key[1] = 64 + lane < n ? keys[64 + lane] : 0;
        above[0] = count_above(keys, n, key[0]);
        if (n > 64) above[1] = count_above(keys, n, key[1]);
        wave_sync();
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (key[i] != 0 && above[i] < k) keys[above[i]] = key[i];
        wave_sync();
        if (n >= k) {
            n = k;
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (const uint64_t at = __ballot(key[i] != 0 && above[i] == k - 1)) at_least(lane_key(key[i], __ffsll((unsigned long long)at) - 1));
        }
    }
};

// A softmax's statistics: the largest logit m and how many logits are it, s = sum exp2((x
// - m) c) over the others (next to a certain token everything lies in them), and t = the
// same sum times (x - m) c.  What is added up over a row is in 64 bits.
struct Stats {
    float m;
    int ones;
    double s, t;
    static __device__ __forceinline__ Stats none() { return {-INFINITY, 0, 0.0, 0.0}; }
    // to a larger maximum; without a logit above -inf the sums are zero (or NaN)
    __device__ __forceinline__ void rescale(float to, float c)
    {
        const float d = fmaxf((m - to) * c, -1e4f);
        const double f = (double)__builtin_amdgcn_exp2f(d), all = s + (double)ones;
        t = f * (t + (double)d * all);
        s = f * all;
        m = to;
        ones = 0;
    }
    __device__ __forceinline__ void join(Stats o, float c)
    {
        const float to = fmaxf(m, o.m);
        if (m != to) rescale(to, c);
        if (o.m != to) o.rescale(to, c);
        s += o.s;
        t += o.t;
        ones += o.ones;
    }
};
// The largest of the wave's values, NaN only where all are.
__device__ __forceinline__ float wave_most(float x)
{
    return over_wave(x, [](float a, float b) { return fmaxf(a, b); });
}
// The sums of the wave's lanes, whose m is the same.
__device__ __forceinline__ Stats wave_total(Stats a)
{
    auto sum = [](auto x, auto y) { return x + y; };
    return {a.m, over_wave(a.ones, sum), over_wave(a.s, sum), over_wave(a.t, sum)};
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

// A workgroup per row and part of it.  A wave holds 64 x 32 logits at a time: their
// maximum (which moves the running sums only where it rises), the exponentials, and, where
// one of them passes the wave's k-th largest so far, their places in its list.  A wave's
// maximum, sums and list are its own, so nothing waits inside the pass.  The last part of
// a row to arrive merges all of them.  Bounded by HBM where there are rows enough, each logit
// being read once: 1000 rows of 131072 (524 MB) 98 us, with the 5 most probable 104, 5.0 to
// 5.3 TB/s; 64 with the 20 most probable 18, 32 19 (34 MB: a pass of the lanes, and the lists' merge),
// one with 5 8.7 (a launch, the pass, two trips to memory and the merge).
template <bool TOP>
__global__ __launch_bounds__(256, 4) void logprobs_kernel(LogprobsView p)
{
    __shared__ uint64_t keys[4][TOP ? kKeys : 1], least[4];
    __shared__ Stats stats[4];
    __shared__ double top_x, log_s; // the row's largest logit, the logarithm of its sum
    __shared__ int count[4], last;
    __shared__ uint32_t first[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_top = p.n_top, row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const float *x0 = p.logits + row * p.ld;
    const int32_t *given = p.given + (size_t)row * p.n_given;
    auto logit_of = [&](int id) { return id >= 0 && id < p.vocab ? x0[id] : NAN; };
    const float asked = tid < p.n_given ? logit_of(given[tid]) : 0.f; // (needed by the row's last part alone, and here by then)

    Stats st = Stats::none();
    Best best(keys[wave], n_top);
    const int w0 = part * p.chunk + wave * (p.chunk / 4), w1 = min(p.vocab, w0 + p.chunk / 4);
    int base = w0;
    do { // (once at least: the first time has a barrier)
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
        float m4[kTile / 4], m; // (NaN only where all are)
#pragma unroll
        for (int i = 0; i < kTile / 4; i++) {
            m4[i] = fmaxf(fmaxf(x[4 * i], x[4 * i + 1]), fmaxf(x[4 * i + 2], x[4 * i + 3]));
            m = i ? fmaxf(m, m4[i]) : m4[i];
        }
        const float most = wave_most(m);
        if (most > st.m) st.rescale(most, p.c);
        // 2^((x - m) c) as 2^(x c - m c): what m c loses by its rounding is put back into the sums
        // (more than 100 only where logits are further apart than that)
        const float mu = st.m == -INFINITY ? 0.f : st.m, mc = mu * p.c, lost = fminf(fmaxf(fmaf(mu, p.c, -mc), -100.f), 100.f);
        float s2[2] = {0.f, 0.f}, t2[2] = {0.f, 0.f};
        auto add = [&](int i, float y, float d) {
            s2[i & 1] += y;
            t2[i & 1] = fmaf(y, fmaxf(d, -1e4f), t2[i & 1]); // (0 times -inf is 0 here)
        };
        if (most == st.m) { // the maximum is among them: it is counted, not added
#pragma unroll
            for (int i = 0; i < kTile; i++) {
                const float d = fmaf(x[i], p.c, -mc), e = __builtin_amdgcn_exp2f(d);
                const bool one = x[i] == mu;
                st.ones += one ? 1 : 0;
                add(i, one ? 0.f : e, d);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kTile; i++) {
                const float d = fmaf(x[i], p.c, -mc);
                add(i, __builtin_amdgcn_exp2f(d), d);
            }
        }
        const float s = s2[0] + s2[1], t = t2[0] + t2[1];
        const double put = (double)__builtin_amdgcn_exp2f(-lost);
        st.s += (double)s * put;
        st.t += ((double)t - (double)lost * (double)s) * put;
        if constexpr (TOP) {
            const bool has_nan = s != s, some = base + 4 * lane < w1; // (else all of its places are past the end)
            const uint32_t up = some ? (uint32_t)(key_of(m, 0) >> 32) : 0;
            if (base == w0) { // a first bound: as many lanes' largest from each wave as make k of them
                const uint32_t mine = __any(has_nan) ? 0 : rank_of(up, (n_top + 3) / 4);
                if (lane == 0) first[wave] = mine;
                __syncthreads();
                best.at_least((uint64_t)min(min(first[0], first[1]), min(first[2], first[3])) << 32);
            }
            // a lane is looked at where its largest is not below the bound, or it has a NaN
            const uint64_t lanes = __ballot(some && (!(m < best.bound) || has_nan));
            if (lanes) {
                auto key = [&](int i) {
                    const int at = base + 256 * (i >> 2) + 4 * lane + (i & 3);
                    float y = x[i];
                    asm("" : "+v"(y)); // made where it is wanted: all keys at once are 64 registers
                    return at < w1 ? key_of(y, at) : 0;
                };
                if (__popcll(lanes) > kLogprobsTop && (__any(has_nan) || !best.raise(up))) { // more than the list has room for
                    uint64_t top = 0;
#pragma unroll
                    for (int i = 0; i < kTile; i++) top = max(top, key(i));
                    best.raise_keys(top);
                }
#pragma unroll
                for (int i = 0; i < kTile; i += 4) {
                    if (!__any(some && (!(m4[i / 4] < best.bound) || has_nan))) continue;
#pragma unroll
                    for (int j = i; j < i + 4; j++) {
                        if (!__any(!(x[j] < best.bound))) continue;
                        const uint64_t k = key(j);
                        best.push(k != 0 && k >= best.least, k);
                    }
                }
                best.cut();
            }
        }
        base += 64 * kTile;
    } while (base < w1);
    st = wave_total(st);
    if (lane == 0) {
        stats[wave] = st;
        count[wave] = best.n;
        least[wave] = best.least;
    }
    __syncthreads();
    if constexpr (TOP) { // the workgroup's list: all four one after the other
        int before = 0, n = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            before += w < wave ? count[w] : 0;
            n += count[w];
        }
        if (wave > 0 && lane < best.n) keys[0][before + lane] = best.keys[lane]; // (at most k, which is at most 32)
        __syncthreads();
        if (wave == 0) {
            best.at_least(max(max(least[0], least[1]), max(least[2], least[3])));
            best.n = n;
            best.cut();
        }
    }
    if (p.parts > 1) {
        LogprobsPart *mine = p.part + blockIdx.x;
        if (tid < 4) {
            store_shared64(&mine->s[tid], __builtin_bit_cast(uint64_t, stats[tid].s));
            store_shared64(&mine->t[tid], __builtin_bit_cast(uint64_t, stats[tid].t));
            store_shared64(&mine->m[tid], (uint64_t)(uint32_t)stats[tid].ones << 32 | __float_as_uint(stats[tid].m));
        }
        if constexpr (TOP)
            if (tid < n_top) store_shared64(&mine->key[tid], tid < best.n ? keys[0][tid] : 0);
        if (!arrives_last(p.tickets + row, p.parts, last)) return;
        const LogprobsPart *from = p.part + (size_t)row * p.parts;
        if constexpr (TOP) {
            // sixteen threads to a list, two of its keys to each
            const int l = min(tid >> 4, p.parts - 1), i0 = tid & 15;
            uint64_t key[2];
#pragma unroll
            for (int i = 0; i < 2; i++) key[i] = tid >> 4 < p.parts && i0 + 16 * i < n_top ? load_shared64(&from[l].key[i0 + 16 * i]) : 0;
            if (wave == 0) {
                // A bound: the lists are in order, so the k / i-th largest of their i-th keys is one
                // for the k-th of all; i = 1, 2, 4, 8 in the wave's four rows of lanes, a list to each.
                const int i = 1 << (lane >> 4), rank = (n_top + i - 1) / i;
                const uint64_t top = (lane & 15) < p.parts && i <= n_top ? load_shared64(&from[lane & 15].key[i - 1]) : 0;
                int above = 0;
                uint64_t y = top;
#pragma unroll
                for (int k = 1; k < 16; k++) {
                    y = (uint64_t)(uint32_t)turned<0x121>((int)(y >> 32)) << 32 | (uint32_t)turned<0x121>((int)(uint32_t)y);
                    above += y > top ? 1 : 0;
                }
                uint64_t floor = 0;
                for (uint64_t at = __ballot(top != 0 && above == rank - 1); at; at &= at - 1)
                    floor = max(floor, lane_key(top, __ffsll((unsigned long long)at) - 1));
                if (lane == 0) {
                    least[0] = floor;
                    count[0] = 0;
                }
            }
            __syncthreads();
            const uint64_t floor = least[0];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const bool take = key[i] != 0 && key[i] >= floor;
                const uint64_t m = __ballot(take);
                if (!m) continue;
                int at = 0;
                if (lane == 0) at = atomicAdd(&count[0], __popcll(m));
                at = __builtin_amdgcn_readfirstlane(at);
                if (take) keys[0][at + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u))] = key[i];
            }
            __syncthreads();
            if (wave == 0) {
                best = Best(keys[0], n_top);
                best.n = count[0];
                best.cut();
            }
        }
        if (wave == 1 && lane < 4 * p.parts) {
            const uint64_t m = load_shared64(&from[lane >> 2].m[lane & 3]);
            st.s = __builtin_bit_cast(double, load_shared64(&from[lane >> 2].s[lane & 3]));
            st.t = __builtin_bit_cast(double, load_shared64(&from[lane >> 2].t[lane & 3]));
            st.m = __uint_as_float((uint32_t)m);
            st.ones = (int)(m >> 32);
        }
    } else if (wave == 1 && lane < 4) st = stats[lane];
    if (wave == 1) { // beside the first wave's list
        if (lane >= 4 * p.parts) st = Stats::none();
        const float most = wave_most(st.m);
        if (most > st.m) st.rescale(most, p.c);
        st = wave_total(st);
        // logp(x) = (x - m) / T - log(1 + s);  H = log(1 + s) - (sum e (x - m) / T) / (1 + s),
        // where s has all of the sum but one logit that is m
        const double rest = st.s + (double)(st.ones - 1), log_of = fabsf(st.m) < INFINITY ? log1p(rest) : NAN;
        if (lane == 0) {
            top_x = (double)st.m;
            log_s = log_of;
            if (p.entropy) p.entropy[row] = (float)(log_of - 0.69314718055994530942 * st.t / (1.0 + rest));
        }
    }
    __syncthreads();

    const double m = top_x, log_sum = log_s;
    auto logp = [&](float x) { return (float)(((double)x - m) * p.inverse - log_sum); };
    float *to = p.logp + (size_t)row * p.n_given;
    if (tid < p.n_given) to[tid] = logp(asked);
    for (int i = tid + 256; i < p.n_given; i += 256) to[i] = logp(logit_of(given[i]));
    if constexpr (TOP)
        if (tid < n_top) {
            const uint64_t key = keys[0][tid];
            if (p.top) p.top[(size_t)row * n_top + tid] = index_of(key);
            if (p.top_logp) p.top_logp[(size_t)row * n_top + tid] = logp(value_of(key));
        }
}

// Parts of a row: few rows are split until the GPU is full, into no more parts than sixteen
// (one wave merges their four waves each) and none of less than 8192 logits, a pass of the
// workgroup's lanes (us, one call after the other in a graph, 131072 logits: 1 row, 5 most
// probable, 2 / 4 / 8 / 16 parts 20.0 / 13.6 / 11.0 / 8.7; 64 rows, 20, 42 / 33 / 28 / 20;
// 200, 5, 1 / 2 / 4 parts 38.6 / 31.2 / 32.1; 400, 1 / 2 parts 47.8 / 53.3; 1 row of 32000,
// 2 / 4 / 8 parts 10.1 / 8.5 / 9.4).
int logprobs_parts(int rows, int vocab)
{
    return rows > kLogprobsParts / 4 ? 1 : std::max(1, std::min({kLogprobsParts / std::max(rows, 1), (vocab + 8191) / 8192, kLogprobsSplit}));
}

hipError_t launch_logprobs(const LogprobsArgs &a, hipStream_t s)
{
    if (a.rows <= 0) return hipSuccess;
    const int parts = logprobs_parts(a.rows, a.vocab);
    const int chunk = ((a.vocab + parts - 1) / parts + 1023) & ~1023;
    const LogprobsView v = {a.logits, a.ld, a.given, a.logp, a.entropy, a.top_logp, a.top, a.part, a.tickets, a.vocab, a.n_given, a.n_top,
                            parts, chunk, (float)(1.4426950408889634074 / (double)a.temperature), 1.0 / (double)a.temperature};
    const dim3 grid((unsigned)a.rows * parts);
    if (a.n_top > 0) hipLaunchKernelGGL(logprobs_kernel<true>, grid, dim3(256), 0, s, v);
    else hipLaunchKernelGGL(logprobs_kernel<false>, grid, dim3(256), 0, s, v);
    return hipGetLastError();
}

} // namespace jev
