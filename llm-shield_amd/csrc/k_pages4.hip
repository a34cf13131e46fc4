// The 4-bit paged KV cache (Pages with bits = 4 in jev_internal.h): rotary positions with
// the store, attention, reading back.  Plans are the 8-bit cache's (k_pages.hip).
//
// A token's row of a KV head (K or V, hd elements) has a power of two 2^e, and each 32
// elements of it a step u (1 .. 15) and a zero point z (0 .. 15): an element's code n (0 ..
// 15) stands for (n - z) u 2^e.  (n - z) u is a whole number of at most 225, exact in fp16,
// so the matrix cores multiply what is stored, and 2^e enters as an exponent.  Rows do not
// depend on each other: storing a token reads and rounds nothing that is there.
#include <algorithm>

#include "jev_pages_dev.h"

namespace jev {

namespace {

// A block's bytes (16 tokens of a KV head, Pages4 in jev_internal.h).  A 32-bit word holds
// eight nibbles, turned two bits to the left so that the second and sixth lie where a
// masked word is two fp16 numbers 16 + n as it stands: pair p of a word is its nibbles p
// (low half) and p + 4 (high half).
constexpr uint32_t kNibble = 0x03c003c0u, kSixteen = 0x4c004c00u;

__device__ __forceinline__ uint32_t turn_left(uint32_t x, int by) { return __builtin_rotateleft32(x, by); }

// Bit of element i (0 .. 7) of a word before the turn: pairs (0, 1), (2, 3), ...
__host__ __device__ constexpr int nibble_at(int i) { return 4 * ((i >> 1) + 4 * (i & 1)); }

// Pair p of a word as fp16: 16 + n.  `k16`: sixteen() in a vector register, so that mask and
// exponent are one v_and_or (an instruction takes one constant from the scalar side).
__device__ __forceinline__ uint32_t sixteen()
{
    uint32_t k = kSixteen;
    asm("" : "+v"(k));
    return k;
}
__device__ __forceinline__ half2_t masked(uint32_t x, uint32_t k16) { return __builtin_bit_cast(half2_t, (x & kNibble) | k16); }
template <int P>
__device__ __forceinline__ half2_t nibble_pair(uint32_t w, uint32_t k16)
{
    return masked(P == 0 ? w << 4 : P == 1 ? w : P == 2 ? w >> 4 : turn_left(w, 24), k16);
}
__device__ __forceinline__ half2_t nibble_pair(uint32_t w, int p, uint32_t k16) { return masked(turn_left(w, (4 - 4 * p) & 31), k16); }

// Steps and zero points turn 16 + n into (n - z) u: (16 + n) u - (16 + z) u, where the
// second product is a whole number below 2^9.
struct Steps {
    half2_t u, m;
    Steps() = default;
    __device__ __forceinline__ Steps(half2_t u16, half2_t z16) : u(u16 - half2_t{(_Float16)16.f, (_Float16)16.f}), m(-z16 * u) {}
    __device__ __forceinline__ uint32_t operator()(half2_t n16) const
    {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n16, u, m));
    }
};

// A word's eight elements: with the same step for all, and with one for each pair's halves.
__device__ __forceinline__ half8_t word_f16(uint32_t w, const Steps &s, uint32_t k16)
{
    return __builtin_bit_cast(half8_t, make_uint4(s(nibble_pair<0>(w, k16)), s(nibble_pair<1>(w, k16)), s(nibble_pair<2>(w, k16)),
                                                  s(nibble_pair<3>(w, k16))));
}
__device__ __forceinline__ half8_t word_f16(uint32_t w, const Steps (&s)[4], uint32_t k16)
{
    return __builtin_bit_cast(half8_t, make_uint4(s[0](nibble_pair<0>(w, k16)), s[1](nibble_pair<1>(w, k16)), s[2](nibble_pair<2>(w, k16)),
                                                  s[3](nibble_pair<3>(w, k16))));
}

// Of a K step word's pair (u of a token's group low, its z high), for all of the group.
__device__ __forceinline__ Steps key_steps(half2_t uz) { return Steps(half2_t{uz[0], uz[0]}, half2_t{uz[1], uz[1]}); }
// V's step and zero words of eight tokens.
__device__ __forceinline__ void value_steps(uint32_t u, uint32_t z, Steps (&s)[4], uint32_t k16)
{
    s[0] = Steps(nibble_pair<0>(u, k16), nibble_pair<0>(z, k16));
    s[1] = Steps(nibble_pair<1>(u, k16), nibble_pair<1>(z, k16));
    s[2] = Steps(nibble_pair<2>(u, k16), nibble_pair<2>(z, k16));
    s[3] = Steps(nibble_pair<3>(u, k16), nibble_pair<3>(z, k16));
}

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ int byte_of(const uint4 &v, int i) { return (int)((word_of(v, i >> 2) >> (8 * (i & 3))) & 255u); }

__device__ __forceinline__ int most_byte(const uint4 &v)
{
    typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
    ushort2_t m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = word_of(v, i);
        m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2_t, w & 0x00ff00ffu));
        m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2_t, (w >> 8) & 0x00ff00ffu));
    }
    return max((int)m[0], (int)m[1]);
}

uint8_t *layer4_of(const Pages &p, int layer) { return p.k + (size_t)layer * p.n_blocks() * pages4_bytes(p.hd); }

// y / u to the nearest whole number, a half to the even one; u whole, 1 .. 15, |y| <= 225.
// The remainder is exact: it is a multiple of y's last bit and not larger than y or u.
__device__ __forceinline__ float whole_steps(float y, float u, float inv)
{
    float q = rintf(y * inv);
    const float rest = fmaf(-q, u, y), twice = 2.f * fabsf(rest);
    if (twice > u || (twice == u && ((int)q & 1))) q += rest > 0.f ? 1.f : -1.f;
    return q;
}

struct Store4View {
    uint8_t *pool;
    PagesPlanHead *head;
    const PagesUnit *unit;
    const double2 *angle;
    const float *q, *k_in, *v_in;
    float *q_out;
    int64_t q_ld, kv_ld;
    size_t in_stride;
    int nin, n_kv, n_heads, group, sub, sub_shift, half, rope_half, orig_ctx;
    float temp_scale;
    int n_tokens, n_requests, wide; // of the call's plan
};

} // namespace

// One workgroup per block that the batch touches and KV head: the block's new tokens'
// queries (of the head's group) rotated, their keys rotated, keys and values stored.
// Sixteen threads hold a token's row; the rotated rows pass through LDS, and a thread
// takes hd / 16 neighbouring elements of them to steps and codes.  Words that hold other
// tokens' nibbles (V's, and all steps) are read first and merged.  Rotations are 64-bit
// and round to fp32 once, quotients are exact: a stored value does not depend on how
// they are formed.
template <int HD, bool VEC>
__global__ __launch_bounds__(256) void pages4_store_kernel(Store4View p)
{
    constexpr int NP = HD / 32, NE = HD / 16, NG = HD / 32, TG = 32 / NE, LD = HD + 4, RING = 2;
    constexpr Pages4 at(HD);
    __shared__ __align__(16) float xs[2][kPageBlock][LD];
    __shared__ uint8_t code[kPageBlock][HD];                    // V's
    __shared__ uint8_t step[2][kPageBlock][NG], zero[2][kPageBlock][NG];
    const int tid = threadIdx.x, j = tid & 15, h = blockIdx.y;
    const PagesUnit un = p.unit[blockIdx.x];
    const PagesPlanHead plan = *p.head; // (the unit's load does not wait for this)
    if (outgrown(p, plan) || (int)blockIdx.x >= plan.n_units) return;
    const int pos0 = un.pos, n = un.n, row0 = un.row, off = pos0 & (kPageBlock - 1);
    const bool kv = p.k_in != nullptr;
    const RowPairs<HD> e(p, j);

    // this thread's token, and its rows: K (-2), V (-1), then the group's queries
    const int nt = n > 8 ? 16 : n > 4 ? 8 : n > 2 ? 4 : n, jump = 16 / nt; // (nt: 1, 2, 4, 8, 16)
    const int t = (tid >> 4) % nt, row = row0 + t, first = (kv ? -2 : 0) + (tid >> 4) / nt, end = t < n && p.q ? p.group : 0;
    const bool mine = t < n;

    // where the block lies, and the words of it that hold other tokens too
    uint8_t *block = p.pool + ((((size_t)(un.block >> p.sub_shift) * p.n_kv + h) << p.sub_shift) | (un.block & (p.sub - 1))) * at.bytes;
    uint32_t *vword = (uint32_t *)(block + at.v) + tid, *sword = (uint32_t *)(block + at.ks) + tid;
    const bool has_v = kv && tid < 2 * HD, has_s = kv && tid < 8 * NG;
    uint32_t old_v = 0, old_s = 0;
    if (off > 0) {
        if (has_v) old_v = *vword;
        if (has_s) old_s = *sword;
    }
    double2 g[NP];
#pragma unroll
    for (int c = 0; c < NP; c++) {
        const int q = NP * j + c;
        g[c] = mine && q < p.half ? p.angle[(size_t)row * p.half + q] : make_double2(0.0, 0.0);
    }
    auto load = [&](int which, float2 (&y)[NP]) {
        const float *src = which == -2 ? p.k_in + row * p.kv_ld + h * HD
                           : which == -1 ? p.v_in + row * p.kv_ld + h * HD
                                         : p.q + row * p.q_ld + (size_t)(h * p.group + which) * HD;
        load_pairs<HD, VEC>(e, src, y);
        for (int i = 1; i < p.nin; i++) {
            float2 w[NP];
            load_pairs<HD, VEC>(e, src + i * p.in_stride, w);
#pragma unroll
            for (int c = 0; c < NP; c++) y[c] = make_float2(y[c].x + w[c].x, y[c].y + w[c].y);
        }
    };
    auto rotate = [&](double f, float2 (&y)[NP]) {
#pragma unroll
        for (int c = 0; c < NP; c++) {
            const double u = y[c].x, v = y[c].y;
            const double m0 = u * g[c].x, m1 = v * g[c].y, m2 = u * g[c].y, m3 = v * g[c].x;
            const bool turned = NP * j + c < p.half;
            y[c] = make_float2((float)((turned ? m0 - m1 : u) * f), (float)((turned ? m2 + m3 : v) * f));
        }
    };

    int w = first;
    if (kv) {
        float2 x[2][NP]; // this thread's rows of K and V
#pragma unroll
        for (int it = 0; it < 2; it++)
            if (mine && w + it * jump < 0) load(w + it * jump, x[it]);
#pragma unroll
        for (int it = 0; it < 2; it++) {
            const int which = w + it * jump;
            if (!mine || which >= 0) continue;
            if (which == -2) rotate(1.0, x[it]);
            store_pairs<HD, VEC>(e, xs[which + 2][t], x[it]);
        }
        while (w < 0) w += jump;
    }
    if (end) {
        double f = 1.0;
        const int pos = pos0 + t;
        if (p.orig_ctx > 0 && p.temp_scale != 0.f && pos >= p.orig_ctx)
            f = 1.0 + (double)p.temp_scale * log(1.0 + (double)(pos / p.orig_ctx));
        // RING rows in flight
        for (; w < end; w += RING * jump) {
            float2 y[RING][NP];
#pragma unroll
            for (int i = 0; i < RING; i++)
                if (w + i * jump < end) load(w + i * jump, y[i]);
#pragma unroll
            for (int i = 0; i < RING; i++)
                if (w + i * jump < end) {
                    rotate(f, y[i]);
                    store_pairs<HD, VEC>(e, p.q_out + ((size_t)row * p.n_heads + h * p.group + w + i * jump) * HD, y[i]);
                }
        }
    }
    if (!kv) return;
    __syncthreads();

    // steps and codes of token tid / 16, elements NE j ..
    const int tk = tid >> 4;
    if (tk < n) {
        unsigned bad = 0; // a value that is not finite has the largest bits
        int power[2];
#pragma unroll
        for (int v = 0; v < 2; v++) {
            float x[NE], hi = 0.f, lo = 0.f;
            unsigned bits = 0;
#pragma unroll
            for (int i = 0; i < NE; i++) {
                x[i] = xs[v][tk][NE * j + i];
                hi = fmaxf(hi, x[i]);
                lo = fmaxf(lo, -x[i]);
                bits = max(bits, __float_as_uint(fabsf(x[i])));
            }
#pragma unroll
            for (int o = 1; o < TG; o <<= 1) {
                hi = fmaxf(hi, __shfl_xor(hi, o, 64));
                lo = fmaxf(lo, __shfl_xor(lo, o, 64));
            }
            const float span = 0.5f * hi + 0.5f * lo; // half the group's span: the whole one may be past fp32's range
            float most = span;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                most = fmaxf(most, __shfl_xor(most, o, 64));
                bits = max(bits, (unsigned)__shfl_xor((int)bits, o, 64));
            }
            bad = max(bad, bits);
            // the least 2^ex with the widest span <= 15 * 15 * 2^ex, 225 = 0.87890625 * 2^8
            const bool some = most > 0.f && bits < 0x7f800000u;
            const int ex = max(__builtin_amdgcn_frexp_expf(most) - (__builtin_amdgcn_frexp_mantf(most) <= 0.87890625f ? 7 : 6), -126);
            const float wide = some ? ldexpf(span, 1 - ex) : 0.f;
            float u = ceilf(wide * (1.f / 15.f)); // then the least u with span <= 15 u exactly
            if (15.f * (u - 1.f) >= wide) u -= 1.f;
            if (15.f * u < wide) u += 1.f;
            u = fmaxf(u, 1.f);
            const float inv = __builtin_amdgcn_rcpf(u), z = some ? whole_steps(ldexpf(lo, -ex), u, inv) : 0.f;
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < NE; i++) {
                const float q = some ? whole_steps(ldexpf(x[i], -ex), u, inv) + z : 0.f;
                const uint32_t c = (uint32_t)(int)fminf(fmaxf(q, 0.f), 15.f);
                if (v) code[tk][NE * j + i] = (uint8_t)c;
                else word |= c << nibble_at((NE * j + i) & 7);
            }
            if (!v) {
                if (NE == 4) word |= (uint32_t)__shfl_xor((int)word, 1, 64);
                if (NE == 8 || !(j & 1)) *(uint32_t *)(block + at.k + (off + tk) * (HD / 2) + 4 * (NE * j / 8)) = turn_left(word, 2);
            }
            if (j % TG == 0) {
                step[v][tk][j / TG] = (uint8_t)(int)u;
                zero[v][tk][j / TG] = (uint8_t)(int)z;
            }
            power[v] = some ? ex + 127 : 0;
        }
        // a value that is not finite: the token's V power says so for both
        if (j < 2) block[(j ? at.ve : at.ke) + off + tk] = (uint8_t)(bad < 0x7f800000u ? power[j] : j ? 255 : 0);
    }
    __syncthreads();

    // words over several tokens: the new ones' nibbles among what is there
    auto merge = [&](uint32_t old, auto token, auto nibble) {
        uint32_t put = 0, mask = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int tk = token(i) - off;
            if (tk < 0 || tk >= n) continue;
            put |= (uint32_t)nibble(i, tk) << nibble_at(i);
            mask |= 15u << nibble_at(i);
        }
        mask = turn_left(mask, 2);
        return make_uint2((old & ~mask) | turn_left(put, 2), mask);
    };
    if (has_v) {
        const int dim = 32 * (tid >> 6) + 16 * ((tid >> 1) & 1) + ((tid >> 2) & 15), t0 = 8 * (tid & 1);
        const uint2 r = merge(old_v, [&](int i) { return t0 + i; }, [&](int, int tk) { return code[tk][dim]; });
        if (r.y) *vword = r.x;
    }
    if (has_s) {
        uint2 r;
        if (tid < 4 * NG) { // K: tokens r, 4 + r, ..: u the even elements (low half), z the odd ones
            const int gr = tid >> 2, r0 = tid & 3;
            r = merge(old_s, [&](int i) { return 4 * (i >> 1) + r0; }, [&](int i, int tk) { return i & 1 ? zero[0][tk][gr] : step[0][tk][gr]; });
        } else {
            const int gr = (tid - 4 * NG) >> 2, t0 = 8 * (tid & 1), z = tid & 2;
            r = merge(old_s, [&](int i) { return t0 + i; }, [&](int, int tk) { return z ? zero[1][tk][gr] : step[1][tk][gr]; });
        }
        if (r.y) *sword = r.x;
    }
}

hipError_t launch_pages4_store(const Pages &p, const PagesStoreArgs &a, hipStream_t s)
{
    const int units = a.n_tokens / kPageBlock + 2 * (a.n_requests < a.n_tokens ? a.n_requests : a.n_tokens);
    const int np = p.hd / 32;
    auto vec = [&](const void *x, int64_t ld) { return !x || ((uintptr_t)x % (4 * np) == 0 && ld % np == 0); };
    // as in the 8-bit store: rows that start aligned, and no thread with pairs on both
    // sides of the rotated part's end
    const bool v = vec(a.q, a.q_ld) && vec(a.k, a.kv_ld) && vec(a.v, a.kv_ld) && vec(a.q_out, 0) && a.in_stride % np == 0 &&
                   (!p.rope_half || p.half % np == 0);
    const Store4View view = {layer4_of(p, a.layer), p.head, p.unit, p.angle, a.q, a.k, a.v, a.q_out, a.q_ld, a.kv_ld, a.in_stride, a.nin,
                             p.n_kv, p.n_heads, p.group, p.sub, p.sub_shift, p.half, p.rope_half, p.orig_ctx, p.temp_scale,
                             a.n_tokens, a.n_requests, 1};
    const dim3 grid(units > 0 ? units : 1, p.n_kv);
    if (p.hd == 128 && v) hipLaunchKernelGGL((pages4_store_kernel<128, true>), grid, dim3(256), 0, s, view);
    else if (p.hd == 128) hipLaunchKernelGGL((pages4_store_kernel<128, false>), grid, dim3(256), 0, s, view);
    else if (v) hipLaunchKernelGGL((pages4_store_kernel<64, true>), grid, dim3(256), 0, s, view);
    else hipLaunchKernelGGL((pages4_store_kernel<64, false>), grid, dim3(256), 0, s, view);
    return hipGetLastError();
}

// ------------------------------------------------------------ attention

namespace {

struct Attend4View {
    const uint8_t *pool;
    const int32_t *table;
    PagesPlanHead *head;
    const PagesItem *item, *wide_item;
    float *part, *wide_part;
    int32_t *tickets, *wide_tickets;
    const float *q;
    float *out;
    int n_kv, n_heads, group, sub, sub_shift, width;
    float scale;
    int wides, tiles;               // workgroups of each kind
    int n_tokens, n_requests, wide; // of the call's plan
};

// A query row as fp16 pairs: scaled by a power of two so that its largest element lies in
// [2^13, 2^14), then by the softmax's scale in powers of two.  A key's 2^e and the row's
// power meet in a score's exponent, in whole numbers.
struct Query4 {
    float scale;
    int ex;
    __device__ __forceinline__ Query4(float m, float softmax)
        : scale(softmax * 1.44269504088896341f), ex(m > 0.f && m < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(m) : 0) {}
    __device__ __forceinline__ int power() const { return -127 - ex; } // with a key's byte
    __device__ __forceinline__ float scaled(float x) const { return __builtin_amdgcn_ldexpf(x, ex) * scale; }
};

// Two values as fp16, to nearest, and `part` times that plus the values: with -1 what fp16
// leaves of them.  (The remainder is taken of the fp32 values: they are rounded to fp32 first.)
__device__ __forceinline__ uint32_t pair_f16(float x0, float x1)
{
    typedef float floatx2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{x0, x1}, half2_t));
}
__device__ __forceinline__ void remainders(uint32_t f, float part, float x0, float x1, float &r0, float &r1)
{
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(f), "v"(part), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(f), "v"(part), "v"(x1));
}
// Eight elements of a query, rounded to fp32, as a pair of fragments; or the one that `part`
// (0: high, -1: low) names.
__device__ __forceinline__ void split_query(const Query4 &q, const float (&x)[8], half8_t &hi, half8_t &lo)
{
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float y0 = q.scaled(x[2 * i]), y1 = q.scaled(x[2 * i + 1]), r0, r1;
        asm("" : "+v"(y0), "+v"(y1)); // hi straight from the product may be another than the one that lo completes
        h[i] = pair_f16(y0, y1);
        remainders(h[i], -1.f, y0, y1, r0, r1);
        l[i] = pair_f16(r0, r1);
    }
    hi = __builtin_bit_cast(half8_t, make_uint4(h[0], h[1], h[2], h[3]));
    lo = __builtin_bit_cast(half8_t, make_uint4(l[0], l[1], l[2], l[3]));
}
__device__ __forceinline__ half8_t split_query(const Query4 &q, const float (&x)[8], float part)
{
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float y0 = q.scaled(x[2 * i]), y1 = q.scaled(x[2 * i + 1]), r0, r1;
        asm("" : "+v"(y0), "+v"(y1));
        remainders(pair_f16(y0, y1), part, y0, y1, r0, r1);
        h[i] = pair_f16(r0, r1);
    }
    return __builtin_bit_cast(half8_t, make_uint4(h[0], h[1], h[2], h[3]));
}

template <int HD>
struct Tile4Lds {
    float lo[4][16][HD + 4];
    float lm[4][kPagesTileRows], ll[4][kPagesTileRows];
    uint2 steps[4][4][HD / 4 + 2]; // a wave's V steps of 64 keys: [block][group of dims][pair of tokens]
    int last;
};

// Up to ROWS (token, head) rows of a request and KV head over keys [key0, key1) of its
// pages; the four waves take 64 keys (four blocks) in turn and merge at the end.
// S^T = K Q^T with the rows of the K operand dealt so that a lane's sixteen scores are the
// sixteen tokens of one block, which makes the weights the P^T operand of O^T += V^T P^T
// as they stand.  q and p enter as fp16 pairs (hi + lo, ~22 bits).  Up to eight rows leave
// half of the operand's sixteen columns, which take the low parts: one matrix instruction a
// product instead of two.  A weight is 2^(score - m); the V operand's 2^e and the row's own
// power are added to its exponent, so that what enters fp16 is relative to the row's
// heaviest product so far (times 2^9), over the keys that the row sees.
template <int HD, int ROWS>
__device__ __forceinline__ void attend4_tile(const Attend4View &p, Tile4Lds<HD> &lds, const PagesItem &r, int h)
{
    constexpr int NC = HD / 32, NS = HD / 16, NI = HD / 32, LD = HD + 4, NQ = ROWS == 8 ? 1 : 2;
    constexpr Pages4 at(HD);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, n = lane & 15;
    const uint32_t k16 = sixteen();
    const int32_t *table = p.table + (size_t)r.id * p.width;
    // columns past the request's rows repeat its last one
    const int n_rows = r.row1, row = min(r.row0 + (n & (ROWS - 1)), n_rows - 1);
    const int token = row / p.group, head = h * p.group + row % p.group;
    const int limit = r.past + token; // last visible key
    // the tile's last visible key; keys up to `clear` are seen by every row
    const int top = r.past + min(n_rows - 1, r.row0 + ROWS - 1) / p.group;
    const int key1 = min(r.key1, top + 1), clear = r.past + r.row0 / p.group;
    const int last = (r.len - 1) / kPageBlock; // blocks past it are read as this one, and masked

    // V's steps of a block are made by its sixteen lanes, NI / 2 pairs of tokens of a group
    // each, and shared through LDS
    const int pair0 = n * (NI / 2), step_at = 16 * (pair0 >> 3) + 4 * ((pair0 >> 2) & 1);
    auto &steps = lds.steps[wave][g];

    // a lane reads K of block n / 4 of the four, V and the powers of block g
    auto page_of = [&](int kb, int i) { return table[min(4 * kb + i, last) >> p.sub_shift]; };
    auto block_of = [&](int kb, int i, int page) {
        return p.pool + ((((size_t)page * p.n_kv + h) << p.sub_shift) + (min(4 * kb + i, last) & (p.sub - 1))) * at.bytes;
    };
    uint4 kr[4], vr[NI], ke, ve;
    uint32_t ks, vu, vz;
    auto fetch_k = [&](int kb, int page) {
        const uint8_t *b = block_of(kb, n >> 2, page);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint8_t *src = b + at.k + (4 * t + (n & 3)) * (HD / 2) + 4 * NC * g;
            if constexpr (NC == 4) kr[t] = *(const uint4 *)src;
            else {
                const uint2 x = *(const uint2 *)src;
                kr[t] = make_uint4(x.x, x.y, 0, 0);
            }
        }
        ks = *(const uint32_t *)(b + at.ks + 4 * (4 * (g * NI / 4) + (n & 3)));
    };
    auto fetch_v = [&](int kb, int page) {
        const uint8_t *b = block_of(kb, g, page);
        ke = *(const uint4 *)(b + at.ke);
        ve = *(const uint4 *)(b + at.ve);
#pragma unroll
        for (int i = 0; i < NI; i++) vr[i] = *(const uint4 *)(b + at.v + 256 * i + 16 * n);
        vu = *(const uint32_t *)(b + at.vs + step_at);
        vz = *(const uint32_t *)(b + at.vs + step_at + 8);
    };
    int kb = r.key0 / 64 + wave;
    int pk = page_of(kb, n >> 2), pv = page_of(kb, g);
    if (kb * 64 < key1) {
        fetch_k(kb, pk);
        fetch_v(kb, pv);
    }
    pk = page_of(kb + 4, n >> 2);
    pv = page_of(kb + 4, g);

    // Q^T fragments: dims 8 NC g + 8 c .. + 7 of column n
    half8_t qf[NQ][NC];
    int query;
    const float part = n < 8 ? 0.f : -1.f; // 8 rows: a column's part of a query or a weight
    {
        const float *src = p.q + ((size_t)(r.start + token) * p.n_heads + head) * HD + 8 * NC * g;
        float x[NC][8], m = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c][i] = src[8 * c + i];
                m = fmaxf(m, fabsf(x[c][i]));
            }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const Query4 scaled(m, p.scale);
        query = scaled.power();
#pragma unroll
        for (int c = 0; c < NC; c++) {
            if constexpr (NQ == 2) split_query(scaled, x[c], qf[0][c], qf[1][c]);
            else qf[0][c] = split_query(scaled, x[c], part);
        }
    }

    floatx4 o[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) o[s] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f, e = -INFINITY; // m and e whole numbers; outputs are held times 2^(9 - e)
    int value = -127;                            // with a V row's byte: the power from a weight to fp16's

    auto row_max = [](float x) {
        x = fmaxf(x, __shfl_xor(x, 16, 64));
        return fmaxf(x, __shfl_xor(x, 32, 64));
    };
    for (; kb * 64 < key1; kb += 4) {
        const bool more = (kb + 4) * 64 < key1;
        float sv[16];
        const Steps kst[4] = {key_steps(nibble_pair<0>(ks, k16)), key_steps(nibble_pair<1>(ks, k16)), key_steps(nibble_pair<2>(ks, k16)),
                              key_steps(nibble_pair<3>(ks, k16))};
#pragma unroll
        for (int t = 0; t < 4; t++) {
            floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const half8_t k = word_f16(word_of(kr[t], c), kst[t], k16);
#pragma unroll
                for (int i = 0; i < NQ; i++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[i][c], acc, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float x = acc[i];
                if constexpr (NQ == 1) // the other part's column is eight lanes on
                    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true));
                sv[4 * t + i] = __builtin_amdgcn_ldexpf(x, byte_of(ke, 4 * t + i) + query);
            }
        }
        if (more) fetch_k(kb + 4, pk);
#pragma unroll
        for (int i = 0; i < NI / 2; i++) {
            const int t = (pair0 & 3) + i;
            const Steps st(nibble_pair(vu, t, k16), nibble_pair(vz, t, k16));
            steps[pair0 + i] = make_uint2(__builtin_bit_cast(uint32_t, st.u), __builtin_bit_cast(uint32_t, st.m));
        }
        if (kb * 64 + 63 > clear) {
            const int left = limit - (kb * 64 + 16 * g); // last visible token of the lane's block
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (i > left) sv[i] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) mx = fmaxf(mx, sv[i]);
        // (m and e move by what their own row sees alone, whichever rows the wave looks for)
        if (__any(mx > m + 6.f)) {
            const float mr = row_max(mx), mn = mr > m + 6.f ? ceilf(mr) : m;
            l *= m == mn ? 1.f : exp2f(m - mn);
            m = mn;
            value = -127 + (e == -INFINITY ? 0 : (int)(9.f - e + m));
        }
        const float mu = m == -INFINITY ? 0.f : m;
        // the largest score with the largest power bounds what the row's products can be (a
        // block without visible keys: -inf, or NaN with a token that is not finite)
        const int mb = most_byte(ve);
        if (__any(mx + (mb == 255 ? INFINITY : (float)(mb - 127)) > e + 6.f)) {
            float mv = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int b = byte_of(ve, i);
                if (b < 255) mv = fmaxf(mv, sv[i] + (float)(b - 127));
                else if (sv[i] > -INFINITY) l = NAN; // a token that is not finite, seen
            }
            const float mr = row_max(mv), en = mr > e + 6.f ? ceilf(mr) : e, up = e == en ? 1.f : exp2f(e - en);
#pragma unroll
            for (int s = 0; s < NS; s++) o[s] *= up;
            e = en;
            value = -127 + (e == -INFINITY ? 0 : (int)(9.f - e + mu));
        }
        float wt[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float x = __builtin_amdgcn_exp2f(sv[i] - mu);
            l += x;
            wt[i] = __builtin_amdgcn_ldexpf(x, byte_of(ve, i) + value);
        }
        half8_t pf[NQ][2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            uint32_t hi[4], lw[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x = wt[8 * c + 2 * i], y = wt[8 * c + 2 * i + 1];
                if constexpr (NQ == 2) split2_mix(x, y, hi[i], lw[i]);
                else { // the high columns keep x, the low ones what fp16 leaves of it
                    float r0, r1;
                    remainders(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y)), part, x, y, r0, r1);
                    hi[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r0, r1));
                }
            }
            pf[0][c] = __builtin_bit_cast(half8_t, make_uint4(hi[0], hi[1], hi[2], hi[3]));
            if constexpr (NQ == 2) pf[1][c] = __builtin_bit_cast(half8_t, make_uint4(lw[0], lw[1], lw[2], lw[3]));
        }
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                Steps st[4];
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const uint4 x = *(const uint4 *)&steps[8 * i + 4 * c + k];
                    st[k].u = __builtin_bit_cast(half2_t, x.x), st[k].m = __builtin_bit_cast(half2_t, x.y);
                    st[k + 1].u = __builtin_bit_cast(half2_t, x.z), st[k + 1].m = __builtin_bit_cast(half2_t, x.w);
                }
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const half8_t v = word_f16(word_of(vr[i], 2 * b + c), st, k16);
#pragma unroll
                    for (int k = 0; k < NQ; k++) o[2 * i + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[k][c], o[2 * i + b], 0, 0, 0);
                }
            }
        if (more) {
            fetch_v(kb + 4, pv);
            pk = page_of(kb + 8, n >> 2);
            pv = page_of(kb + 8, g);
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // the four waves' results, in wave order
    const MeanScale mean(e, m, l);
#pragma unroll
    for (int s = 0; s < NS; s++) *(floatx4 *)&lds.lo[wave][n][16 * s + 4 * g] = o[s] * mean.f1 * mean.f2;
    if (g == 0) {
        lds.lm[wave][n] = m;
        lds.ll[wave][n] = l;
    }
    __syncthreads();
    for (int i = tid; i < ROWS * (HD / 4); i += 256) {
        const int c = i / (HD / 4), d = 4 * (i % (HD / 4)), rr = r.row0 + c;
        if (rr >= n_rows) continue;
        float mm = lds.lm[0][c];
#pragma unroll
        for (int w = 1; w < 4; w++) mm = fmaxf(mm, lds.lm[w][c]);
        const float mu = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f, f[4];
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = lds.ll[w][c] * exp2f(lds.lm[w][c] - mu);
            sum += f[w];
        }
        const float inv = sum == 0.f && r.part >= 0 ? 0.f : 1.f / sum;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            floatx4 y = *(const floatx4 *)&lds.lo[w][c][d];
            if constexpr (NQ == 1) y += *(const floatx4 *)&lds.lo[w][c + 8][d];
            x += y * (f[w] * inv);
        }
        if (r.part < 0) {
            const int tk = rr / p.group, hd = h * p.group + rr % p.group;
            float *dst = p.out + ((size_t)(r.start + tk) * p.n_heads + hd) * HD + d;
#pragma unroll
            for (int k = 0; k < 4; k++) dst[k] = x[k];
        } else {
            float *dst = p.part + (((size_t)r.part * p.n_kv + h) * kPagesTileRows + c) * LD;
            store_shared(dst + d, x[0], x[1]);
            store_shared(dst + d + 2, x[2], x[3]);
            if (d == 0) store_shared(dst + HD, mm, sum);
        }
    }
    if (r.part >= 0) {
        // the tile's last part to arrive merges them all, in their order
        const int tiles = div_up(n_rows, kPagesTileRows), tile = r.row0 / kPagesTileRows;
        if (arrives_last(p.tickets + (size_t)(r.part0 + tile) * p.n_kv + h, r.n_parts, lds.last))
            for (int c = tid >> 4; c < min(ROWS, n_rows - r.row0); c += 16) {
                const int rr = r.row0 + c, tk = rr / p.group;
                merge_parts<HD>(
                    [&](int k) { return p.part + (((size_t)(r.part0 + k * tiles + tile) * p.n_kv + h) * kPagesTileRows + c) * LD; },
                    r.n_parts, p.out + ((size_t)(r.start + tk) * p.n_heads + h * p.group + rr % p.group) * HD, tid & 15);
            }
    }
    __syncthreads();
}

template <int HD>
struct Wide4Lds {
    union {
        struct {
            uint4 kf[2][2 * (HD / 16) * 64], vf[2][4 * (HD / 32) * 64];
            uint4 power[2][2][4]; // of 64 keys: K's, V's bytes
            int top[2][4];        // a block's largest V byte
        };
        float rows[kPagesWideRows * (HD + 4)]; // a part: means, maximum, sum
        float factor[8][kPagesWideRows];
    };
    int last;
};

// 128 (token, head) rows of a request and KV head, 32 to a wave, over its keys in blocks
// of 64: as above, with K and V turned into fp16 fragments (codes less zero points times
// steps) in LDS once for the four waves, double buffered: the next block's codes are in
// flight during a block's products and become fragments beside its scores' matrix
// instructions.  v_mfma_f32_32x32x16_f16: S^T is two tiles of 32 keys, their rows dealt so
// that a lane's sixteen scores are one block's tokens in order.
template <int HD>
__device__ __forceinline__ void attend4_wide(const Attend4View &p, Wide4Lds<HD> &lds, const PagesItem &r, int first)
{
    constexpr int NC = HD / 16, ND = HD / 32;
    constexpr Pages4 at(HD);
    auto &kf = lds.kf;
    auto &vf = lds.vf;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hh = lane >> 5, n = lane & 31, h = first % p.n_kv, item = first / p.n_kv;
    const int32_t *table = p.table + (size_t)r.id * p.width;

    const int n_rows = r.row1, wrow = r.row0 + 32 * wave;
    const bool active = wrow < n_rows;
    const int row = min(wrow + n, n_rows - 1), token = row / p.group, head = h * p.group + row % p.group;
    const int limit = r.past + token; // last visible key
    const int key1 = min(r.key1, r.past + min(n_rows - 1, r.row0 + kPagesWideRows - 1) / p.group + 1);
    const int clear = r.past + min(wrow, n_rows - 1) / p.group; // keys up to it are seen by every row of the wave
    const int last = (r.len - 1) / kPageBlock;

    // A wave stages one of 64 keys' four 16-token blocks.  Buffer loads, as in the 8-bit
    // cache: their bases are the wave's.
    const rsrc_t rt = make_rsrc(table, 4 * p.width);
    auto page_of = [&](int kb) {
        return __builtin_amdgcn_raw_buffer_load_b32(rt, 0, 4 * (min(4 * kb + wave, last) >> p.sub_shift), 0);
    };
    // A lane's share: the codes of a quarter of token lane / 4 (K) and, of all tokens, of
    // dims 32 i + n and 16 on (V, hd 64: of one), i = lane / 16; their steps.
    const int vi = lane / (HD == 128 ? 16 : 32), quarter = lane & 3;
    const int ks_at = at.ks + 4 * (4 * (HD == 128 ? quarter : quarter >> 1) + ((lane >> 2) & 3));
    uint32_t kr[HD / 32], vr[HD / 32], ks;
    uint4 vs, er;
    auto fetch = [&](int kb, int page) {
        const int c = min(4 * kb + wave, last) & (p.sub - 1);
        const size_t b = (((size_t)__builtin_amdgcn_readfirstlane(page) * p.n_kv + h) << p.sub_shift) + c;
        const rsrc_t rb = make_rsrc(p.pool + b * at.bytes, at.bytes);
        if constexpr (HD == 128) {
            const uint4 k = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rb, 16 * lane, at.k, 0));
            const uint4 v = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rb, 16 * lane, at.v, 0));
            kr[0] = k.x, kr[1] = k.y, kr[2] = k.z, kr[3] = k.w, vr[0] = v.x, vr[1] = v.y, vr[2] = v.z, vr[3] = v.w;
        } else {
            const uint2 k = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rb, 8 * lane, at.k, 0));
            const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rb, 8 * lane, at.v, 0));
            kr[0] = k.x, kr[1] = k.y, vr[0] = v.x, vr[1] = v.y;
        }
        ks = __builtin_amdgcn_raw_buffer_load_b32(rb, ks_at, 0, 0);
        vs = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rb, 16 * vi, at.vs, 0));
        er = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rb, 16 * (lane & 1), at.ke, 0));
    };
    // K's rows of the tile are dealt by quarter so that neighbouring lanes' writes take all
    // banks.  NC pieces: a lane's words of K, then of V.
    const int krow = (8 * (lane >> 4) + 4 * (wave & 1) + ((lane >> 2) & 3)) ^ (quarter << 1);
    const int vcol = 32 * (wave & 1) + (HD == 128 ? lane & 15 : 16 * (lane & 1) + ((lane >> 1) & 15));
    const uint32_t k16 = sixteen();
    Steps kst, vst[4];
    auto put = [&](int buf, int piece) {
        if (piece < NC / 2) {
            if (piece == 0) {
                kst = key_steps(nibble_pair(ks, lane >> 4, k16));
                const int most = most_byte(er);
                if (lane < 2) lds.power[buf][lane][wave] = er;
                if (lane == 1) lds.top[buf][wave] = most;
            }
            const int c = HD == 128 ? 2 * quarter + (piece >> 1) : quarter;
            (kf[buf] + ((wave >> 1) * NC + c) * 64 + krow)[32 * (piece & 1)] = __builtin_bit_cast(uint4, word_f16(kr[piece], kst, k16));
        } else {
            const int i = piece - NC / 2, j = HD == 128 ? i >> 1 : i, b = HD == 128 ? i & 1 : 0; // tokens 8 j .., dims 16 b ..
            if (b == 0) value_steps(j ? vs.y : vs.x, j ? vs.w : vs.z, vst, k16);
            (vf[buf] + ((2 * vi + (wave >> 1)) * 2 + j) * 64 + vcol)[16 * b] = __builtin_bit_cast(uint4, word_f16(vr[HD == 128 ? 2 * b + j : j], vst, k16));
        }
    };

    int kb = r.key0 / 64;
    int next = page_of(kb);
    fetch(kb, next);
    next = page_of(kb + 1);

    // Q^T fragments: dims 16 c + 8 hh .. + 7 of row n
    half8_t qh[NC], ql[NC];
    int query;
    {
        const float *src = p.q + ((size_t)(r.start + token) * p.n_heads + head) * HD + 8 * hh;
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(src[16 * c + i]));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const Query4 scaled(m, p.scale);
        query = scaled.power();
#pragma unroll
        for (int c = 0; c < NC; c++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = src[16 * c + i];
            split_query(scaled, x, qh[c], ql[c]);
        }
    }

    floatx16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = floatx16{};
    float m = -INFINITY, l = 0.f, e = -INFINITY; // m and e whole numbers; outputs are held times 2^(9 - e)
    int value = -127;                            // with a V row's byte: the power from a weight to fp16's
#pragma unroll
    for (int i = 0; i < NC; i++) put(0, i);
    fetch(kb + 1, next); // (past the last block: the last again, which nobody reads)
    next = page_of(kb + 2);
    __syncthreads();

    if (!active) { // no rows of its own: it stages for the others
        for (int buf = 0; kb * 64 < key1; kb++, buf ^= 1) {
#pragma unroll
            for (int i = 0; i < NC; i++) put(buf ^ 1, i);
            fetch(kb + 2, next);
            next = page_of(kb + 3);
            __syncthreads();
        }
    }
    for (int buf = 0; kb * 64 < key1; kb++, buf ^= 1) {
        floatx16 s[2] = {floatx16{}, floatx16{}};
        auto kfrag = [&](int t, int c) {
            return __builtin_bit_cast(half8_t, kf[buf][(t * NC + c) * 64 + (lane ^ (((HD == 128 ? c >> 1 : c) & 3) << 1))]);
        };
        half8_t k0 = kfrag(0, 0), k1 = kfrag(1, 0);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const half8_t n0 = kfrag(0, min(c + 1, NC - 1)), n1 = kfrag(1, min(c + 1, NC - 1));
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qh[c], s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qh[c], s[1], 0, 0, 0);
            put(buf ^ 1, c);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, ql[c], s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, ql[c], s[1], 0, 0, 0);
            k0 = n0, k1 = n1;
            __builtin_amdgcn_sched_barrier(0);
        }
        fetch(kb + 2, next);
        next = page_of(kb + 3);
        uint4 ve[2];
        int top[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint4 ke = lds.power[buf][0][2 * t + hh];
            ve[t] = lds.power[buf][1][2 * t + hh];
            top[t] = lds.top[buf][2 * t + hh];
#pragma unroll
            for (int i = 0; i < 16; i++) s[t][i] = __builtin_amdgcn_ldexpf(s[t][i], byte_of(ke, i) + query);
        }
        if (kb * 64 + 63 > clear) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int left = limit - (kb * 64 + 32 * t + 16 * hh); // last visible token of the lane's block
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (i > left) s[t][i] = -INFINITY;
            }
        }
        float mx[2];
        bool past_e = false;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            mx[t] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) mx[t] = fmaxf(mx[t], s[t][i]);
            // (as in attend4_tile: a bound on the row's products, NaN where a block without
            // visible keys has a token that is not finite)
            past_e |= mx[t] + (top[t] == 255 ? INFINITY : (float)(top[t] - 127)) > e + 6.f;
        }
        auto halves = [](float x) { // the larger of the lane's and the other half's
            const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
        };
        const bool past_m = fmaxf(mx[0], mx[1]) > m + 6.f;
        if (__any(past_m || past_e)) {
            if (__any(past_m)) {
                const float mr = halves(fmaxf(mx[0], mx[1])), mn = mr > m + 6.f ? ceilf(mr) : m;
                l *= m == mn ? 1.f : exp2f(m - mn);
                m = mn;
            }
            if (__any(past_e)) {
                float mv = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int b = byte_of(ve[t], i);
                        if (b < 255) mv = fmaxf(mv, s[t][i] + (float)(b - 127));
                        else if (s[t][i] > -INFINITY) l = NAN; // a token that is not finite, seen
                    }
                const float mr = halves(mv), en = mr > e + 6.f ? ceilf(mr) : e, up = e == en ? 1.f : exp2f(e - en);
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= up;
                e = en;
            }
            value = -127 + (e == -INFINITY ? 0 : (int)(9.f - e + (m == -INFINITY ? 0.f : m)));
        }
        const float mu = m == -INFINITY ? 0.f : m;
        uint32_t hi[2][8], lw[2][8];
        auto weights = [&](int t, int i) { // of tokens 2 i and 2 i + 1 of the lane's block
            const float x = __builtin_amdgcn_exp2f(s[t][2 * i] - mu), y = __builtin_amdgcn_exp2f(s[t][2 * i + 1] - mu);
            l += x;
            l += y;
            split2_mix(__builtin_amdgcn_ldexpf(x, byte_of(ve[t], 2 * i) + value),
                       __builtin_amdgcn_ldexpf(y, byte_of(ve[t], 2 * i + 1) + value), hi[t][i], lw[t][i]);
        };
        auto pfrag = [&](const uint32_t (&x)[8], int j) {
            return __builtin_bit_cast(half8_t, make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]));
        };
        auto vfrag = [&](int t, int k) { // k = ND j + d
            return __builtin_bit_cast(half8_t, vf[buf][(((k % ND) * 2 + t) * 2 + k / ND) * 64 + lane]);
        };
        half8_t v = vfrag(0, 0);
#pragma unroll
        for (int i = 0; i < 8; i++) weights(0, i);
        __builtin_amdgcn_sched_barrier(0);
        // the second tile's exponentials run beside the first's V^T P^T
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < 2 * ND; k++) {
                const half8_t ahead = t && k == 2 * ND - 1 ? v : vfrag(k == 2 * ND - 1 ? 1 : t, (k + 1) % (2 * ND));
                o[k % ND] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pfrag(hi[t], k / ND), o[k % ND], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4 / ND; i++)
                    if (!t) weights(1, 8 / ND / 2 * k + i);
                o[k % ND] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pfrag(lw[t], k / ND), o[k % ND], 0, 0, 0);
                v = ahead;
                __builtin_amdgcn_sched_barrier(0);
            }
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    wide_result<HD>(p, lds, item, h, o, MeanScale(e, m, l), m, l);
}

} // namespace

// The attention of a plan in one launch: wide tiles first, then 16-row tiles, `tiles`
// workgroups of which take turns.
template <int HD, bool WIDE>
__global__ __launch_bounds__(256, 2) void pages4_attend_kernel(Attend4View p)
{
    union Lds {
        Tile4Lds<HD> tile;
        Wide4Lds<WIDE ? HD : 32> wide;
    };
    __shared__ __align__(16) char mem[sizeof(Lds)];
    // (the first item, which is there if not of this plan, does not wait for the head)
    const bool wide = WIDE && (int)blockIdx.x < p.wides;
    const int first = wide ? blockIdx.x : (int)blockIdx.x - p.wides, h = first % p.n_kv, stride = p.tiles / p.n_kv;
    int item = first / p.n_kv;
    PagesItem it = wide ? p.wide_item[item] : p.item[item];
    const PagesPlanHead plan = *p.head;
    if (outgrown(p, plan) || item >= (wide ? plan.n_wide : plan.n_items)) return;
    if constexpr (WIDE) {
        if (wide) {
            attend4_wide<HD>(p, *(Wide4Lds<HD> *)mem, it, first);
            return;
        }
    }
    Tile4Lds<HD> &lds = *(Tile4Lds<HD> *)mem;
    while (item < plan.n_items) {
        if (it.row1 - it.row0 <= 8) attend4_tile<HD, 8>(p, lds, it, h);
        else attend4_tile<HD, 16>(p, lds, it, h);
        item += stride;
        if (item < plan.n_items) it = p.item[item];
    }
}

hipError_t launch_pages4_attend(const Pages &p, const PagesAttendArgs &a, hipStream_t s)
{
    // as many workgroups as the call's requests can need (launch_pages_attend)
    const int64_t split = (int64_t)((p.group + kPagesTileRows - 1) / kPagesTileRows) * std::min(a.n_requests, a.n_tokens);
    const int64_t parts = std::min((int64_t)p.max_parts, split * pages_most_parts(p.max_context));
    const int64_t most = a.n_tokens == 0 ? 1 : std::max<int64_t>(1, parts + (int64_t)a.n_tokens * p.group / kPagesTileRows + a.n_requests);
    const int64_t most_wide = (int64_t)a.n_tokens * p.group / kPagesWideRows + a.n_requests + pages_wide_target(p.n_kv);
    const int wides = a.wide ? (int)(most_wide * p.n_kv) : 0, tiles = (int)(most < 2048 ? most : 2048) * p.n_kv;
    const Attend4View view = {layer4_of(p, a.layer), p.table, p.head, p.item, p.wide, p.part, p.wide_part, p.tickets, p.wide_tickets,
                              a.q, a.out, p.n_kv, p.n_heads, p.group, p.sub, p.sub_shift, p.width, p.scale,
                              wides, tiles, a.n_tokens, a.n_requests, a.wide};
    auto launch = [&](auto kernel) { launch_stamped(a.ev_start, a.ev_stop, kernel, dim3(wides + tiles), dim3(256), 0, s, view); };
    if (p.hd == 128) launch(a.wide ? pages4_attend_kernel<128, true> : pages4_attend_kernel<128, false>);
    else launch(a.wide ? pages4_attend_kernel<64, true> : pages4_attend_kernel<64, false>);
    return hipGetLastError();
}

// ------------------------------------------------------------ reading back

namespace {
struct Read4View {
    const uint8_t *pool;
    const int32_t *slot;
    float *k_out, *v_out;
    int n, n_kv, page, sub, n_pages;
};
} // namespace

// Sixteen slots and one KV head to a workgroup, a slot to sixteen threads, hd / 16
// neighbouring elements to each.
template <int HD>
__global__ __launch_bounds__(256) void pages4_read_kernel(Read4View p)
{
    constexpr int NE = HD / 16;
    constexpr Pages4 at(HD);
    const int tid = threadIdx.x, h = blockIdx.y, i = blockIdx.x * 16 + (tid >> 4), d0 = NE * (tid & 15), gr = d0 / 32;
    if (i >= p.n) return;
    const int slot = p.slot[i];
    float x[2][NE] = {};
    if (slot >= 0 && slot / p.page < p.n_pages) {
        const int tk = slot % kPageBlock;
        const uint8_t *b = p.pool + (((size_t)(slot / p.page) * p.n_kv + h) * p.sub + slot % p.page / kPageBlock) * at.bytes;
        auto nibble = [](uint32_t w, int i) { return (int)((turn_left(w, 30) >> nibble_at(i)) & 15u); };
        const uint32_t kw = *(const uint32_t *)(b + at.k + tk * (HD / 2) + 4 * (d0 / 8));
        const uint32_t ks = *(const uint32_t *)(b + at.ks + 4 * (4 * gr + (tk & 3)));
        const uint32_t *vs = (const uint32_t *)(b + at.vs) + 4 * gr + (tk >> 3);
        const uint32_t vu = vs[0], vz = vs[2];
        const int ke = b[at.ke + tk], ve = b[at.ve + tk];
        uint32_t vw[NE];
#pragma unroll
        for (int k = 0; k < NE; k++) {
            const int d = d0 + k;
            vw[k] = *((const uint32_t *)(b + at.v) + 64 * gr + 4 * (d & 15) + 2 * ((d >> 4) & 1) + (tk >> 3));
        }
        const int ku = nibble(ks, 2 * (tk >> 2)), kz = nibble(ks, 2 * (tk >> 2) + 1), u = nibble(vu, tk & 7), z = nibble(vz, tk & 7);
#pragma unroll
        for (int k = 0; k < NE; k++) {
            x[0][k] = ve == 255 ? NAN : ldexpf((float)((nibble(kw, (d0 + k) & 7) - kz) * ku), ke - 127);
            x[1][k] = ve == 255 ? NAN : ldexpf((float)((nibble(vw[k], tk & 7) - z) * u), ve - 127);
        }
    }
    const size_t to = ((size_t)i * p.n_kv + h) * HD + d0;
#pragma unroll
    for (int k = 0; k < NE; k++) {
        p.k_out[to + k] = x[0][k];
        p.v_out[to + k] = x[1][k];
    }
}

hipError_t launch_pages4_read(const Pages &p, int layer, const int32_t *slot, int n, float *k, float *v, hipStream_t s)
{
    if (n <= 0) return hipSuccess;
    const Read4View view = {layer4_of(p, layer), slot, k, v, n, p.n_kv, p.page, p.sub, p.n_pages};
    const dim3 grid((n + 15) / 16, p.n_kv);
    if (p.hd == 128) hipLaunchKernelGGL(pages4_read_kernel<128>, grid, dim3(256), 0, s, view);
    else hipLaunchKernelGGL(pages4_read_kernel<64>, grid, dim3(256), 0, s, view);
    return hipGetLastError();
}

} // namespace jev
