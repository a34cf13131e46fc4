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

// A word's eight elements, with the same step for all.
__device__ __forceinline__ half8_t word_f16(uint32_t w, const Steps &s, uint32_t k16)
{
    return __builtin_bit_cast(half8_t, make_uint4(s(nibble_pair<0>(w, k16)), s(nibble_pair<1>(w, k16)), s(nibble_pair<2>(w, k16)),
                                                  s(nibble_pair<3>(w, k16))));
}
// Of a K step word's pair (u of a token's group low, its z high), for all of the group.
__device__ __forceinline__ Steps key_steps(half2_t uz) { return Steps(half2_t{uz[0], uz[0]}, half2_t{uz[1], uz[1]}); }
// V's step word of a quad and group: pairs u of tokens 0 and 1, of 2 and 3, z of the same.
struct QuadSteps {
    Steps s[2];
    QuadSteps() = default;
    __device__ __forceinline__ QuadSteps(uint32_t w, uint32_t k16)
        : s{Steps(nibble_pair<0>(w, k16), nibble_pair<2>(w, k16)), Steps(nibble_pair<1>(w, k16), nibble_pair<3>(w, k16))} {}
    // A V code word: tokens 0 .. 3 of a dim, then of the dim 16 on, two words of fp16 each.
    __device__ __forceinline__ uint4 operator()(uint32_t w, uint32_t k16) const
    {
        return make_uint4(s[0](nibble_pair<0>(w, k16)), s[1](nibble_pair<1>(w, k16)), s[0](nibble_pair<2>(w, k16)), s[1](nibble_pair<3>(w, k16)));
    }
};

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ int byte_of(uint32_t w, int i) { return (int)((w >> (8 * i)) & 255u); }

// The largest of the words' bytes.
template <int N>
__device__ __forceinline__ int most_byte(const uint32_t (&w)[N])
{
    typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
    ushort2_t m = {0, 0};
#pragma unroll
    for (int i = 0; i < N; i++) {
        m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2_t, w[i] & 0x00ff00ffu));
        m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2_t, (w[i] >> 8) & 0x00ff00ffu));
    }
    return max((int)m[0], (int)m[1]);
}

uint8_t *layer4_of(const Pages &p, int layer) { return p.k + (size_t)layer * p.n_blocks() * pages4_bytes(p.hd); }

// The largest of four, eight or sixteen neighbouring lanes' values (aligned), on all of them.
template <int N>
__device__ __forceinline__ unsigned most_of(unsigned x)
{
    auto other = [&](auto ctrl) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true); };
    x = max(x, other(std::integral_constant<int, 0xb1>())); // lane ^ 1
    x = max(x, other(std::integral_constant<int, 0x4e>())); // lane ^ 2
    if (N >= 8) x = max(x, other(std::integral_constant<int, 0x141>())); // the half row mirrored
    if (N >= 16) x = max(x, other(std::integral_constant<int, 0x140>())); // the row mirrored
    return x;
}

// y / u to the nearest whole number, a half to the even one; u whole, 1 .. 15, |y| <= 225.
// The remainder is exact: it is a multiple of y's last bit and not larger than y or u.
__device__ __forceinline__ float whole_steps(float y, float u, float inv)
{
    const float q = rintf(y * inv), rest = fmaf(-q, u, y), twice = 2.f * fabsf(rest);
    const bool other = (twice > u) | ((twice == u) & (bool)((int)q & 1));
    return q + (other ? copysignf(1.f, rest) : 0.f);
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
// they are formed.  One token (32 query heads, 8 KV heads of 128) takes 6.3 us, a launch and
// a chain of trips to memory (arguments, plan and unit, rows and the block's words); 64 7.5;
// 8000 of a prompt 81, 326 MB at 4.1 TB/s.
template <int HD, bool VEC>
__global__ __launch_bounds__(256) void pages4_store_kernel(Store4View p)
{
    constexpr int NP = HD / 32, NE = HD / 16, NG = HD / 32, TG = 32 / NE, LD = HD + 4, RING = 2;
    constexpr Pages4 at(HD);
    __shared__ __align__(16) float xs[2][kPageBlock][LD];
    __shared__ uint8_t code[kPageBlock][HD];                    // V's
    __shared__ uint8_t step[2][kPageBlock][NG], zero[2][kPageBlock][NG];
    __shared__ uint16_t power[2][kPageBlock]; // bytes, or kNotFinite
    constexpr uint16_t kNotFinite = 256;
    const int tid = threadIdx.x, j = tid & 15, h = blockIdx.y;
    const PagesUnit un = p.unit[blockIdx.x];
    PagesPlanHead plan = *p.head;
    asm volatile("" : "+s"(plan.n_tokens), "+s"(plan.n_requests), "+s"(plan.n_units), "+s"(plan.n_wide) : "s"(un.row)); // one wait for all
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

    // steps and codes of a token's elements NE j ..: of its key and value, or with up to
    // eight tokens of one of them
    const bool apart = n <= 8;
    const int tk = apart ? tid >> 4 & 7 : tid >> 4, v0 = apart ? tid >> 7 : 0, v1 = apart ? v0 + 1 : 2;
    if (tk < n) {
        for (int v = v0; v < v1; v++) {
            float x[NE], hi = 0.f, lo = 0.f;
            unsigned bits = 0; // a value that is not finite has the largest
#pragma unroll
            for (int i = 0; i < NE; i++) {
                x[i] = xs[v][tk][NE * j + i];
                hi = fmaxf(hi, x[i]);
                lo = fmaxf(lo, -x[i]);
                bits = max(bits, __float_as_uint(fabsf(x[i])));
            }
            // (numbers from zero are ordered as their bits)
            hi = __uint_as_float(most_of<TG>(__float_as_uint(hi)));
            lo = __uint_as_float(most_of<TG>(__float_as_uint(lo)));
            const float span = 0.5f * hi + 0.5f * lo; // half the group's span: the whole one may be past fp32's range
            const float most = __uint_as_float(most_of<16>(__float_as_uint(span)));
            bits = most_of<16>(bits);
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
                const float q = whole_steps(ldexpf(x[i], -ex), u, inv) + z;
                const uint32_t c = some ? (uint32_t)(int)fminf(fmaxf(q, 0.f), 15.f) : 0u;
                if (v) code[tk][NE * j + i] = (uint8_t)c;
                else word |= c << nibble_at((NE * j + i) & 7);
            }
            if (!v) {
                if (NE == 4) word |= (uint32_t)__shfl_xor((int)word, 1, 64);
                const int w8 = NE * j / 8; // eight dims of them
                if (NE == 8 || !(j & 1)) *((uint32_t *)(block + at.k) + (w8 / NG * kPageBlock + off + tk) * NG + w8 % NG) = turn_left(word, 2);
            }
            if (j % TG == 0) {
                step[v][tk][j / TG] = (uint8_t)(int)u;
                zero[v][tk][j / TG] = (uint8_t)(int)z;
            }
            if (j == 0) power[v][tk] = (uint16_t)(bits >= 0x7f800000u ? kNotFinite : some ? ex + 127 : 0);
        }
    }
    __syncthreads();

    // a value that is not finite: the token's V power says so for both
    if (tid < 2 * n) {
        const int t = tid >> 1, v = tid & 1;
        const bool bad = max(power[0][t], power[1][t]) == kNotFinite;
        block[at.pw + (off + t) / 4 * 8 + 4 * v + (off + t) % 4] = (uint8_t)(bad ? v ? 255 : 0 : power[v][t]);
    }
    // words over several tokens: the new ones' nibbles among what is there
    auto merge = [&](uint32_t old, auto token, auto nibble) {
        uint32_t put = 0, mask = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int tk = token(i) - off;
            const uint32_t x = nibble(i, tk & 15); // (read whether it is one or not: the reads go out together)
            const uint32_t m = tk < 0 || tk >= n ? 0u : 15u << nibble_at(i);
            put |= (x << nibble_at(i)) & m;
            mask |= m;
        }
        mask = turn_left(mask, 2);
        return make_uint2((old & ~mask) | turn_left(put, 2), mask);
    };
    if (has_v) {
        const int q = tid / (16 * NG), dim = 32 * (tid % NG) + tid / NG % 16;
        const uint2 r = merge(old_v, [&](int i) { return 4 * q + (i & 3); }, [&](int i, int tk) { return code[tk][dim + 4 * (i & 4)]; });
        if (r.y) *vword = r.x;
    }
    if (has_s) {
        uint2 r;
        if (tid < 4 * NG) { // K: u of a token, z of it, the quad's next token
            const int gr = tid >> 2, q = tid & 3;
            r = merge(old_s, [&](int i) { return 4 * q + (i >> 1); }, [&](int i, int tk) { return i & 1 ? zero[0][tk][gr] : step[0][tk][gr]; });
        } else {
            const int gr = tid % NG, q = (tid - 4 * NG) / NG;
            r = merge(old_s, [&](int i) { return 4 * q + (i & 3); }, [&](int i, int tk) { return i & 4 ? zero[1][tk][gr] : step[1][tk][gr]; });
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

// x of the lanes whose number differs in bits 16 and 32, joined by `op`, on all of them.
template <typename Op>
__device__ __forceinline__ float over_quarters(float x, Op op)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// x of T neighbouring lanes (16, 32 or 64, aligned) joined by `op`, on all of them.
template <int T, typename Op>
__device__ __forceinline__ float over_lanes(float x, Op op)
{
    auto other = [&](auto ctrl) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
    x = op(x, other(std::integral_constant<int, 0xb1>()));  // lane ^ 1
    x = op(x, other(std::integral_constant<int, 0x4e>()));  // lane ^ 2
    x = op(x, other(std::integral_constant<int, 0x141>())); // the half row mirrored
    x = op(x, other(std::integral_constant<int, 0x140>())); // the row mirrored
    if constexpr (T == 64) x = over_quarters(x, op);
    else if constexpr (T == 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    return x;
}

// One row's parts (merge_parts) by T threads of a wave, at most T of them, their maxima whole
// numbers or -inf: a part's maximum and sum to a thread, and the first parts' rows under way
// beside them, so that memory is waited for once (four parts of four rows 10000 -> 2500 cycles).
template <int HD, int T, typename At>
__device__ __forceinline__ void merge4_parts(At at, int n_parts, float *dst, int j)
{
    constexpr int N = HD / 2 / T, B = 8;
    const int first = 4 * (threadIdx.x & 63 & ~(T - 1)); // of the row's lanes
    float2 ml = make_float2(-INFINITY, 0.f), y[B][N];
    if (j < n_parts) ml = load_shared(at(j) + HD);
    auto fetch = [&](int k0) {
#pragma unroll
        for (int k = 0; k < B; k++)
            if (k0 + k < n_parts)
#pragma unroll
                for (int i = 0; i < N; i++) y[k][i] = load_shared(at(k0 + k) + 2 * (T * i + j));
    };
    fetch(0);
    const float m = over_lanes<T>(ml.x, fmaxf), mu = m == -INFINITY ? 0.f : m;
    const float w = ldexpf(ml.y, (int)fmaxf(ml.x - mu, -300.f)), f = w * (1.f / over_lanes<T>(w, [](float a, float b) { return a + b; }));
    float2 x[N] = {};
    for (int k0 = 0; k0 < n_parts; k0 += B) {
        if (k0) fetch(k0);
#pragma unroll
        for (int k = 0; k < B; k++) {
            if (k0 + k >= n_parts) break;
            const float fk = __int_as_float(__builtin_amdgcn_ds_bpermute(first + 4 * (k0 + k), __float_as_int(f)));
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = make_float2(x[i].x + y[k][i].x * fk, x[i].y + y[k][i].y * fk);
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        dst[2 * (T * i + j)] = x[i].x;
        dst[2 * (T * i + j) + 1] = x[i].y;
    }
}

template <int HD>
struct Tile4Lds {
    uint4 q[2][HD / 32][64]; // [part][dims][lane]; eight rows: both parts in [0]
    struct Wave {
        union {
            uint4 steps[4][4][HD / 32]; // V's of 64 keys: [block][quad][group of dims]
            float rows[16][HD + 4];     // at the end: the means
        };
        float m[16], l[16];
    } wave[4];
    int last;
};

// Up to sixteen (token, head) rows of a request and KV head over keys [key0, key1) of its
// pages; the four waves take 64 keys (four blocks) in turn and merge at the end.  S^T =
// K Q^T, a block of sixteen keys to a product: a lane's scores are four tokens of each of the
// four blocks, and its weights the P^T operand of O^T += V^T P^T as they stand.  q and p
// enter as fp16 pairs (hi + lo, ~22 bits): up to eight rows (!BOTH) as the high and low eight
// of the operand's sixteen columns, one matrix instruction a product, more (BOTH) as two
// operands.  A weight is 2^(score - m); the V operand's 2^e and the row's own power are
// added to its exponent, so that what enters fp16 is relative to the row's heaviest product
// so far (times 2^9), over the keys that the row sees.
// Codes become fp16 by a mask and a fused multiply-add a pair: of 64 keys' ~640 vector
// instructions (hd 128) 350, and with scores and weights they take longer than the matrix
// cores' 32 and, below three waves a SIMD, than memory.  So 168 registers: queries
// in LDS, V's steps made once for sixteen lanes, block addresses the wave's (two waves a SIMD
// 94 us for 64 tokens over 500 to 12000 keys, three 84; with loads free of branches 80, 285 MB
// at 3.6 TB/s).  One token over 120000 keys 44 us (133 MB, 3 TB/s and the parts' merge), over
// 4000 14.3, over 300 8.6: there waves wait for each other's trips to memory, ~1800 cycles an
// iteration of 2400 of work.  K and V a 64-key block further ahead, in LDS, gained nothing.
template <int HD, bool BOTH>
__device__ __forceinline__ void attend4_tile(const Attend4View &p, Tile4Lds<HD> &lds, const PagesItem &r, int h)
{
    constexpr int NC = HD / 32, NS = HD / 16, LD = HD + 4, ROWS = BOTH ? 16 : 8;
    constexpr Pages4 at(HD);
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid)); // what follows from it is not kept from item to item: registers
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, n = lane & 15;
    const int n_rows = r.row1;
    const uint32_t k16 = sixteen();
    auto &own = lds.wave[wave];
    const int32_t *table = p.table + (size_t)r.id * p.width;
    // columns past the request's rows repeat its last one
    const int row = min(r.row0 + (n & (ROWS - 1)), n_rows - 1);
    const int token = row / p.group, head = h * p.group + row % p.group;
    const int limit = r.past + token; // last visible key
    // the tile's last visible key; keys up to `clear` are seen by every row
    const int top = r.past + min(n_rows - 1, r.row0 + ROWS - 1) / p.group;
    const int key1 = min(r.key1, top + 1), clear = r.past + r.row0 / p.group;
    const int last = (r.len - 1) / kPageBlock; // blocks past it are read as this one, and masked

    // the pages of 64 keys' four blocks, a lane each; then the blocks are the wave's, and a
    // lane's place in all of them is the same
    auto pages_of = [&](int kb) { return table[min(4 * kb + (lane & 3), last) >> p.sub_shift]; };
    const uint32_t page_bytes = (uint32_t)(p.n_kv << p.sub_shift) * at.bytes;
    const uint8_t *const pool = p.pool + (size_t)((h << p.sub_shift) * at.bytes);
    const uint32_t codes_at = 4 * NC * lane, ks_at = at.ks + 4 * (4 * (g * NC / 4) + (n >> 2)), vs_at = at.vs + 4 * (lane & (4 * NC - 1));
    uint32_t kr[4][NC], vr[4][NC], ks[4], vs[4];
    uint2 power[4]; // K's of the lane's tokens of a block, V's
    rsrc_t block[4];
    // (past the wave's keys buffers without bytes, which cost no traffic: as branches the
    // loads' waits would be for the worst way through them)
    auto blocks_of = [&](int kb, int pages) {
        const int bytes = kb * 64 < key1 ? at.bytes : 0;
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const uint32_t page = __builtin_amdgcn_readlane(pages, b), sub = min(4 * kb + b, last) & (p.sub - 1);
            block[b] = make_rsrc(pool + (uint64_t)page * page_bytes + sub * at.bytes, bytes);
        }
    };
    auto load = [&](uint32_t (&to)[NC], const rsrc_t &from, int offset) {
        if constexpr (NC == 4) {
            const uint4 x = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(from, codes_at, offset, 0));
            to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
        } else {
            const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(from, codes_at, offset, 0));
            to[0] = x.x, to[1] = x.y;
        }
    };
    auto fetch_k = [&] {
#pragma unroll
        for (int b = 0; b < 4; b++) {
            load(kr[b], block[b], at.k);
            ks[b] = __builtin_amdgcn_raw_buffer_load_b32(block[b], ks_at, 0, 0);
        }
    };
    auto fetch_v = [&] {
#pragma unroll
        for (int b = 0; b < 4; b++) {
            power[b] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(block[b], 8 * g, at.pw, 0));
            load(vr[b], block[b], at.v);
            vs[b] = __builtin_amdgcn_raw_buffer_load_b32(block[b], vs_at, 0, 0);
        }
    };
    int kb = r.key0 / 64 + wave;
    int pages = pages_of(kb);
    float qx[NC][8]; // under way while the page's number is
    {
        const float *src = p.q + ((size_t)(r.start + token) * p.n_heads + head) * HD + 8 * NC * g;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) qx[c][i] = src[8 * c + i];
    }
    blocks_of(kb, pages);
    pages = pages_of(kb + 4);
    fetch_k();
    fetch_v();

    // Q^T fragments: dims 8 NC g + 8 c .. + 7 of column n
    int query;
    const float part = n < 8 ? 0.f : -1.f; // a column's part of a query or a weight
    {
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(qx[c][i]));
        const Query4 scaled(over_quarters(m, fmaxf), p.scale);
        query = scaled.power();
        asm("" : "+v"(query)); // one number: its -127 would be added to each byte by itself
        // a wave makes a quarter of the fragments, in LDS for all (and for each 64 keys'
        // products again: registers)
#pragma unroll
        for (int c = 0; c < NC; c++) {
            if (c != wave) continue;
            if constexpr (BOTH) {
                half8_t hi, lo;
                split_query(scaled, qx[c], hi, lo);
                lds.q[0][c][lane] = __builtin_bit_cast(uint4, hi);
                lds.q[1][c][lane] = __builtin_bit_cast(uint4, lo);
            } else lds.q[0][c][lane] = __builtin_bit_cast(uint4, split_query(scaled, qx[c], part));
        }
    }
    __syncthreads();

    floatx4 o[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) o[s] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f, e = -INFINITY; // m and e whole numbers; outputs are held times 2^(9 - e)
    int value = -127;                            // with a V row's byte: the power from a weight to fp16's

    auto row_max = [](float x) { return over_quarters(x, fmaxf); };
    auto both = [](float x) { // both parts' sum: the other's column is eight lanes on
        if constexpr (!BOTH) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true));
        return x;
    };
    for (; kb * 64 < key1; kb += 4) {
        float sv[16]; // [block][token of the lane's quad]
        {
            half8_t qf[1 + BOTH][NC];
#pragma unroll
            for (int i = 0; i <= BOTH; i++)
#pragma unroll
                for (int c = 0; c < NC; c++) qf[i][c] = __builtin_bit_cast(half8_t, lds.q[i][c][lane]);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const Steps st = key_steps(nibble_pair(ks[b], n & 3, k16));
                floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const half8_t k = word_f16(kr[b][c], st, k16);
#pragma unroll
                    for (int i = 0; i <= BOTH; i++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[i][c], acc, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) sv[4 * b + i] = __builtin_amdgcn_ldexpf(both(acc[i]), byte_of(power[b].x, i) + query);
            }
        }
        blocks_of(kb + 4, pages);
        pages = pages_of(kb + 8);
        fetch_k();
        // V's steps, a quad's and group's to a lane, for the sixteen lanes that want them
        {
            const int b = lane / (4 * NC) & 3;
            const uint32_t w = b == 0 ? vs[0] : b == 1 ? vs[1] : b == 2 ? vs[2] : vs[3];
            const QuadSteps st(w, k16);
            if (NC == 4 || lane < 32)
                (&own.steps[0][0][0])[lane] = make_uint4(__builtin_bit_cast(uint32_t, st.s[0].u), __builtin_bit_cast(uint32_t, st.s[0].m),
                                                         __builtin_bit_cast(uint32_t, st.s[1].u), __builtin_bit_cast(uint32_t, st.s[1].m));
        }
        if (kb * 64 + 63 > clear) {
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int left = limit - (kb * 64 + 16 * b + 4 * g); // last visible token of the lane's quad
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (i > left) sv[4 * b + i] = -INFINITY;
            }
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
        // the largest score with the largest power bounds what the row's products can be
        // (without visible keys: -inf, or NaN with a token that is not finite)
        uint32_t vp[4] = {power[0].y, power[1].y, power[2].y, power[3].y};
        const int mb = most_byte(vp);
        if (__any(mx + (mb == 255 ? INFINITY : (float)(mb - 127)) > e + 6.f)) {
            float mv = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int b = byte_of(vp[i >> 2], i & 3);
                if (b < 255) mv = fmaxf(mv, sv[i] + (float)(b - 127));
                else if (sv[i] > -INFINITY) l = NAN; // a token that is not finite, seen
            }
            const float mr = row_max(mv), en = mr > e + 6.f ? ceilf(mr) : e, up = e == en ? 1.f : exp2f(e - en);
#pragma unroll
            for (int s = 0; s < NS; s++) o[s] *= up;
            e = en;
            value = -127 + (e == -INFINITY ? 0 : (int)(9.f - e + mu));
        }
        asm("" : "+v"(vp[0]), "+v"(vp[1]), "+v"(vp[2]), "+v"(vp[3])); // (bytes taken above are not kept: 16 registers)
        half8_t pf[1 + BOTH][2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            uint32_t w[4], lw[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = 8 * c + 2 * i;
                float x = __builtin_amdgcn_exp2f(sv[t] - mu), z = __builtin_amdgcn_exp2f(sv[t + 1] - mu), r0, r1;
                l += x;
                l += z;
                x = __builtin_amdgcn_ldexpf(x, byte_of(vp[t >> 2], t & 3) + value);
                z = __builtin_amdgcn_ldexpf(z, byte_of(vp[t >> 2], (t & 3) + 1) + value);
                if constexpr (BOTH) split2_mix(x, z, w[i], lw[i]);
                else { // the high columns keep the weights, the low ones what fp16 leaves of them
                    remainders(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, z)), part, x, z, r0, r1);
                    w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r0, r1));
                }
            }
            pf[0][c] = __builtin_bit_cast(half8_t, make_uint4(w[0], w[1], w[2], w[3]));
            if constexpr (BOTH) pf[1][c] = __builtin_bit_cast(half8_t, make_uint4(lw[0], lw[1], lw[2], lw[3]));
        }
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int j = 0; j < NC; j++) { // dims 32 j .., of two blocks
                uint4 v[2];
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const uint4 x = own.steps[2 * c + b][g][j];
                    QuadSteps st;
                    st.s[0].u = __builtin_bit_cast(half2_t, x.x), st.s[0].m = __builtin_bit_cast(half2_t, x.y);
                    st.s[1].u = __builtin_bit_cast(half2_t, x.z), st.s[1].m = __builtin_bit_cast(half2_t, x.w);
                    v[b] = st(vr[2 * c + b][j], k16);
                }
                const half8_t v0 = __builtin_bit_cast(half8_t, make_uint4(v[0].x, v[0].y, v[1].x, v[1].y)); // dims 32 j + n
                const half8_t v1 = __builtin_bit_cast(half8_t, make_uint4(v[0].z, v[0].w, v[1].z, v[1].w)); // and 16 on
#pragma unroll
                for (int i = 0; i <= BOTH; i++) {
                    o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[i][c], o[2 * j], 0, 0, 0);
                    o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[i][c], o[2 * j + 1], 0, 0, 0);
                }
            }
        fetch_v();
    }
    l = over_quarters(l, [](float a, float b) { return a + b; });

    // the waves' results, in wave order
    const MeanScale mean(e, m, l);
#pragma unroll
    for (int s = 0; s < NS; s++) {
        floatx4 x = o[s] * mean.f1 * mean.f2;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = both(x[i]);
        if (n < ROWS) *(floatx4 *)&own.rows[n][16 * s + 4 * g] = x;
    }
    if (lane < ROWS) {
        own.m[lane] = m;
        own.l[lane] = l;
    }
    __syncthreads();
    for (int i = tid; i < ROWS * (HD / 4); i += 256) {
        const int c = i / (HD / 4), d = 4 * (i % (HD / 4)), rr = r.row0 + c;
        if (rr >= n_rows) continue;
        float mm = -INFINITY;
        for (int w = 0; w < 4; w++) mm = fmaxf(mm, lds.wave[w].m[c]);
        const float mu = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f, f[4];
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = ldexpf(lds.wave[w].l[c], (int)fmaxf(lds.wave[w].m[c] - mu, -300.f)); // (whole numbers)
            sum += f[w];
        }
        const float inv = sum == 0.f && r.part >= 0 ? 0.f : 1.f / sum;
#pragma unroll
        for (int w = 0; w < 4; w++) x += *(const floatx4 *)&lds.wave[w].rows[c][d] * (f[w] * inv);
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
        if (arrives_last(p.tickets + (size_t)(r.part0 + tile) * p.n_kv + h, r.n_parts, lds.last)) {
            const int rows = min(ROWS, n_rows - r.row0);
            auto merge = [&](auto threads) { // a row to that many
                constexpr int T = decltype(threads)::value;
                const int c = tid / T, rr = r.row0 + c, tk = rr / p.group;
                if (c >= rows) return;
                auto at = [&](int k) { return p.part + (((size_t)(r.part0 + k * tiles + tile) * p.n_kv + h) * kPagesTileRows + c) * LD; };
                float *dst = p.out + ((size_t)(r.start + tk) * p.n_heads + h * p.group + rr % p.group) * HD;
                if (r.n_parts <= T) merge4_parts<HD, T>(at, r.n_parts, dst, tid % T);
                else if (tid % T < 16) merge_parts<HD>(at, r.n_parts, dst, tid % T);
            };
            if constexpr (BOTH) merge(std::integral_constant<int, 16>());
            else if (HD == 128 && rows <= 4) merge(std::integral_constant<int, HD == 128 ? 64 : 32>());
            else merge(std::integral_constant<int, 32>());
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
// that a lane's sixteen scores are one block's tokens in order.  Four prompts of 300 to 4000
// tokens behind 1 to 700 take 330 to 350 us (123 GFLOP, each twice: 740 TFLOP/s) where 16-row
// tiles took 633.  The matrix cores are busy 47 % of the time at 1.93 GHz: under them the
// clock falls with the power drawn, and vector work adds to it (without the products' low
// halves 254 us, without the staging 314, without the weights' exponents 312).
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
    // A lane's share: a part of a token's codes (K), and four tokens' of dims 16 s + t (V)
    const int t = lane & 15, quad = lane >> 4;
    const int ks_at = at.ks + 4 * (4 * (quad * ND / 4) + (t >> 2));
    uint32_t kr[ND], vr[ND], vs, ks, er;
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
        vs = __builtin_amdgcn_raw_buffer_load_b32(rb, 4 * (ND * quad + t % ND), at.vs, 0);
        er = __builtin_amdgcn_raw_buffer_load_b32(rb, 4 * (lane & 7), at.pw, 0); // a quad's powers, K's and V's in turn
    };
    // NC pieces: a lane's words of K, then of V (four tokens of two dims each).
    const int krow = 8 * (t >> 2) + 4 * (wave & 1) + (t & 3), vcol = 32 * (wave & 1) + t;
    const uint32_t k16 = sixteen();
    Steps kst;
    uint4 vst; // of group t % ND, for the lanes beside
    auto put = [&](int buf, int piece) {
        if (piece < ND) {
            if (piece == 0) {
                kst = key_steps(nibble_pair(ks, t & 3, k16));
                const uint32_t w[1] = {er};
                const int most = most_byte(w);
                const int top = max(max(__builtin_amdgcn_readlane(most, 1), __builtin_amdgcn_readlane(most, 3)),
                                    max(__builtin_amdgcn_readlane(most, 5), __builtin_amdgcn_readlane(most, 7)));
                if (lane < 8) ((uint32_t *)&lds.power[buf][lane & 1][wave])[lane >> 1] = er;
                if (lane == 0) lds.top[buf][wave] = top;
            }
            const int c = HD == 128 ? 2 * quad + (piece >> 1) : quad;
            (kf[buf] + ((wave >> 1) * NC + c) * 64 + krow)[32 * (piece & 1)] = __builtin_bit_cast(uint4, word_f16(kr[piece], kst, k16));
        } else {
            const int j = piece - ND;
            if (j == 0) {
                const QuadSteps own(vs, k16);
                vst = make_uint4(__builtin_bit_cast(uint32_t, own.s[0].u), __builtin_bit_cast(uint32_t, own.s[0].m),
                                 __builtin_bit_cast(uint32_t, own.s[1].u), __builtin_bit_cast(uint32_t, own.s[1].m));
            }
            auto of = [&](uint32_t x) { // lane j's of four
                const int y = (int)x;
                return __builtin_bit_cast(half2_t, j == 0   ? __builtin_amdgcn_mov_dpp(y, 0x00, 0xf, 0xf, true)
                                                   : j == 1 ? __builtin_amdgcn_mov_dpp(y, 0x55, 0xf, 0xf, true)
                                                   : j == 2 ? __builtin_amdgcn_mov_dpp(y, 0xaa, 0xf, 0xf, true)
                                                            : __builtin_amdgcn_mov_dpp(y, 0xff, 0xf, 0xf, true));
            };
            QuadSteps st;
            st.s[0].u = of(vst.x), st.s[0].m = of(vst.y), st.s[1].u = of(vst.z), st.s[1].m = of(vst.w);
            const uint4 v = st(vr[j], k16);
            uint2 *to = (uint2 *)(vf[buf] + ((2 * j + (wave >> 1)) * 2 + (quad >> 1)) * 64 + vcol) + (quad & 1);
            to[0] = make_uint2(v.x, v.y);
            to[32] = make_uint2(v.z, v.w);
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
        asm("" : "+v"(query)); // one number: its -127 would be added to each byte by itself
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
            return __builtin_bit_cast(half8_t, kf[buf][(t * NC + c) * 64 + lane]);
        };
        half8_t k0 = kfrag(0, 0), k1 = kfrag(1, 0);
        __builtin_amdgcn_s_setprio(1); // of two waves, the one with products to issue goes first (9 prompts of 48 over 4096 keys 104 -> 100 us)
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
        __builtin_amdgcn_s_setprio(0);
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
            for (int i = 0; i < 16; i++) s[t][i] = __builtin_amdgcn_ldexpf(s[t][i], byte_of(word_of(ke, i >> 2), i & 3) + query);
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
                        const int b = byte_of(word_of(ve[t], i >> 2), i & 3);
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
            split2_mix(__builtin_amdgcn_ldexpf(x, byte_of(word_of(ve[t], i >> 1), 2 * (i & 1)) + value),
                       __builtin_amdgcn_ldexpf(y, byte_of(word_of(ve[t], i >> 1), 2 * (i & 1) + 1) + value), hi[t][i], lw[t][i]);
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
        __builtin_amdgcn_s_setprio(1);
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
        __builtin_amdgcn_s_setprio(0);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    wide_result<HD>(p, lds, item, h, o, MeanScale(e, m, l), m, l);
}

} // namespace

// The attention of a plan in one launch: wide tiles first, then 16-row tiles, `tiles`
// workgroups of which take turns.
template <int HD, bool WIDE>
__global__ __launch_bounds__(256, WIDE ? 2 : 3) void pages4_attend_kernel(Attend4View p)
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
    auto scalar = [](int &x) { x = __builtin_amdgcn_readfirstlane(x); };
    while (item < plan.n_items) {
        // the workgroup's, so held in scalar registers
        scalar(it.id), scalar(it.start), scalar(it.past), scalar(it.len), scalar(it.row0), scalar(it.row1);
        scalar(it.key0), scalar(it.key1), scalar(it.part), scalar(it.part0), scalar(it.n_parts);
        if (it.row1 - it.row0 > 8) attend4_tile<HD, true>(p, lds, it, h);
        else attend4_tile<HD, false>(p, lds, it, h);
        item += stride;
        if (item < plan.n_items) it = p.item[item];
    }
}

hipError_t launch_pages4_attend(const Pages &p, const PagesAttendArgs &a, hipStream_t s)
{
    // as many workgroups as the call's requests can need (launch_pages_attend; with a token
    // each: where one has more, the workgroups take turns)
    const int64_t each = (int64_t)std::min(a.n_requests, a.n_tokens) * pages_most_parts(p.max_context);
    const int64_t few = a.n_tokens > a.n_requests ? std::min(each * p.few, (int64_t)kPagesFewWgs / p.n_kv) : 0;
    const int64_t split = a.wide ? p.split : (p.group + kPagesTileRows - 1) / kPagesTileRows;
    const int64_t parts = std::min((int64_t)p.max_parts, std::max(each * split, few));
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

// Sixteen slots and one KV head to a workgroup, a slot to sixteen threads: hd / 16
// neighbouring elements of K to each, and of V the dims that its words hold, 16 apart (V
// gathered word by word for neighbouring dims: 47 us for 8000 tokens of 8 heads of 128, so
// 17, 65 MB of values at 4 TB/s).
template <int HD>
__global__ __launch_bounds__(256) void pages4_read_kernel(Read4View p)
{
    constexpr int NE = HD / 16, NG = HD / 32;
    constexpr Pages4 at(HD);
    typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4))); // the caller's alignment
    const int tid = threadIdx.x, h = blockIdx.y, i = blockIdx.x * 16 + (tid >> 4), j = tid & 15, d0 = NE * j, gr = d0 / 32;
    if (i >= p.n) return;
    const int slot = p.slot[i];
    float x[2][NE] = {};
    if (slot >= 0 && slot / p.page < p.n_pages) {
        const int tk = slot % kPageBlock, q = tk / 4, t = tk % 4, w8 = d0 / 8;
        const uint8_t *b = p.pool + (((size_t)(slot / p.page) * p.n_kv + h) * p.sub + slot % p.page / kPageBlock) * at.bytes;
        auto nibble = [](uint32_t w, int i) { return (int)((turn_left(w, 30) >> nibble_at(i)) & 15u); };
        const uint32_t kw = ((const uint32_t *)(b + at.k))[(w8 / NG * kPageBlock + tk) * NG + w8 % NG];
        const uint32_t ks = ((const uint32_t *)(b + at.ks))[4 * gr + q];
        const int ke = b[at.pw + 8 * q + t], ve = b[at.pw + 8 * q + 4 + t];
        uint32_t vw[NG], vs[NG];
#pragma unroll
        for (int g = 0; g < NG; g++) {
            vw[g] = ((const uint32_t *)(b + at.v))[(16 * q + j) * NG + g];
            vs[g] = ((const uint32_t *)(b + at.vs))[NG * q + g];
        }
        const int ku = nibble(ks, 2 * t), kz = nibble(ks, 2 * t + 1);
#pragma unroll
        for (int k = 0; k < NE; k++) {
            const int g = k / 2;
            x[0][k] = ve == 255 ? NAN : ldexpf((float)((nibble(kw, (d0 + k) & 7) - kz) * ku), ke - 127);
            x[1][k] = ve == 255 ? NAN : ldexpf((float)((nibble(vw[g], t + 4 * (k & 1)) - nibble(vs[g], 4 + t)) * nibble(vs[g], t)), ve - 127);
        }
    }
    const size_t to = ((size_t)i * p.n_kv + h) * HD;
#pragma unroll
    for (int k = 0; k < NE; k += 4) {
        const floatx4_any y = {x[0][k], x[0][k + 1], x[0][k + 2], x[0][k + 3]};
        *(floatx4_any *)(p.k_out + to + d0 + k) = y;
    }
#pragma unroll
    for (int k = 0; k < NE; k++) p.v_out[to + 16 * k + j] = x[1][k];
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
