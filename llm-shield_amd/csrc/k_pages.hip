// The 8-bit paged KV cache (Pages in jev_internal.h): a step's plan from the
// requests' lengths, rotary positions with the store, attention, reading back.
#include <algorithm>

#include "jev_pages_dev.h"

namespace jev {

namespace {

// Kernels take what they need of a cache and a call (the layer's base in the
// pointers) instead of all of it: a launch costs by its arguments' bytes (an empty
// kernel's with 400 of them 3.8 us, with 16 2.8; the attention's call 3.5 -> 3.4),
// and one or two launches are all there is to a small step's layer.
struct PlanView {
    int32_t *table, *length, *n_free, *fresh_pages, *prefix;
    uint32_t *used;
    PagesPlanHead *head;
    PagesRequest *req;
    PagesUnit *unit;
    PagesItem *item, *wide;
    double2 *angle;
    const double *freqs;
    double mscale;
    int page, sub, sub_shift, n_pages, max_requests, max_context, width, half, group, split, few, wide_keys, n_kv;
};
// Exclusive prefix sums over the workgroup's threads of N values at once, in
// place, and their totals.  `ws`: N words per wave.
template <int NT, int N, typename T>
__device__ __forceinline__ void block_scan(T (&v)[N], T (&total)[N], T *ws)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T x[N];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = v[i];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < N; i++) {
            const T y = __shfl_up(x[i], o, 64);
            if (lane >= o) x[i] += y;
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++)
        if (lane == 63) ws[wave * N + i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        T before = 0;
        total[i] = 0;
        for (int w = 0; w < NT / 64; w++) {
            const T y = ws[w * N + i];
            before += w < wave ? y : 0;
            total[i] += y;
        }
        v[i] = before + x[i] - v[i];
    }
}

// The last index b with prefix[b] <= i (prefix ascending, prefix[0] = 0, i < prefix[n]).
__device__ __forceinline__ int find(const int *prefix, int n, int i)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (prefix[m] <= i) lo = m;
        else hi = m;
    }
    return lo;
}

// What a batch row adds to the lists: blocks its new tokens touch; 16-row or
// wide tiles of a KV head, times their parts; partial results.
struct Counts {
    int units, items, wides, parts, wide_parts, n_parts, wide;
};
// `wide`: the most 16-row tiles of a request without wide ones, 0: of any.
__device__ __forceinline__ bool is_wide(const PlanView &p, int fresh, int wide)
{
    return wide && div_up(fresh * p.group, kPagesTileRows) > wide;
}
__device__ __forceinline__ Counts counts(const PlanView &p, int past, int fresh, int wide, int wide_keys, int small = 0)
{
    Counts c = {0, 0, 0, 0, 0, 1, 0};
    if (fresh <= 0) return c;
    const int len = past + fresh, rows = fresh * p.group;
    c.units = (len - 1) / kPageBlock - past / kPageBlock + 1;
    if (is_wide(p, fresh, wide)) {
        c.wide = 1;
        c.n_parts = div_up(len, wide_keys);
        c.wides = div_up(rows, kPagesWideRows) * c.n_parts;
        c.wide_parts = c.n_parts > 1 ? c.wides : 0;
        return c;
    }
    const int tiles = div_up(rows, kPagesTileRows);
    if (small || tiles <= max(wide, p.split)) c.n_parts = div_up(len, pages_part_keys(len));
    c.items = tiles * c.n_parts;
    c.parts = c.n_parts > 1 ? c.items : 0;
    return c;
}

// The lists that follow from a valid plan, by `n` threads of which this is
// number `i0`: the blocks to store, the attention's workgroups, the angles, and
// what the caller asked for.  px: tokens, units, items and wide items before
// each batch row (`stride` apart), R + 1 entries each; req: the batch rows, in
// LDS or in memory.
__device__ __forceinline__ void plan_lists(const PlanView &p, const PagesPlanArgs &a, const PagesPlanHead &h, const int *px,
                                           int stride, const PagesRequest *req, int i0, int n)
{
    const int R = h.n_requests;
    const int *start = px, *unit0 = px + stride, *item0 = px + 2 * stride, *wide0 = px + 3 * stride;
    for (int u = i0; u < h.n_units; u += n) {
        const int b = find(unit0, R, u);
        const PagesRequest r = req[b];
        const int block = r.past / kPageBlock + u - unit0[b], pos = max(r.past, block * kPageBlock);
        const int page = p.table[(size_t)r.id * p.width + (block >> p.sub_shift)];
        const PagesUnit un = {r.start + pos - r.past, pos, min(r.len, (block + 1) * kPageBlock) - pos,
                              (page << p.sub_shift) + (block & (p.sub - 1))};
        p.unit[u] = un;
    }
    for (int i = i0; i < h.n_items; i += n) {
        const int b = find(item0, R, i), k = i - item0[b];
        const PagesRequest r = req[b];
        const int tiles = (item0[b + 1] - item0[b]) / r.n_parts, t = k % tiles, part = k / tiles;
        const int keys = r.n_parts > 1 ? pages_part_keys(r.len) : r.len;
        const int key0 = part * keys;
        const PagesItem it = {t * kPagesTileRows, key0, min(r.len, key0 + keys), r.n_parts > 1 ? r.part0 + k : -1,
                              r.id, r.past, r.len, r.start, r.n_parts, r.part0, (r.len - r.past) * p.group, 0};
        p.item[i] = it;
    }
    for (int i = i0; i < h.n_wide; i += n) {
        const int b = find(wide0, R, i), k = i - wide0[b];
        const PagesRequest r = req[b];
        const int tiles = (wide0[b + 1] - wide0[b]) / r.n_parts, part = k % r.n_parts;
        const int keys = (div_up(r.len, r.n_parts) + 63) & ~63; // parts of a length, in whole blocks of 64
        // a request's tiles take like numbers of rows, whole waves' of 32; the longest come first
        const int rows = (r.len - r.past) * p.group, per = (div_up(rows, tiles) + 31) & ~31;
        const int key0 = part * keys, row0 = (tiles - 1 - k / r.n_parts) * per;
        const PagesItem it = {row0, key0, min(r.len, key0 + keys), r.n_parts > 1 ? r.part0 + k : -1,
                              r.id, r.past, r.len, r.start, r.n_parts, r.part0, min(rows, row0 + per), 0};
        p.wide[i] = it;
    }
    // Angles in 64 bits: a far position times a frequency keeps its fraction.
    // Once a plan, not once a layer and head: the library's 64-bit sine and
    // cosine are ~150 instructions.
    for (int i = i0; i < h.n_tokens * p.half; i += n) { // (at most 2^22 tokens x 64)
        const int t = i / p.half, j = i - t * p.half, b = find(start, R, t);
        double sn, cs;
        sincos((double)(req[b].past + t - start[b]) * p.freqs[j], &sn, &cs);
        p.angle[i] = make_double2(cs * p.mscale, sn * p.mscale);
    }
    if (a.slot || a.position || a.row)
        for (int t = i0; t < a.n_tokens; t += n) {
            int b = -1, pos = -1, slot = -1;
            if (t < h.n_tokens) {
                b = find(start, R, t);
                const PagesRequest r = req[b];
                pos = r.past + t - start[b];
                slot = p.table[(size_t)r.id * p.width + pos / p.page] * p.page + pos % p.page;
            }
            if (a.slot) a.slot[t] = slot;
            if (a.position) a.position[t] = pos;
            if (a.row) a.row[t] = b;
        }
    if (a.start)
        for (int b = i0; b <= a.n_requests; b += n) a.start[b] = R > 0 ? start[b] : 0;
    if (a.table) // a wave to a row, four rows' loads in flight
        for (int b0 = i0 >> 6; b0 < a.n_requests; b0 += 4 * (n >> 6))
            for (int j = i0 & 63; j < p.width; j += 64) {
                int page[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int b = b0 + u * (n >> 6);
                    page[u] = -1;
                    if (b < R && j < div_up(req[b].len, p.page)) page[u] = p.table[(size_t)req[b].id * p.width + j];
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int b = b0 + u * (n >> 6);
                    if (b < a.n_requests) a.table[(size_t)b * p.width + j] = page[u];
                }
            }
}

} // namespace

// A step's bookkeeping in one workgroup: pages given back and taken, prefix
// sums, and with LISTS everything that follows from them (many tokens: a
// launch of its own, over the whole GPU).  Checks first: a plan that does not
// fit changes nothing and plans no tokens.  Bounded by latency: a few trips to
// memory, each of which every thread makes at once (12 requests of a token each,
// every output among it, 8.9 us in a graph; 700 of up to 150 tokens 17 us, their lists 11).
template <int NT, bool LISTS>
__global__ __launch_bounds__(NT) void pages_plan_kernel(PlanView p, PagesPlanArgs a)
{
    constexpr int C = NT == 256 ? 1 : 8, S = NT * C + 1; // requests of a thread; entries of a prefix sum
    constexpr bool FEW = NT == 256;                      // the batch rows fit LDS
    __shared__ PagesRequest few[FEW ? NT : 1];
    PagesRequest *req;
    if constexpr (FEW) req = few;
    else req = p.req;
    __shared__ int px[4 * S];
    __shared__ unsigned seen[kPagesMaxRequests / 32];
    __shared__ long long ws[5 * NT / 64];
    __shared__ int bad;
    const int tid = threadIdx.x, R = a.n_requests, per = div_up(R, NT);
    int *start = px, *need0 = px + S, *gone0 = px + 2 * S;
    for (int i = tid; i < kPagesMaxRequests / 32; i += NT) seen[i] = 0;
    if (tid == 0) bad = 0;
    const int n_free = *p.n_free;
    __syncthreads();

    // the requests of this thread: b = tid * per + i
    int id[C], past[C], fresh[C], keep[C], need[C], own[C];
    long long sum[3] = {0, 0, 0}, all_of[3]; // tokens, pages taken, pages given back: 64 bits before they are checked
#pragma unroll
    for (int i = 0; i < C; i++) {
        const int b = tid * per + i;
        id[i] = past[i] = fresh[i] = keep[i] = need[i] = own[i] = 0;
        if (i >= per || b >= R) continue;
        id[i] = a.request[b];
        fresh[i] = a.fresh[b];
        bool ok = id[i] >= 0 && id[i] < p.max_requests;
        if (ok) ok = !(atomicOr(&seen[id[i] >> 5], 1u << (id[i] & 31)) >> (id[i] & 31) & 1u);
        if (ok) {
            const int len = p.length[id[i]];
            past[i] = a.past ? a.past[b] : len;
            ok = past[i] >= 0 && past[i] <= len && fresh[i] >= 0 && fresh[i] <= p.max_context - past[i];
        }
        if (!ok) {
            bad = 1;
            continue;
        }
        own[i] = div_up(p.length[id[i]], p.page);
        keep[i] = div_up(past[i], p.page);
        need[i] = div_up(past[i] + fresh[i], p.page);
        sum[0] += fresh[i];
        sum[1] += need[i] - keep[i];
        sum[2] += own[i] - keep[i];
    }
    block_scan<NT, 3>(sum, all_of, ws);
    const long long tokens = all_of[0], more = all_of[1], gone = all_of[2];
    const int status = bad || tokens > a.n_tokens ? JEV_EINVAL : more > n_free + gone ? JEV_ENOMEM : JEV_OK;
    if (status != JEV_OK) {
        PagesPlanHead h = {status, 0, 0, 0, 0, 0};
        if (tid == 0) *p.head = h;
        if (LISTS) plan_lists(p, a, h, px, S, req, tid, NT);
        return;
    }

    int s0 = (int)sum[0], s1 = (int)sum[1], s2 = (int)sum[2];
#pragma unroll
    for (int i = 0; i < C; i++) {
        const int b = tid * per + i;
        if (i >= per || b >= R) continue;
        start[b] = s0;
        need0[b] = s1;
        gone0[b] = s2;
        s0 += fresh[i];
        s1 += need[i] - keep[i];
        s2 += own[i] - keep[i];
        PagesRequest r = {id[i], past[i], past[i] + fresh[i], start[b], 0, 1};
        req[b] = r;
    }
    if (tid == 0) {
        start[R] = (int)tokens;
        need0[R] = (int)more;
        gone0[R] = (int)gone;
    }
    __syncthreads();

    for (int k = tid; k < (int)gone; k += NT) {
        const int b = find(gone0, R, k);
        const int page = p.table[(size_t)req[b].id * p.width + div_up(req[b].past, p.page) + k - gone0[b]];
        atomicAnd(&p.used[page >> 5], ~(1u << (page & 31)));
    }
    __syncthreads(); // every page is back before the free ones are counted
    if (more > 0) {
        const int words = div_up(p.n_pages, 32), per_w = div_up(words, NT);
        const int w0 = min(words, tid * per_w), w1 = min(words, w0 + per_w);
        // past the first-level cache, which the atomics went around
        auto word = [&](int w) { return __hip_atomic_load(&p.used[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        int n = 0;
        for (int w = w0; w < w1; w++) n += __popc(~word(w));
        int rank_of[1] = {n}, free_of[1];
        block_scan<NT, 1>(rank_of, free_of, (int *)ws);
        int rank = rank_of[0];
        for (int w = w0; w < w1 && rank < (int)more; w++) {
            uint32_t u = word(w);
            for (; ~u && rank < (int)more; rank++) {
                const int bit = __ffs(~u) - 1;
                u |= 1u << bit;
                p.fresh_pages[rank] = 32 * w + bit;
            }
            __hip_atomic_store(&p.used[w], u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        for (int k = tid; k < (int)more; k += NT) {
            const int b = find(need0, R, k);
            p.table[(size_t)req[b].id * p.width + div_up(req[b].past, p.page) + k - need0[b]] = p.fresh_pages[k];
        }
    }
    __syncthreads(); // need0 and gone0 are done with

    // the lists' prefix sums take their place
    int *unit0 = px + S, *item0 = px + 2 * S, *wide0 = px + 3 * S;
    int wide_keys = p.wide_keys, wide = 0; // (a small call's requests are all split)
    if (a.wide) {
        wide = p.split;
        if (p.few > p.split) {
            long long of[1] = {0}, total[1]; // tiles' parts of the requests between
#pragma unroll
            for (int i = 0; i < C; i++)
                if (is_wide(p, fresh[i], p.split) && !is_wide(p, fresh[i], p.few)) of[0] += counts(p, past[i], fresh[i], p.few, 0).items;
            block_scan<NT, 1>(of, total, ws);
            if (total[0] * p.n_kv <= kPagesFewWgs) wide = p.few;
        }
    }
    if (a.wide) {
        long long of[2] = {0, 0}, total[2]; // keys over the tiles, tiles
#pragma unroll
        for (int i = 0; i < C; i++)
            if (is_wide(p, fresh[i], wide)) {
                const int n = div_up(fresh[i] * p.group, kPagesWideRows);
                of[0] += (long long)n * (past[i] + fresh[i]);
                of[1] += n;
            }
        block_scan<NT, 2>(of, total, ws);
        const long long keys = total[0], tiles = total[1];
        // a tile's last part may be short: with keys / room of them each there are
        // at most room + tiles parts, one round; many tiles split only where one
        // is twice as long as their mean
        const long long target = pages_wide_target(p.n_kv), room = max(target - tiles, (target + 1) / 2);
        wide_keys = (int)min((long long)p.max_context, max((long long)wide_keys, (keys + room - 1) / room));
    }
    int n0[5] = {0, 0, 0, 0, 0}; // units, items, wide items, parts, wide parts
    Counts c[C];
#pragma unroll
    for (int i = 0; i < C; i++) {
        c[i] = counts(p, past[i], fresh[i], wide, wide_keys, a.small);
        n0[0] += c[i].units;
        n0[1] += c[i].items;
        n0[2] += c[i].wides;
        n0[3] += c[i].parts;
        n0[4] += c[i].wide_parts;
    }
    int all_n[5];
    block_scan<NT, 5>(n0, all_n, (int *)ws);
    __shared__ PagesPlanHead all;
    if (tid == 0) {
        PagesPlanHead h = {JEV_OK, (int)tokens, all_n[0], all_n[1], all_n[2], R};
        all = h;
        *p.head = h;
        unit0[R] = h.n_units;
        item0[R] = h.n_items;
        wide0[R] = h.n_wide;
        *p.n_free = n_free + (int)(gone - more);
    }
#pragma unroll
    for (int i = 0; i < C; i++) {
        const int b = tid * per + i;
        if (i >= per || b >= R) continue;
        unit0[b] = n0[0];
        item0[b] = n0[1];
        wide0[b] = n0[2];
        req[b].part0 = c[i].wide ? n0[4] : n0[3];
        req[b].n_parts = c[i].n_parts;
        n0[0] += c[i].units;
        n0[1] += c[i].items;
        n0[2] += c[i].wides;
        n0[3] += c[i].parts;
        n0[4] += c[i].wide_parts;
        p.length[id[i]] = past[i] + fresh[i];
    }
    __syncthreads();
    if (LISTS) plan_lists(p, a, all, px, S, req, tid, NT);
    else {
        for (int j = 0; j < 4; j++)
            for (int i = tid; i <= R; i += NT) p.prefix[j * (kPagesMaxRequests + 1) + i] = px[j * S + i];
        if (FEW && tid < R) p.req[tid] = req[tid];
    }
}

// The lists of a plan with many tokens, over the whole GPU.
__global__ __launch_bounds__(256) void pages_lists_kernel(PlanView p, PagesPlanArgs a)
{
    constexpr int S = kPagesMaxRequests + 1;
    __shared__ int px[4 * S];
    const PagesPlanHead h = *p.head;
    if (h.n_requests > 0)
        for (int j = 0; j < 4; j++)
            for (int i = threadIdx.x; i <= h.n_requests; i += 256) px[j * S + i] = p.prefix[j * S + i];
    __syncthreads();
    plan_lists(p, a, h, px, S, p.req, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

hipError_t launch_pages_plan(const Pages &p, const PagesPlanArgs &a, hipStream_t s)
{
    if (a.n_requests < 0 || a.n_requests > p.max_requests || a.n_tokens < 0 || a.n_tokens > p.max_tokens)
        return hipErrorInvalidValue;
    const PlanView v = {p.table, p.length, p.n_free, p.fresh_pages, p.prefix, p.used, p.head, p.req, p.unit, p.item, p.wide, p.angle, p.freqs,
                        p.mscale, p.page, p.sub, p.sub_shift, p.n_pages, p.max_requests, p.max_context, p.width, p.half, p.group, p.split, p.few, p.wide_keys, p.n_kv};
    // What the lists write, in words; an angle counts for several.  Short lists are written
    // by the plan's own workgroup (in a graph, so / with a launch of their own: 12 requests
    // of a token and 64 pairs 6.7 / 7.6 us, 16 9.4 / 10.0, 24 10.8 / 9.8, 64 18.6 / 10.2; one
    // of 20 tokens 8.1 / 9.5, of 60 11.7 / 9.5).
    const double work = (double)a.n_tokens * (4 + 8.0 * p.half) + (a.table ? (double)a.n_requests * p.width : 0.0);
    const bool lists = work <= 9216;
    // A request to a thread of 256, or up to eight to one of 512: 200 requests 12.5 / 13.3 us,
    // 12 6.7 / 9.0.
    const bool small = a.n_requests <= 256;
    if (small && lists) hipLaunchKernelGGL((pages_plan_kernel<256, true>), dim3(1), dim3(256), 0, s, v, a);
    else if (small) hipLaunchKernelGGL((pages_plan_kernel<256, false>), dim3(1), dim3(256), 0, s, v, a);
    else if (lists) hipLaunchKernelGGL((pages_plan_kernel<512, true>), dim3(1), dim3(512), 0, s, v, a);
    else hipLaunchKernelGGL((pages_plan_kernel<512, false>), dim3(1), dim3(512), 0, s, v, a);
    // (2048 words to a workgroup of the lists: 64 requests' tables 12.6 us instead of 11.4;
    // 128: 64 requests of 300 tokens 42.6 instead of 37.9)
    if (!lists) hipLaunchKernelGGL(pages_lists_kernel, dim3((int)fmin(1024.0, ceil(work / 512))), dim3(256), 0, s, v, a);
    return hipGetLastError();
}

// ------------------------------------------------------------ rotary positions and the store

namespace {

// x / by in 64 bits, rounded to the nearest whole number, a half to the even
// one, as the byte q + 128; `inv` = 1 / by.  The product is within 2^-51 of the
// quotient, and two fp32 numbers' quotient (or one times a code) is further
// than that from a half unless it is one: then x - q by is exactly half of by.
__device__ __forceinline__ uint32_t code_of(double x, double by, double inv)
{
    double q = rint(x * inv);
    const double rest = fma(-q, by, x);
    if (fabs(rest) * 2.0 == by && ((int)q & 1)) q += rest > 0.0 ? 1.0 : -1.0;
    return (uint32_t)(int)(fmin(fmax(q, -127.0), 127.0) + 128.0);
}

// Byte of dim d of token t in a block's K and V codes.
template <int HD>
__device__ __forceinline__ int k_at(int t, int d) { return (d >> 6) * 1024 + t * 64 + (d & 63); }
template <int HD>
__device__ __forceinline__ int v_at(int t, int d) { return d * 16 + t; }

} // namespace

namespace {
struct StoreView {
    uint8_t *k, *v;
    float2 *ks;
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

// One workgroup per block that the batch touches and KV head: the block's new
// tokens' queries (of the head's group) rotated, their keys rotated and stored,
// their values stored.  Sixteen threads hold a token's row, and keep to one
// token, so its angles are loaded once for all rows; with fewer tokens in the
// block its rows are dealt over the idle sixteens.  Products of the rotation
// are 64-bit and round to fp32 once, so a stored code does not depend on how
// they are formed.  A block's scale only grows while the block fills; codes it
// already holds are then rounded to the new one.  Bounded by memory: 4 B in per
// element, 1 B (K, V) or 4 B (q) out, a begun block's codes both ways (queries alone, 8200 tokens x 32 x 128: 54 us,
// 5.0 TB/s; 9400 tokens of 11 prompts with 8 KV heads 95 us, 4.2 TB/s; with a row of
// its own for each thread, and its angles, 67 and 198 with the reading back).  A single
// token has its whole block read, coded and written again, a chain of trips to memory and
// barriers in small workgroups: 64 requests 7.5 us, 700 34 (where every scale grows, and
// every code with it, 3.5 and 14 more).
template <int HD, bool VEC>
__global__ __launch_bounds__(256) void pages_store_kernel(StoreView p)
{
    constexpr int NP = HD / 32, BYTES = kPageBlock * HD, RING = 2;
    __shared__ __align__(16) uint8_t code[2][BYTES];
    __shared__ unsigned most[2];
    const int tid = threadIdx.x, j = tid & 15, h = blockIdx.y;
    const PagesUnit un = p.unit[blockIdx.x];
    const PagesPlanHead plan = *p.head; // (the unit's load does not wait for this)
    if (outgrown(p, plan) || (int)blockIdx.x >= plan.n_units) return;
    const int pos0 = un.pos, n = un.n, row0 = un.row, off = pos0 & (kPageBlock - 1);
    const bool kv = p.k_in != nullptr;
    const RowPairs<HD> e(p, j);

    // this thread's token, and its rows: K (-2), V (-1), then the group's queries
    const int nt = n > 8 ? 16 : n > 4 ? 8 : n > 2 ? 4 : n, step = 16 / nt; // (nt: 1, 2, 4, 8, 16)
    const int t = (tid >> 4) % nt, row = row0 + t, first = (kv ? -2 : 0) + (tid >> 4) / nt, end = t < n && p.q ? p.group : 0;
    const bool mine = t < n;

    // where the block lies
    const size_t block = ((((size_t)(un.block >> p.sub_shift) * p.n_kv + h) << p.sub_shift) | (un.block & (p.sub - 1)));
    const bool begun = kv && off > 0;
    float2 s_old = make_float2(0.f, 0.f);
    if (kv) {
        if (tid < 2) most[tid] = 0;
        if (begun) s_old = p.ks[block];
        if (tid < 2 * BYTES / 16) {
            const bool v = tid >= BYTES / 16;
            const int i = v ? tid - BYTES / 16 : tid;
            uint4 w = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
            if (begun) w = ((const uint4 *)((v ? p.v : p.k) + block * BYTES))[i];
            ((uint4 *)code[v])[i] = w;
        }
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
        for (int z = 1; z < p.nin; z++) {
            float2 w[NP];
            load_pairs<HD, VEC>(e, src + z * p.in_stride, w);
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

    float2 x[2][NP]; // this thread's rows of K and V
    int w = first;
    if (kv) {
        __syncthreads(); // `most` is zero
#pragma unroll
        for (int it = 0; it < 2; it++)
            if (mine && w + it * step < 0) load(w + it * step, x[it]);
#pragma unroll
        for (int it = 0; it < 2; it++) {
            const int which = w + it * step;
            if (!mine || which >= 0) continue;
            if (which == -2) rotate(1.0, x[it]);
            unsigned m = 0; // a value that is not finite has the largest bits
#pragma unroll
            for (int c = 0; c < NP; c++)
                m = max(m, max(__float_as_uint(fabsf(x[it][c].x)), __float_as_uint(fabsf(x[it][c].y))));
            for (int o = 1; o < 16; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
            if (j == 0) atomicMax(&most[which + 2], m);
        }
        while (w < 0) w += step;
    }
    if (end) {
        double f = 1.0;
        const int pos = pos0 + t;
        if (p.orig_ctx > 0 && p.temp_scale != 0.f && pos >= p.orig_ctx)
            f = 1.0 + (double)p.temp_scale * log(1.0 + (double)(pos / p.orig_ctx));
        // RING rows in flight
        for (; w < end; w += RING * step) {
            float2 y[RING][NP];
#pragma unroll
            for (int i = 0; i < RING; i++)
                if (w + i * step < end) load(w + i * step, y[i]);
#pragma unroll
            for (int i = 0; i < RING; i++)
                if (w + i * step < end) {
                    rotate(f, y[i]);
                    store_pairs<HD, VEC>(e, p.q_out + ((size_t)row * p.n_heads + h * p.group + w + i * step) * HD, y[i]);
                }
        }
    }
    if (!kv) return;
    __syncthreads(); // `most` and the old codes are whole

    float s[2];
    double by[2], inv[2];
#pragma unroll
    for (int v = 0; v < 2; v++) {
        const float old = v ? s_old.y : s_old.x;
        const float now = most[v] >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(most[v]) / 127.0f;
        s[v] = now > old || now != now ? now : old; // NaN stays
        by[v] = (double)s[v];
        inv[v] = s[v] > 0.f ? 1.0 / by[v] : 0.0;
    }
    if (begun && tid < 2 * BYTES / 16) {
        const bool v = tid >= BYTES / 16;
        const float old = v ? s_old.y : s_old.x, now = v ? s[1] : s[0];
        const double d = v ? by[1] : by[0], id = v ? inv[1] : inv[0];
        if (now != old) { // also where either is NaN
            uint32_t *word = (uint32_t *)code[v] + 4 * (v ? tid - BYTES / 16 : tid);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t y = 0;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int q = (int)((word[i] >> (8 * c)) & 255u) - 128;
                    y |= (now > 0.f ? code_of((double)q * (double)old, d, id) : 128u) << (8 * c);
                }
                word[i] = y;
            }
        }
    }
    // places from the first new token on held nothing, or what the request was
    // cut back from: the new codes come over them, the rest is past its end
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 2; it++) {
        const int which = first + it * step;
        if (!mine || which >= 0) continue;
        const bool v = which == -1;
        const double d = v ? by[1] : by[0], id = v ? inv[1] : inv[0];
        const bool zero = !(d > 0.0);
        const int tk = off + t;
#pragma unroll
        for (int c = 0; c < NP; c++) {
            const uint32_t q0 = zero ? 128u : code_of((double)x[it][c].x, d, id);
            const uint32_t q1 = zero ? 128u : code_of((double)x[it][c].y, d, id);
            code[v][v ? v_at<HD>(tk, e.e0[c]) : k_at<HD>(tk, e.e0[c])] = (uint8_t)q0;
            code[v][v ? v_at<HD>(tk, e.e1[c]) : k_at<HD>(tk, e.e1[c])] = (uint8_t)q1;
        }
    }
    __syncthreads();
    if (tid < 2 * BYTES / 16) {
        const bool v = tid >= BYTES / 16;
        const int i = v ? tid - BYTES / 16 : tid;
        ((uint4 *)((v ? p.v : p.k) + block * BYTES))[i] = ((const uint4 *)code[v])[i];
    }
    if (tid == 0) p.ks[block] = make_float2(s[0], s[1]);
}

hipError_t launch_pages_store(const Pages &p, const PagesStoreArgs &a, hipStream_t s)
{
    if (p.bits == 4) return launch_pages4_store(p, a, s);
    const int units = a.n_tokens / kPageBlock + 2 * (a.n_requests < a.n_tokens ? a.n_requests : a.n_tokens);
    const int np = p.hd / 32;
    auto vec = [&](const void *x, int64_t ld) { return !x || ((uintptr_t)x % (4 * np) == 0 && ld % np == 0); };
    // a thread's pairs in vector accesses: rows that start aligned, and no
    // thread with pairs on both sides of the rotated part's end
    const bool v = vec(a.q, a.q_ld) && vec(a.k, a.kv_ld) && vec(a.v, a.kv_ld) && vec(a.q_out, 0) && a.in_stride % np == 0 &&
                   (!p.rope_half || p.half % np == 0);
    const size_t bytes = (size_t)kPageBlock * p.hd;
    const StoreView view = {layer_of(p, p.k, a.layer, bytes), layer_of(p, p.v, a.layer, bytes), layer_of(p, p.ks, a.layer, 1), p.head, p.unit,
                            p.angle, a.q, a.k, a.v, a.q_out, a.q_ld, a.kv_ld, a.in_stride, a.nin, p.n_kv, p.n_heads, p.group,
                            p.sub, p.sub_shift, p.half, p.rope_half, p.orig_ctx, p.temp_scale, a.n_tokens, a.n_requests, 1};
    const dim3 grid(units > 0 ? units : 1, p.n_kv);
    if (p.hd == 128 && v) hipLaunchKernelGGL((pages_store_kernel<128, true>), grid, dim3(256), 0, s, view);
    else if (p.hd == 128) hipLaunchKernelGGL((pages_store_kernel<128, false>), grid, dim3(256), 0, s, view);
    else if (v) hipLaunchKernelGGL((pages_store_kernel<64, true>), grid, dim3(256), 0, s, view);
    else hipLaunchKernelGGL((pages_store_kernel<64, false>), grid, dim3(256), 0, s, view);
    return hipGetLastError();
}

// ------------------------------------------------------------ attention

namespace {

// Sixteen codes (two words each) as fp16: exact.
__device__ __forceinline__ uint4 codes_f16(uint32_t w0, uint32_t w1)
{
    uint4 u;
    bytes_to_f16(w0, (_Float16)1152.f, u.x, u.y);
    bytes_to_f16(w1, (_Float16)1152.f, u.z, u.w);
    return u;
}

// A query row as fp16 pairs: scaled by a power of two so that its largest
// element m lies in [2^13, 2^14); rows of zeros and rows with infinities stay as
// they are.  `scores` undoes it in a block's K scale (the power alone may be
// outside fp32's range) and turns scores into exponents of two; f1 f2 is the factor,
// in two steps that stay inside that range.
struct QueryScale {
    float f1, f2, scale;
    int ex;
    QueryScale() = default;
    __device__ __forceinline__ QueryScale(float m, float softmax)
        : scale(softmax * 1.44269504088896341f), ex(m > 0.f && m < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(m) : 0)
    {
        f1 = ldexpf(1.f, ex / 2), f2 = ldexpf(1.f, ex - ex / 2);
    }
    __device__ __forceinline__ float scores(float ks) const { return ldexpf(ks, -ex) * scale; }
    __device__ __forceinline__ void split(float x, _Float16 &hi, _Float16 &lo) const
    {
        const float y = x * f1 * f2;
        hi = (_Float16)y;
        lo = (_Float16)(y - (float)hi);
    }
};

// A block's weights are 2^(score + log2(V scale) + 9 - e) = 2^(score + c), where e, whole,
// lies between the row's largest score + log2(V scale) so far, less 6, and that plus 1:
// a weight falls under fp16's last bit only where it is less than 2^-32 of the heaviest
// one, however large the scales of blocks without weight are.
struct ValueScale {
    int exp;
    float lg;                                          // log2 of the mantissa; -inf for 0
    __device__ __forceinline__ ValueScale(float vs)    // vs: the block's V scale, 0 where the row sees none of it
        : exp(__builtin_amdgcn_frexp_expf(vs)), lg(__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(vs))) {}
    __device__ __forceinline__ float top(float mx) const { return mx + ((float)exp + lg); } // mx: the block's largest score
    // The row's sum takes the block's weights times 2^(-c - mu), so c may be any number where
    // the outputs do not see them: weights below 2^-31, and a scale of zero's (codes of zero).
    __device__ __forceinline__ float c(float vs, float mx, float e, float mu) const
    {
        if (vs > 0.f && mx > -INFINITY) return fmaxf((float)exp + 9.f - e + lg, -31.f - mx);
        return vs != vs ? vs : -mu;
    }
};
} // namespace

namespace {
struct AttendView {
    const uint8_t *k, *v;
    const float2 *ks;
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
} // namespace

// Sixteen (token, head) rows of a request and KV head over keys [key0, key1) of
// its pages; the four waves take 64 keys (four blocks) in turn and merge at the
// end.  S^T = K Q^T: with the rows of the K operand (token i, block b) dealt so
// that a lane's sixteen scores are the sixteen tokens of ONE block, the
// accumulators are the P^T operand of O^T += V^T P^T as they stand -- no
// exchange between lanes -- and a lane has one K and one V scale per 64 keys.
// Codes are exact in fp16; q and p enter as fp16 pairs (hi + lo), ~22 bits, so
// each product is two matrix instructions.  p carries the V scale through its
// exponent (ValueScale): one fused multiply-add and one exp2 a score; the maxima move
// only when a score passes one by 2^6.  Statistics, scores and outputs are fp32.  The
// next 64 keys' K is in flight during the softmax and V^T P^T, their V during the next
// scores.  Many single tokens are bound by HBM: 2 hd bytes a key and KV head (32 heads
// over 8 x 128, one call after the other over different layers: 64 tokens over 500 to
// 12000 keys 98 us, 5.1 TB/s; 64 of another draw, 899 MB, 162 us, 5.5).  Few of them wait
// for their trips to memory instead, and for their parts' merge: one over 300 keys 7.5 us,
// over 4000 13.3, over 30000 25, over 120002 58 (4.2 TB/s), 12 over 500 to 2000 15.4.
template <int HD>
struct TileLds {
    float lo[4][kPagesTileRows][HD + 4];
    float lm[4][kPagesTileRows], ll[4][kPagesTileRows];
    int last;
};
template <int HD>
__device__ __forceinline__ void attend_tiles(const AttendView &p, TileLds<HD> &lds, PagesItem it, int n_items, int first, int count)
{
    constexpr int NJ = HD / 64, NS = HD / 16, BYTES = kPageBlock * HD, LD = HD + 4;
    auto &lo = lds.lo;
    auto &lm = lds.lm, &ll = lds.ll;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, n = lane & 15, h = first % p.n_kv;
    const int stride = count / p.n_kv;
    const uint8_t *kbase = p.k;
    const uint8_t *vbase = p.v;
    const float2 *sbase = p.ks;

    for (int item = first / p.n_kv; item < n_items;) {
        const PagesItem &r = it;
        const int32_t *table = p.table + (size_t)r.id * p.width;
        // lanes past the request's rows repeat its last one
        const int n_rows = it.row1, row = min(it.row0 + n, n_rows - 1);
        const int token = row / p.group, head = h * p.group + row % p.group;
        const int limit = r.past + token; // last visible key
        // the tile's last visible key; keys up to `clear` are seen by every row
        const int top = r.past + min(n_rows - 1, it.row0 + kPagesTileRows - 1) / p.group;
        const int key1 = min(it.key1, top + 1), clear = r.past + it.row0 / p.group;
        const int last = (r.len - 1) / kPageBlock; // blocks past it are read as this one, and masked

        // a lane reads K of block n / 4 of the four, V of block g
        auto page_of = [&](int kb, int i) { return table[min(4 * kb + i, last) >> p.sub_shift]; };
        auto block_of = [&](int kb, int i, int page) {
            return (((size_t)page * p.n_kv + h) << p.sub_shift) + (min(4 * kb + i, last) & (p.sub - 1));
        };
        uint4 kr[4][NJ], vr[NS];
        float2 sc;
        auto fetch_k = [&](int kb, int page) {
            const uint8_t *src = kbase + block_of(kb, n >> 2, page) * BYTES + (n & 3) * 64 + 16 * g;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int j = 0; j < NJ; j++) kr[t][j] = *(const uint4 *)(src + j * 1024 + 256 * t);
        };
        auto fetch_v = [&](int kb, int page) {
            const size_t b = block_of(kb, g, page);
            const uint8_t *src = vbase + b * BYTES + 16 * n;
            sc = sbase[b];
#pragma unroll
            for (int s = 0; s < NS; s++) vr[s] = *(const uint4 *)(src + 256 * s);
        };
        int kb = it.key0 / 64 + wave;
        int pk = page_of(kb, n >> 2), pv = page_of(kb, g);
        if (kb * 64 < key1) {
            fetch_k(kb, pk);
            fetch_v(kb, pv);
        }
        pk = page_of(kb + 4, n >> 2);
        pv = page_of(kb + 4, g);

        // Q^T fragments: dims 64 j + 16 g + 8 c .. + 7 of row n
        half8_t qh[2 * NJ], ql[2 * NJ];
        QueryScale query;
        {
            const float *src = p.q + ((size_t)(r.start + token) * p.n_heads + head) * HD + 16 * g;
            float x[2 * NJ][8], m = 0.f;
#pragma unroll
            for (int c = 0; c < 2 * NJ; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[c][i] = src[64 * (c >> 1) + 8 * (c & 1) + i];
                    m = fmaxf(m, fabsf(x[c][i]));
                }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            query = QueryScale(m, p.scale);
#pragma unroll
            for (int c = 0; c < 2 * NJ; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    _Float16 hi, lw;
                    query.split(x[c][i], hi, lw);
                    qh[c][i] = hi;
                    ql[c][i] = lw;
                }
        }

        floatx4 o[NS];
#pragma unroll
        for (int s = 0; s < NS; s++) o[s] = floatx4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f, e = -INFINITY; // outputs are held times 2^(9 - e)

        for (; kb * 64 < key1; kb += 4) {
            const bool more = (kb + 4) * 64 < key1;
            floatx4 sv[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const half8_t k0 = __builtin_bit_cast(half8_t, codes_f16(kr[t][j].x, kr[t][j].y));
                    const half8_t k1 = __builtin_bit_cast(half8_t, codes_f16(kr[t][j].z, kr[t][j].w));
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[2 * j], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[2 * j + 1], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[2 * j], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[2 * j + 1], acc, 0, 0, 0);
                }
                sv[t] = acc;
            }
            if (more) fetch_k(kb + 4, pk);
            // a scale of zero has codes of zero: any other does as well
            float ks = query.scores(sc.x), vs = sc.y;
            ks = ks < 1e-37f ? 1e-37f : ks;
            if (kb * 64 + 63 > clear) {
                const int left = limit - (kb * 64 + 16 * g); // last visible token of the lane's block
                if (left < 0) { // none: whatever its scales are
                    ks = 1.f;
                    vs = 0.f;
                }
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (4 * t + i > left) sv[t][i] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, sv[t][i]);
            mx *= ks;
            const ValueScale value(vs);
            const float mv = value.top(mx);
            if (__any(mx > m + 6.f || mv > e + 6.f)) {
                float mn = fmaxf(m, mx), en = fmaxf(e, ceilf(mv));
                mn = fmaxf(mn, __shfl_xor(mn, 16, 64));
                en = fmaxf(en, __shfl_xor(en, 16, 64));
                mn = fmaxf(mn, __shfl_xor(mn, 32, 64));
                en = fmaxf(en, __shfl_xor(en, 32, 64));
                l *= m == -INFINITY ? 0.f : exp2f(m - mn);
                const float up = e == -INFINITY ? 0.f : exp2f(e - en);
#pragma unroll
                for (int s = 0; s < NS; s++) o[s] *= up;
                m = mn;
                e = en;
            }
            const float mu = m == -INFINITY ? 0.f : m, c = value.c(vs, mx, e, mu);
            float w[16], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                w[i] = __builtin_amdgcn_exp2f(fmaf(sv[i >> 2][i & 3], ks, c));
                sum += w[i];
            }
            l += sum * __builtin_amdgcn_exp2f(-c - mu);
            uint32_t hi[8], lw[8];
#pragma unroll
            for (int i = 0; i < 8; i++) split2_mix(w[2 * i], w[2 * i + 1], hi[i], lw[i]);
            const half8_t ph0 = __builtin_bit_cast(half8_t, make_uint4(hi[0], hi[1], hi[2], hi[3]));
            const half8_t ph1 = __builtin_bit_cast(half8_t, make_uint4(hi[4], hi[5], hi[6], hi[7]));
            const half8_t pl0 = __builtin_bit_cast(half8_t, make_uint4(lw[0], lw[1], lw[2], lw[3]));
            const half8_t pl1 = __builtin_bit_cast(half8_t, make_uint4(lw[4], lw[5], lw[6], lw[7]));
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const half8_t v0 = __builtin_bit_cast(half8_t, codes_f16(vr[s].x, vr[s].y));
                const half8_t v1 = __builtin_bit_cast(half8_t, codes_f16(vr[s].z, vr[s].w));
                o[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph0, o[s], 0, 0, 0);
                o[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph1, o[s], 0, 0, 0);
                o[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl0, o[s], 0, 0, 0);
                o[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl1, o[s], 0, 0, 0);
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
        for (int s = 0; s < NS; s++) *(floatx4 *)&lo[wave][n][16 * s + 4 * g] = o[s] * mean.f1 * mean.f2;
        if (g == 0) {
            lm[wave][n] = m;
            ll[wave][n] = l;
        }
        __syncthreads();
        for (int i = tid; i < kPagesTileRows * (HD / 4); i += 256) {
            const int c = i / (HD / 4), d = 4 * (i % (HD / 4)), rr = it.row0 + c;
            if (rr >= n_rows) continue;
            float mm = lm[0][c];
#pragma unroll
            for (int w = 1; w < 4; w++) mm = fmaxf(mm, lm[w][c]);
            const float mu = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f, f[4];
            floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                f[w] = ll[w][c] * exp2f(lm[w][c] - mu);
                sum += f[w];
            }
            const float inv = sum == 0.f && it.part >= 0 ? 0.f : 1.f / sum;
#pragma unroll
            for (int w = 0; w < 4; w++) x += *(const floatx4 *)&lo[w][c][d] * (f[w] * inv);
            if (it.part < 0) {
                const int tk = rr / p.group, hd = h * p.group + rr % p.group;
                float *dst = p.out + ((size_t)(r.start + tk) * p.n_heads + hd) * HD + d;
#pragma unroll
                for (int k = 0; k < 4; k++) dst[k] = x[k];
            } else {
                float *dst = p.part + (((size_t)it.part * p.n_kv + h) * kPagesTileRows + c) * LD;
                store_shared(dst + d, x[0], x[1]);
                store_shared(dst + d + 2, x[2], x[3]);
                if (d == 0) store_shared(dst + HD, mm, sum);
            }
        }
        if (it.part >= 0) {
            // the tile's last part to arrive merges them all, in their order
            const int tiles = div_up(n_rows, kPagesTileRows), tile = it.row0 / kPagesTileRows;
            if (arrives_last(p.tickets + (size_t)(r.part0 + tile) * p.n_kv + h, r.n_parts, lds.last))
                for (int c = tid >> 4; c < min(kPagesTileRows, n_rows - it.row0); c += 16) {
                    const int rr = it.row0 + c, tk = rr / p.group;
                    merge_parts<HD>(
                        [&](int k) { return p.part + (((size_t)(r.part0 + k * tiles + tile) * p.n_kv + h) * kPagesTileRows + c) * LD; },
                        r.n_parts, p.out + ((size_t)(r.start + tk) * p.n_heads + h * p.group + rr % p.group) * HD, tid & 15);
                }
        }
        __syncthreads();
        item += stride;
        if (item < n_items) it = p.item[item];
    }
}

// 128 (token, head) rows of a request and KV head, 32 to a wave, over its keys
// in blocks of 64: as above, with K and V turned into fp16 fragments in LDS once
// for the four waves (double buffered: the next block's codes are in flight
// during a block's products and written as it ends).  v_mfma_f32_32x32x16_f16:
// S^T is two tiles of 32 keys, their rows dealt so that a lane's sixteen scores
// are one block's tokens in order, which is again the P^T operand.  The V scale
// enters through the exponent (one fused multiply-add and one exp2 a score), and
// the maximum moves only when a score passes it by 2^6, so most blocks rescale
// nothing.  Bound by the matrix cores at two instructions a product, with the
// exponentials and fp16 pairs of ~9 vector instructions a score beside them: four
// prompts of 300 to 4000 tokens 312 to 328 us by the card, 530 to 556 TFLOP/s (a product
// counted once), the matrix cores 56 % busy and the clock at what the power allows
// (1.91 GHz).  64 rows to a wave halve the LDS reads and are slower (315 -> 345 us: one
// workgroup a compute unit).  Tens of tokens behind a long cache are bound by what is not
// split: 9 x 48 over 4096 keys 98 us, of 52, for waves without rows, 80 of 512 places
// empty, and one workgroup that merges each tile's parts.
template <int HD>
struct WideLds {
    union {
        struct {
            uint4 kf[2][2 * (HD / 16) * 64], vf[2][4 * (HD / 32) * 64];
            float2 sc[2][4];
        };
        float rows[kPagesWideRows * (HD + 4)]; // a part: means, maximum, sum
        float factor[8][kPagesWideRows];
    };
    int last;
};

template <int HD>
__device__ __forceinline__ void attend_wide(const AttendView &p, WideLds<HD> &lds, const PagesItem &it, int first)
{
    constexpr int NC = HD / 16, ND = HD / 32, NL = HD / 64, BYTES = kPageBlock * HD;
    auto &kf = lds.kf;
    auto &vf = lds.vf;
    auto &sc = lds.sc;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hh = lane >> 5, n = lane & 31, h = first % p.n_kv, item = first / p.n_kv;
    const PagesItem &r = it;
    const int32_t *table = p.table + (size_t)r.id * p.width;
    const uint8_t *kbase = p.k;
    const uint8_t *vbase = p.v;
    const float2 *sbase = p.ks;

    const int n_rows = it.row1, wrow = it.row0 + 32 * wave;
    const bool active = wrow < n_rows;
    const int row = min(wrow + n, n_rows - 1), token = row / p.group, head = h * p.group + row % p.group;
    const int limit = r.past + token; // last visible key
    const int key1 = min(it.key1, r.past + min(n_rows - 1, it.row0 + kPagesWideRows - 1) / p.group + 1);
    const int clear = r.past + min(wrow, n_rows - 1) / p.group; // keys up to it are seen by every row of the wave
    const int last = (r.len - 1) / kPageBlock;

    // A wave stages one of a block's four 16-token blocks.  Buffer loads: their
    // bases are the wave's, so no vector registers hold addresses, and its page and
    // scales do not become scalar loads, which were waited for where they were
    // issued, at the top of every block.
    const rsrc_t rt = make_rsrc(table, 4 * p.width);
    auto page_of = [&](int kb) {
        return __builtin_amdgcn_raw_buffer_load_b32(rt, 0, 4 * (min(4 * kb + wave, last) >> p.sub_shift), 0);
    };
    uint4 kr[NL], vr[NL];
    float2 sr;
    auto fetch = [&](int kb, int page) {
        const int c = min(4 * kb + wave, last) & (p.sub - 1);
        const size_t b = (((size_t)__builtin_amdgcn_readfirstlane(page) * p.n_kv + h) << p.sub_shift) + c;
        const rsrc_t rk = make_rsrc(kbase + b * BYTES, BYTES), rv = make_rsrc(vbase + b * BYTES, BYTES), rs = make_rsrc(sbase + b, 8);
#pragma unroll
        for (int i = 0; i < NL; i++) kr[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, 16 * lane, 1024 * i, 0));
#pragma unroll
        for (int i = 0; i < NL; i++) vr[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, 16 * lane, 1024 * i, 0));
        sr = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rs, 0, 0, 0));
    };
    // K: sixteen dims of token lane / 4, chunk 4 i + lane % 4; its row of the tile,
    // dealt by chunk so that neighbouring lanes' writes take all banks.  V: sixteen
    // tokens of dim 64 i + lane.  One of the 4 NL halves of these to a piece.
    const int krow = (8 * (lane >> 4) + 4 * (wave & 1) + ((lane >> 2) & 3)) ^ ((lane & 3) << 1);
    auto put = [&](int buf, int piece) {
        const int i = piece >> 2, half = piece & 1;
        if (piece & 2)
            (vf[buf] + ((2 * i + hh) * 4 + (wave >> 1) * 2) * 64 + 32 * (wave & 1) + n)[64 * half] =
                half ? codes_f16(vr[i].z, vr[i].w) : codes_f16(vr[i].x, vr[i].y);
        else
            (kf[buf] + ((wave >> 1) * NC + 4 * i + (lane & 3)) * 64 + krow)[32 * half] =
                half ? codes_f16(kr[i].z, kr[i].w) : codes_f16(kr[i].x, kr[i].y);
        if (piece == 0 && lane == 0) sc[buf][wave] = sr;
    };

    int kb = it.key0 / 64;
    int next = page_of(kb);
    fetch(kb, next);
    next = page_of(kb + 1);

    // Q^T fragments: dims 16 c + 8 hh .. + 7 of row n
    half8_t qh[NC], ql[NC];
    QueryScale query;
    {
        const float *src = p.q + ((size_t)(r.start + token) * p.n_heads + head) * HD + 8 * hh;
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(src[16 * c + i]));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        query = QueryScale(m, p.scale);
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                _Float16 hi, lw;
                query.split(src[16 * c + i], hi, lw);
                qh[c][i] = hi;
                ql[c][i] = lw;
            }
    }

    floatx16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = floatx16{};
    float m = -INFINITY, l = 0.f, e = -INFINITY; // outputs are held times 2^(9 - e)
#pragma unroll
    for (int i = 0; i < 4 * NL; i++) put(0, i);
    fetch(kb + 1, next); // (past the last block: the last again, which nobody reads)
    next = page_of(kb + 2);
    __syncthreads();

    if (!active) { // no rows of its own: it stages for the others
        for (int buf = 0; kb * 64 < key1; kb++, buf ^= 1) {
#pragma unroll
            for (int i = 0; i < 4 * NL; i++) put(buf ^ 1, i);
            fetch(kb + 2, next);
            next = page_of(kb + 3);
            __syncthreads();
        }
    }
    for (int buf = 0; kb * 64 < key1; kb++, buf ^= 1) {
        // the scores; beside their matrix instructions the next block's codes,
        // here by now, become fragments, and the block after it is asked for
        floatx16 s[2] = {floatx16{}, floatx16{}};
        auto kfrag = [&](int t, int c) { return __builtin_bit_cast(half8_t, kf[buf][(t * NC + c) * 64 + (lane ^ ((c & 3) << 1))]); };
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
        const float4 s01 = *(const float4 *)&sc[buf][0], s23 = *(const float4 *)&sc[buf][2];
        const float2 s0 = hh ? make_float2(s01.z, s01.w) : make_float2(s01.x, s01.y);
        const float2 s1 = hh ? make_float2(s23.z, s23.w) : make_float2(s23.x, s23.y);
        float ks[2] = {query.scores(s0.x), query.scores(s1.x)}, vs[2] = {s0.y, s1.y};
#pragma unroll
        for (int t = 0; t < 2; t++) ks[t] = ks[t] < 1e-37f ? 1e-37f : ks[t]; // a scale of zero has codes of zero
        if (kb * 64 + 63 > clear) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int left = limit - (kb * 64 + 32 * t + 16 * hh); // last visible token of the lane's block
                if (left < 0) { // none: whatever its scales are
                    ks[t] = 1.f;
                    vs[t] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (i > left) s[t][i] = -INFINITY;
            }
        }
        float mx[2], mv[2];
        const ValueScale value[2] = {ValueScale(vs[0]), ValueScale(vs[1])};
#pragma unroll
        for (int t = 0; t < 2; t++) {
            float y = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) y = fmaxf(y, s[t][i]);
            mx[t] = y * ks[t];
            mv[t] = value[t].top(mx[t]);
        }
        if (__any(fmaxf(mx[0], mx[1]) > m + 6.f || fmaxf(mv[0], mv[1]) > e + 6.f)) {
            auto halves = [](float x) { // the larger of the lane's and the other half's
                const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
                return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
            };
            const float mn = halves(fmaxf(m, fmaxf(mx[0], mx[1]))), en = halves(fmaxf(e, ceilf(fmaxf(mv[0], mv[1]))));
            l *= m == -INFINITY ? 0.f : exp2f(m - mn);
            const float g = e == -INFINITY ? 0.f : exp2f(e - en);
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= g;
            m = mn;
            e = en;
        }
        const float mu = m == -INFINITY ? 0.f : m;
        const float c0 = value[0].c(vs[0], mx[0], e, mu), c1 = value[1].c(vs[1], mx[1], e, mu);
        float sum[2] = {0.f, 0.f};
        uint32_t hi[2][8], lw[2][8];
        auto weights = [&](int t, int i) { // of tokens 2 i and 2 i + 1 of the lane's block
            const float x = __builtin_amdgcn_exp2f(fmaf(s[t][2 * i], ks[t], t ? c1 : c0));
            const float y = __builtin_amdgcn_exp2f(fmaf(s[t][2 * i + 1], ks[t], t ? c1 : c0));
            sum[t] += x;
            sum[t] += y;
            split2_mix(x, y, hi[t][i], lw[t][i]);
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
        l += sum[0] * __builtin_amdgcn_exp2f(-c0 - mu);
        l += sum[1] * __builtin_amdgcn_exp2f(-c1 - mu);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    wide_result<HD>(p, lds, item, h, o, MeanScale(e, m, l), m, l);
}

// The attention of a plan in one launch: wide tiles first, then 16-row tiles,
// `tiles` workgroups of which take turns.
template <int HD, bool WIDE>
__global__ __launch_bounds__(256, 2) void pages_attend_kernel(AttendView p)
{
    union Lds {
        TileLds<HD> tile;
        WideLds<WIDE ? HD : 16> wide;
    };
    __shared__ __align__(16) char mem[sizeof(Lds)];
    Lds &lds = *(Lds *)mem;
    // (the first item, which is there if not of this plan, does not wait for the head)
    const bool wide = WIDE && (int)blockIdx.x < p.wides;
    const int first = wide ? blockIdx.x : (int)blockIdx.x - p.wides, item = first / p.n_kv;
    const PagesItem it = wide ? p.wide_item[item] : p.item[item];
    const PagesPlanHead plan = *p.head;
    if (outgrown(p, plan) || item >= (wide ? plan.n_wide : plan.n_items)) return;
    if constexpr (WIDE) {
        if (wide) {
            attend_wide<HD>(p, *(WideLds<HD> *)mem, it, first);
            return;
        }
    }
    attend_tiles<HD>(p, lds.tile, it, plan.n_items, first, p.tiles);
}

hipError_t launch_pages_attend(const Pages &p, const PagesAttendArgs &a, hipStream_t s)
{
    if (p.bits == 4) return launch_pages4_attend(p, a, s);
    // Workgroups for the parts that the call's requests can have, whatever the pool has
    // room for: one token over 300 keys in a pool of 2^21 tokens and requests of at most
    // 8192 7.4 us, with a workgroup for every part of the pool (16384 of them) 10.4.
    // (No tokens: a workgroup a KV head, for `outgrown`.)
    const int64_t split = (int64_t)p.split * std::min(a.n_requests, a.n_tokens);
    const int64_t parts = std::min((int64_t)p.max_parts, split * pages_most_parts(p.max_context));
    const int64_t most = a.n_tokens == 0 ? 1 : std::max<int64_t>(1, parts + (int64_t)a.n_tokens * p.group / kPagesTileRows + a.n_requests);
    const int64_t most_wide = (int64_t)a.n_tokens * p.group / kPagesWideRows + a.n_requests + pages_wide_target(p.n_kv);
    const int wides = a.wide ? (int)(most_wide * p.n_kv) : 0, tiles = (int)(most < 2048 ? most : 2048) * p.n_kv;
    const size_t bytes = (size_t)kPageBlock * p.hd;
    const AttendView view = {layer_of(p, p.k, a.layer, bytes), layer_of(p, p.v, a.layer, bytes), layer_of(p, p.ks, a.layer, 1), p.table, p.head,
                             p.item, p.wide, p.part, p.wide_part, p.tickets, p.wide_tickets, a.q, a.out, p.n_kv, p.n_heads, p.group,
                             p.sub, p.sub_shift, p.width, p.scale, wides, tiles, a.n_tokens, a.n_requests, a.wide};
    auto launch = [&](auto kernel) { launch_stamped(a.ev_start, a.ev_stop, kernel, dim3(wides + tiles), dim3(256), 0, s, view); };
    if (p.hd == 128) launch(a.wide ? pages_attend_kernel<128, true> : pages_attend_kernel<128, false>);
    else launch(a.wide ? pages_attend_kernel<64, true> : pages_attend_kernel<64, false>);
    return hipGetLastError();
}

// ------------------------------------------------------------ reading back

namespace {
struct ReadView {
    const uint8_t *k, *v;
    const float2 *ks;
    const int32_t *slot;
    float *k_out, *v_out;
    int n, n_kv, page, sub, n_pages;
};
} // namespace

// Sixteen slots and one KV head to a workgroup.  K rows lie in runs of 64
// dims.  V lies dim by dim, so its bytes are read with the tokens along the
// lanes (neighbouring slots: one 64-byte run per load) and turned in LDS.  Bounded
// by what it writes (9400 slots of 8 x 128: 23 us, 3.4 TB/s).
template <int HD>
__global__ __launch_bounds__(256) void pages_read_kernel(ReadView p)
{
    constexpr int ND = HD / 16, BYTES = kPageBlock * HD, LD = HD + 4;
    __shared__ __align__(16) float lv[16][LD];
    const int tid = threadIdx.x, h = blockIdx.y, first = blockIdx.x * 16;
    struct Place {
        size_t block;
        int token;
        float2 s;
    };
    auto place = [&](int i) { // of the workgroup's slot i
        Place r = {0, 0, make_float2(0.f, 0.f)};
        const int sl = first + i < p.n ? p.slot[first + i] : -1;
        if (sl >= 0 && sl / p.page < p.n_pages) {
            r.token = sl % kPageBlock;
            r.block = ((size_t)(sl / p.page) * p.n_kv + h) * p.sub + sl % p.page / kPageBlock;
            r.s = p.ks[r.block];
        }
        return r; // elsewhere the pool's first block with scales of zero
    };
    {
        const Place r = place(tid & 15);
        const uint8_t *src = p.v + r.block * BYTES + r.token;
        uint8_t c[ND];
#pragma unroll
        for (int i = 0; i < ND; i++) c[i] = src[(i * 16 + (tid >> 4)) * 16];
#pragma unroll
        for (int i = 0; i < ND; i++) lv[tid & 15][i * 16 + (tid >> 4)] = (float)((int)c[i] - 128) * r.s.y;
    }
    const int i = tid >> 4, j = tid & 15;
    const Place r = place(i);
    uint32_t w[ND / 4];
#pragma unroll
    for (int c = 0; c < ND / 4; c++) w[c] = *(const uint32_t *)(p.k + r.block * BYTES + k_at<HD>(r.token, ND * j + 4 * c));
    __syncthreads();
    if (first + i >= p.n) return;
    const size_t to = ((size_t)(first + i) * p.n_kv + h) * HD + ND * j;
#pragma unroll
    for (int c = 0; c < ND; c++) p.k_out[to + c] = (float)((int)((w[c / 4] >> (8 * (c % 4))) & 255u) - 128) * r.s.x;
#pragma unroll
    for (int c = 0; c < ND; c++) p.v_out[to + c] = lv[i][ND * j + c];
}

hipError_t launch_pages_read(const Pages &p, int layer, const int32_t *slot, int n, float *k, float *v, hipStream_t s)
{
    if (p.bits == 4) return launch_pages4_read(p, layer, slot, n, k, v, s);
    if (n <= 0) return hipSuccess;
    const size_t bytes = (size_t)kPageBlock * p.hd;
    const ReadView view = {layer_of(p, p.k, layer, bytes), layer_of(p, p.v, layer, bytes), layer_of(p, p.ks, layer, 1), slot, k, v,
                           n, p.n_kv, p.page, p.sub, p.n_pages};
    const dim3 grid((n + 15) / 16, p.n_kv);
    if (p.hd == 128) hipLaunchKernelGGL(pages_read_kernel<128>, grid, dim3(256), 0, s, view);
    else hipLaunchKernelGGL(pages_read_kernel<64>, grid, dim3(256), 0, s, view);
    return hipGetLastError();
}

} // namespace jev
