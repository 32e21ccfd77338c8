// How the work of attention over pages is cut (sm_100a). The rows of a step meet keys in two kinds of sets: a request's own tokens, which its rows see
// up to their own place, and a group's prefix, which all rows of the group see whole. (A request whose rows fill tiles by themselves meets the prefix and its own
// tokens in one set: there is nothing to share then, and nothing to join.) A set's query rows are (row, query head of the key / value head) pairs, in that
// order. Sets of few query rows go to single warps, in tiles of 16 rows and units of 16 keys; sets of many go to the tensor cores' wide form, in tiles
// of 256 rows and units of 64 keys (the two ways).
//
// All units of a way's sets lie on one line: set after set, and in it key / value head after head, tile after tile, with a gap before each tile for what
// starting and storing it costs. The SMs are divided between the ways by the work on their lines, and a way's workers take equal stretches of its line,
// whatever the lengths are. A tile that the ends of stretches cut leaves pieces -- largest score, sum, weighted sum --, which are joined afterwards. Lengths
// are known on the device alone, so every block lays out the lines for itself: one read of the lengths and one prefix sum over the sets.
#pragma once
#include "stream_core.cuh"
#include "../../include/llmb200_paged_kernels.h"

#include <limits.h>

// Division by a number that stays: q = n / d for 0 <= n < 2^31 (Granlund and Montgomery, 1994).
struct Div {
    int d;
    unsigned m, s;
};
inline Div div_of(int d)
{
    Div r = {d, 0, 0};
    while ((1LL << r.s) < d) ++r.s;
    r.m = (unsigned)(((1ULL << 32) * ((1ULL << r.s) - d)) / d + 1);
    return r;
}

// What the host says of a step: query heads of a key / value head, and key / value heads; sets of more than few_most query rows go the second way; a request
// of `big` of them or more meets its prefix by itself; blocks of the kernel, and workers of the first way in one (of the second: one); what a unit
// of the second way costs in units of the first. each: sets of a thread. row_step: rows of a way's tile, in
// 256ths, rounded up.
struct Shape {
    Div by_g, by_kv;
    int few_most, big, blocks, few_warps, each;
    int row_step[2];
    int ratio;
};

// Where a way's pieces lie in d_work: [slot][rows of a tile][hd] sums and [slot][rows of a tile] (largest score, sum), scores in units of log 2. A tile's piece of
// worker w is in slot tile + w: the number of a piece never falls from one to the next on the line, and one of the two grows.
struct Pieces { float *acc; float2 *top; };

namespace {

// The two ways: rows of a tile, keys of a unit, fewest units of a worker, units' worth of a gap (two at least: see line_before). Fewest 2 and 3 of the first way
// take 24.3 us where 4 takes 22.9 and 8 takes 23.2 (24 requests, hd 256), 8 takes 17.0 and 4 14.3 for four chats; gaps of 6 units of the second way 1 % more than 8.
template <int WAY> struct Cut;
template <> struct Cut<0> { static constexpr int ROWS = 16, KEYS = 16, LEAST = 4, GAP = 2; };
template <> struct Cut<1> { static constexpr int ROWS = 256, KEYS = 64, LEAST = 8, GAP = 8; };

// What a block knows of the step, in shared memory.
struct Plan {
    int *row, *len, *group, *prefix;     // [n_req + 1], [n_req], [n_groups + 1], [n_groups]
    int *small;                          // [n_req + 1]: rows of requests that are not big, before each request
    int *unit[2], *tile[2];              // [sets + 1] of a way: place on the line of each set, (head, tile) pairs before it; groups' prefixes first, then requests
    int n_req, n_groups;
    int per[2], units[2];                // units of a worker, of the line
    int many_blocks;                     // blocks of the second way, the first ones
    Shape shape;
};

__host__ __device__ inline size_t plan_bytes(int n_req, int n_groups)
{
    return (((size_t)n_req * 7 + (size_t)n_groups * 6 + 12) * 4 + 15) & ~(size_t)15;
}

__device__ __forceinline__ int over(int n, const Div &d) { return (int)((__umulhi((unsigned)n, d.m) + (unsigned)n) >> d.s); }
// n / d, where the quotient is below 2^22
__device__ __forceinline__ int quotient(int n, int d)
{
    int q = (int)__fdividef((float)n, (float)d);
    const int r = n - q * d;
    q += (r >= d) - (r < 0);
    return q;
}

// The last e < n with start[e] <= at; start is ascending, start[0] = 0.
__device__ __forceinline__ int last_at(const int *start, int n, int at)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}
// Whether the rows of a request have keys in a prefix: its group, or -1.
__device__ __forceinline__ int group_of(const Plan &p, int r)
{
    if (!p.n_groups || r < p.group[0] || r >= p.group[p.n_groups]) return -1;
    const int g = last_at(p.group, p.n_groups, r);
    return p.prefix[g] > 0 ? g : -1;
}

struct Set {
    int rows, nr, keys;                  // new rows, query rows (rows * G), keys: of a request its own
    int before;                          // keys of the prefix that come before the own ones: big requests
    bool own;
};
__device__ __forceinline__ Set set_at(const Plan &p, int e)
{
    Set s;
    s.own = e >= p.n_groups;
    s.before = 0;
    if (s.own) {
        const int r = e - p.n_groups;
        s.rows = p.row[r + 1] - p.row[r]; s.keys = p.len[r];
        if (s.rows * p.shape.by_g.d >= p.shape.big) {
            const int g = group_of(p, r);
            if (g >= 0) s.before = p.prefix[g];
        }
    } else {
        s.rows = p.small[p.group[e + 1]] - p.small[p.group[e]]; s.keys = p.prefix[e];
    }
    s.nr = s.rows * p.shape.by_g.d;
    return s;
}
__device__ __forceinline__ int way_of(const Plan &p, const Set &s) { return s.nr > p.shape.few_most; }
// The row of d_q that a set's i-th row is.
__device__ __forceinline__ int row_at(const Plan &p, int e, int i)
{
    if (e >= p.n_groups) return p.row[e - p.n_groups] + i;
    const int j = p.small[p.group[e]] + i, r = last_at(p.small, p.n_req, j);
    return p.row[r] + j - p.small[r];
}
template <int WAY> __device__ __forceinline__ int tiles_of(const Set &s) { return (s.nr + Cut<WAY>::ROWS - 1) / Cut<WAY>::ROWS; }
// own keys (of a prefix: all) that the last query row of a tile sees; units before the own keys; the tile's units
template <int WAY> __device__ __forceinline__ int seen_by(const Plan &p, const Set &s, int t)
{
    return s.own ? s.keys - s.rows + over(min((t + 1) * Cut<WAY>::ROWS, s.nr) - 1, p.shape.by_g) + 1 : s.keys;
}
template <int WAY> __device__ __forceinline__ int units_before_own(const Set &s) { return (s.before + Cut<WAY>::KEYS - 1) / Cut<WAY>::KEYS; }
template <int WAY> __device__ __forceinline__ int units_of(const Plan &p, const Set &s, int t)
{
    return units_before_own<WAY>(s) + (seen_by<WAY>(p, s, t) + Cut<WAY>::KEYS - 1) / Cut<WAY>::KEYS;
}
// Where the t-th tile of a head begins on the line, its gap included. A request's tiles see about row_step / 256 keys more from one to the next: their places come
// from the sum of that progression, with one unit more a tile for what rounding takes, and a tile's gap is what its units leave (GAP - 2 at least).
template <int WAY, typename Place = int> __device__ __forceinline__ Place line_before(const Plan &p, const Set &s, int t)
{
    constexpr int GAP = Cut<WAY>::GAP, KEYS = Cut<WAY>::KEYS;
    if (!s.own) return (Place)t * (GAP + units_of<WAY>(p, s, 0));
    const long long keys = (long long)(s.keys - s.rows) * t + (((long long)p.shape.row_step[WAY] * t * (t + 1)) >> 9);
    return (Place)t * (GAP + 1 + units_before_own<WAY>(s)) + (Place)(keys / KEYS);
}

// Units of a worker: equal stretches, and none so short that joining costs more than it spreads.
template <int WAY> __device__ __forceinline__ int stretch(int units, int workers)
{
    return max(Cut<WAY>::LEAST, (int)(((unsigned)units + workers - 1) / (unsigned)workers));
}

// Reads the lengths and lays the lines; false (for the whole block) if something does not fit. `mem` holds plan_bytes; for blocks of up to 16 warps.
// Two kernels lay the same plan with unlike numbers of threads, and the second looks for the pieces where the first has left them: so all sums are of whole numbers, whose
// order does not matter. (tests/test_cpu_paged_plan.py compares them.)
// This runs at the head of every launch, from cold instruction caches: short code counts, so loops stay loops. 3.5 thousand clocks for 33 sets (as a function of its
// own, which reads the launch's arguments from memory, 8).
__device__ __forceinline__ bool make_plan(const b200_paged_attn_args &a, const Shape &shape, char *mem, Plan &plan)
{
    __shared__ int4 red[16];
    __shared__ longlong2 red_w[16];
    const int sets = a.n_req + a.n_groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int *const unit = reinterpret_cast<int *>(mem), *const row = unit + 4 * (sets + 1), *const group = row + 3 * a.n_req + 2;
    if (threadIdx.x == 0) {
        plan.n_req = a.n_req; plan.n_groups = a.n_groups; plan.shape = shape;
        plan.unit[0] = unit; plan.tile[0] = unit + sets + 1; plan.unit[1] = unit + 2 * (sets + 1); plan.tile[1] = unit + 3 * (sets + 1);
        plan.row = plan.small = row; plan.len = row + a.n_req + 1;
        plan.group = group; plan.prefix = group + a.n_groups + 1;
    }
    int bad = 0, big = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i <= a.n_req; i += blockDim.x) {           // (n_groups <= n_req)
        const bool is_req = i < a.n_req, is_group = i < a.n_groups;
        const int r0 = a.d_row_start[i], r1 = is_req ? a.d_row_start[i + 1] : r0, len = is_req ? a.d_len[i] : 0;
        const int g0 = i <= a.n_groups && a.n_groups ? a.d_group_start[i] : 0, g1 = is_group ? a.d_group_start[i + 1] : g0, prefix = is_group ? a.d_prefix_len[i] : 0;
        row[i] = r0;
        if (is_req) row[a.n_req + 1 + i] = len;
        if (i <= a.n_groups) group[i] = g0;
        if (is_group) group[a.n_groups + 1 + i] = prefix;
        bad |= (i == 0 && r0 != 0) || r1 < r0 || r1 > a.max_rows || (r1 > r0 && (len < r1 - r0 || len > a.table_ld * a.page));
        bad |= g0 < 0 || g1 < g0 || g1 > a.n_req || prefix < 0 || prefix > a.prefix_ld * a.page;
        big |= !bad && (r1 - r0) * shape.by_g.d >= shape.big;
    }
    if (__syncthreads_or(bad | big)) {
        bad = __syncthreads_or(bad);
        if (bad) {
            if (blockIdx.x == 0 && threadIdx.x == 0 && a.d_status) atomicOr(a.d_status, B200_PAGED_BAD_LENGTH);
            return false;
        }
        if (a.n_groups) {                                    // rows that are not big ones, 32 requests at a time
            int *const small = row + 2 * a.n_req + 1;
            if (warp == 0) {
                int before = 0;
#pragma unroll 1
                for (int r = lane; r - lane < a.n_req; r += 32) {
                    const int rows = r < a.n_req ? row[r + 1] - row[r] : 0, mine = rows * shape.by_g.d >= shape.big && group_of(plan, r) >= 0 ? 0 : rows;
                    int in = mine;
#pragma unroll 1
                    for (int o = 1; o < 32; o <<= 1) {
                        const int x = __shfl_up_sync(0xffffffffu, in, o);
                        if (lane >= o) in += x;
                    }
                    if (r <= a.n_req) small[r] = before + in - mine;
                    before += __shfl_sync(0xffffffffu, in, 31);
                }
                if (lane == 0) { small[a.n_req] = before; plan.small = small; }
            }
            __syncthreads();
        }
    }
    // the two lines: (units, tiles) of each, for the sets of this thread, of the warp, of the block
    const int e0 = min(sets, (int)threadIdx.x * shape.each), e1 = min(sets, e0 + shape.each);
    int4 mine = make_int4(0, 0, 0, 0);
    long long size = 0, many_cost = 0;                       // many_cost: in twentieths of a unit of the first way
#pragma unroll 1
    for (int e = e0; e < e1; ++e) {
        const Set s = set_at(plan, e);
        int n = 0, k = 0;
        long long line = 0;                                  // of a head
        const int way = way_of(plan, s);
        if (s.nr > 0 && s.keys > 0) {
            if (way) {
                k = tiles_of<1>(s);
                line = line_before<1, long long>(plan, s, k);
                // a tile whose rows fit into one stream costs two thirds
                const int last = s.nr - (k - 1) * Cut<1>::ROWS;
                n = (int)line;
                many_cost += (20LL * n - (last > Cut<1>::ROWS / 2 ? 0 : 7 * (n / k))) * (shape.ratio * shape.by_kv.d);
            } else {
                k = tiles_of<0>(s);
                line = line_before<0, long long>(plan, s, k);
                n = (int)line;
            }
            size += line * shape.by_kv.d;
            n *= shape.by_kv.d; k *= shape.by_kv.d;
        }
        int *const at = unit + e + way * 2 * (sets + 1);     // summed up below, by the same thread
        at[0] = n; at[sets + 1] = k;
        int *const other = unit + e + (way ^ 1) * 2 * (sets + 1);
        other[0] = 0; other[sets + 1] = 0;
        if (way) { mine.z += n; mine.w += k; } else { mine.x += n; mine.y += k; }
    }
    int4 in = mine;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, in.x, o), y = __shfl_up_sync(0xffffffffu, in.y, o);
        const int z = __shfl_up_sync(0xffffffffu, in.z, o), w = __shfl_up_sync(0xffffffffu, in.w, o);
        const long long f = __shfl_up_sync(0xffffffffu, size, o), g = __shfl_up_sync(0xffffffffu, many_cost, o);
        if (lane >= o) { in.x += x; in.y += y; in.z += z; in.w += w; size += f; many_cost += g; }
    }
    if (lane == 31) { red[warp] = in; red_w[warp] = make_longlong2(size, many_cost); }
    __syncthreads();
    int4 all = make_int4(0, 0, 0, 0);
    in.x -= mine.x; in.y -= mine.y; in.z -= mine.z; in.w -= mine.w;
    size = many_cost = 0;
#pragma unroll 1
    for (int w = 0; w * 32 * shape.each < sets; ++w) {       // (the others have none)
        const int4 x = red[w];
        if (w < warp) { in.x += x.x; in.y += x.y; in.z += x.z; in.w += x.w; }
        all.x += x.x; all.y += x.y; all.z += x.z; all.w += x.w;
        size += red_w[w].x; many_cost += red_w[w].y;
    }
    if (size > INT_MAX) {                                    // places on the lines are 32-bit numbers
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.d_status) atomicOr(a.d_status, B200_PAGED_BAD_LENGTH);
        return false;
    }
#pragma unroll 1
    for (int e = e0; e < e1; ++e) {
        int *const at = unit + e;
        const int x = at[0], y = at[sets + 1], z = at[2 * (sets + 1)], w = at[3 * (sets + 1)];
        at[0] = in.x; at[sets + 1] = in.y; at[2 * (sets + 1)] = in.z; at[3 * (sets + 1)] = in.w;
        in.x += x; in.y += y; in.z += z; in.w += w;
    }
    if (threadIdx.x == 0) {
        unit[sets] = all.x; unit[2 * sets + 1] = all.y; unit[3 * sets + 2] = all.z; unit[4 * sets + 3] = all.w;
        // blocks for each way: by their shares of the work, no more than have units to begin with, one at least
        int many = 0;
        if (all.z > 0) {
            const unsigned long long both = 20ULL * all.x + many_cost;
            const int down = max(0, 42 - __clzll(both));     // 22 bits of each are enough
            const unsigned part = (unsigned)((unsigned long long)many_cost >> down), whole = (unsigned)(both >> down);
            many = all.x == 0 ? shape.blocks : max(1, min(shape.blocks - 1, (int)((shape.blocks * part + whole / 2) / whole)));
            many = min(many, (all.z + Cut<1>::LEAST - 1) / Cut<1>::LEAST);
        }
        plan.many_blocks = many;
        plan.units[0] = all.x; plan.units[1] = all.z;
        plan.per[0] = stretch<0>(all.x, max(1, shape.blocks - many) * shape.few_warps);
        plan.per[1] = stretch<1>(all.z, max(1, many));
    }
    __syncthreads();
    return true;
}

// One worker's way along a line: the pieces of its stretch, one after the other.
struct Piece {
    int e, h, t, tiles;                  // set, key / value head, tile, tiles of a head
    int k0, n, ut;                       // its units k0 .. k0 + n - 1 of the tile's ut
    Set s;
};
template <int WAY> struct Walk {
    int at, end, e;
    __device__ __forceinline__ Walk(const Plan &p, int worker)
    {
        at = (int)min((long long)worker * p.per[WAY], (long long)p.units[WAY]);
        end = p.units[WAY] - at > p.per[WAY] ? at + p.per[WAY] : p.units[WAY];
        e = at < end ? last_at(p.unit[WAY], p.n_req + p.n_groups, at) : 0;
    }
    __device__ __forceinline__ bool next(const Plan &p, Piece &q)
    {
        while (at < end) {
            const int *unit = p.unit[WAY];
            while (unit[e + 1] <= at) ++e;
            q.e = e;
            q.s = set_at(p, e);
            q.tiles = tiles_of<WAY>(q.s);
            const int head = over(unit[e + 1] - unit[e], p.shape.by_kv);
            q.h = quotient(at - unit[e], head);
            int rest = at - unit[e] - q.h * head, end_of = head;
            q.t = 0;
            if (q.tiles > 1) {                               // the last tile that begins at or before the place
                int hi = q.tiles;
#pragma unroll 1
                while (hi - q.t > 1) {
                    const int mid = (q.t + hi) >> 1;
                    if (line_before<WAY>(p, q.s, mid) <= rest) q.t = mid; else hi = mid;
                }
                const int begin = line_before<WAY>(p, q.s, q.t);
                rest -= begin;
                end_of = line_before<WAY>(p, q.s, q.t + 1) - begin;
            }
            q.ut = units_of<WAY>(p, q.s, q.t);
            const int gap = end_of - q.ut, n = min(end_of - rest, end - at);
            at += n;
            q.k0 = max(0, rest - gap);
            q.n = rest + n - gap - q.k0;
            if (q.n > 0) return true;                        // (not only a gap)
        }
        return false;
    }
};

// Where the keys of a piece lie: in the prefix's pages, or behind `first` units of them in the request's own, and how many of each the tile's last row sees.
struct Keys {
    const int *prefix, *table;
    int first, before, seen;
};
template <int WAY> __device__ __forceinline__ Keys keys_of(const b200_paged_attn_args &a, const Plan &p, const Piece &q)
{
    if (!q.s.own) return {a.d_prefix_table + (size_t)q.e * a.prefix_ld, nullptr, INT_MAX, q.s.keys, 0};
    const int r = q.e - a.n_groups;
    return {q.s.before ? a.d_prefix_table + (size_t)group_of(p, r) * a.prefix_ld : nullptr, a.d_table + (size_t)r * a.table_ld, units_before_own<WAY>(q.s), q.s.before, seen_by<WAY>(p, q.s, q.t)};
}
// A unit of a piece: its page table, its first key there, and how many keys the tile's last row sees there.
struct Part { const int *table; int key0, seen; bool own; };
template <int WAY> __device__ __forceinline__ Part part_at(const Keys &k, const Piece &q, int unit)
{
    const int u = q.k0 + unit;
    if (u < k.first) return {k.prefix, u * Cut<WAY>::KEYS, k.before, false};
    return {k.table, (u - k.first) * Cut<WAY>::KEYS, k.seen, true};
}
// Whether a set's rows have all of their keys in it.
__device__ __forceinline__ bool alone(const Plan &p, const Piece &q) { return q.s.own && (q.s.before > 0 || group_of(p, q.e - p.n_groups) < 0); }

}  // namespace
