// How the work of attention over pages is cut (sm_100a). The rows of a step meet keys in two kinds of sets: a request's own tokens, which its rows see
// up to their own place, and a group's prefix, which all rows of the group see whole. (A request whose rows fill tiles by themselves meets the prefix and its own
// tokens in one set: there is nothing to share then, and nothing to join.) A set's query rows -- (row, query head of the key / value head) pairs, in
// that order -- are cut into tiles of RT, the keys that a tile sees into units of KU, and all units of all sets lie on one line: set after set, and in it
// key / value head after head, tile after tile, with a gap before each tile for what starting and storing it costs. Workers take equal stretches of that line,
// whatever the lengths are; a tile that the ends of stretches cut leaves pieces -- largest score, sum, weighted sum --, which are joined afterwards. Lengths are known on the device alone, so every block
// lays out the line for itself: one read of the lengths and a prefix sum, about a microsecond.
#pragma once
#include "stream_core.cuh"
#include "../../include/llmb200_paged_kernels.h"

#include <limits.h>

// The sets that a kernel deals with: those of more than `lo` and at most `hi` query rows, in tiles of RT rows and units of KU keys.
// A worker takes `least` units at least; `gap` units stand before each tile.
struct Cut { int rt, ku, lo, hi, least, gap; };

// Where a cut's pieces lie in d_work: [slot][rt][hd] sums and [slot][rt] (largest score, sum), scores in units of log 2. A tile's piece of worker w is in
// slot tile + w: the number of a piece never falls from one to the next on the line, and one of the two grows.
struct Pieces { float *acc; float2 *top; int workers; };

namespace {

// What a block knows of the step, in shared memory.
struct Plan {
    int *row, *len, *group, *prefix;     // [n_req + 1], [n_req], [n_groups + 1], [n_groups]
    int *small;                          // [n_req + 1]: rows of requests that are not big, before each request
    char *lines;                         // room for the lines
    int n_req, n_groups, n_kv, G, big;   // a request of `big` query rows or more meets its prefix by itself
};
// One cut's line.
struct Line {
    int *unit;                           // [sets + 1]: units before each set; groups' prefixes first, then requests
    int *tile;                           // [sets + 1]: (head, tile) pairs before each set
    int units, per;                      // all units; those of a worker
};

__host__ __device__ inline size_t plan_bytes(int n_req, int n_groups, int cuts)
{
    const size_t sets = (size_t)n_req + n_groups;
    const size_t n = (size_t)cuts * 2 * (sets + 1) * 4 + ((size_t)n_req * 3 + 3 + 2 * (size_t)n_groups + 2) * 4;
    return (n + 15) & ~(size_t)15;
}

// The last e < n with start[e] <= at; start is ascending, start[0] = 0.
template <typename I> __device__ __forceinline__ int last_at(const I *start, int n, I at)
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

__device__ __forceinline__ bool is_big(const Plan &p, int r, int group) { return group >= 0 && (p.row[r + 1] - p.row[r]) * p.G >= p.big; }
__device__ __forceinline__ Set set_at(const Plan &p, int e)
{
    Set s;
    s.own = e >= p.n_groups;
    s.before = 0;
    if (s.own) {
        const int r = e - p.n_groups;
        s.rows = p.row[r + 1] - p.row[r]; s.keys = p.len[r];
        if (s.rows * p.G >= p.big) {
            const int g = group_of(p, r);
            if (g >= 0) s.before = p.prefix[g];
        }
    } else {
        s.rows = p.small[p.group[e + 1]] - p.small[p.group[e]]; s.keys = p.prefix[e];
    }
    s.nr = s.rows * p.G;
    return s;
}
// The row of d_q that a set's i-th row is.
__device__ __forceinline__ int row_at(const Plan &p, int e, int i)
{
    if (e >= p.n_groups) return p.row[e - p.n_groups] + i;
    const int j = p.small[p.group[e]] + i, r = last_at(p.small, p.n_req, j);
    return p.row[r] + j - p.small[r];
}
__device__ __forceinline__ bool in_cut(const Set &s, const Cut &c) { return s.nr > c.lo && s.nr <= c.hi && s.keys > 0; }
__device__ __forceinline__ int tiles_of(const Set &s, const Cut &c) { return (s.nr + c.rt - 1) / c.rt; }
// own keys (of a prefix: all) that the last query row of a tile sees; units before the own keys; the tile's units
__device__ __forceinline__ int seen_by(const Plan &p, const Set &s, const Cut &c, int t)
{
    return s.own ? s.keys - s.rows + (min((t + 1) * c.rt, s.nr) - 1) / p.G + 1 : s.keys;
}
__device__ __forceinline__ int units_before_own(const Set &s, const Cut &c) { return (s.before + c.ku - 1) / c.ku; }
__device__ __forceinline__ int units_of(const Plan &p, const Set &s, const Cut &c, int t) { return units_before_own(s, c) + (seen_by(p, s, c, t) + c.ku - 1) / c.ku; }
// where the t-th tile of a head begins on the line, its gap included
__device__ __forceinline__ long long line_before(const Plan &p, const Set &s, const Cut &c, int t)
{
    if (!s.own) return (long long)t * (c.gap + units_of(p, s, c, 0));
    long long n = (long long)t * c.gap;
    for (int i = 0; i < t; ++i) n += units_of(p, s, c, i);
    return n;
}

// Reads the lengths; false (for the whole block) if one of them does not fit. `mem` holds plan_bytes. `red`: 32 ints.
__device__ inline bool load_plan(const b200_paged_attn_args &a, Plan &p, char *mem, int cuts, int big, int *red)
{
    const int sets = a.n_req + a.n_groups;
    p.n_req = a.n_req; p.n_groups = a.n_groups; p.n_kv = a.n_kv; p.G = a.n_q / a.n_kv; p.big = big;
    p.lines = mem;
    p.row = reinterpret_cast<int *>(mem) + (size_t)cuts * 2 * (sets + 1);
    p.len = p.row + a.n_req + 1;
    p.small = p.len + a.n_req + 1;
    p.group = p.small + a.n_req + 1;
    p.prefix = p.group + a.n_groups + 1;
    for (int i = threadIdx.x; i <= a.n_req; i += blockDim.x) {
        p.row[i] = a.d_row_start[i];
        if (i < a.n_req) p.len[i] = a.d_len[i];
    }
    for (int i = threadIdx.x; i < a.n_groups + (a.n_groups > 0); i += blockDim.x) {
        p.group[i] = a.d_group_start[i];
        if (i < a.n_groups) p.prefix[i] = a.d_prefix_len[i];
    }
    __syncthreads();
    int bad = 0;
    for (int i = threadIdx.x; i < a.n_req; i += blockDim.x) {
        const int r0 = p.row[i], r1 = p.row[i + 1], len = p.len[i];
        bad |= (i == 0 && r0 != 0) || r1 < r0 || r1 > a.max_rows;
        bad |= r1 > r0 && (len < r1 - r0 || len > (long long)a.table_ld * a.page);
    }
    for (int i = threadIdx.x; i < a.n_groups; i += blockDim.x) {
        const int g0 = p.group[i], g1 = p.group[i + 1];
        bad |= g0 < 0 || g1 < g0 || g1 > a.n_req || p.prefix[i] < 0 || p.prefix[i] > (long long)a.prefix_ld * a.page;
    }
    bad = __syncthreads_or(bad);
    if (bad && blockIdx.x == 0 && threadIdx.x == 0 && a.d_status) atomicOr(a.d_status, B200_PAGED_BAD_LENGTH);
    if (bad) return false;
    // rows of small requests: all of them where none can be big
    if (big == INT_MAX || !a.n_groups) { p.small = p.row; return true; }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const int each = (a.n_req + blockDim.x - 1) / blockDim.x, r0 = min(a.n_req, (int)threadIdx.x * each), r1 = min(a.n_req, r0 + each);
    int n = 0;
    for (int r = r0; r < r1; ++r) n += is_big(p, r, group_of(p, r)) ? 0 : p.row[r + 1] - p.row[r];
    int in = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += x;
    }
    if (lane == 31) red[warp] = in;
    __syncthreads();
    in -= n;
    for (int w = 0; w < warp; ++w) in += red[w];
    for (int r = r0; r < r1; ++r) {
        p.small[r] = in;
        in += is_big(p, r, group_of(p, r)) ? 0 : p.row[r + 1] - p.row[r];
        if (r == a.n_req - 1) p.small[a.n_req] = in;
    }
    __syncthreads();
    return true;
}

// Units of a worker: equal stretches, and none so short that joining costs more than it spreads.
__device__ __forceinline__ int stretch(int units, int workers, int least) { return max(least, units / workers + (units % workers != 0)); }

// Lays the line of a cut that `workers` share, in the k-th room for one; false (for the whole block) if it has more than 2^31 - 1 units. `red`: 32 long
// longs and 32 ints.
__device__ inline bool lay_line(const b200_paged_attn_args &a, const Plan &p, const Cut &c, int k, int workers, Line &line, long long *red, int *red_t)
{
    const int sets = p.n_req + p.n_groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    line.unit = reinterpret_cast<int *>(p.lines) + (size_t)2 * k * (sets + 1);
    line.tile = line.unit + sets + 1;
    const int each = (sets + blockDim.x - 1) / blockDim.x, e0 = min(sets, (int)threadIdx.x * each), e1 = min(sets, e0 + each);
    long long u = 0;
    int t = 0;
    for (int e = e0; e < e1; ++e) {
        const Set s = set_at(p, e);
        long long n = 0;
        int m = 0;
        if (in_cut(s, c)) { m = tiles_of(s, c); n = line_before(p, s, c, m) * p.n_kv; m *= p.n_kv; }
        line.unit[e] = (int)n; line.tile[e] = m;                  // summed up below, by the same thread
        u += n; t += m;
    }
    long long iu = u;
    int it = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, iu, o);
        const int y = __shfl_up_sync(0xffffffffu, it, o);
        if (lane >= o) { iu += x; it += y; }
    }
    __syncthreads();                                         // `red` of an earlier line
    if (lane == 31) { red[warp] = iu; red_t[warp] = it; }
    __syncthreads();
    long long all = 0;
    int all_t = 0;
    iu -= u; it -= t;
    for (int w = 0; w < nw; ++w) {
        if (w == warp) { iu += all; it += all_t; }
        all += red[w]; all_t += red_t[w];
    }
    for (int e = e0; e < e1; ++e) {
        const int n = line.unit[e], m = line.tile[e];
        line.unit[e] = (int)iu; line.tile[e] = it;
        iu += n; it += m;
    }
    if (threadIdx.x == 0) { line.unit[sets] = (int)all; line.tile[sets] = all_t; }
    __syncthreads();
    if (all > 0x7fffffff) {
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.d_status) atomicOr(a.d_status, B200_PAGED_BAD_LENGTH);
        return false;
    }
    line.units = (int)all;
    line.per = stretch(line.units, workers, c.least);
    return true;
}

// One worker's way along a line: the pieces of its stretch, one after the other.
struct Piece {
    int e, h, t, tiles;                  // set, key / value head, tile, tiles of a head
    int k0, n, ut;                       // its units k0 .. k0 + n - 1 of the tile's ut
    Set s;
};
struct Walk {
    int at, end, e;
    __device__ __forceinline__ Walk(const Plan &p, const Line &line, int worker)
    {
        at = (int)min((long long)worker * line.per, (long long)line.units);
        end = line.units - at > line.per ? at + line.per : line.units;
        e = at < end ? last_at(line.unit, p.n_req + p.n_groups, at) : 0;
    }
    __device__ __forceinline__ bool next(const Plan &p, const Line &line, const Cut &c, Piece &q)
    {
        while (at < end) {
            while (line.unit[e + 1] <= at) ++e;
            q.e = e;
            q.s = set_at(p, e);
            q.tiles = tiles_of(q.s, c);
            const int head = (line.unit[e + 1] - line.unit[e]) / p.n_kv;
            q.h = (at - line.unit[e]) / head;
            int rest = at - line.unit[e] - q.h * head;
            q.t = 0;
            q.ut = units_of(p, q.s, c, 0);
            while (rest >= c.gap + q.ut) { rest -= c.gap + q.ut; q.ut = units_of(p, q.s, c, ++q.t); }
            const int n = min(c.gap + q.ut - rest, end - at);
            at += n;
            q.k0 = max(0, rest - c.gap);
            q.n = rest + n - c.gap - q.k0;
            if (q.n > 0) return true;                        // (not only a gap)
        }
        return false;
    }
};

// A unit of a piece: its page table, its first key there, and how many keys the tile's last row sees there.
struct Part { const int *table; int key0, seen; bool own; };
__device__ __forceinline__ Part part_at(const b200_paged_attn_args &a, const Plan &p, const Cut &c, const Piece &q, int unit)
{
    const int first = units_before_own(q.s, c), u = q.k0 + unit, r = q.e - a.n_groups;
    if (!q.s.own) return {a.d_prefix_table + (size_t)q.e * a.prefix_ld, u * c.ku, q.s.keys, false};
    if (u < first) return {a.d_prefix_table + (size_t)group_of(p, r) * a.prefix_ld, u * c.ku, q.s.before, false};
    return {a.d_table + (size_t)r * a.table_ld, (u - first) * c.ku, seen_by(p, q.s, c, q.t), true};
}
// Whether a set's rows have all of their keys in it.
__device__ __forceinline__ bool alone(const Plan &p, const Piece &q) { return q.s.own && (q.s.before > 0 || group_of(p, q.e - p.n_groups) < 0); }

}  // namespace
