// Attention of a step's new rows over pages (sm_100a): each row over its request's own tokens, and over a prefix that its group shares. One launch works on all keys
// (paged_plan.cuh: how they are cut; paged_attention_few.cuh and paged_attention_many.cuh: the two ways), one block to an SM, and a second one joins the pieces
// of tiles that were cut. (Two launches for the two ways, one after the other, and plans and joins without care for cold instruction caches: 77 us for 32
// answers to a prompt of 8199 tokens that take 42 now, 28 for four short chats that take 14; floors 16 and 0.5.)
#include "paged_attention_few.cuh"
#include "paged_attention_many.cuh"

#include <atomic>
#include <cmath>

extern unsigned long long g_b200_launches;

namespace {

constexpr int JOIN_WARPS = 4, JOIN_BLOCKS = 4, JOIN_CHUNK = 8;
// Sets of more query rows than FEW_MOST go the second way, where hd is one of its own (two tiles of 16 rows read their keys twice, mostly from L2). Us, hd 128,
// 8 key / value heads, by single warps and on tcgen05: 8 requests of 6000 tokens, 32 query rows each 54 and 66, 48 rows 74 and 70, 64 rows 134 and 70; 64 of
// 1500 tokens, 32 rows 137 and 132, 48 rows 217 and 140; hd 64, 64 requests of 32 rows 74 and 107, of 48 rows 124 and 115.
// A request of BIG_ROWS query rows fills a stream there by itself: portions that met prefix and own tokens in two sets, and were joined, took 520 us
// where one set takes 287 (four requests of 125 .. 811 new tokens behind 4096).
constexpr int FEW_MOST = 32, BIG_ROWS = 128;

__host__ __device__ constexpr int block_threads(int hd) { return hd > 128 ? 128 : MANY_THREADS; }
__host__ __device__ constexpr int most_few_warps(int hd) { return hd > 128 ? 4 : 8; }

struct Room { int slots, plan_off; };
// Dynamic shared memory: what is left of an SM's besides static memory and the alignment to 1024 bytes.
constexpr size_t ROOM = 227 * 1024 - 2048 - 1024;

template <typename T, int HD>
__global__ void __launch_bounds__(block_threads(HD), 1)
attn_pages_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ b200_paged_attn_args a, const __grid_constant__ Shape shape,
                  const Pieces few, const Pieces many, const Room room)
{
    extern __shared__ __align__(1024) char smem[];
    __shared__ Plan plan;                                    // not in registers: those are for the scores
    char *base = smem + ((1024 - (smem_u32(smem) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_launch_dependents();                                 // after the wait: attn_join_kernel reads the lengths ahead of its own
    if (!make_plan(a, shape, base + room.plan_off, plan)) return;
    if constexpr (HD > 128) {
        if (warp < shape.few_warps) few_worker<T, HD>(a, plan, few, blockIdx.x * shape.few_warps + warp, smem_u32(base) + warp * few_ring(HD));
    }
    else if ((int)blockIdx.x < plan.many_blocks) many_block<T, HD>(map_k, map_v, a, plan, many, base, room.slots);
    else if (warp >= 4) {                                    // registers as in many_block
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        if (warp - 4 < shape.few_warps)
            few_worker<T, HD>(a, plan, few, ((int)blockIdx.x - plan.many_blocks) * shape.few_warps + warp - 4, smem_u32(base) + (warp - 4) * few_ring(HD));
    } else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
}

// The pieces of a tile that a row of it has: where the first one lies, how many, how far apart; whether there is more than the one that covers all.
struct Cuts { const float *acc; const float2 *top; int count, step; bool several; };
template <int WAY> __device__ __forceinline__ Cuts cuts_of(const Plan &p, const Set &s, const Pieces &in, int e, int h, int i, int hd)
{
    constexpr int ROWS = Cut<WAY>::ROWS;
    const int t = i / ROWS, per_head = over(p.unit[WAY][e + 1] - p.unit[WAY][e], p.shape.by_kv);
    const int end = p.unit[WAY][e] + h * per_head + line_before<WAY>(p, s, t + 1);           // the tile's units end where the next tile's gap begins
    const int w0 = quotient(end - units_of<WAY>(p, s, t), p.per[WAY]), w1 = quotient(end - 1, p.per[WAY]);
    // a tile of 128 rows at most, in places for 256: two pieces in each, of every other unit
    const bool halves = WAY == 1 && s.nr - t * ROWS <= ROWS / 2;
    const long long place = (long long)(p.tile[WAY][e] + h * tiles_of<WAY>(s) + t + w0) * ROWS + i % ROWS;
    return {in.acc + place * hd, in.top + place, (w1 - w0 + 1) * (halves ? 2 : 1), halves ? ROWS / 2 : ROWS, w1 > w0 || halves};
}

// A warp to each (row, query head) whose keys were cut, over the pieces in the order of the lines.
template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
attn_join_kernel(const __grid_constant__ b200_paged_attn_args a, const __grid_constant__ Shape shape, const Pieces few, const Pieces many)
{
    constexpr int N = HD / 32, AHEAD = 8;                    // numbers of a lane, next to one another; pieces on their way
    extern __shared__ __align__(1024) char smem[];
    __shared__ Plan p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // The lengths are older than the kernel before this one, which started after all that came before it had ended: only its pieces are waited for.
    if (!make_plan(a, shape, smem, p)) { pdl_wait(); return; }
    pdl_launch_dependents();
    bool waited = false;
    const int G = shape.by_g.d, all = p.row[p.n_req] * a.n_q, workers = gridDim.x * JOIN_WARPS;
#pragma unroll 1
    for (int at = blockIdx.x * JOIN_WARPS + warp; at < all; at += workers) {
        const int row = at / a.n_q, head = at - row * a.n_q, h = over(head, shape.by_g), r = last_at(p.row, p.n_req, row);
        int group = group_of(p, r);
        const Set own = set_at(p, p.n_groups + r);
        if (own.before > 0) group = -1;                      // one set
        const int i = (row - p.row[r]) * G + head - h * G;
        Cuts x = {}, y = way_of(p, own) ? cuts_of<1>(p, own, many, p.n_groups + r, h, i, HD) : cuts_of<0>(p, own, few, p.n_groups + r, h, i, HD);
        if (group >= 0) {
            const Set shared = set_at(p, group);
            const int j = i + (p.small[r] - p.small[p.group[group]]) * G;
            x = way_of(p, shared) ? cuts_of<1>(p, shared, many, group, h, j, HD) : cuts_of<0>(p, shared, few, group, h, j, HD);
        }
        x.acc += lane * N; y.acc += lane * N;
        if (group < 0 && !y.several) continue;           // stored where it was formed
        if (!waited) { pdl_wait(); waited = true; }
        const int n = x.count + y.count;
        auto top_of = [&](int j) { return j < x.count ? x.top + (long long)j * x.step : y.top + (long long)(j - x.count) * y.step; };
        auto acc_of = [&](int j) { return j < x.count ? x.acc + (long long)j * x.step * HD : y.acc + (long long)(j - x.count) * y.step * HD; };
        float top = -INFINITY, l = 0.0f, o[N];
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] = 0.0f;
#pragma unroll 1
        for (int j0 = 0; j0 < n; j0 += AHEAD) {
            float2 ml[AHEAD];
            float v[AHEAD][N];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {            // behind the last one it again, with no weight
                const int k = min(j0 + j, n - 1);
                const float *from = acc_of(k);
                ml[j] = *top_of(k);
                if constexpr (N >= 4) {
#pragma unroll
                    for (int q = 0; q < N; q += 4) *reinterpret_cast<float4 *>(&v[j][q]) = *reinterpret_cast<const float4 *>(from + q);
                } else *reinterpret_cast<float2 *>(v[j]) = *reinterpret_cast<const float2 *>(from);
            }
            asm volatile("" ::: "memory");                  // all of them before the first is used: left to itself the compiler puts each before its use
            float higher = top;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) higher = fmaxf(higher, ml[j].x);
            const float base = higher == -INFINITY ? 0.0f : higher, down = ex2(top - base);
            top = higher;
            l *= down;
#pragma unroll
            for (int q = 0; q < N; ++q) o[q] *= down;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const bool on = j0 + j < n;
                const float f = on ? ex2(ml[j].x - base) : 0.0f;
                l = fmaf(on ? ml[j].y : 0.0f, f, l);
#pragma unroll
                for (int q = 0; q < N; ++q) o[q] = fmaf(on ? v[j][q] : 0.0f, f, o[q]);
            }
        }
        const float inv = 1.0f / l;
        uint32_t *to = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.d_out) + (long long)row * a.out_ld + (size_t)head * HD + lane * N);
#pragma unroll
        for (int q = 0; q < N; q += 2) to[q / 2] = pack2<T>(o[q] * inv, o[q + 1] * inv);
    }
    if (!waited) pdl_wait();
}

// Joins the pieces of R query rows next to one another in their tiles -- those of x, then those of y -- and stores them. AHEAD pieces of each are on their way at a time.
template <typename T, int HD, int R, int AHEAD>
__device__ __forceinline__ void join_rows(const Cuts &x, const Cuts &y, uint16_t *const (&to)[R])
{
    constexpr int N = HD / 32;                               // numbers of a lane, next to one another
    const int lane = threadIdx.x & 31, n = x.count + y.count;
    float top[R], l[R], o[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        top[r] = -INFINITY; l[r] = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) o[r][k] = 0.0f;
    }
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += AHEAD) {
        float2 ml[R][AHEAD];
        float v[R][AHEAD][N];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {                    // behind the last one it again, with no weight
            const int k = min(j0 + j, n - 1);
            const long long at = k < x.count ? (long long)k * x.step : (long long)(k - x.count) * y.step;
            const float *from = (k < x.count ? x.acc : y.acc) + at * HD + lane * N;
            const float2 *tops = (k < x.count ? x.top : y.top) + at;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                ml[r][j] = tops[r];
                if constexpr (N >= 4) {
#pragma unroll
                    for (int q = 0; q < N; q += 4) *reinterpret_cast<float4 *>(&v[r][j][q]) = *reinterpret_cast<const float4 *>(from + r * HD + q);
                } else *reinterpret_cast<float2 *>(v[r][j]) = *reinterpret_cast<const float2 *>(from + r * HD);
            }
        }
        asm volatile("" ::: "memory");                      // all of them before the first is used
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float higher = top[r];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) higher = fmaxf(higher, ml[r][j].x);
            const float base = higher == -INFINITY ? 0.0f : higher, down = ex2(top[r] - base);
            top[r] = higher;
            l[r] *= down;
#pragma unroll
            for (int q = 0; q < N; ++q) o[r][q] *= down;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const bool on = j0 + j < n;
                const float f = on ? ex2(ml[r][j].x - base) : 0.0f;
                l[r] = fmaf(on ? ml[r][j].y : 0.0f, f, l[r]);
#pragma unroll
                for (int q = 0; q < N; ++q) o[r][q] = fmaf(on ? v[r][j][q] : 0.0f, f, o[r][q]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float inv = 1.0f / l[r];
        uint32_t *out = reinterpret_cast<uint32_t *>(to[r] + lane * N);
#pragma unroll
        for (int q = 0; q < N; q += 2) out[q / 2] = pack2<T>(o[r][q] * inv, o[r][q + 1] * inv);
    }
}

// The same where there are more query rows than warps: a key / value head's query rows of all requests are one sequence, of which a warp takes up to JOIN_CHUNK in a
// row, looks up their places together and joins two at a time. Four portions, 38 000 rows of two or three pieces: 31 us, and 51 one by one; 96 rows of 35
// pieces, hd 256: 12 one by one, and 21 so.
template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
attn_join_rows_kernel(const __grid_constant__ b200_paged_attn_args a, const __grid_constant__ Shape shape, const Pieces few, const Pieces many)
{
    extern __shared__ __align__(1024) char smem[];
    __shared__ Plan p;
    const int warp = threadIdx.x >> 5;
    // The lengths are older than the kernel before this one, which started after all that came before it had ended: only its pieces are waited for.
    if (!make_plan(a, shape, smem, p)) { pdl_wait(); return; }
    pdl_launch_dependents();
    bool waited = false;
    const int G = shape.by_g.d, per_head = p.row[p.n_req] * G, workers = gridDim.x * JOIN_WARPS;
    const int chunk = (int)min(((long long)per_head * a.n_kv + workers - 1) / workers, (long long)JOIN_CHUNK), chunks = chunk ? (per_head + chunk - 1) / chunk : 0;      // of a head
    for (long long c = blockIdx.x * JOIN_WARPS + warp; c < (long long)chunks * a.n_kv; c += workers) {
        const int h = (int)(c / chunks), begin = ((int)(c % chunks)) * chunk, end = min(begin + chunk, per_head);
        int r = 0, past = 0, group = -1, shift = 0, y_from = 0, y_past = 0, x_from = 0, x_past = 0;     // request, end of its rows; where the cuts looked up hold
        Cuts x = {}, y = {};
        for (int at = begin; at < end;) {
            if (at >= past) {                                // another request
                r = last_at(p.row, p.n_req, over(at, shape.by_g));
                past = p.row[r + 1] * G;
                group = group_of(p, r);
                if (set_at(p, p.n_groups + r).before > 0) group = -1;    // one set
                shift = group >= 0 ? (p.small[r] - p.small[p.group[group]]) * G : 0;
                y_past = x_past = -1;
                x = {};
            }
            const int i = at - p.row[r] * G, j = i + shift;
            if (i >= y_past) {
                const Set own = set_at(p, p.n_groups + r);
                const int way = way_of(p, own), rows = way ? MANY_ROWS : FEW_ROWS;
                y = way ? cuts_of<1>(p, own, many, p.n_groups + r, h, i, HD) : cuts_of<0>(p, own, few, p.n_groups + r, h, i, HD);
                y_from = i; y_past = (i / rows + 1) * rows;
            }
            if (group >= 0 && j >= x_past) {
                const Set shared = set_at(p, group);
                const int way = way_of(p, shared), rows = way ? MANY_ROWS : FEW_ROWS;
                x = way ? cuts_of<1>(p, shared, many, group, h, j, HD) : cuts_of<0>(p, shared, few, group, h, j, HD);
                x_from = j; x_past = (j / rows + 1) * rows;
            }
            int left = min(min(end, past) - at, y_past - i); // rows that are found at the same places
            if (group >= 0) left = min(left, x_past - j);
            if (group < 0 && !y.several) { at += left; continue; }       // stored where they were formed
            if (!waited) { pdl_wait(); waited = true; }
            auto out = [&](int k) {
                const int row = over(at + k, shape.by_g);
                return static_cast<uint16_t *>(a.d_out) + (long long)row * a.out_ld + (size_t)(h * G + at + k - row * G) * HD;
            };
            const Cuts xs = {x.acc + (long long)(j - x_from) * HD, x.top + (j - x_from), x.count, x.step, true};
            const Cuts ys = {y.acc + (long long)(i - y_from) * HD, y.top + (i - y_from), y.count, y.step, true};
            if (left >= 2) {
                uint16_t *const to[2] = {out(0), out(1)};
                join_rows<T, HD, 2, (HD > 128 ? 2 : 4)>(xs, ys, to);
                at += 2;
            } else {
                uint16_t *const to[1] = {out(0)};
                join_rows<T, HD, 1, 8>(xs, ys, to);
                ++at;
            }
        }
    }
    if (!waited) pdl_wait();
}

constexpr int DEVICES = 64;              // beyond these nothing is remembered

int sm_count()
{
    static std::atomic<int> known[DEVICES];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev < DEVICES && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    if (dev < DEVICES) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Lets a kernel have all of an SM's shared memory, once a device.
template <typename K> cudaError_t allow_all(K kern, std::atomic<unsigned long long> &done)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < DEVICES && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
    cudaFuncAttributes at;
    if ((e = cudaFuncGetAttributes(&at, kern)) != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)at.sharedSizeBytes);
    if (e == cudaSuccess && dev < DEVICES) done.fetch_or(1ULL << dev, std::memory_order_relaxed);
    return e;
}

// Sizes alone: 0, or why they are refused.
int check_sizes(const b200_paged_attn_args &a)
{
    if ((a.wtype != B200_WT_F16 && a.wtype != B200_WT_BF16) || (a.hd != 64 && a.hd != 128 && a.hd != 256)) return B200_E_BADARG;
    if (a.n_q < 1 || a.n_kv < 1 || a.n_q % a.n_kv || a.n_q > 1024 || a.max_rows < 0 || a.max_rows > (1 << 20) || a.n_pages < 1) return B200_E_BADARG;
    if (a.page < 16 || a.page > 256 || (a.page & (a.page - 1))) return B200_E_BADARG;
    if (a.n_req < 0 || a.n_req > B200_PAGED_MAX_REQ || a.n_groups < 0 || a.n_groups > a.n_req) return B200_E_BADARG;
    if (a.table_ld < 0 || a.table_ld > (1 << 20) || a.prefix_ld < 0 || a.prefix_ld > (1 << 20)) return B200_E_BADARG;
    if ((long long)a.n_pages * a.page > INT_MAX || (long long)a.n_pages * a.n_kv > INT_MAX || (long long)a.table_ld * a.page > INT_MAX || (long long)a.prefix_ld * a.page > INT_MAX)
        return B200_E_TOOLARGE;
    return 0;
}

struct Layout { Shape shape; size_t few_acc, few_top, many_acc, many_top, bytes; };

Layout layout_of(const b200_paged_attn_args &a)
{
    const long long G = a.n_q / a.n_kv, all = a.max_rows * G * (a.n_groups ? 2 : 1);         // query rows of all sets
    const long long sets = (a.n_req < a.max_rows ? a.n_req : a.max_rows) + (a.n_groups < a.max_rows ? a.n_groups : a.max_rows);
    const bool wide = a.hd <= 128;
    Layout L = {};
    L.shape.by_g = div_of((int)G); L.shape.by_kv = div_of(a.n_kv);
    L.shape.few_most = wide ? FEW_MOST : INT_MAX; L.shape.big = wide ? BIG_ROWS : INT_MAX;
    L.shape.blocks = sm_count(); 
    const int rings = (int)((ROOM - plan_bytes(a.n_req, a.n_groups)) / few_ring(a.hd));       // hundreds of requests leave less than all of the warps a ring
    L.shape.few_warps = rings < most_few_warps(a.hd) ? rings : most_few_warps(a.hd);
    L.shape.ratio = a.hd == 64 ? 16 : 10;              // from the ends of both kinds of blocks, 64 requests of one prefix of 65521 tokens: together within a tenth
    L.shape.row_step[0] = (int)((FEW_ROWS * 256 + G - 1) / G); L.shape.row_step[1] = (int)((MANY_ROWS * 256 + G - 1) / G);
    L.shape.each = 1;
    // tiles: all rows in full ones, and one that is not full for each set that has rows; a piece more for each worker
    const long long few_tiles = sets * ((FEW_MOST + FEW_ROWS - 1) / FEW_ROWS), full = (all + FEW_ROWS - 1) / FEW_ROWS + sets;
    const long long few_slots = (wide && few_tiles < full ? few_tiles : full) * a.n_kv + L.shape.blocks * most_few_warps(a.hd);
    const long long many_sets = all / (FEW_MOST + 1) < sets ? all / (FEW_MOST + 1) : sets;
    const long long many_slots = wide && all > FEW_MOST ? ((all + MANY_ROWS - 1) / MANY_ROWS + many_sets) * a.n_kv + L.shape.blocks : 0;
    L.few_acc = 0;
    L.few_top = L.few_acc + (size_t)few_slots * FEW_ROWS * a.hd * 4;
    L.many_acc = L.few_top + (size_t)few_slots * FEW_ROWS * 8;
    L.many_top = L.many_acc + (size_t)many_slots * MANY_ROWS * a.hd * 4;
    L.bytes = L.many_top + (size_t)many_slots * MANY_ROWS * 8;
    return L;
}

template <typename T, int HD>
int launch(const b200_paged_attn_args &a, cudaStream_t st)
{
    Layout L = layout_of(a);
    if (a.work_bytes < L.bytes) return B200_E_BADARG;
    char *work = static_cast<char *>(a.d_work);
    const Pieces few = {reinterpret_cast<float *>(work + L.few_acc), reinterpret_cast<float2 *>(work + L.few_top)};
    const Pieces many = {reinterpret_cast<float *>(work + L.many_acc), reinterpret_cast<float2 *>(work + L.many_top)};
    const size_t plan = plan_bytes(a.n_req, a.n_groups), rings = (size_t)L.shape.few_warps * few_ring(HD);
    Room room = {0, (int)rings};
    CUtensorMap map_k = {}, map_v = {};
    if constexpr (HD <= 128) {
        constexpr size_t SLOT = KEY64 * (HD / 64), QUERIES = 2 * QUERY64 * (HD / 64);
        const size_t left = ROOM - plan - QUERIES;
        room.slots = (int)(left / SLOT) < MOST_SLOTS ? (int)(left / SLOT) : MOST_SLOTS;
        if (QUERIES + room.slots * SLOT > rings) room.plan_off = (int)(QUERIES + room.slots * SLOT);
        const int box = a.page < MANY_KEYS ? a.page : MANY_KEYS;
        if (!pool_map(&map_k, a.d_k_pool, a, box) || !pool_map(&map_v, a.d_v_pool, a, box)) return B200_E_STATE;
    }
    const size_t smem = room.plan_off + plan + 1024;
    static std::atomic<unsigned long long> pages_done, join_done, join_rows_done;
    cudaError_t e = allow_all(attn_pages_kernel<T, HD>, pages_done);
    if (e == cudaSuccess) e = allow_all(attn_join_kernel<T, HD>, join_done);
    if (e == cudaSuccess) e = allow_all(attn_join_rows_kernel<T, HD>, join_rows_done);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    const int sets = a.n_req + a.n_groups;
    L.shape.each = (sets + block_threads(HD) - 1) / block_threads(HD);
    cfg.gridDim = dim3((unsigned)L.shape.blocks);
    cfg.blockDim = dim3(block_threads(HD));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = a.use_pdl != 0;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, attn_pages_kernel<T, HD>, map_k, map_v, a, L.shape, few, many, room);
    if (e != cudaSuccess) return (int)e;
    ++g_b200_launches;
    L.shape.each = (sets + JOIN_WARPS * 32 - 1) / (JOIN_WARPS * 32);
    const long long blocks = ((long long)a.max_rows * a.n_q + JOIN_WARPS - 1) / JOIN_WARPS, most = (long long)JOIN_BLOCKS * L.shape.blocks;
    e = launch_chained(blocks > most ? attn_join_rows_kernel<T, HD> : attn_join_kernel<T, HD>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(JOIN_WARPS * 32), plan, st, a,
                       L.shape, few, many);
    if (e != cudaSuccess) return (int)e;
    ++g_b200_launches;
    return (int)cudaGetLastError();
}

}  // namespace

extern "C" size_t b200_paged_attn_work_bytes(const b200_paged_attn_args *a)
{
    return a && check_sizes(*a) == 0 ? layout_of(*a).bytes : 0;
}

extern "C" int b200_paged_attn(const b200_paged_attn_args *ap, void *stream)
{
    if (!ap) return B200_E_BADARG;
    const b200_paged_attn_args &a = *ap;
    if (const int rc = check_sizes(a)) return rc;
    if (!std::isfinite(a.scale * 1.4426950408889634f)) return B200_E_BADARG;        // (weights are powers of two)
    if (a.max_rows == 0 || a.n_req == 0) return 0;
    if (!a.d_q || !a.d_k_pool || !a.d_v_pool || !a.d_out || !a.d_row_start || !a.d_len || !a.d_table || !a.d_work) return B200_E_BADARG;
    if (a.n_groups && (!a.d_group_start || !a.d_prefix_len || (a.prefix_ld && !a.d_prefix_table))) return B200_E_BADARG;
    if (a.q_ld < (long long)a.n_q * a.hd || a.q_ld % 8 || a.out_ld < (long long)a.n_q * a.hd || a.out_ld % 8) return B200_E_BADARG;
    if (((uintptr_t)a.d_q | (uintptr_t)a.d_k_pool | (uintptr_t)a.d_v_pool | (uintptr_t)a.d_out | (uintptr_t)a.d_work) % 16) return B200_E_BADARG;
    cudaStream_t st = (cudaStream_t)stream;
    if (a.wtype == B200_WT_F16) return a.hd == 64 ? launch<__half, 64>(a, st) : a.hd == 128 ? launch<__half, 128>(a, st) : launch<__half, 256>(a, st);
    return a.hd == 64 ? launch<__nv_bfloat16, 64>(a, st) : a.hd == 128 ? launch<__nv_bfloat16, 128>(a, st) : launch<__nv_bfloat16, 256>(a, st);
}
