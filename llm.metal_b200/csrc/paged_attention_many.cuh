// Attention over pages for sets of many query rows: the prefix that a group shares, and the own tokens of requests that bring portions of prompts
// (paged_plan.cuh). Both products run on tcgen05.
//
// A block works on two streams that take turns on the tensor core, so that one's softmax runs under the other's products: the two halves of a tile of 256 query
// rows on the same keys, or, where a tile has 128 rows at most, the same rows on every other unit of 64 keys, each stream with a maximum, sum and result of its own.
// Per unit and stream: S = Q K^T (128 x 64, one of two places in tensor memory, so that the next scores are there when these are done with), the weights
// P = 2^(c S - m) back into S's place as 16-bit pairs, O += P V with P as the operand from tensor memory and V as it lies, [key][hd] (the product's
// second operand along its rows). m is the largest score so far, less 7 in binary16 (weight_lift), and that only as far as it must be: O is rescaled when the largest weight would
// be more than 2^8 times that, 2^15. Weights are rounded by half a step down to 2^-21 of the largest one in binary16 and by 2^-32 of it at most below that.
//   warp 0      pages into a ring of shared memory: TMA, a box of 64 numbers by up to 64 tokens a lane, keys and values by turns
//   warps 1, 2  the products of stream 0, of stream 1: one lane issues them
//   warps 4-7   stream 0: queries into shared memory, softmax, results; warps 8-11 stream 1. A thread to a row.
// What bounds it: for tiles of 128 rows memory, once the copies are under way; for full ones the chain weights -> product -> next scores. A unit of 64 keys by 256 rows
// takes 1.9 thousand clocks (hd 128), of which the tensor core is busy most (scores of 64 columns seem to cost it as much as 128 would) and the rows' warps 1.6, 1.0 of them exponentials; four
// portions of 125 .. 811 tokens behind 4096, 32 / 8 heads, 179 us: 840 TFLOP/s, 0.52 of the measured product. On the way there, the same launch: units of
// 128 keys, whose next scores wait for the products of these, 224 us; units of 64 issued by one lane that divides and makes addresses for each step 314,
// by a whole warp in uniform registers 210, by one for each stream 185. A quarter of the weights by a polynomial, and scores read from tensor memory a unit early, gave nothing.
// Every wait is bounded; on a timeout the block reports it, lets copies in flight land, frees its tensor memory and returns.
#pragma once
#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int MANY_ROWS = Cut<1>::ROWS, MANY_KEYS = Cut<1>::KEYS, MANY_THREADS = 384, HALF_ROWS = MANY_ROWS / 2, MOST_SLOTS = 12;
constexpr uint32_t QUERY64 = HALF_ROWS * 128, KEY64 = MANY_KEYS * 128;       // 64 numbers of a tile's rows, of a unit's keys
constexpr int S_COL = 0, O_COL = 256;                        // tensor memory: S of stream s at 128 s and 128 s + 64, O at 256 + 128 s

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
// Second operand that lies along its rows ([k][n], 128-byte swizzle): 8 rows of k 1024 bytes apart, 64 columns of n `block` bytes apart.
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t saddr, uint32_t block)
{
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(block >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// first operand from tensor memory
__device__ __forceinline__ void umma_from_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) { tmem_st16(taddr, r); tmem_st16(taddr + 16, r + 16); }
// 64 columns of the lanes' rows
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
                 "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
                 "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
                   "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
                   "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
                   "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                   "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr)
{
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    return r;
}
// One lane of a converged warp. (By the whole warp up to here, so that addresses and descriptors stay in uniform registers, which is where the products take them from.)
__device__ __forceinline__ bool one_lane()
{
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on != 0;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// chunk ch of a row of a tile whose 64 numbers a row lie `block` bytes apart
__device__ __forceinline__ uint32_t swizzled(int row, int ch, uint32_t block) { return (ch >> 3) * block + row * 128 + (((ch & 7) ^ (row & 7)) * 16); }
__device__ __forceinline__ void zero16(uint32_t at) { asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory"); }

// The rows' results times f: by the whole warp. Eight columns at a time: a row of scores is held meanwhile.
template <int HD> __device__ __forceinline__ void scale_rows(uint32_t o_at, float f)
{
#pragma unroll 1
    for (int k = 0; k < HD; k += 8) {
        uint32_t x[8];
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]) : "r"(o_at + k) : "memory");
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = __float_as_uint(__uint_as_float(x[q]) * f);
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"r"(o_at + k), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]) : "memory");
    }
}

// The rows' results plus weight times value of one key, for rows that see it: by the whole warp.
template <typename T, int HD> __device__ __noinline__ void add_key(uint32_t s_at, uint32_t o_at, uint32_t v_at, int key, bool sees)
{
    const uint32_t two = tmem_ld1(s_at + key / 2);
    const float e = to_float<T>((uint16_t)(key & 1 ? two >> 16 : two));
#pragma unroll 1
    for (int k = 0; k < HD; k += 32) {
        uint32_t x[32];
        tmem_ld32(o_at + k, x);
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
            const uint4 v = lds_128(v_at + swizzled(key, k / 8 + ch, KEY64));
            const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float a = __uint_as_float(x[8 * ch + 2 * q]), b = __uint_as_float(x[8 * ch + 2 * q + 1]);
                x[8 * ch + 2 * q] = __float_as_uint(sees ? fmaf(e, to_float<T>((uint16_t)word[q]), a) : a);
                x[8 * ch + 2 * q + 1] = __float_as_uint(sees ? fmaf(e, to_float<T>((uint16_t)(word[q] >> 16)), b) : b);
            }
        }
        tmem_st32(o_at + k, x);
    }
    tmem_wait_st();
}

// Which units of a piece a stream has, and the order in which the piece's keys and values pass through the ring: `lead` units of keys, then values and keys by turns.
struct Streams {
    bool halves;                         // one tile of rows, every other unit to a stream
    int units[2], n, lead, ahead;        // lead: `ahead`, or all that there are
    __device__ __forceinline__ uint32_t values(int j) const { return lead + j + min(j, n - lead); }
};
// (Four units ahead where every other one is a stream's, if the ring has 7 places: what lay before the values of a unit whose scores are there was asked for before
// its keys then, which is_there relies on.)
__device__ __forceinline__ Streams streams_of(const Plan &p, const Piece &q, int slots)
{
    Streams w;
    w.n = q.n;
    w.halves = min(MANY_ROWS, q.s.nr - q.t * MANY_ROWS) <= HALF_ROWS;
    w.ahead = w.halves && slots >= 7 ? 4 : 2;
    w.lead = min(q.n, w.ahead);
    if (w.halves) { w.units[0] = (q.n + 1) / 2; w.units[1] = q.n / 2; return w; }
    const int seen = q.s.own ? q.s.keys - q.s.rows + over(q.t * MANY_ROWS + HALF_ROWS - 1, p.shape.by_g) + 1 : q.s.keys;
    w.units[0] = max(0, min(q.n, units_before_own<1>(q.s) + (seen + MANY_KEYS - 1) / MANY_KEYS - q.k0));
    w.units[1] = q.n;
    return w;
}

// A place in the ring, and the phase of its barriers.
struct Place {
    int slot;
    uint32_t phase;
    __device__ __forceinline__ void next(int slots) { if (++slot == slots) { slot = 0; phase ^= 1; } }
};

// A block's stretch of the second line. `base`: two tiles of queries and `slots` places of keys or values, 1024-byte aligned.
template <typename T, int HD>
__device__ __forceinline__ void many_block(const CUtensorMap &map_k, const CUtensorMap &map_v, const b200_paged_attn_args &a, const Plan &p, const Pieces &out, char *base, int slots)
{
    constexpr int NB = HD / 64;
    constexpr uint32_t SLOT = KEY64 * NB, Q_TILE = QUERY64 * NB;
    constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t IDESC_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t)(MANY_KEYS >> 3) << 17) | (8u << 24);
    constexpr uint32_t IDESC_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
    __shared__ uint64_t full_bar[MOST_SLOTS], empty_bar[MOST_SLOTS], q_bar[2], s_bar[2][2], p_bar[2][2], o_bar[2][2], alone_bar[2], both_bar, both_done;
    __shared__ uint32_t tmem_sh;
    __shared__ int abort_sh;
    __shared__ uint32_t special_sh[6][2];                    // marks of values that are not finite: two of each stream's own, two of both's
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort_flag = &abort_sh;
    const uint32_t q_tiles = smem_u32(base), ring = q_tiles + 2 * Q_TILE;

    if (threadIdx.x == 0) {
        abort_sh = 0;
        for (int s = 0; s < slots; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 2); }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_bar[s], 128); mbar_init(&s_bar[s][0], 1); mbar_init(&s_bar[s][1], 1); mbar_init(&alone_bar[s], 128);
            for (int k = 0; k < 2; ++k) { mbar_init(&p_bar[s][k], 128); mbar_init(&o_bar[s][k], 1); }
        }
        mbar_init(&both_bar, 256); mbar_init(&both_done, 2);
        for (int i = 0; i < 12; ++i) special_sh[i >> 1][i & 1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = tmem_sh;
    // Whether what passes as the phase-th through a place of the ring has arrived. Where each stream reads every other unit, the other stream's keys or values may have been there before
    // and may still be on their way, as copies do not land in order; the parity of the barrier of arrivals is then that of the phase before it, which is over. That
    // the place was given back first decides: it was asked for before something that this stream has seen arrive, and is not given back again without this stream.
    auto is_there = [&](int slot, uint32_t phase, bool halves) {
        return __all_sync(0xffffffffu, (!halves || wait_or_abort(&empty_bar[slot], phase ^ 1, abort_flag)) && wait_or_abort(&full_bar[slot], phase, abort_flag)) != 0;
    };
    auto give_up = [&]() { if (!*abort_flag) { *abort_flag = 1; if (a.d_status) atomicOr(a.d_status, B200_PAGED_TIMED_OUT); } };

    // Registers: 168 a thread at the launch, 384 threads; 72 for four warps and 216 for the eight with a row of scores a thread are as many.
    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- a stream's rows ----
        const int s = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;       // stream, row of its tile = lane of tensor memory
        const uint32_t tm = tmem + ((uint32_t)(warp & 3) << 21), o_at = tm + O_COL + s * 128;
        // the sign goes into the queries; a scale of zero weighs all seen keys alike, and hidden ones, at minus infinity, not at all
        const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.17549435e-38f);
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        constexpr float LIFT = weight_lift<T>(7);
        uint32_t turn = 0, item = 0, s_phase = 0, even = 0, odd = 0, alone_phase = 0, both_phase = 0;      // even, odd: products with weights of the first and of the second place, before this piece
        bool ok = true;
        Walk<1> walk(p, blockIdx.x);
        Piece piece;
        while (ok && walk.next(p, piece)) {
            const Streams w = streams_of(p, piece, slots);
            const Set &st = piece.s;
            const int i0 = piece.t * MANY_ROWS, i = i0 + (w.halves ? 0 : s * HALF_ROWS) + r, mine = w.units[s];
            const bool valid = i < st.nr, warp_valid = __any_sync(0xffffffffu, valid);
            const Div by_g = p.shape.by_g;
            const int last = min(i, st.nr - 1), local = over(last, by_g), row = row_at(p, piece.e, local);
            const int column = (piece.h * by_g.d + last - local * by_g.d) * HD;
            // own keys that this row sees, that the first row of this warp sees, that the first row of the whole tile sees (all rows see)
            const Keys keys = keys_of<1>(a, p, piece);
            const int own_limit = st.keys - st.rows + local + 1, own_warp = __shfl_sync(0xffffffffu, own_limit, 0), own_all = st.keys - st.rows + over(i0, by_g) + 1;
            // a warp's rows, HD / 8 lanes to each so that whole lines are read; all loads before the first store
            constexpr int CH = HD / 8, RL = 32 / CH;         // 16-byte chunks of a row, rows of a load
            const long long q_off = (long long)row * a.q_ld + column;
            if (warp_valid && !(w.halves && s == 1)) {
                uint4 v[32 / RL];
#pragma unroll
                for (int k = 0; k < 32 / RL; ++k) {
                    const long long off = __shfl_sync(0xffffffffu, q_off, k * RL + lane / CH);
                    v[k] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.d_q) + off + (lane % CH) * 8);
                }
#pragma unroll
                for (int k = 0; k < 32 / RL; ++k)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_tiles + s * Q_TILE + swizzled((warp & 3) * 32 + k * RL + lane / CH, lane % CH, QUERY64)),
                                 "r"(v[k].x ^ flip), "r"(v[k].y ^ flip), "r"(v[k].z ^ flip), "r"(v[k].w ^ flip) : "memory");
            }
            async_proxy_fence();
            {
                uint32_t zero[32] = {};
#pragma unroll
                for (int k = 0; k < HD; k += 32) tmem_st32(o_at + k, zero);
                tmem_wait_st();
            }
            before_sync();
            mbar_arrive(&q_bar[s]);
            float top = -INFINITY, l = 0.0f;
            auto settled = [&](int j) {                      // the sums of this piece's first j units are in O
                if (j == 0) return true;
                const int i = j - 1;
                const bool there = __all_sync(0xffffffffu, wait_or_abort(&o_bar[s][i & 1], ((i & 1 ? odd : even) + i / 2) & 1, abort_flag));
                after_sync();
                return there;
            };
            for (int j = 0; j < mine; ++j) {
                const int unit = w.halves ? 2 * j + s : j, place = j & 1;
                const uint32_t s_at = tm + S_COL + s * 128 + place * 64;
                const Part u = part_at<1>(keys, piece, unit);
                const int key0 = u.key0, limit = u.own ? own_limit : u.seen, limit_warp = u.own ? own_warp : u.seen, limit_all = u.own ? own_all : u.seen;
                if (!__all_sync(0xffffffffu, wait_or_abort(&s_bar[s][place], (s_phase >> place) & 1, abort_flag))) { ok = false; break; }
                s_phase ^= 1u << place;
                after_sync();
                const bool some_hidden = key0 + MANY_KEYS > limit_warp;
                const int cols = limit - key0;               // columns below this are seen
                if (warp_valid) {
                    uint32_t x[64];
                    tmem_ld64(s_at, x);
                    if (some_hidden) {
#pragma unroll
                        for (int q = 0; q < 64; ++q) x[q] = q < cols ? x[q] : 0xff800000u;
                    }
                    float big4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int q = 0; q < 64; ++q) big4[q & 3] = fmaxf(big4[q & 3], __uint_as_float(x[q]));
                    const float big = valid ? fmaxf(fmaxf(big4[0], big4[1]), fmaxf(big4[2], big4[3])) * c - LIFT : -INFINITY;   // (what lies in other rows must not decide)
                    if (__any_sync(0xffffffffu, big > top + 8.0f)) {     // (true too for the first)
                        const float higher = fmaxf(top, big), f = top == -INFINITY ? 0.0f : ex2(top - higher);
                        if (__any_sync(0xffffffffu, top != -INFINITY)) {
                            if (!settled(j)) { ok = false; break; }
                            scale_rows<HD>(o_at, f);
                        }
                        l *= f;
                        top = higher;
                    }
                    const float b = top == -INFINITY ? 0.0f : -top;
                    float2 sum[2] = {};
#pragma unroll
                    for (int k = 0; k < MANY_KEYS; k += 32) {
                        uint32_t y[16];
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            float2 e = __ffma2_rn(make_float2(__uint_as_float(x[k + 2 * q]), __uint_as_float(x[k + 2 * q + 1])), make_float2(c, c), make_float2(b, b));
                            e.x = ex2(e.x); e.y = ex2(e.y);
                            sum[q & 1] = __fadd2_rn(sum[q & 1], e);
                            y[q] = pack2<T>(e.x, e.y);
                        }
                        tmem_st16(s_at + k / 2, y);
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    tmem_wait_st();
                }
                if (key0 + MANY_KEYS > limit_all) {
                    // Not all rows see all of these keys: zero weights must not meet infinities or NaN. Values behind the last seen key are made zero; of those
                    // that some rows see, the ones that are not finite are added row by row and then made zero too.
                    const uint32_t v_item = item + w.values(unit), v_at = ring + (v_item % slots) * SLOT;
                    if (!is_there(v_item % slots, (v_item / slots) & 1, w.halves)) { ok = false; break; }
                    const bool both = !w.halves && unit < w.units[0];
                    auto meet = [&]() {                      // of all threads that read this unit
                        if (both) { mbar_arrive(&both_bar); ok = __all_sync(0xffffffffu, wait_or_abort(&both_bar, both_phase, abort_flag)); both_phase ^= 1; }
                        else { mbar_arrive(&alone_bar[s]); ok = __all_sync(0xffffffffu, wait_or_abort(&alone_bar[s], alone_phase, abort_flag)); alone_phase ^= 1; }
                    };
                    const int there = u.seen - key0;         // a thread to a key
                    const bool looks = !both || s == 0;
                    // By turns (a unit meets once or three times): a warp may write the next unit's marks while another has yet to read these, and who writes those of the
                    // unit after that has met everyone in between.
                    uint32_t *found = special_sh[both ? 4 + both_phase : 2 * s + alone_phase];
                    if (looks) {
                        bool special = false;
                        if (r < there && r < MANY_KEYS && u.own) {
#pragma unroll
                            for (int ch = 0; ch < HD / 8; ++ch) special |= any_special<T>(lds_128(v_at + swizzled(r, ch, KEY64)));
                        }
                        const uint32_t word = __ballot_sync(0xffffffffu, special);
                        if (lane == 0 && r < MANY_KEYS) found[warp & 3] = word;
                        if (r >= there && r < MANY_KEYS) {
#pragma unroll
                            for (int ch = 0; ch < HD / 8; ++ch) zero16(v_at + swizzled(r, ch, KEY64));
                        }
                        async_proxy_fence();
                    }
                    meet();
                    if (!ok) break;
                    volatile uint32_t *marks = found;
                    if (marks[0] | marks[1]) {                   // the same for all who meet
                        if (!settled(j)) { ok = false; break; }
#pragma unroll 1
                        for (int key = 0; key < MANY_KEYS; ++key)
                            if (marks[key >> 5] >> (key & 31) & 1) add_key<T, HD>(s_at, o_at, v_at, key, key < cols);
                        const bool clear = looks && r < MANY_KEYS && (marks[r >> 5] >> (r & 31) & 1);
                        meet();                              // nobody needs them any more
                        if (!ok) break;
                        if (clear) {
#pragma unroll
                            for (int ch = 0; ch < HD / 8; ++ch) zero16(v_at + swizzled(r, ch, KEY64));
                        }
                        async_proxy_fence();
                        meet();
                        if (!ok) break;
                    }
                }
                before_sync();
                mbar_arrive(&p_bar[s][place]);
            }
            if (!ok) break;

            // ---- the piece's results ----
            ok = settled(mine);
            if (!ok) break;
            const bool whole = piece.n == piece.ut && !w.halves && alone(p, piece);          // nothing to join with
            const long long place = (long long)(p.tile[1][piece.e] + piece.h * piece.tiles + piece.t + (int)blockIdx.x) * MANY_ROWS + s * HALF_ROWS + r;
            // All products of the piece are done: waited for once in every piece, so that no stream, not even one without units, runs two ahead of the products. Where
            // the other stream reads this one's queries, before the results pass through their room.
            auto finished = [&]() { return __all_sync(0xffffffffu, wait_or_abort(&both_done, turn & 1, abort_flag)); };
            const bool early = w.halves && s == 0;
            if (early && !finished()) { ok = false; break; }
            if (warp_valid) {
                // Through the room of the warp's own queries, 32 columns at a time: a thread holds a row, a store covers 128 bytes of four.
                const float inv = whole ? 1.0f / l : 1.0f;
                const long long out_off = (long long)row * a.out_ld + column;
                const int rows = min(32, st.nr - (i - lane)), ch = lane & 7;
#pragma unroll 1
                for (int k = 0; k < HD; k += 32) {
                    const uint32_t stage = q_tiles + s * Q_TILE + (k / 32) % NB * QUERY64 + (warp & 3) * 4096;
                    uint32_t x[32];
                    tmem_ld32(o_at + k, x);
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((q ^ (lane & 7)) * 16)), "r"(x[4 * q]), "r"(x[4 * q + 1]),
                                     "r"(x[4 * q + 2]), "r"(x[4 * q + 3]) : "memory");
                    __syncwarp();
                    float *acc = out.acc + (place - lane) * HD + k + ch * 4;
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int k_row = 4 * q + (lane >> 3);
                        const long long off = __shfl_sync(0xffffffffu, out_off, k_row);
                        const float f = __shfl_sync(0xffffffffu, inv, k_row);
                        const uint4 v = lds_128(stage + k_row * 128 + ((ch ^ (k_row & 7)) * 16));
                        if (k_row < rows) {
                            if (whole) {
                                uint2 y;
                                y.x = pack2<T>(__uint_as_float(v.x) * f, __uint_as_float(v.y) * f);
                                y.y = pack2<T>(__uint_as_float(v.z) * f, __uint_as_float(v.w) * f);
                                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.d_out) + off + k + ch * 4) = y;
                            } else *reinterpret_cast<uint4 *>(acc + (long long)k_row * HD) = v;
                        }
                    }
                    __syncwarp();
                }
                if (valid && !whole) out.top[place] = make_float2(top, l);
            }
            before_sync();
            if (!early && !finished()) { ok = false; break; }
            ++turn;
            even += (mine + 1) / 2; odd += mine / 2;
            item += 2 * piece.n;
        }
        if (!ok && lane == 0) give_up();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            // ---- pages into the ring ----
            // A copy takes up to 64 tokens of a page by 64 numbers; a lane to each. A unit's page numbers are asked for one unit ahead, once for its keys and once for its
            // values: with that round trip in each step the ring would fill at half of its rate.
            const int page_shift = 31 - __clz(a.page), box_shift = min(page_shift, 6), box = 1 << box_shift;
            const int mine = lane / NB, part = lane % NB;
            asm volatile("fence.proxy.async;" ::: "memory");     // rows that an earlier kernel stored, read by the copy engine
            Place at = {0, 0};
            bool outside = false, ok = true;
            Walk<1> walk(p, blockIdx.x);
            Piece piece;
            while (ok && walk.next(p, piece)) {
                const Streams w = streams_of(p, piece, slots);
                const int n = piece.n, lead = w.lead;
                const Keys keys = keys_of<1>(a, p, piece);
                struct Unit { int there, y, id; };               // copies, the first token in the page, this lane's page
                auto unit_at = [&](int unit) {
                    const Part u = part_at<1>(keys, piece, unit);
                    Unit x;
                    x.there = min(MANY_KEYS >> box_shift, (u.seen - u.key0 + box - 1) >> box_shift);
                    const int key = u.key0 + (mine << box_shift);
                    x.y = key & (a.page - 1);
                    x.id = mine < x.there ? __ldg(u.table + (key >> page_shift)) : 0;
                    return x;
                };
                Unit next[2] = {unit_at(0), unit_at(0)};
                auto load = [&](int unit, int values) {          // by the whole warp
                    const Unit u = values ? next[1] : next[0];
                    if (unit + 1 < n) { if (values) next[1] = unit_at(unit + 1); else next[0] = unit_at(unit + 1); }
                    const bool there = u.id >= 0 && u.id < a.n_pages;
                    outside |= !there;
                    if (!__all_sync(0xffffffffu, wait_or_abort(&empty_bar[at.slot], at.phase ^ 1, abort_flag))) { ok = false; return; }
                    if (lane == 0) mbar_expect_tx(&full_bar[at.slot], (uint32_t)u.there << box_shift << 7 << (NB - 1));
                    __syncwarp();
                    if (mine < u.there)                          // a page of -1 is outside the map and reads as zeros
                        tma_load_3d(ring + at.slot * SLOT + part * KEY64 + (mine << box_shift << 7), values ? &map_v : &map_k, part * 64, u.y, there ? u.id * a.n_kv + piece.h : -1,
                                    &full_bar[at.slot]);
                    at.next(slots);
                };
#pragma unroll 1
                for (int j = -lead; j < n && ok; ++j) {          // keys `lead` units ahead of values
                    if (j >= 0) load(j, 1);
                    if (ok && j + lead < n) load(j + lead, 0);
                }
            }
            if (!ok) give_up();
            if (outside && a.d_status) atomicOr(a.d_status, B200_PAGED_BAD_PAGE);
        } else if (warp < 3) {
            // ---- the products of a stream ----
            // A division or an address made anew for each step would keep the tensor core waiting. Places in the ring are counted, descriptors are the
            // first place's plus an offset, the whole warp follows and one lane issues.
            const int s = warp - 1;
            uint32_t turn = 0, p_phase = 0;
            bool ok = true;
            Walk<1> walk(p, blockIdx.x);
            Piece piece;
            Place at = {0, 0};
            const uint64_t k_desc = smem_desc_sw128(ring), v_desc = smem_desc_rows(ring, KEY64);
            const uint32_t s_at = tmem + S_COL + s * 128, o_at = tmem + O_COL + s * 128;
            auto arrived = [&](uint64_t *bar, uint32_t phase) { return (bool)__all_sync(0xffffffffu, wait_or_abort(bar, phase, abort_flag)); };
            while (ok && walk.next(p, piece)) {
                const Streams w = streams_of(p, piece, slots);
                const int n = uniform(piece.n), mine = uniform(w.units[s]), lead = uniform(w.lead), ahead = uniform(w.ahead), halves = uniform(w.halves);
                const uint64_t q_desc = smem_desc_sw128(q_tiles + (halves ? 0 : s * Q_TILE));
                ok = arrived(&q_bar[0], turn & 1) && arrived(&q_bar[1], turn & 1);
                ++turn;
                if (!ok) break;
                after_sync();
                // A place is free again when both streams have said so, a stream that has no use for it too; the only reader of one says it twice.
                auto scores = [&](int place, const Place &k) {
                    if (!ok || !(ok = is_there(k.slot, k.phase, halves))) return;
                    after_sync();
                    const uint64_t kd = k_desc + k.slot * (SLOT >> 4);
                    if (one_lane()) {
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int x = 0; x < 4; ++x) umma_f16(s_at + place * 64, q_desc + b * (QUERY64 >> 4) + 2 * x, kd + b * (KEY64 >> 4) + 2 * x, IDESC_S, (b | x) != 0);
                        umma_commit(&s_bar[s][place]);
                        umma_commit(&empty_bar[k.slot]);
                        if (halves) umma_commit(&empty_bar[k.slot]);
                    }
                    __syncwarp();
                };
                auto sums = [&](int place, const Place &v) {
                    if (!ok || !(ok = is_there(v.slot, v.phase, halves) && arrived(&p_bar[s][place], (p_phase >> place) & 1))) return;
                    p_phase ^= 1u << place;
                    after_sync();
                    const uint64_t vd = v_desc + v.slot * (SLOT >> 4);
                    if (one_lane()) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) umma_from_tmem(o_at, s_at + place * 64 + 8 * x, vd + 128 * x, IDESC_O);
                        umma_commit(&o_bar[s][place]);
                        umma_commit(&empty_bar[v.slot]);
                        if (halves) umma_commit(&empty_bar[v.slot]);
                    }
                    __syncwarp();
                };
                auto pass = [&](const Place &x) {            // (arrived first: the word is for this occupant)
                    if (!ok || !(ok = arrived(&full_bar[x.slot], x.phase))) return;
                    if (lane == 0) mbar_arrive(&empty_bar[x.slot]);
                    __syncwarp();
                };
                if (halves) {
#pragma unroll 1
                    for (int u = 0; u < lead; ++u, at.next(slots))
                        if ((u & 1) == s) scores(u >> 1, at);
#pragma unroll 1
                    for (int u = 0; u < n && ok; ++u) {
                        if ((u & 1) == s) sums((u >> 1) & 1, at);
                        at.next(slots);
                        if (u + ahead < n) {
                            if ((u & 1) == s) scores(((u + ahead) >> 1) & 1, at);
                            at.next(slots);
                        }
                    }
                } else {
#pragma unroll 1
                    for (int j = 0; j < lead; ++j, at.next(slots)) {
                        if (j < mine) scores(j, at); else pass(at);
                    }
#pragma unroll 1
                    for (int j = 0; j < n && ok; ++j) {
                        if (j < mine) sums(j & 1, at); else pass(at);
                        at.next(slots);
                        if (j + 2 < n) {
                            if (j + 2 < mine) scores(j & 1, at); else pass(at);
                            at.next(slots);
                        }
                    }
                }
                if (!ok) break;
                if (one_lane()) umma_commit(&both_done);
                __syncwarp();
            }
            if (!ok && lane == 0) give_up();
        }
    }

    before_sync();
    __syncthreads();
    if (*abort_flag)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);     // copies in flight land before the memory is released
    if (warp == 1) {
        after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// pool [n_pages * n_kv][page][hd]; a box is 64 numbers of `box` tokens
bool pool_map(CUtensorMap *map, const void *pool, const b200_paged_attn_args &a, int box)
{
    encode_fn_t enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)a.hd, (cuuint64_t)a.page, (cuuint64_t)a.n_pages * a.n_kv};
    const cuuint64_t strides[2] = {(cuuint64_t)a.hd * 2, (cuuint64_t)a.hd * 2 * a.page};
    const cuuint32_t extent[3] = {64, (cuuint32_t)box, 1}, step[3] = {1, 1, 1};
    return enc(map, a.wtype == B200_WT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(pool), dims, strides, extent, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
