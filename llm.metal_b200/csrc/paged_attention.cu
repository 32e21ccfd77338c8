// Attention of a step's new rows over pages (sm_100a): each row over its request's own tokens, and over a prefix that its group shares
// (paged_plan.cuh: how the work is cut).
//
// attn_few_kernel: a warp to itself, 16 query rows against a stretch of keys on mma.sync, m16n8k16, 16 keys a unit. Keys and values come with cp.async
// into a ring of the warp's own, two units ahead; scores, weights and sums stay in registers, one pass with a running maximum. What bounds it
// is memory: 16 rows take 64 operations a byte of cache at most, and the few warps of an SM hold enough bytes in flight. Warps share nothing, so that there is
// no barrier in the loop. Scores, maxima, sums and results are fp32; weights are rounded to the cache's type for the second product, by at most
// half a step each, which is what the results' own rounding is.
// attn_join_kernel: a warp to each (row, query head) whose keys were cut, over the pieces in the order of the line.
#include "paged_attention.cuh"

namespace {

constexpr int FEW_ROWS = 16, FEW_KEYS = 16, FEW_WARPS = 4, FEW_STAGES = 3, FEW_LEAST = 4, FEW_GAP = 1;
constexpr int JOIN_WARPS = 8, JOIN_BLOCKS = 4;

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool on)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T, int HD>
__global__ void __launch_bounds__(FEW_WARPS * 32)
attn_few_kernel(const __grid_constant__ b200_paged_attn_args a, const Cut cut, const Pieces out, int big, int beside)
{
    constexpr int CH = HD / 8;                               // 16-byte chunks of a key
    constexpr int HALF_STAGE = FEW_KEYS * HD * 2, STAGE = 2 * HALF_STAGE;
    extern __shared__ __align__(128) char smem[];
    __shared__ long long red[32];
    __shared__ int red_t[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    // Beside attn_many_kernel, launched before: its blocks let this grid start when they have waited for what came before, so that everything that is read here
    // is there. Its results are waited for at the end, for the join's sake, whose own wait covers this grid alone.
    if (!beside) pdl_wait();
    Plan p;
    if (!load_plan(a, p, smem + FEW_WARPS * FEW_STAGES * STAGE, 1, big, red_t)) { pdl_wait(); return; }
    Line line;
    if (!lay_line(a, p, cut, 0, out.workers, line, red, red_t)) { pdl_wait(); return; }
    const int worker = blockIdx.x * FEW_WARPS + warp;
    const uint32_t ring = smem_u32(smem) + warp * FEW_STAGES * STAGE;
    const uint16_t *kp = static_cast<const uint16_t *>(a.d_k_pool), *vp = static_cast<const uint16_t *>(a.d_v_pool);
    const float c = a.scale * 1.4426950408889634f;
    const int g = lane >> 2, cq = lane & 3;
    const int page_shift = 31 - __clz(a.page);

    Walk walk(p, line, worker);                              // warps are independent from here on
    Piece piece;
    while (walk.next(p, line, cut, piece)) {
        // ---- query rows t * 16 .. of head h, units k0 .. k0 + n - 1 ----
        const Set &s = piece.s;
        const int e = piece.e, h = piece.h, t = piece.t, k0 = piece.k0, n = piece.n;
        const int i0 = t * FEW_ROWS, valid = min(FEW_ROWS, s.nr - i0);
        const int seen = seen_by(p, s, cut, t), seen_first = s.own ? s.keys - s.rows + i0 / p.G + 1 : s.keys;
        const int *table = part_at(a, p, cut, piece, 0).table;
        int limit[2], row_of[2];
        uint32_t q[CH / 2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = i0 + g + 8 * half;
            const bool on = g + 8 * half < valid;
            limit[half] = !on ? 0 : s.own ? s.keys - s.rows + i / p.G + 1 : s.keys;
            row_of[half] = row_at(p, e, on ? i / p.G : 0);
            const uint16_t *src = static_cast<const uint16_t *>(a.d_q) + (long long)row_of[half] * a.q_ld + (size_t)(h * p.G + (on ? i % p.G : 0)) * HD + 2 * cq;
#pragma unroll
            for (int ks = 0; ks < CH / 2; ++ks) {
                q[ks][half] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * ks) : 0u;
                q[ks][2 + half] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * ks + 8) : 0u;
            }
        }
        int ids = 0;
        bool outside = false;
        auto issue = [&](int i) {                            // unit k0 + i of the tile into its place of the ring
            if (i < n) {
                if ((i & 31) == 0) {                         // page numbers, 32 units at a time
                    const int key = (k0 + i + lane) * FEW_KEYS;
                    ids = i + lane < n ? __ldg(table + (key >> page_shift)) : 0;
                }
                const int id = __shfl_sync(0xffffffffu, ids, i & 31), key = (k0 + i) * FEW_KEYS;
                const bool there = id >= 0 && id < a.n_pages;
                outside |= !there;
                const size_t at = (((size_t)(there ? id : 0) * a.n_kv + h) * a.page + (key & (a.page - 1))) * HD;
                const uint32_t dst = ring + (i % FEW_STAGES) * STAGE;
#pragma unroll
                for (int j = 0; j < FEW_KEYS * CH / 32; ++j) {
                    const int row = (lane + 32 * j) / CH, ch = (lane + 32 * j) % CH;
                    const bool on = there && key + row < seen;           // what is not seen is not read: zeros
                    const uint32_t to = dst + row * HD * 2 + ((ch ^ (row & 7)) * 16);
                    cp16(to, kp + at + (size_t)row * HD + ch * 8, on);
                    cp16(to + HALF_STAGE, vp + at + (size_t)row * HD + ch * 8, on);
                }
            }
            cp_commit();
        };
        float o[CH][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < CH; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        __syncwarp();                                        // the ring's last reads, of the piece before
#pragma unroll
        for (int i = 0; i < FEW_STAGES - 1; ++i) issue(i);
        for (int i = 0; i < n; ++i) {
            cp_wait<FEW_STAGES - 2>();
            __syncwarp();
            issue(i + FEW_STAGES - 1);
            const uint32_t kt = ring + (i % FEW_STAGES) * STAGE, vt = kt + HALF_STAGE;
            const int key = (k0 + i) * FEW_KEYS, mi = lane >> 3, rr = lane & 7;
            float sc[2][4] = {};
#pragma unroll
            for (int ks = 0; ks < CH / 2; ++ks) {
                uint32_t b[4];
                const int row = (mi >> 1) * 8 + rr, ch = ks * 2 + (mi & 1);
                ldsm4(kt + row * HD * 2 + ((ch ^ (row & 7)) * 16), b);
                mma16<T>(sc[0], q[ks], b[0], b[1]);
                mma16<T>(sc[1], q[ks], b[2], b[3]);
            }
            float top[2] = {m[0], m[1]};
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = sc[nt][j] * c;
                    sc[nt][j] = key + nt * 8 + 2 * cq + (j & 1) < limit[j >> 1] ? x : -INFINITY;
                    top[j >> 1] = fmaxf(top[j >> 1], sc[nt][j]);
                }
            float base[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                base[r] = top[r] == -INFINITY ? 0.0f : top[r];
            }
            if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
                const float f0 = ex2(m[0] - base[0]), f1 = ex2(m[1] - base[1]);
                l[0] *= f0; l[1] *= f1;
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) { o[ch][0] *= f0; o[ch][1] *= f0; o[ch][2] *= f1; o[ch][3] *= f1; }
                m[0] = top[0]; m[1] = top[1];
            }
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sc[nt][j] = ex2(sc[nt][j] - base[j >> 1]);
                    l[j >> 1] += sc[nt][j];
                }
            if (key + FEW_KEYS > seen_first && seen_first < seen) {
                // Some rows see keys of this unit that others do not: zero weights must not meet infinities or NaN. Values of such keys are added
                // row by row where they are seen, and taken out of the product.
                uint32_t special = 0;
#pragma unroll 1
                for (int row = 0; row < FEW_KEYS; ++row) {
                    const bool mine = lane < CH && any_special<T>(lds_128(vt + row * HD * 2 + (lane % CH) * 16));
                    if (__any_sync(0xffffffffu, mine)) special |= 1u << row;
                }
                while (special) {
                    const int row = __ffs(special) - 1;
                    special &= special - 1;
                    float w[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float even = row < 8 ? sc[0][2 * r] : sc[1][2 * r], odd = row < 8 ? sc[0][2 * r + 1] : sc[1][2 * r + 1];
                        w[r] = __shfl_sync(0xffffffffu, row & 1 ? odd : even, (lane & ~3) | ((row & 7) >> 1));
                    }
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch) {
                        uint32_t two;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(two) : "r"(vt + row * HD * 2 + ((ch ^ (row & 7)) * 16) + 4 * cq));
                        const float v0 = to_float<T>((uint16_t)two), v1 = to_float<T>((uint16_t)(two >> 16));
                        if (key + row < limit[0]) { o[ch][0] = fmaf(w[0], v0, o[ch][0]); o[ch][1] = fmaf(w[0], v1, o[ch][1]); }
                        if (key + row < limit[1]) { o[ch][2] = fmaf(w[1], v0, o[ch][2]); o[ch][3] = fmaf(w[1], v1, o[ch][3]); }
                    }
                    __syncwarp();
                    if (lane < CH) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vt + row * HD * 2 + lane * 16), "r"(0u) : "memory");
                    __syncwarp();
                }
            }
            const uint32_t w[4] = {pack2<T>(sc[0][0], sc[0][1]), pack2<T>(sc[0][2], sc[0][3]), pack2<T>(sc[1][0], sc[1][1]), pack2<T>(sc[1][2], sc[1][3])};
#pragma unroll
            for (int cp = 0; cp < CH / 2; ++cp) {
                uint32_t b[4];
                const int row = (mi & 1) * 8 + rr, ch = cp * 2 + (mi >> 1);
                ldsm4_t(vt + row * HD * 2 + ((ch ^ (row & 7)) * 16), b);
                mma16<T>(o[2 * cp], w, b[0], b[1]);
                mma16<T>(o[2 * cp + 1], w, b[2], b[3]);
            }
        }
        cp_wait<0>();
        if (outside && lane == 0 && a.d_status) atomicOr(a.d_status, B200_PAGED_BAD_PAGE);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        const bool whole = n == piece.ut && alone(p, piece);          // nothing to join with
        const long long slot = line.tile[e] + (long long)h * piece.tiles + t + worker;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int k = g + 8 * r, i = i0 + k;
            if (k >= valid) continue;
            if (whole) {
                const float inv = 1.0f / l[r];
                uint16_t *to = static_cast<uint16_t *>(a.d_out) + (long long)row_of[r] * a.out_ld + (size_t)(h * p.G + i % p.G) * HD + 2 * cq;
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) *reinterpret_cast<uint32_t *>(to + 8 * ch) = pack2<T>(o[ch][2 * r] * inv, o[ch][2 * r + 1] * inv);
            } else {
                float *to = out.acc + (slot * FEW_ROWS + k) * HD + 2 * cq;
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) *reinterpret_cast<float2 *>(to + 8 * ch) = make_float2(o[ch][2 * r], o[ch][2 * r + 1]);
                if (cq == 0) out.top[slot * FEW_ROWS + k] = make_float2(m[r], l[r]);
            }
        }
    }
    pdl_wait();
}

template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
attn_join_kernel(const __grid_constant__ b200_paged_attn_args a, const Cut cut0, const Pieces in0, const Cut cut1, const Pieces in1, int big)
{
    constexpr int N = HD / 32;                               // numbers of a lane, next to one another
    extern __shared__ __align__(128) char smem[];
    __shared__ long long red[32];
    __shared__ int red_t[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    pdl_wait();
    Plan p;
    if (!load_plan(a, p, smem, 2, big, red_t)) return;
    Line few, many;
    if (!lay_line(a, p, cut0, 0, in0.workers, few, red, red_t) || !lay_line(a, p, cut1, 1, in1.workers, many, red, red_t)) return;
    const long long all = (long long)p.row[p.n_req] * a.n_q;
    for (long long at = (long long)blockIdx.x * JOIN_WARPS + warp; at < all; at += (long long)gridDim.x * JOIN_WARPS) {
        const int row = (int)(at / a.n_q), head = (int)(at % a.n_q);
        const int r = last_at(p.row, p.n_req, row), h = head / p.G;
        int group = group_of(p, r);
        if (is_big(p, r, group)) group = -1;                 // one set
        // the row's pieces of the prefix and of the own tokens: where the first one lies, how many, how far apart
        const float *acc[2] = {};
        const float2 *tops[2] = {};
        int count[2] = {0, 0}, step[2] = {0, 0};
        bool cut_up = false;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = k == 0 ? group : p.n_groups + r;
            if (e < 0) continue;
            const Set s = set_at(p, e);
            const bool is_few = in_cut(s, cut0);
            const Cut &cut = is_few ? cut0 : cut1;
            const Line &line = is_few ? few : many;
            const Pieces &in = is_few ? in0 : in1;
            const int i = (row - p.row[r] + (s.own ? 0 : p.small[r] - p.small[p.group[e]])) * p.G + head % p.G, t = i / cut.rt, tiles = tiles_of(s, cut);
            const int per_head = (line.unit[e + 1] - line.unit[e]) / p.n_kv;
            const int b = line.unit[e] + h * per_head + (int)line_before(p, s, cut, t) + cut.gap, w0 = b / line.per, w1 = (b + units_of(p, s, cut, t) - 1) / line.per;
            // a tile of 128 rows at most, in places for 256: two pieces in each, of every other unit
            const bool halves = !is_few && s.nr - t * MANY_ROWS <= MANY_ROWS / 2;
            const long long place = (long long)(line.tile[e] + h * tiles + t + w0) * cut.rt + i % cut.rt;
            acc[k] = in.acc + place * HD;
            tops[k] = in.top + place;
            step[k] = halves ? cut.rt / 2 : cut.rt;
            count[k] = (w1 - w0 + 1) * (halves ? 2 : 1);
            cut_up |= w1 > w0 || halves;
        }
        const int n = count[0] + count[1];
        if (group < 0 && !cut_up) continue;                      // stored where it was formed
        auto top_of = [&](int j) { return j < count[0] ? tops[0][(long long)j * step[0]] : tops[1][(long long)(j - count[0]) * step[1]]; };
        auto acc_of = [&](int j) { return j < count[0] ? acc[0] + (long long)j * step[0] * HD : acc[1] + (long long)(j - count[0]) * step[1] * HD; };
        float top = -INFINITY;
        for (int j = lane; j < n; j += 32) top = fmaxf(top, top_of(j).x);
        top = warp_max(top);
        const float base = top == -INFINITY ? 0.0f : top;
        float l = 0.0f, o[N];
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = 0.0f;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const float2 ml = top_of(j);
            const float f = ex2(ml.x - base);
            const float *v = acc_of(j) + lane * N;
            l = fmaf(ml.y, f, l);
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = fmaf(v[i], f, o[i]);
        }
        const float inv = 1.0f / l;
        uint32_t *to = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.d_out) + (long long)row * a.out_ld + (size_t)head * HD + lane * N);
#pragma unroll
        for (int i = 0; i < N; i += 2) to[i / 2] = pack2<T>(o[i] * inv, o[i + 1] * inv);
    }
}

int sm_count()
{
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    return n;
}

// Sizes alone: 0, or why they are refused.
int check_sizes(const b200_paged_attn_args &a)
{
    if ((a.wtype != B200_WT_F16 && a.wtype != B200_WT_BF16) || (a.hd != 64 && a.hd != 128 && a.hd != 256)) return B200_E_BADARG;
    if (a.n_q < 1 || a.n_kv < 1 || a.n_q % a.n_kv || a.n_q > 1024 || a.max_rows < 0 || a.max_rows > (1 << 20) || a.n_pages < 1) return B200_E_BADARG;
    if (a.page < 16 || a.page > 256 || (a.page & (a.page - 1))) return B200_E_BADARG;
    if (a.n_req < 0 || a.n_req > B200_PAGED_MAX_REQ || a.n_groups < 0 || a.n_groups > a.n_req) return B200_E_BADARG;
    if (a.table_ld < 0 || a.table_ld > (1 << 20) || a.prefix_ld < 0 || a.prefix_ld > (1 << 20)) return B200_E_BADARG;
    if ((long long)a.n_pages * a.page > INT_MAX || (long long)a.n_pages * a.n_kv > INT_MAX || (long long)a.table_ld * a.page > INT_MAX || (long long)a.prefix_ld * a.page > INT_MAX) return B200_E_TOOLARGE;
    return 0;
}

// Sets of more query rows than this go to attn_many_kernel, where hd is one of its own.
constexpr int FEW_MOST = 16;

struct Layout { int few_workers, many_workers; size_t few_acc, few_top, many_acc, many_top, bytes; };

Layout layout_of(const b200_paged_attn_args &a)
{
    const long long G = a.n_q / a.n_kv, all = a.max_rows * G * (a.n_groups ? 2 : 1);         // query rows of all sets
    const long long sets = (a.n_req < a.max_rows ? a.n_req : a.max_rows) + (a.n_groups < a.max_rows ? a.n_groups : a.max_rows);
    Layout L = {};
    L.few_workers = 2 * sm_count() * FEW_WARPS;
    L.many_workers = a.hd <= 128 && all > FEW_MOST ? sm_count() : 0;
    // tiles: all rows in full ones, and one that is not full for each set that has rows; a piece more for each worker
    const long long few_most = L.many_workers ? FEW_MOST : all;
    const long long few_tiles = sets * ((few_most + FEW_ROWS - 1) / FEW_ROWS), full = (all + FEW_ROWS - 1) / FEW_ROWS + sets;
    const long long few_slots = (few_tiles < full ? few_tiles : full) * a.n_kv + L.few_workers;
    const long long many_sets = all / (FEW_MOST + 1) < sets ? all / (FEW_MOST + 1) : sets;
    const long long many_slots = L.many_workers ? ((all + MANY_ROWS - 1) / MANY_ROWS + many_sets) * a.n_kv + L.many_workers : 0;
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
    const Layout L = layout_of(a);
    if (a.work_bytes < L.bytes) return B200_E_BADARG;
    char *work = static_cast<char *>(a.d_work);
    const Pieces few = {reinterpret_cast<float *>(work + L.few_acc), reinterpret_cast<float2 *>(work + L.few_top), L.few_workers};
    const Pieces many = {reinterpret_cast<float *>(work + L.many_acc), reinterpret_cast<float2 *>(work + L.many_top), L.many_workers};
    const Cut few_cut = {FEW_ROWS, FEW_KEYS, 0, L.many_workers ? FEW_MOST : INT_MAX, FEW_LEAST, FEW_GAP};
    const Cut many_cut = {MANY_ROWS, MANY_KEYS, L.many_workers ? FEW_MOST : INT_MAX, INT_MAX, MANY_LEAST, MANY_GAP};
    const int big = L.many_workers ? BIG_ROWS : INT_MAX;
    if (L.many_workers)
        if (const int rc = attn_many_launch(a, many_cut, many, big, st)) return rc;
    const size_t plan = plan_bytes(a.n_req, a.n_groups, 1), smem = (size_t)FEW_WARPS * FEW_STAGES * 2 * FEW_KEYS * HD * 2 + plan;
    cudaError_t e = cudaFuncSetAttribute(attn_few_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(L.few_workers / FEW_WARPS));
    cfg.blockDim = dim3(FEW_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = a.use_pdl != 0 || L.many_workers;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, attn_few_kernel<T, HD>, a, few_cut, few, big, (int)(L.many_workers != 0));
    if (e != cudaSuccess) return (int)e;
    ++g_b200_launches;
    const size_t both = plan_bytes(a.n_req, a.n_groups, 2);
    if (both > 48 * 1024 && (e = cudaFuncSetAttribute(attn_join_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)both)) != cudaSuccess) return (int)e;
    const long long blocks = ((long long)a.max_rows * a.n_q + JOIN_WARPS - 1) / JOIN_WARPS, most = JOIN_BLOCKS * sm_count();
    e = launch_chained(attn_join_kernel<T, HD>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(JOIN_WARPS * 32), both, st, a, few_cut, few, many_cut, many, big);
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
    if (a.max_rows == 0 || a.n_req == 0) return 0;
    if (!a.d_q || !a.d_k_pool || !a.d_v_pool || !a.d_out || !a.d_row_start || !a.d_len || !a.d_table || !a.d_work) return B200_E_BADARG;
    if (a.n_groups && (!a.d_group_start || !a.d_prefix_len || (a.prefix_ld && !a.d_prefix_table))) return B200_E_BADARG;
    if (a.q_ld < (long long)a.n_q * a.hd || a.q_ld % 8 || a.out_ld < (long long)a.n_q * a.hd || a.out_ld % 8) return B200_E_BADARG;
    if (((uintptr_t)a.d_q | (uintptr_t)a.d_k_pool | (uintptr_t)a.d_v_pool | (uintptr_t)a.d_out | (uintptr_t)a.d_work) % 16) return B200_E_BADARG;
    cudaStream_t st = (cudaStream_t)stream;
    if (a.wtype == B200_WT_F16) return a.hd == 64 ? launch<__half, 64>(a, st) : a.hd == 128 ? launch<__half, 128>(a, st) : launch<__half, 256>(a, st);
    return a.hd == 64 ? launch<__nv_bfloat16, 64>(a, st) : a.hd == 128 ? launch<__nv_bfloat16, 128>(a, st) : launch<__nv_bfloat16, 256>(a, st);
}
