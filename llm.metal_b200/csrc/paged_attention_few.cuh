// Attention over pages for sets of few query rows: a warp to itself, 16 query rows against a stretch of keys on mma.sync, m16n8k16, 16 keys a unit
// (paged_plan.cuh). Keys and values come with cp.async into a ring of the warp's own, two units ahead; scores, weights and sums stay in registers, one
// pass with a running maximum. What bounds it is memory: 16 rows take 64 operations a byte of cache at most, and the eight warps of an SM hold enough bytes in
// flight: 64 requests of 1500 tokens, 8 key / value heads of 128, 4 query heads to each, 82 us, 4.8 TB/s with the head of the launch and the join (floor 60). Warps
// share nothing, so that there is no barrier in the loop. Scores, maxima, sums and results are fp32; weights are rounded to the
// cache's type for the second product, as its two operands have one type: by half a step each, which is what the results' own rounding is, down to 2^-29 of the largest weight in
// binary16 and by 2^-40 of it at most below that (weight_lift).
#pragma once
#include "paged_attention.cuh"

namespace {

constexpr int FEW_ROWS = Cut<0>::ROWS, FEW_KEYS = Cut<0>::KEYS, FEW_STAGES = 3;
__host__ __device__ constexpr int few_ring(int hd) { return FEW_STAGES * 2 * FEW_KEYS * hd * 2; }    // bytes of a warp's ring

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
// The pieces of one worker. `ring`: few_ring(HD) bytes of shared memory, 128-byte aligned.
template <typename T, int HD>
__device__ void few_worker(const b200_paged_attn_args &a, const Plan &p, const Pieces &out, int worker, uint32_t ring)
{
    constexpr int CH = HD / 8;                               // 16-byte chunks of a key
    constexpr int HALF_STAGE = FEW_KEYS * HD * 2, STAGE = 2 * HALF_STAGE;
    const int lane = threadIdx.x & 31, g = lane >> 2, cq = lane & 3;
    const uint16_t *kp = static_cast<const uint16_t *>(a.d_k_pool), *vp = static_cast<const uint16_t *>(a.d_v_pool);
    const float c = a.scale * 1.4426950408889634f, lift = weight_lift<T>(15);
    const int page_shift = 31 - __clz(a.page);
    const Div by_g = p.shape.by_g;

    Walk<0> walk(p, worker);
    Piece piece;
    while (walk.next(p, piece)) {
        // ---- query rows t * 16 .. of head h, units k0 .. k0 + n - 1 ----
        const Set &s = piece.s;
        const int e = piece.e, h = piece.h, t = piece.t, k0 = piece.k0, n = piece.n;
        const int i0 = t * FEW_ROWS, valid = min(FEW_ROWS, s.nr - i0);
        const int seen = seen_by<0>(p, s, t), seen_first = s.own ? s.keys - s.rows + over(i0, by_g) + 1 : s.keys;
        const Keys keys = keys_of<0>(a, p, piece);                // (none comes before a request's own here)
        const int *table = s.own ? keys.table : keys.prefix;
        // the first page numbers, then the queries: one round trip for both
        int ids = lane < n ? __ldg(table + ((k0 + lane) * FEW_KEYS >> page_shift)) : 0;
        int limit[2], row_of[2], column[2];
        uint32_t q[CH / 2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = i0 + g + 8 * half;
            const bool on = g + 8 * half < valid;
            limit[half] = !on ? 0 : s.own ? s.keys - s.rows + over(i, by_g) + 1 : s.keys;
            const int local = on ? over(i, by_g) : 0, head = on ? i - local * by_g.d : 0;
            row_of[half] = row_at(p, e, local);
            column[half] = (h * by_g.d + head) * HD + 2 * cq;
            const uint16_t *src = static_cast<const uint16_t *>(a.d_q) + (long long)row_of[half] * a.q_ld + column[half];
#pragma unroll
            for (int ks = 0; ks < CH / 2; ++ks) {
                q[ks][half] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * ks) : 0u;
                q[ks][2 + half] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * ks + 8) : 0u;
            }
        }
        bool outside = false;
        auto issue = [&](int i) {                            // unit k0 + i of the tile into its place of the ring
            if (i < n) {
                if ((i & 31) == 0 && i > 0) {                // page numbers, 32 units at a time
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
            float top[2] = {-INFINITY, -INFINITY};
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
                top[r] = fmaxf(m[r], top[r] - lift);
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
        const bool whole = n == piece.ut && alone(p, piece); // nothing to join with
        const long long slot = p.tile[0][e] + h * piece.tiles + t + worker;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int k = g + 8 * r;
            if (k >= valid) continue;
            if (whole) {
                const float inv = 1.0f / l[r];
                uint16_t *to = static_cast<uint16_t *>(a.d_out) + (long long)row_of[r] * a.out_ld + column[r];
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
}

}  // namespace
