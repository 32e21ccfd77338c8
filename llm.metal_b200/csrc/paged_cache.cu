// Caches in pages (sm_100a): the tables of a step from the requests' lengths, and the new rows' way into their slots.
//
// Tables (extend, release): prefix sums over at most 1024 requests, one a thread, and then one (row or page) a thread, which finds its request by
// bisection in shared memory. A step of 32 requests is two dependent round trips to L2 and a launch; large ones are stores. One cluster of blocks:
// all of them scan for themselves, and nothing that was read is written before all have read it, so that lengths and the stack's height
// can be updated in place. Whole numbers throughout: the same result in every run. A step of 32 requests is bound by its launch (7 us with the host's part), 1000
// requests with 100 000 new tokens take 14 us (20 with an entry at a time to a thread), 90 000 pages given back 10.
#include "stream_core.cuh"
#include "../../include/llmb200_paged_kernels.h"

#include <cuda_bf16.h>

#include <limits.h>
#include <type_traits>

extern unsigned long long g_b200_launches;

namespace {

// Exclusive sums of x and y over the threads of a block; the totals go to `total`. `red`: 64 ints.
__device__ __forceinline__ int2 block_scan2(int x, int y, int *red, int2 &total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int ix = x, iy = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, ix, o), b = __shfl_up_sync(0xffffffffu, iy, o);
        if (lane >= o) { ix += a; iy += b; }
    }
    if (lane == 31) { red[warp] = ix; red[32 + warp] = iy; }
    __syncthreads();
    int bx = lane < nw ? red[lane] : 0, by = lane < nw ? red[32 + lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, bx, o), b = __shfl_up_sync(0xffffffffu, by, o);
        if (lane >= o) { bx += a; by += b; }
    }
    total.x = __shfl_sync(0xffffffffu, bx, 31);
    total.y = __shfl_sync(0xffffffffu, by, 31);
    const int px = __shfl_sync(0xffffffffu, bx, max(warp - 1, 0)), py = __shfl_sync(0xffffffffu, by, max(warp - 1, 0));
    return make_int2(ix - x + (warp ? px : 0), iy - y + (warp ? py : 0));
}

// The last r < n with start[r] <= at (start ascending, start[0] = 0).
__device__ __forceinline__ int owner_of(const int *start, int n, int at)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void report(unsigned *status, unsigned bits)
{
    if (status && bits) atomicOr(status, bits);
}

constexpr int TABLE_BLOCKS = 8;          // a portable cluster
// Up to this many rows (pages for release) one block does it, which a launch starts sooner. Us in a captured run, one block and the cluster, extend: 32 requests and 32 rows 2.6 and 3.3, 2048
// rows 4.1 and 4.2, 3000 rows 4.3 and 4.3, 4096 rows 4.5 and 4.3, 8192 rows 6.3 and 4.1; 1024 requests and 2048 rows 4.4 and 4.6, 3000 rows 4.8 and 4.6; release: 1024 requests and 2048
// pages 3.8 and 4.1, 4096 pages 4.4 and 4.1.
constexpr int TABLE_ROWS = 2048;

template <bool RELEASE>
__global__ void __launch_bounds__(1024) pages_kernel(const __grid_constant__ b200_pages_args a)
{
    __shared__ int s_len[B200_PAGED_MAX_REQ], s_row[B200_PAGED_MAX_REQ], s_page[B200_PAGED_MAX_REQ];
    __shared__ int red[64];
    const int r = threadIdx.x, n = a.n_req;
    pdl_launch_dependents();
    pdl_wait();
    const int free_n = *a.d_free_n;
    int len = 0, rows = 0, pages = 0;
    unsigned bad = 0;
    if (r < n) {
        len = a.d_len[r];
        const int given = a.d_new[r];
        const long long room = (long long)a.table_ld * a.page;
        if (RELEASE) {
            if (given) {
                if (len < 0 || len > room) bad = B200_PAGED_BAD_LENGTH;
                else pages = (len + a.page - 1) / a.page;
            }
        } else if (len < 0 || given < 0 || given > a.max_rows || (long long)len + given > room) {
            bad = B200_PAGED_BAD_LENGTH;
        } else {
            rows = given;
            pages = (len + given + a.page - 1) / a.page - (len + a.page - 1) / a.page;
        }
    }
    int2 total;                                              // at most 1024 * 2^20 each
    const int2 at = block_scan2(rows, pages, red, total);
    if (r < n) { s_len[r] = len; s_row[r] = at.x; s_page[r] = at.y; }
    if (total.x > a.max_rows) bad |= B200_PAGED_BAD_LENGTH;
    if (free_n < 0 || free_n > a.n_pages || (RELEASE ? free_n + total.y > a.n_pages : total.y > free_n)) bad |= B200_PAGED_NO_PAGES;
    const unsigned why = (__syncthreads_or(bad & B200_PAGED_BAD_LENGTH) ? B200_PAGED_BAD_LENGTH : 0u) | (__syncthreads_or(bad & B200_PAGED_NO_PAGES) ? B200_PAGED_NO_PAGES : 0u);
    if (gridDim.x > 1) cluster_sync();                       // all blocks have read what is updated in place
    if (blockIdx.x == 0) {
        if (r < n) {
            a.d_len_out[r] = why ? len : RELEASE ? (a.d_new[r] ? 0 : len) : len + rows;
            if (!RELEASE) a.d_row_start[r] = why ? 0 : at.x;
        }
        if (r == 0) {
            *a.d_free_n_out = why ? free_n : RELEASE ? free_n + total.y : free_n - total.y;
            if (!RELEASE) a.d_row_start[n] = why ? 0 : total.x;
            report(a.d_status, why);
        }
    }
    if (why) return;
    // Where there is more than one to a thread, four at a time: one search, one round trip to the table and the stack, and 16-byte stores where the arrays are
    // aligned for them.
    const int thread = blockIdx.x * blockDim.x + threadIdx.x, threads = gridDim.x * blockDim.x, shift = 31 - __clz(a.page);
    const int pages_each = total.y > threads ? 4 : 1, rows_each = total.x > threads ? 4 : 1;
    unsigned outside = 0;
#pragma unroll 1
    for (int p = pages_each * thread; p < total.y; p += pages_each * threads) {
        int q = owner_of(s_page, n, p);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= pages_each || p + k >= total.y) break;
            while (q + 1 < n && s_page[q + 1] <= p + k) ++q;
            if (RELEASE) {
                const int id = a.d_table[(size_t)q * a.table_ld + (p + k - s_page[q])];
                a.d_free[free_n + p + k] = id;
                if (id < 0 || id >= a.n_pages) outside = B200_PAGED_BAD_PAGE;
            } else a.d_table[(size_t)q * a.table_ld + ((s_len[q] + a.page - 1) >> shift) + (p + k - s_page[q])] = a.d_free[free_n - 1 - p - k];
        }
    }
    if (RELEASE) { report(a.d_status, outside); return; }
    const bool wide = ((reinterpret_cast<uintptr_t>(a.d_slot) | reinterpret_cast<uintptr_t>(a.d_pos)) & 15) == 0;
#pragma unroll 1
    for (int m = rows_each * thread; m < total.x; m += rows_each * threads) {
        int q = owner_of(s_row, n, m), slot[4], pos[4], token_in_page[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= rows_each) break;
            const int at_row = min(m + k, total.x - 1);
            while (q + 1 < n && s_row[q + 1] <= at_row) ++q;
            const int token = s_len[q] + (at_row - s_row[q]), page = token >> shift, held = (s_len[q] + a.page - 1) >> shift;
            // the pages of this call come from the stack: their numbers in the table may not be there yet
            slot[k] = page < held ? a.d_table[(size_t)q * a.table_ld + page] : a.d_free[free_n - 1 - (s_page[q] + page - held)];
            pos[k] = (a.d_base ? a.d_base[q] : 0) + token;
            token_in_page[k] = token & (a.page - 1);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= rows_each) break;
            const bool ok = slot[k] >= 0 && slot[k] < a.n_pages;
            slot[k] = ok ? (slot[k] << shift) + token_in_page[k] : -1;
            if (!ok) outside = B200_PAGED_BAD_PAGE;
        }
        if (rows_each == 4 && wide && m + 4 <= total.x) {
            *reinterpret_cast<int4 *>(a.d_slot + m) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4 *>(a.d_pos + m) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < rows_each && m + k < total.x) { a.d_slot[m + k] = slot[k]; a.d_pos[m + k] = pos[k]; }
        }
    }
    report(a.d_status, outside);
}

template <bool RELEASE>
int launch_pages(const b200_pages_args *ap, void *stream)
{
    if (!ap) return B200_E_BADARG;
    const b200_pages_args &a = *ap;
    if (a.n_req < 0 || a.n_req > B200_PAGED_MAX_REQ || a.n_pages < 0 || a.table_ld < 0 || a.table_ld > (1 << 20)) return B200_E_BADARG;
    if (a.page < 16 || a.page > 256 || (a.page & (a.page - 1))) return B200_E_BADARG;
    if ((long long)a.n_pages * a.page > INT_MAX || (long long)a.table_ld * a.page > INT_MAX) return B200_E_TOOLARGE;
    if (!a.d_free_n || !a.d_free_n_out || (a.n_req && (!a.d_len || !a.d_len_out || !a.d_new)) || (a.n_req && a.table_ld && !a.d_table) || (a.n_pages && !a.d_free)) return B200_E_BADARG;
    if (!RELEASE) {
        if (a.max_rows < 0 || a.max_rows > (1 << 20)) return B200_E_BADARG;
        if (!a.d_row_start || (a.max_rows && (!a.d_slot || !a.d_pos))) return B200_E_BADARG;
    }
    const long long most = RELEASE ? (long long)a.n_req * a.table_ld : a.max_rows;
    const bool one = most <= TABLE_ROWS;
    int threads = 1024;
    if (one) {
        const int want = a.n_req > (int)most ? a.n_req : (int)most;
        threads = want >= 1024 ? 1024 : want < 64 ? 64 : (want + 31) & ~31;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(one ? 1 : TABLE_BLOCKS);
    cfg.blockDim = dim3(threads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = a.use_pdl != 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = TABLE_BLOCKS; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = one ? 1 : 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, pages_kernel<RELEASE>, a);
    if (e != cudaSuccess) return (int)e;
    ++g_b200_launches;
    return (int)cudaGetLastError();
}

// ---- new rows into their slots ------------------------------------------------------------------------------------------------
// Bound by memory: 4 bytes read and 2 written a number; 8191 rows of 32 heads of 128 take 41 us, 4.9 TB/s, where a copy reaches 6.6. hd / 8 lanes hold a
// head, each four numbers of its lower half and the four that they turn with, so that the norm is a few shuffles and the rotation stays in
// the lane. (A warp to a head of 128, four numbers a lane: 140 instructions a head, 50 us.) The angle pos * inv_freq is formed in 64 bits (exact) and brought
// into one turn before the 32-bit sine and cosine: as a 32-bit product it is off by pos * 2^-24, more than binary16's step from position 8000 on. q, k and v are rounded once, to the type of the cache that the tensor cores read.
template <typename T> __device__ __forceinline__ uint16_t to_bits(float x)
{
    if constexpr (std::is_same<T, __half>::value) return __half_as_ushort(__float2half_rn(x));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

constexpr int STORE_WARPS = 8, STORE_AHEAD = 2;
// Up to STORE_FEW rows a block has one round of heads, or 32 rows would run on 32 SMs; above, all heads of a row, which forms the angles once. Us in a captured run, one round and all heads:
// 32 / 8 heads of 128, 32 rows 2.1 and 3.0, 128 rows 2.9 and 3.3, 256 rows 4.2 and 3.8, 512 rows 6.2 and 4.8; 16 / 8 heads of 128, 32 rows 2.3 and 2.5, 128 rows 2.6 and
// 2.7, 256 rows 3.2 and 3.0, 512 rows 4.7 and 3.8; 16 / 2 heads of 64 and 4 / 1 of 256 are one round or little more, and the same either way.
constexpr int STORE_FEW = 192;

template <typename T, int HD>
__global__ void __launch_bounds__(STORE_WARPS * 32) paged_store_kernel(const __grid_constant__ b200_paged_store_args a, int heads_per_block)
{
    constexpr int HALF = HD / 2, N = 4, LANES = HD / 8, HEADS = 32 / LANES, STEP = STORE_WARPS * HEADS;        // lanes of a head, heads of a warp, of a round
    __shared__ __align__(16) float s_cos[HALF], s_sin[HALF];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane % LANES * N;
    const int m = blockIdx.x;
    pdl_launch_dependents();
    float gq[2 * N], gk[2 * N];                              // weights: constants, read ahead of the wait
#pragma unroll
    for (int j = 0; j < 2 * N; ++j) gq[j] = gk[j] = 1.0f;
    auto weights = [&](float *g, const float *from) {
        if (!from) return;
        *reinterpret_cast<float4 *>(g) = *reinterpret_cast<const float4 *>(from + d);
        *reinterpret_cast<float4 *>(g + N) = *reinterpret_cast<const float4 *>(from + HALF + d);
    };
    weights(gq, a.d_q_gamma);
    weights(gk, a.d_k_gamma);
    const float freq = a.d_inv_freq && threadIdx.x < HALF ? a.d_inv_freq[threadIdx.x] : 0.0f;
    pdl_wait();
    // all loads at once, the count's among them: rows up to max_rows exist, and what lies behind the last one is only not stored
    const int rows = *a.d_rows, slot = a.d_slot[m], pos = a.d_pos[m];
    const int heads = a.n_q + 2 * a.n_kv, h1 = min(heads, ((int)blockIdx.y + 1) * heads_per_block);
    const float *row = a.d_qkv + (long long)m * a.qkv_ld + d;
    float x[STORE_AHEAD][2 * N];                             // heads on their way: the first ones under the angles
    auto load = [&](int h0) {
#pragma unroll
        for (int k = 0; k < STORE_AHEAD; ++k) {
            const int h = h0 + k * STEP;
            if (h < h1) {
                *reinterpret_cast<float4 *>(x[k]) = *reinterpret_cast<const float4 *>(row + h * HD);
                *reinterpret_cast<float4 *>(x[k] + N) = *reinterpret_cast<const float4 *>(row + h * HD + HALF);
            }
        }
    };
    int h0 = blockIdx.y * heads_per_block + warp * HEADS + lane / LANES;
    load(h0);
    if (rows < 0 || rows > a.max_rows) {
        if (m == 0 && blockIdx.y == 0 && threadIdx.x == 0) report(a.d_status, B200_PAGED_BAD_LENGTH);
        return;
    }
    if (m >= rows) return;
    if (threadIdx.x < HALF && a.d_inv_freq) {
        constexpr double TURN = 6.283185307179586476925, PER_TURN = 0.15915494309189533577;
        const double t = (double)pos * (double)freq;
        float sn, cs;
        sincosf((float)(t - rint(t * PER_TURN) * TURN), &sn, &cs);
        s_cos[threadIdx.x] = cs; s_sin[threadIdx.x] = sn;
    }
    const bool in_pool = slot >= 0 && slot < a.n_pages * a.page;
    if (!in_pool && threadIdx.x == 0 && blockIdx.y == 0) report(a.d_status, B200_PAGED_BAD_PAGE);
    __syncthreads();
    float cs[N], sn[N];
    *reinterpret_cast<float4 *>(cs) = *reinterpret_cast<const float4 *>(s_cos + d);
    *reinterpret_cast<float4 *>(sn) = *reinterpret_cast<const float4 *>(s_sin + d);
    const int shift = 31 - __clz(a.page);
    const long long at = ((long long)(slot >> shift) * a.n_kv << shift) + (slot & (a.page - 1));       // of head 0: heads are a page apart
#pragma unroll 1
    for (; __any_sync(0xffffffffu, h0 < h1); h0 += STORE_AHEAD * STEP) {
#pragma unroll
        for (int k = 0; k < STORE_AHEAD; ++k) {
            const int h = h0 + k * STEP;
            const bool is_q = h < a.n_q, turns = h < a.n_q + a.n_kv;
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * N; ++j) ss = fmaf(x[k][j], x[k][j], ss);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (h >= h1) continue;
            if (turns) {
                if (is_q ? a.d_q_gamma != nullptr : a.d_k_gamma != nullptr) {
                    const float inv = rsqrtf(fmaf(ss, 1.0f / (float)HD, a.eps));       // 2 ulp
#pragma unroll
                    for (int j = 0; j < 2 * N; ++j) x[k][j] *= (is_q ? gq[j] : gk[j]) * inv;
                }
                if (a.d_inv_freq) {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float lo = x[k][j], hi = x[k][N + j];
                        x[k][j] = lo * cs[j] - hi * sn[j]; x[k][N + j] = lo * sn[j] + hi * cs[j];
                    }
                }
            }
            uint16_t *to;
            if (is_q) to = static_cast<uint16_t *>(a.d_q) + (long long)m * a.q_ld + h * HD;
            else {
                if (!in_pool) continue;
                to = static_cast<uint16_t *>(turns ? a.d_k_pool : a.d_v_pool) + (at + ((long long)(h - a.n_q - (turns ? 0 : a.n_kv)) << shift)) * HD;
            }
            uint2 w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                w[j].x = (uint32_t)to_bits<T>(x[k][N * j]) | (uint32_t)to_bits<T>(x[k][N * j + 1]) << 16;
                w[j].y = (uint32_t)to_bits<T>(x[k][N * j + 2]) | (uint32_t)to_bits<T>(x[k][N * j + 3]) << 16;
            }
            *reinterpret_cast<uint2 *>(to + d) = w[0];
            *reinterpret_cast<uint2 *>(to + HALF + d) = w[1];
        }
        load(h0 + STORE_AHEAD * STEP);
    }
}

template <typename T>
int launch_store(const b200_paged_store_args &a, cudaStream_t st)
{
    const int heads = a.n_q + 2 * a.n_kv, per = a.max_rows <= STORE_FEW ? STORE_WARPS * 256 / a.hd : heads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.max_rows, (heads + per - 1) / per);
    cfg.blockDim = dim3(STORE_WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = a.use_pdl != 0;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = a.hd == 64 ? cudaLaunchKernelEx(&cfg, paged_store_kernel<T, 64>, a, per)
                        : a.hd == 128 ? cudaLaunchKernelEx(&cfg, paged_store_kernel<T, 128>, a, per) : cudaLaunchKernelEx(&cfg, paged_store_kernel<T, 256>, a, per);
    if (e != cudaSuccess) return (int)e;
    ++g_b200_launches;
    return (int)cudaGetLastError();
}

}  // namespace

extern "C" int b200_pages_extend(const b200_pages_args *a, void *stream) { return launch_pages<false>(a, stream); }
extern "C" int b200_pages_release(const b200_pages_args *a, void *stream) { return launch_pages<true>(a, stream); }

extern "C" int b200_paged_store(const b200_paged_store_args *ap, void *stream)
{
    if (!ap) return B200_E_BADARG;
    const b200_paged_store_args &a = *ap;
    if ((a.wtype != B200_WT_F16 && a.wtype != B200_WT_BF16) || (a.hd != 64 && a.hd != 128 && a.hd != 256)) return B200_E_BADARG;
    if (a.n_q < 1 || a.n_kv < 1 || a.n_q % a.n_kv || a.n_q > 1024 || a.max_rows < 0 || a.max_rows > (1 << 20) || a.n_pages < 1) return B200_E_BADARG;
    if (a.page < 16 || a.page > 256 || (a.page & (a.page - 1))) return B200_E_BADARG;
    if ((long long)a.n_pages * a.page > INT_MAX) return B200_E_TOOLARGE;
    if (a.max_rows == 0) return 0;
    if (!a.d_qkv || !a.d_rows || !a.d_slot || !a.d_pos || !a.d_k_pool || !a.d_v_pool || !a.d_q) return B200_E_BADARG;
    if (a.qkv_ld < (long long)(a.n_q + 2 * a.n_kv) * a.hd || a.qkv_ld % 4 || a.q_ld < (long long)a.n_q * a.hd || a.q_ld % 8) return B200_E_BADARG;
    if (((uintptr_t)a.d_qkv | (uintptr_t)a.d_k_pool | (uintptr_t)a.d_v_pool | (uintptr_t)a.d_q | (uintptr_t)a.d_q_gamma | (uintptr_t)a.d_k_gamma | (uintptr_t)a.d_inv_freq) % 16)
        return B200_E_BADARG;
    return a.wtype == B200_WT_F16 ? launch_store<__half>(a, (cudaStream_t)stream) : launch_store<__nv_bfloat16>(a, (cudaStream_t)stream);
}
