/*
 * llmb200_paged_kernels.h -- kernel-level C ABI of caches in pages that requests share (sm_100a).
 *
 * For callers that serve many requests of unlike lengths, or sample a group of answers to one prompt: the keys and
 * values of a layer lie in two pools of pages, a request owns the pages that its own tokens fill, and the tokens that a
 * group of requests begins with lie in pages of their own, stored once and read once for all of the group. Beside
 * b200_attn_decode and b200_rows_attn (llmb200_kernels.h), whose caches are one block a sequence.
 *
 * One step: b200_pages_extend (once), then per layer the fused q / k / v product, b200_paged_store and b200_paged_attn.
 * When requests end: b200_pages_release. No counterpart in the reference, which copies its cache per sequence
 * (src/nn/fast_inference.c:696-985).
 *
 * Everything that a step decides -- lengths, rows, pages -- is read on the device: a step can be captured into a CUDA
 * graph and replayed while requests grow. What the host gives are bounds.
 *
 *   pool       [n_pages][n_kv][page][hd] elements of the type `wtype` names (B200_WT_F16 or B200_WT_BF16), 16-byte
 *              aligned; page is 16, 32, 64, 128 or 256, hd is 64, 128 or 256
 *   table      int [n_req][table_ld]: page numbers of each request's own tokens, in order; what lies behind the last
 *              page of a request is not read
 *   slot       number of a token's place in a pool: page number * page + place within the page
 *   rows       the new tokens of all requests, request after request: request r has rows d_row_start[r] ..
 *              d_row_start[r + 1] - 1. Rows behind the last request's, up to max_rows, exist in every array of rows, are
 *              never written, and what they hold has no influence.
 *
 * Every function enqueues on `stream` (a cudaStream_t) of the current device and returns 0, a positive cudaError_t, or a
 * negative B200_E_* code for rejected arguments; nothing allocates or waits. What only the device can see is reported
 * through *d_status (optional): bits are added to it, never taken away. Arrays that are written overlap no other array
 * of the call, but where it is said.
 */
#ifndef LLMB200_PAGED_KERNELS_H
#define LLMB200_PAGED_KERNELS_H

#include "llmb200_kernels.h"   /* B200_E_*, B200_WT_* */

#ifdef __cplusplus
extern "C" {
#endif

#define B200_PAGED_MAX_REQ 1024

#define B200_PAGED_NO_PAGES   1u   /* extend: fewer free pages than needed; release: more pages than there are */
#define B200_PAGED_BAD_LENGTH 2u   /* a length, a row count or a range that does not fit its buffer */
#define B200_PAGED_BAD_PAGE   4u   /* a page number outside the pool */
#define B200_PAGED_TIMED_OUT  8u   /* a wait inside a kernel ran out: the call's results are invalid */

/* ------------------------------------------------------------------------
 * b200_pages_extend: request r holds d_len[r] tokens of its own and takes d_new[r] more (0: none). It gets the pages that
 * it lacks, in order of requests, from the top of the stack d_free[0 .. *d_free_n), and
 *   d_table                  its new pages' numbers
 *   d_row_start[r]           sum of d_new before r, r <= n_req
 *   d_slot, d_pos [row]      slot of every new token and its position, d_base[r] + d_len[r] + i (d_base NULL: 0)
 *   d_len_out[r]             d_len[r] + d_new[r]
 *   *d_free_n_out            what is left of the stack; the stack itself is only read
 * All or nothing: if pages run out or a length does not fit (negative, more than table_ld pages, more than max_rows new
 * tokens in all), *d_status says so, d_row_start becomes all zero -- the calls that follow have no rows --, d_len_out and
 * *d_free_n_out repeat what was there, and nothing else is written. A page number outside the pool on the stack or in
 * the last page that a request fills further gives slot -1, which b200_paged_store leaves out, and B200_PAGED_BAD_PAGE.
 *
 * b200_pages_release: requests with d_new[r] != 0 give their pages back, request after request, to the top of the stack
 * (d_free has room for n_pages), and d_len_out[r] becomes 0, d_len[r] for the others. The table keeps its
 * numbers. d_base, d_row_start, d_slot, d_pos and max_rows are not used. All or nothing, likewise. A page number outside the
 * pool goes onto the stack as the table has it, so that the stack's height stays that of the lengths, with B200_PAGED_BAD_PAGE.
 *
 * d_len_out may be d_len and d_free_n_out may be d_free_n; no other two arrays may overlap.
 * ---------------------------------------------------------------------- */
typedef struct b200_pages_args {
    int n_req;                     /* 0 .. B200_PAGED_MAX_REQ */
    int page, table_ld, n_pages, max_rows;
    const int *d_len; int *d_len_out;
    const int *d_new, *d_base;
    int *d_table;
    int *d_free; const int *d_free_n; int *d_free_n_out;
    int *d_row_start;              /* [n_req + 1] */
    int *d_slot, *d_pos;           /* [max_rows] */
    unsigned *d_status;
    int use_pdl;                   /* programmatic dependent launch: may start while the kernel before it drains */
} b200_pages_args;
int b200_pages_extend(const b200_pages_args *a, void *stream);
int b200_pages_release(const b200_pages_args *a, void *stream);

/* ------------------------------------------------------------------------
 * New rows of a layer's fused projection into its pools. Row m of d_qkv is fp32 [n_q * hd | n_kv * hd | n_kv * hd]:
 *   q, k   RMS norm over each head times gamma (gamma NULL: no norm), then the rotation of b200_attn_decode: the pair
 *          (d, d + hd / 2) turns by the angle d_pos[m] * d_inv_freq[d], formed exactly (d_inv_freq NULL: no rotation)
 *   k, v   rounded to the pool's type, stored at slot d_slot[m]; a slot outside the pool is left out
 *   q      rounded likewise, stored to row m of d_q: what b200_paged_attn reads
 * With use_pdl the weights (d_q_gamma, d_k_gamma, d_inv_freq) are read ahead of the wait for the kernel before.
 * *d_rows rows (a device word): the last of b200_pages_extend's d_row_start. If it is negative or more than max_rows, nothing
 * is stored and *d_status says so. b200_pages_extend gives no slot twice; of two rows of one slot each element is one of the two's.
 * ---------------------------------------------------------------------- */
typedef struct b200_paged_store_args {
    int wtype, n_q, n_kv, hd, page, n_pages, max_rows;
    float eps;
    const float *d_qkv; long long qkv_ld;                    /* rows qkv_ld floats apart, a multiple of 4; 16-byte aligned */
    const float *d_q_gamma, *d_k_gamma, *d_inv_freq;         /* [hd], [hd], [hd / 2]; 16-byte aligned */
    const int *d_rows, *d_slot, *d_pos;
    void *d_k_pool, *d_v_pool;
    void *d_q; long long q_ld;                               /* rows q_ld elements apart, a multiple of 8; 16-byte aligned */
    unsigned *d_status;
    int use_pdl;
} b200_paged_store_args;
int b200_paged_store(const b200_paged_store_args *a, void *stream);

/* ------------------------------------------------------------------------
 * Attention of the new rows. Request r owns d_len[r] tokens, its new rows' included (b200_pages_extend's d_len_out): row i
 * of its n sees its own tokens 0 .. d_len[r] - n + i, and before them all of its group's prefix:
 *   out[m][h] = sum over those keys of softmax(scale * q[m][h] . k) v,   head h reads key / value head h / (n_q / n_kv)
 * Group g is the requests d_group_start[g] .. d_group_start[g + 1] - 1, its prefix the first d_prefix_len[g] tokens (0:
 * none) of the pages d_prefix_table[g][prefix_ld]. Requests outside every group have no prefix; n_groups 0: no
 * request has. The pages of a prefix are read once for every 256 query rows (rows times n_q / n_kv) of its group, up to hd 128, and
 * for every 16 above; a request that brings 128 of them by itself, a portion of a prompt, reads its prefix for itself.
 * Tokens that a row does not see have no influence on it, whatever their slots hold (infinities and NaN too). Scores, largest scores and
 * sums are fp32; each weight is rounded to the pool's type before it meets its value (half a step; in binary16 2^-32 of the row's
 * largest weight at least), and the result once more. (b200_rows_attn has two planes of queries, and weights and results of fp32.)
 *
 * If a length or a range does not fit its buffer, the call leaves all of its output as it was and *d_status says
 * so. So it does for work of 2^31 units (16 query rows by 16 keys, from 33 query rows of a request or group on and up to hd 128 256 by 64, and up to 13
 * more for each 16 or 256 rows): a prompt of 185 000 tokens as one portion, at 32 query heads of 256. A page number outside the pool is not read; what the rows that would see it come out as is undefined.
 * d_work: b200_paged_attn_work_bytes(a) bytes, 16-byte aligned, for this call alone while it runs; nothing is kept in it
 * from one call to the next. Calls that may run at the same time need a d_work each.
 * ---------------------------------------------------------------------- */
typedef struct b200_paged_attn_args {
    int wtype, n_q, n_kv, hd, page, n_pages, max_rows;
    float scale;                                             /* finite, times log2(e) too: below 2.3e38 */
    const void *d_q; long long q_ld;                         /* rows q_ld elements apart, a multiple of 8; 16-byte aligned */
    const void *d_k_pool, *d_v_pool;
    void *d_out; long long out_ld;                           /* likewise; n_q * hd elements of the pool's type a row */
    int n_req; const int *d_row_start, *d_len;
    const int *d_table; int table_ld;
    int n_groups; const int *d_group_start, *d_prefix_len;   /* n_groups <= n_req */
    const int *d_prefix_table; int prefix_ld;
    void *d_work; size_t work_bytes;
    unsigned *d_status;
    int use_pdl;
} b200_paged_attn_args;
/* Bytes of d_work for these sizes (the pointers, d_work's among them, are not looked at); 0 for sizes that b200_paged_attn refuses. */
size_t b200_paged_attn_work_bytes(const b200_paged_attn_args *a);
int b200_paged_attn(const b200_paged_attn_args *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* LLMB200_PAGED_KERNELS_H */
