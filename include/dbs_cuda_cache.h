/* SPDX-License-Identifier: MIT
 *
 * dbs_cuda_cache.h -- a paged key/value cache for the beams of a search, and the
 * attention that reads it. The reference has no counterpart: its search hands
 * parents to the caller, who reorders the model's states. These entry points do
 * that on the device, from the parents a search step wrote, and attend over the
 * result, so a transformer behind a step-by-step search needs no other cache.
 *
 * Conventions as in dbs_cuda.h: device pointers, asynchronous on the caller's
 * stream, a status code back, no allocation. Calls on one cache must be ordered
 * (one stream, or streams that wait for one another).
 */
#ifndef DBS_CUDA_CACHE_H
#define DBS_CUDA_CACHE_H

#include "dbs_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DBS_CUDA_CACHE_MAX_HEAD_DIM 256
#define DBS_CUDA_CACHE_WORKSPACE_ZEROED 8192 /* bytes at the front of a workspace that the caller zeroes once */
/* Bits of the status word. */
#define DBS_CUDA_CACHE_STATUS_POOL 1     /* the pool ran out of pages: some columns have none */
#define DBS_CUDA_CACHE_STATUS_CAPACITY 2 /* a beam was to grow past max_pages columns */
#define DBS_CUDA_CACHE_STATUS_INDEX 4    /* a parent, count, path entry, table entry or length was out of range */
#define DBS_CUDA_CACHE_STATUS_SHARED 8   /* a page that is not complete has several holders, or one twice */
#define DBS_CUDA_CACHE_STATUS_TIMEOUT 16 /* a bounded wait inside a kernel gave up */

/* What dbs_cuda_cache_refresh does about the pool's values. */
#define DBS_CUDA_CACHE_VALUES_ALL 1
#define DBS_CUDA_CACHE_VALUES_IF_SET 2

/* The cache of one search: batch_size examples of beam_size beams. A beam's
 * token at position p lies in row p % page_size of page table[b, k, p / page_size],
 * for every layer and head. The caller owns all arrays:
 *   pages       [num_layers, 2, num_pages, num_heads, page_size, head_dim], keys
 *               then values, of data_type; 16-byte aligned
 *   table       [batch_size, beam_size, max_pages] int32, -1: no page
 *   lengths     [batch_size, beam_size] int32: committed tokens
 *   references  [num_pages] int32: table entries that name the page
 *   plan        dbs_cuda_cache_plan_bytes() bytes, 256-byte aligned, zeroed once
 *   status      2 int32, zeroed once: the bits above (sticky); 1 once a value that
 *               is not finite was written, until dbs_cuda_cache_refresh finds none:
 *               attention then takes every row for itself, right but many times slower
 * A page at or behind a beam's last incomplete page belongs to that beam alone;
 * complete pages may be shared. page_size is 16, 32 or 64, head_dim a multiple of
 * 8 up to 256. */
typedef struct DBSCudaCache {
    int32_t batch_size;
    int32_t beam_size;
    int32_t max_pages;
    int32_t num_pages;
    int32_t num_layers;
    int32_t num_heads;
    int32_t head_dim;
    int32_t page_size;
    int32_t data_type;
    int32_t reserved0;
    void* pages;
    int32_t* table;
    int32_t* lengths;
    int32_t* references;
    void* plan;
    int64_t plan_bytes;
    int32_t* status;
} DBSCudaCache;

/* Bytes of the plan array; negative when the sizes are refused. */
DBS_CUDA_EXPORT int64_t dbs_cuda_cache_plan_bytes(const DBSCudaCache* cache);

/* References and plan from table and lengths, after the caller wrote those. Entries out of range become
 * -1 and lengths outside [0, max_pages * page_size] the nearer end, with the INDEX bit. values: 0, or
 * DBS_CUDA_CACHE_VALUES_ALL: also status[1] from the values of the whole pool, after the caller wrote
 * pages (values that are not finite in pages without a holder become 0, in others they set it), or
 * DBS_CUDA_CACHE_VALUES_IF_SET: the same where status[1] is set, nothing where it is not. */
DBS_CUDA_EXPORT int dbs_cuda_cache_refresh(const DBSCudaCache* cache, int values, void* stream);

/* One step of the beams. First written_s tokens after each beam's committed ones become
 * committed (written [B, K] int32, or NULL: written_all for every beam). Then beam
 * (b, k) becomes a copy of beam (b, parents[b, k]) (NULL: itself; negative: empty):
 * complete pages are shared, the first child in beam order keeps its parent's other
 * pages, every other child gets pages of its own and a copy of the rows in use.
 * Pages without a holder are free at once. Last, every beam with a parent gets pages
 * for room_s more tokens (room [B, K], or NULL: room_all); what it held beyond that is
 * freed. New pages are the lowest free ones, in (beam, column) order. */
DBS_CUDA_EXPORT int dbs_cuda_cache_fork(const DBSCudaCache* cache, const int32_t* parents, const int32_t* written,
                                        int32_t written_all, const int32_t* room, int32_t room_all, void* stream);

/* Accepts a path of the drafted tokens: row lengths + path[b, k, a] moves to row
 * lengths + a for a < counts[b, k], in every layer (path [B, K, path_stride] int32,
 * strictly increasing within the count); then dbs_cuda_cache_fork with no parents,
 * written = counts and room_all. Of a beam whose count is not in [0, path_stride], whose path
 * does not rise or names a token without a page nothing is accepted or moved (the INDEX bit);
 * a beam without tokens and pages stays empty, whatever its count. */
DBS_CUDA_EXPORT int dbs_cuda_cache_commit(const DBSCudaCache* cache, const int32_t* path, int32_t path_stride,
                                          const int32_t* counts, int32_t room_all, void* stream);

/* Moves the pages in use to the front of the pool: with n pages in use, the i-th of
 * those at or above n goes to the i-th free page below n. */
DBS_CUDA_EXPORT int dbs_cuda_cache_compact(const DBSCudaCache* cache, void* stream);

/* New tokens of the first `beams` beams of every example, and attention over the cache.
 * Token j < counts[b, k] (NULL: new_tokens) takes position lengths[b, k] + j: its key and
 * value are written to layer `layer` (k, v NULL: they are there already). Query i sees the
 * committed tokens and the new tokens j with mask[b, k, i, j] (bytes [B, beams, N, N];
 * NULL: j <= i); queries at or past the count, and all that sees nothing, give 0 and an lse
 * of -inf. Tokens without a page are not written and not seen. A score of -inf (or below what
 * 32 bits hold) weighs nothing, and a row of such alone is as one that sees nothing; one of
 * +inf or NaN makes the row's out and lse NaN.
 *   out = softmax(scale * q k^T) v,  lse = log sum exp(scale * q k^T)
 * q, out: [B, beams, N, query_heads, head_dim]; k, v: [B, beams, N, num_heads, head_dim];
 * query head h reads head h / (query_heads / num_heads). Strides are in elements, for
 * the four leading axes; the last axis is contiguous; q, k and v rows start on 16-byte
 * boundaries. out is contiguous, lse [B, beams, N, query_heads] float32 or NULL. */
typedef struct DBSCudaAttendArgs {
    int32_t layer;
    int32_t beams;
    int32_t new_tokens;
    int32_t query_heads;
    float scale;
    int32_t reserved0;
    const void* q;
    const void* k;
    const void* v;
    int64_t q_strides[4];
    int64_t k_strides[4];
    int64_t v_strides[4];
    const uint8_t* mask;
    const int32_t* counts;
    void* out;
    float* lse;
    void* workspace; /* dbs_cuda_cache_attend_workspace_size() bytes, 256-byte aligned; the first
                        DBS_CUDA_CACHE_WORKSPACE_ZEROED of them (counters, 0 between calls) zeroed once */
    int64_t workspace_bytes;
} DBSCudaAttendArgs;

/* Workspace of an attend call of these sizes (of one cache: the same for all); negative when they
 * are refused. One workspace serves all calls on a cache, which are ordered. */
DBS_CUDA_EXPORT int64_t dbs_cuda_cache_attend_workspace_size(const DBSCudaCache* cache, const DBSCudaAttendArgs* args);

DBS_CUDA_EXPORT int dbs_cuda_cache_attend(const DBSCudaCache* cache, const DBSCudaAttendArgs* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif
