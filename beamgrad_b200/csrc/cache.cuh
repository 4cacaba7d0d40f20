// SPDX-License-Identifier: MIT
//
// Shared pieces of the paged beam cache (include/dbs_cuda_cache.h): the kernel's view of a
// cache, the layout of its plan array, and launch helpers.
//
// The plan is what the state kernels leave for the attention. The beams of an example are taken
// in groups of 32 (a bit each); for every group it lists the distinct pages, in column order:
// one unit per page, with the beams that hold it. A page that 8 beams share is then read once
// for all 8 instead of once each, whatever the pattern of sharing that the search left.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "dbs_cuda.h"
#include "dbs_cuda_cache.h"

namespace dbsb {

constexpr int kGroupBeams = 32;  // beams of a group (bits of a unit's mask)

// A distinct page of a group of beams. limit: -1 when every position of it is committed for all
// its beams; else the committed tokens of the one beam that holds it.
struct __align__(16) CacheUnit {
    int32_t page;
    int32_t start;   // position of its first row
    uint32_t mask;   // beams of the group that hold it
    int32_t limit;
};

struct CacheView {
    int B, K, M, P, L, H, D, page, page_log2;
    int elem;        // bytes of an element
    int groups;      // groups of an example
    int unit_cap;    // units a group has room for
    void* pages;
    int32_t* table;
    int32_t* lengths;
    int32_t* references;
    int32_t* status;
    // plan array
    int32_t* words;       // kWord* below
    int32_t* unit_count;  // [B * groups]
    CacheUnit* units;     // [B * groups, unit_cap]
    int32_t* want_count;  // [S] pages a slot asks for
    int32_t* want_first;  // [S] the first column it asks for, or -1 (cache_state.cu)
    int32_t* want_rank;   // [S] rank of its first new page
    int32_t* copy_from;   // [S] page whose rows the slot copies, or -1
    int32_t* copy_rows;   // [S]
    int4* copies;         // [S] {from, to, rows, slot} of the slots that copy
    int32_t* accepted;    // [S] tokens that a commit accepts
    int32_t* free_list;   // [P] fork: free pages; compact: holes
    int32_t* move_list;   // [P] compact: pages that move, in order of their holes
    int32_t* move_to;     // [P] compact: where a page at or above the live count goes
};

// Words of the plan array.
constexpr int kWordArrive = 0;   // CTAs of a state kernel that are done (zero between calls)
constexpr int kWordCopies = 1;   // entries of copies
constexpr int kWordFree = 2;     // entries of free_list that were handed out
constexpr int kWordLive = 3;     // compact: pages in use
constexpr int kWordMoves = 4;    // compact: entries of move_list
constexpr int kWordOdd = 5;     // refresh: a page that is held has a value that is not finite
constexpr int kWords = 64;

inline int64_t cache_plan_layout(CacheView& v, void* base) {
    const int64_t S = static_cast<int64_t>(v.B) * v.K;
    char* at = static_cast<char*>(base);
    int64_t off = 0;
    auto take = [&](int64_t bytes) {
        char* p = at ? at + off : nullptr;
        off = (off + bytes + 255) / 256 * 256;
        return static_cast<void*>(p);
    };
    v.words = static_cast<int32_t*>(take(kWords * 4));
    v.unit_count = static_cast<int32_t*>(take(static_cast<int64_t>(v.B) * v.groups * 4));
    v.units = static_cast<CacheUnit*>(take(static_cast<int64_t>(v.B) * v.groups * v.unit_cap * sizeof(CacheUnit)));
    int32_t** per_slot[] = {&v.want_count, &v.want_first, &v.want_rank, &v.copy_from, &v.copy_rows, &v.accepted};
    for (int32_t** p : per_slot) *p = static_cast<int32_t*>(take(S * 4));
    v.copies = static_cast<int4*>(take(S * 16));
    int32_t** per_page[] = {&v.free_list, &v.move_list, &v.move_to};
    for (int32_t** p : per_page) *p = static_cast<int32_t*>(take(static_cast<int64_t>(v.P) * 4));
    return off;
}

// Everything an attend call needs beside the cache.
struct AttendParams {
    int layer, beams, N, Hq, G;  // G: query heads per key head
    float scale;
    const void* q;
    const void* k;
    const void* v;
    int64_t qs[4], ks[4], vs[4];
    const uint8_t* mask;
    const int32_t* counts;
    void* out;
    float* lse;
    void* workspace;
    int64_t workspace_bytes;
};

// ---------------------------------------------------------------------------
// Programmatic dependent launch: a kernel launched with launch_after() may start while its
// predecessor in the stream still runs, and waits for its memory at grid_wait().
// ---------------------------------------------------------------------------
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... Params, class... Args>
cudaError_t launch_after(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
                         Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Exclusive prefix sum of v over the block (blockDim.x a multiple of 32, at most 1024 threads);
// sums: 33 ints of shared memory; *total: the sum of all.
__device__ __forceinline__ int block_scan(int v, int* sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += o;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int s = lane < warps ? sums[lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += o;
        }
        sums[lane] = s;
    }
    __syncthreads();
    const int before = warp > 0 ? sums[warp - 1] : 0;
    *total = sums[warps - 1];
    __syncthreads();
    return before + x - v;
}

cudaError_t launch_cache_fork(const CacheView& c, const int32_t* parents, const int32_t* written, int written_all,
                              const int32_t* room, int room_all, int sm_count, cudaStream_t stream);
cudaError_t launch_cache_commit(const CacheView& c, const int32_t* path, int path_stride, const int32_t* counts,
                                int room_all, int sm_count, cudaStream_t stream);
cudaError_t launch_cache_compact(const CacheView& c, int sm_count, cudaStream_t stream);
cudaError_t launch_cache_refresh(const CacheView& c, int dtype, int values, int sm_count, cudaStream_t stream);
// Whether the tiles of all segments of a call (attend.cuh) are counted in 31 bits, were every table full.
bool attend_counts_tiles(const CacheView& c, const AttendParams& a);
int64_t attend_workspace(const CacheView& c, const AttendParams& a, int sm_count);
cudaError_t launch_attend(const CacheView& c, int dtype, const AttendParams& a, int sm_count, cudaStream_t stream);

}  // namespace dbsb
