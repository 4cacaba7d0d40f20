// SPDX-License-Identifier: MIT
//
// State of the paged beam cache: forking beams by their parents, accepting a drafted path,
// compacting the pool (include/dbs_cuda_cache.h gives the rules).
//
// References need no recount. Of the old entry (r, c), a complete page, every child of r keeps a
// reference; of an incomplete or spare page only the first child does, if it needs the column. So
// the entry's page changes by (holders - 1), known from three numbers a beam (children, first
// child, columns the first child needs): one atomic an entry at the most, of integers, so their order
// does not show.
//
// New pages are handed out by the last CTA to finish: one scan of the slots' wishes, one scan of
// the references for zeros that stops as soon as there are enough. Nothing else is serial.
#include <climits>

#include "cache.cuh"

namespace dbsb {

namespace {

constexpr int kMetaThreads = 512;
constexpr int kStageInts = 8192;  // table entries of an example staged at a time
constexpr int kCopyThreads = 256;

struct ForkArgs {
    const int32_t* parents;
    const int32_t* written;
    const int32_t* room;
    int written_all, room_all;
};

__device__ __forceinline__ void raise(const CacheView& c, int bit) { atomicOr(c.status, bit); }

// The last CTA of fork_meta_kernel: ranks of the wishes, free pages for them, the copy list.
__device__ void hand_out(const CacheView& c, int* sums) {
    const int S = c.B * c.K, tid = threadIdx.x;
    // The first references are on their way while the wishes are counted.
    auto zeros_at = [&](int at) {  // a bit each
        unsigned zero = 0;
        if (at + 16 <= c.P) {
            int4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __ldcg(reinterpret_cast<const int4*>(c.references + at) + i);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                zero |= ((v[i].x == 0) | (v[i].y == 0) << 1 | (v[i].z == 0) << 2 | (v[i].w == 0) << 3) << (4 * i);
        } else {
            for (int i = 0; i < 16 && at + i < c.P; ++i) zero |= (__ldcg(c.references + at + i) == 0) << i;
        }
        return zero;
    };
    unsigned zero = zeros_at(tid * 16);
    int wanted = 0;
    for (int base = 0; base < S; base += kMetaThreads) {
        const int s = base + tid;
        const int n = s < S ? __ldcg(c.want_count + s) : 0;
        int total;
        const int before = block_scan(n, sums, &total);
        if (s < S) c.want_rank[s] = wanted + before;
        wanted += total;
    }
    // Zeros of the references, 16 a thread and round.
    int found = 0;
    for (int base = 0; base < c.P && found < wanted; base += kMetaThreads * 16) {
        if (base > 0) zero = zeros_at(base + tid * 16);
        int total;
        int rank = found + block_scan(__popc(zero), sums, &total);
        for (; zero != 0 && rank < wanted; zero &= zero - 1, ++rank) {
            const int p = base + tid * 16 + __ffs(zero) - 1;
            c.free_list[rank] = p;
            c.references[p] = 1;
        }
        found += total;
    }
    const int handed = found < wanted ? found : wanted;
    __syncthreads();
    // A slot that copies takes its first new page for the rows.
    int copies = 0;
    for (int base = 0; base < S; base += kMetaThreads) {
        const int s = base + tid;
        const int rows = s < S ? __ldcg(c.copy_rows + s) : 0;
        const int rank = rows > 0 ? c.want_rank[s] : 0;
        const bool copy = rows > 0 && rank < handed;
        int total;
        const int at = copies + block_scan(copy, sums, &total);
        if (copy) c.copies[at] = make_int4(__ldcg(c.copy_from + s), c.free_list[rank], rows, s);
        copies += total;
    }
    if (tid == 0) {
        c.words[kWordCopies] = copies;
        c.words[kWordFree] = handed;
        c.words[kWordArrive] = 0;
        if (found < wanted) raise(c, DBS_CUDA_CACHE_STATUS_POOL);
    }
}

// One CTA an example. Entries that ask for a new page become -2 until cache_finish_kernel, which finds a slot's
// new pages by the columns from the first such one on. Where pages that the slot keeps lie between them (a table
// that a caller wrote), its first column is noted as -1 and the entries are -2 less their number.
__global__ void __launch_bounds__(kMetaThreads) fork_meta_kernel(CacheView c, ForkArgs a) {
    extern __shared__ int32_t smem[];
    __shared__ int sums[33];
    __shared__ int last;
    const int K = c.K, M = c.M, b = blockIdx.x, tid = threadIdx.x, log2 = c.page_log2;
    int32_t* length = smem;         // [K] committed tokens of each beam, with the written ones
    int32_t* children = length + K; // [K]
    int32_t* first = children + K;  // [K] first child or INT_MAX
    int32_t* src = first + K;       // [K] parent of each new beam or -1
    int32_t* need = src + K;        // [K] columns of each new beam
    int32_t* want = need + K;       // [K] new pages it asks for
    int32_t* want_at = want + K;    // [K] the first such column
    int32_t* copied = want_at + K;  // [K] page whose rows it copies or -1
    int32_t* stage = copied + K;    // [K, width]
    const int64_t slot0 = static_cast<int64_t>(b) * K;
    grid_wait();   // what ran before may have written the parents
    grid_release();
    const int width = K * M <= kStageInts ? M : (kStageInts / K > 1 ? kStageInts / K : 1);
    int32_t* table = c.table + slot0 * M;
    auto load_stage = [&](int base, int cols) {
        for (int i = tid; i < K * cols; i += kMetaThreads) {
            const int r = i / cols;
            stage[r * width + i - r * cols] = table[static_cast<int64_t>(r) * M + base + i - r * cols];
        }
    };
    // All that is read is asked for at once.
    for (int k = tid; k < K; k += kMetaThreads) {
        int64_t w = a.written ? a.written[slot0 + k] : a.written_all;
        int64_t m = a.room ? a.room[slot0 + k] : a.room_all;
        const int old = c.lengths[slot0 + k], p = a.parents ? a.parents[slot0 + k] : k;
        if (w < 0 || (p >= 0 && m < 0) || p >= K) raise(c, DBS_CUDA_CACHE_STATUS_INDEX);
        if (w < 0) w = 0;
        const int64_t most = static_cast<int64_t>(M) << log2;
        int64_t n = old + w;
        if (n > most) {
            raise(c, DBS_CUDA_CACHE_STATUS_CAPACITY);
            n = most;
        }
        length[k] = static_cast<int32_t>(n < 0 ? 0 : n);
        src[k] = p < 0 || p >= K ? -1 : p;
        need[k] = static_cast<int>(m < 0 ? 0 : m);  // the room, until the lengths are known
        children[k] = 0;
        first[k] = INT_MAX;
        want[k] = 0;
        want_at[k] = INT_MAX;
        copied[k] = -1;
    }
    load_stage(0, M < width ? M : width);
    __syncthreads();
    for (int k = tid; k < K; k += kMetaThreads) {
        const int p = src[k];
        int columns = 0;
        if (p >= 0) {
            atomicAdd(&children[p], 1);
            atomicMin(&first[p], k);
            const int64_t n = (static_cast<int64_t>(length[p]) + need[k] + c.page - 1) >> log2;
            if (n > M) raise(c, DBS_CUDA_CACHE_STATUS_CAPACITY);
            columns = static_cast<int>(n > M ? M : n);
        }
        need[k] = columns;
    }
    __syncthreads();
    for (int base = 0; base < M; base += width) {
        const int cols = M - base < width ? M - base : width;
        if (base > 0) {
            load_stage(base, cols);
            __syncthreads();
        }
        for (int i = tid; i < K * cols; i += kMetaThreads) {
            const int r = i / cols, at = i - r * cols, col = base + at;
            const int old = stage[r * width + at];
            if (old >= 0) {  // as the entry of the old beam r
                const int heir = first[r];
                const int holders = col < (length[r] >> log2) ? children[r] : (heir < K && col < need[heir]);
                if (holders != 1) atomicAdd(c.references + old, holders - 1);
            }
            const int p = src[r];  // as the entry of the new beam r
            int e = -1;
            if (p >= 0 && col < need[r]) {
                const int held = stage[p * width + at], full = length[p] >> log2;
                if (col < full || first[p] == r) e = held;
                if (col >= full && e < 0) {
                    e = -2;
                    atomicAdd(&want[r], 1);
                    atomicMin(&want_at[r], col);
                }
                if (col == full && first[p] != r && (length[p] & (c.page - 1)) != 0) copied[r] = held;
            }
            if (e != old) table[static_cast<int64_t>(r) * M + col] = e;
        }
        __syncthreads();
    }
    for (int r = tid >> 5; r < K; r += kMetaThreads / 32) {
        const int from = want_at[r], to = need[r], lane = tid & 31;
        if (want[r] == 0 || want[r] == to - from) continue;
        int32_t* row = table + static_cast<int64_t>(r) * M;
        int before = 0;
        for (int base = from; base < to; base += 32) {
            const bool asks = base + lane < to && row[base + lane] == -2;
            const unsigned all = __ballot_sync(0xffffffffu, asks);
            if (asks) row[base + lane] = -2 - (before + __popc(all & ((1u << lane) - 1)));
            before += __popc(all);
        }
        if (lane == 0) want_at[r] = -1;
    }
    __syncthreads();
    for (int s = tid; s < K; s += kMetaThreads) {
        const int p = src[s];
        c.lengths[slot0 + s] = p >= 0 ? length[p] : 0;
        c.want_count[slot0 + s] = want[s];
        c.want_first[slot0 + s] = want_at[s];
        c.copy_from[slot0 + s] = copied[s];
        c.copy_rows[slot0 + s] = copied[s] >= 0 ? length[p] & (c.page - 1) : 0;
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(c.words + kWordArrive, 1) == c.B - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    hand_out(c, sums);
}

// The units of a group of beams, from its final table rows (column order, then first beam).
// resolve: entries below -1 take their slot's new pages first. A warp takes a column at a time, a lane a
// beam: the lanes with one page find each other in one instruction.
constexpr int kPlanPitch = kCopyThreads + 1;  // of a beam's staged columns: a column's lie in different banks

__device__ void write_plan(const CacheView& c, int group, bool resolve, int* sums, int32_t* shared) {
    const int b = group / c.groups, k0 = (group - b * c.groups) * kGroupBeams;
    const int n = c.K - k0 < kGroupBeams ? c.K - k0 : kGroupBeams;
    const int64_t slot0 = static_cast<int64_t>(b) * c.K + k0;
    int32_t* table = c.table + slot0 * c.M;
    CacheUnit* units = c.units + static_cast<int64_t>(group) * c.unit_cap;
    int32_t* length = shared;                   // [32]
    int32_t* rank = shared + kGroupBeams;       // [32] rank of the first new page
    int32_t* from = shared + 2 * kGroupBeams;   // [32] its column, or -1
    int32_t* place = shared + 3 * kGroupBeams;  // [columns] units of each, then the first one's number
    int32_t* stage = place + kCopyThreads;      // [n][kPlanPitch]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < n) {
        length[tid] = c.lengths[slot0 + tid];
        rank[tid] = resolve ? c.want_rank[slot0 + tid] : 0;
        from[tid] = resolve ? c.want_first[slot0 + tid] : 0;
    }
    const int handed = resolve ? c.words[kWordFree] : 0;
    __syncthreads();
    int count = 0;
    for (int base = 0; base < c.M; base += kCopyThreads) {
        const int cols = c.M - base < kCopyThreads ? c.M - base : kCopyThreads;
        for (int i = tid; i < n * cols; i += kCopyThreads) {
            const int k = i / cols, at = i - k * cols, col = base + at;
            int e = table[static_cast<int64_t>(k) * c.M + col];
            if (resolve && e < -1) {
                const int new_page = rank[k] + (from[k] < 0 ? -2 - e : col - from[k]);
                e = new_page < handed ? c.free_list[new_page] : -1;
                table[static_cast<int64_t>(k) * c.M + col] = e;
            }
            stage[k * kPlanPitch + at] = e;
        }
        __syncthreads();
        // Lanes without a page get numbers that no other lane has.
        auto holders_of = [&](int at, int* page) {
            const int e = lane < n ? stage[lane * kPlanPitch + at] : -1;
            *page = e;
            return __match_any_sync(0xffffffffu, e >= 0 ? e : -1 - lane);
        };
        for (int at = warp; at < cols; at += kCopyThreads / 32) {
            int e;
            const unsigned holders = holders_of(at, &e);
            const unsigned firsts = __ballot_sync(0xffffffffu, e >= 0 && __ffs(holders) - 1 == lane);
            if (lane == 0) place[at] = __popc(firsts);
        }
        __syncthreads();
        int total;
        const int at_first = count + block_scan(tid < cols ? place[tid] : 0, sums, &total);
        if (tid < cols) place[tid] = at_first;
        __syncthreads();
        for (int at = warp; at < cols; at += kCopyThreads / 32) {
            int e;
            const unsigned holders = holders_of(at, &e);
            const int end = (base + at + 1) << c.page_log2;
            const unsigned whole = __ballot_sync(0xffffffffu, lane < n && end <= length[lane]);
            const bool first = e >= 0 && __ffs(holders) - 1 == lane, complete = (holders & ~whole) == 0;
            const unsigned firsts = __ballot_sync(0xffffffffu, first);
            if (first) {
                units[place[at] + __popc(firsts & ((1u << lane) - 1))] =
                    CacheUnit{e, (base + at) << c.page_log2, holders, complete ? -1 : length[lane]};
                // (Other holders may be beams of another group or example, or another column.)
                if (!complete && __ldcg(c.references + e) > 1) raise(c, DBS_CUDA_CACHE_STATUS_SHARED);
            }
        }
        count += total;
        __syncthreads();
    }
    if (tid == 0) c.unit_count[group] = count;
}

constexpr size_t plan_smem() { return (3 * kGroupBeams + kCopyThreads + kGroupBeams * kPlanPitch) * sizeof(int32_t); }

// After fork_meta_kernel: the plan and the new pages of the table (one CTA a group), and the
// copies of incomplete pages (the other CTAs; a warp takes the rows of one layer, kind and head,
// which are contiguous).
__global__ void __launch_bounds__(kCopyThreads) cache_finish_kernel(CacheView c, int plan_blocks) {
    extern __shared__ int32_t smem[];
    __shared__ int sums[33];
    grid_wait();
    if (static_cast<int>(blockIdx.x) < plan_blocks) {
        write_plan(c, blockIdx.x, true, sums, smem);
        return;
    }
    const int copies = c.words[kWordCopies];
    const int per = c.L * 2 * c.H;
    const int64_t items = static_cast<int64_t>(copies) * per;
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x - plan_blocks) * (kCopyThreads / 32);
    const int row_vecs = c.D * c.elem / 16;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - plan_blocks) * (kCopyThreads / 32) + (threadIdx.x >> 5);
         i < items; i += warps) {
        const int which = static_cast<int>(i / per), part = static_cast<int>(i - static_cast<int64_t>(which) * per);
        const int4 copy = __ldg(c.copies + which);
        const int64_t block = part / c.H, head = part - block * c.H;  // block: layer * 2 + kind
        const int64_t vecs = static_cast<int64_t>(c.page) * row_vecs;
        const uint4* x = static_cast<const uint4*>(c.pages) + ((block * c.P + copy.x) * c.H + head) * vecs;
        uint4* y = static_cast<uint4*>(c.pages) + ((block * c.P + copy.y) * c.H + head) * vecs;
        const int n = copy.z * row_vecs;
        int v = lane;
        for (; v + 7 * 32 < n; v += 8 * 32) {
            uint4 t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = x[v + 32 * j];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[v + 32 * j] = t[j];
        }
        for (; v < n; v += 32) y[v] = x[v];
    }
}

// Rows of an accepted path to the front of the drafted area. A CTA takes one slot and a part of its
// layers, kinds and heads. The whole path is looked at before a row moves: one that does not rise, or names a
// token without a page, is refused as a whole (0 accepted, for the fork behind this). A thread owns 16 bytes
// of every row of one layer, kind and head, and moves eight rows a round: row path[a] >= a lies at or behind
// every row that earlier rounds wrote, and a round reads all its rows before it writes.
constexpr int kMoveRows = kCopyThreads;  // accepted rows whose places are looked up at a time

__global__ void __launch_bounds__(kCopyThreads) commit_move_kernel(CacheView c, const int32_t* path, int path_stride,
                                                                   const int32_t* counts, int parts) {
    __shared__ int2 moves[kMoveRows];  // row numbers of a layer, kind and head (page * H * page_size + row), -1: none
    __shared__ int bad;
    grid_wait();
    grid_release();
    const int slot = blockIdx.x / parts, piece = blockIdx.x - slot * parts, tid = threadIdx.x;
    const int row_vecs = c.D * c.elem / 16;
    int count = counts[slot];
    const int n = c.lengths[slot];
    const int32_t* row = c.table + static_cast<int64_t>(slot) * c.M;
    const int32_t* steps = path + static_cast<int64_t>(slot) * path_stride;
    const bool empty = n <= 0 && row[0] < 0;  // no tokens, no pages: nothing of this beam was drafted
    if (tid == 0) bad = !empty && (count < 0 || count > path_stride);
    if (empty || count > path_stride) count = 0;
    __syncthreads();
    // The move of entry a; (all threads with a bad one store 1).
    auto look = [&](int a) {
        const int from = steps[a], before = a > 0 ? steps[a - 1] : -1;
        const int64_t at = static_cast<int64_t>(n) + from, to = static_cast<int64_t>(n) + a;
        int p = -1, q = -1;
        if (from > before && from >= a && (at >> c.page_log2) < c.M) p = row[at >> c.page_log2], q = row[to >> c.page_log2];
        if (p < 0 || q < 0) bad = 1;
        if (p < 0 || q < 0 || from == a) return make_int2(-1, -1);
        return make_int2(p * c.H * c.page + static_cast<int>(at & (c.page - 1)), q * c.H * c.page + static_cast<int>(to & (c.page - 1)));
    };
    for (int a = tid; a < count; a += kMoveRows) {
        const int2 m = look(a);
        if (a < kMoveRows) moves[a] = m;
    }
    __syncthreads();
    const bool refused = bad != 0;
    if (tid == 0 && piece == 0) {
        c.accepted[slot] = refused ? 0 : count;
        if (refused) raise(c, DBS_CUDA_CACHE_STATUS_INDEX);
    }
    if (refused) return;
    const int items = c.L * 2 * c.H * row_vecs;
    for (int base = 0; base < count; base += kMoveRows) {
        if (base > 0) {
            __syncthreads();
            if (base + tid < count) moves[tid] = look(base + tid);
            __syncthreads();
        }
        const int rows = count - base < kMoveRows ? count - base : kMoveRows;
        for (int i = piece * kCopyThreads + tid; i < items; i += parts * kCopyThreads) {
            const int part = i / row_vecs, vec = i - part * row_vecs, block = part / c.H, head = part - block * c.H;
            uint4* pages = static_cast<uint4*>(c.pages) + vec +
                           (static_cast<int64_t>(block) * c.P * c.H + head) * c.page * row_vecs;
            for (int a0 = 0; a0 < rows; a0 += 8) {
                uint4 t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (a0 + j < rows && moves[a0 + j].x >= 0) t[j] = pages[static_cast<int64_t>(moves[a0 + j].x) * row_vecs];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (a0 + j < rows && moves[a0 + j].x >= 0) pages[static_cast<int64_t>(moves[a0 + j].y) * row_vecs] = t[j];
            }
        }
    }
}

// Ranks of holes and movers from one prefix count of the pages in use: with n in use, hole h < n
// has rank h - live_before(h), mover m >= n rank live_before(m) - live_before(n).
__global__ void __launch_bounds__(1024) compact_meta_kernel(CacheView c) {
    __shared__ int sums[33];
    __shared__ int below;
    grid_wait();
    grid_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int span = (c.P + 32 * 32 - 1) / (32 * 32) * 32;  // pages of a warp
    const int lo = warp * span, hi = lo + span < c.P ? lo + span : c.P;
    int mine = 0;
    for (int p = lo + lane; p < hi; p += 32) mine += c.references[p] > 0;
    for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    int n;
    const int scanned = block_scan(lane == 0 ? mine : 0, sums, &n);
    const int before = __shfl_sync(0xffffffffu, scanned, 0);
    if (tid == 0) below = n;  // when every live page is below n already
    __syncthreads();
    auto walk = [&](auto&& visit) {
        int live = before;
        for (int base = lo; base < hi; base += 32) {
            const int p = base + lane;
            const int refs = p < hi ? c.references[p] : 0;
            const unsigned bits = __ballot_sync(0xffffffffu, refs > 0);
            if (p < hi) visit(p, refs, live + __popc(bits & ((1u << lane) - 1)));
            live += __popc(bits);
        }
    };
    if (lo <= n && n < hi) walk([&](int p, int, int rank) {
        if (p == n) below = rank;
    });
    __syncthreads();
    walk([&](int p, int refs, int rank) {
        if (p < n && refs <= 0) c.free_list[p - rank] = p;
        if (p >= n && refs > 0) c.move_list[rank - below] = p;
    });
    __threadfence_block();
    __syncthreads();
    const int moves = n - below;
    for (int i = tid; i < moves; i += 1024) {
        const int from = c.move_list[i], to = c.free_list[i];
        c.move_to[from] = to;
        c.references[to] = c.references[from];
        c.references[from] = 0;
    }
    if (tid == 0) {
        c.words[kWordLive] = n;
        c.words[kWordMoves] = moves;
    }
}

// The moves (a CTA takes 16 KB of a page's block of one layer and kind at a time), and the new
// page numbers in table and plan.
__global__ void __launch_bounds__(kCopyThreads) compact_move_kernel(CacheView c) {
    grid_wait();
    const int n = c.words[kWordLive], moves = c.words[kWordMoves];
    if (moves == 0) return;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kCopyThreads;
    const int64_t entries = static_cast<int64_t>(c.B) * c.K * c.M;
    for (int64_t i = first; i < entries; i += step) {
        const int p = c.table[i];
        if (p >= n) c.table[i] = c.move_to[p];
    }
    const int64_t units = static_cast<int64_t>(c.B) * c.groups * c.unit_cap;
    for (int64_t i = first; i < units; i += step) {
        const int64_t group = i / c.unit_cap;
        if (i - group * c.unit_cap >= c.unit_count[group]) continue;
        const int p = c.units[i].page;
        if (p >= n) c.units[i].page = c.move_to[p];
    }
    const int64_t vecs = static_cast<int64_t>(c.H) * c.page * c.D * c.elem / 16;  // of a block
    constexpr int kPiece = kCopyThreads * 4;
    const int64_t pieces = (vecs + kPiece - 1) / kPiece;
    const int64_t items = static_cast<int64_t>(moves) * c.L * 2 * pieces;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const int64_t piece = i % pieces, rest = i / pieces;
        const int64_t block = rest % (c.L * 2), move = rest / (c.L * 2);
        const uint4* x = static_cast<const uint4*>(c.pages) + (block * c.P + c.move_list[move]) * vecs;
        uint4* y = static_cast<uint4*>(c.pages) + (block * c.P + c.free_list[move]) * vecs;
        const int64_t at = piece * kPiece + threadIdx.x;
        uint4 t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j * kCopyThreads < vecs) t[j] = x[at + j * kCopyThreads];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j * kCopyThreads < vecs) y[at + j * kCopyThreads] = t[j];
    }
}

// Table entries and lengths that are out of range never reach an index: the entries become -1, the lengths the
// nearest one that the table has room for.
__global__ void refresh_count_kernel(CacheView c) {
    const int64_t slots = static_cast<int64_t>(c.B) * c.K;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < slots;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int n = c.lengths[i], most = c.M << c.page_log2;
        if (n < 0 || n > most) {
            raise(c, DBS_CUDA_CACHE_STATUS_INDEX);
            c.lengths[i] = n < 0 ? 0 : most;
        }
    }
    const int64_t entries = static_cast<int64_t>(c.B) * c.K * c.M;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < entries;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int p = c.table[i];
        if (p >= c.P || p < -1) {
            raise(c, DBS_CUDA_CACHE_STATUS_INDEX);
            c.table[i] = -1;
        } else if (p >= 0) {
            atomicAdd(c.references + p, 1);
        }
    }
}

__global__ void __launch_bounds__(kCopyThreads) refresh_plan_kernel(CacheView c) {
    extern __shared__ int32_t smem[];
    __shared__ int sums[33];
    write_plan(c, blockIdx.x, false, sums, smem);
}

// Whether the values of the pool hold one that is not finite (exponent bits all set). In pages that nobody
// holds such values mean nothing and become 0: the pages may be handed out again. if_set: only where
// status[1] says that there may be some.
__global__ void refresh_values_kernel(CacheView c, uint32_t exponent_lo, uint32_t exponent_hi, bool if_set) {
    if (if_set && c.status[1] == 0) return;
    const int64_t each = static_cast<int64_t>(c.H) * c.page * c.D * c.elem / 16, vecs = c.P * each;  // of a page; of a layer and kind
    bool odd = false;
    for (int layer = 0; layer < c.L; ++layer) {
        uint4* x = static_cast<uint4*>(c.pages) + (2 * layer + 1) * vecs;
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < vecs;
             i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
            const uint4 v = x[i];
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            bool here = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool lo = (w[j] & exponent_lo) == exponent_lo, hi = (w[j] & exponent_hi) == exponent_hi;
                here |= lo || hi;
                if (exponent_lo == exponent_hi ? lo : lo && hi) w[j] = 0;  // float32: one element
                else if (lo) w[j] &= 0xffff0000u;
                else if (hi) w[j] &= 0x0000ffffu;
            }
            if (!here) continue;
            if (c.references[i / each] == 0) x[i] = make_uint4(w[0], w[1], w[2], w[3]);
            else odd = true;
        }
    }
    if (odd) c.words[kWordOdd] = 1;
}

size_t meta_smem(const CacheView& c) {
    const int64_t all = static_cast<int64_t>(c.K) * c.M;
    const int64_t stage = all <= kStageInts ? all : (c.K > kStageInts ? c.K : kStageInts);
    return (8 * static_cast<size_t>(c.K) + stage) * sizeof(int32_t);
}

unsigned copy_blocks(int64_t work, int sm_count) {
    const int64_t cap = static_cast<int64_t>(sm_count) * 8;
    return static_cast<unsigned>(work < 1 ? 1 : (work < cap ? work : cap));
}

}  // namespace

cudaError_t launch_cache_fork(const CacheView& c, const int32_t* parents, const int32_t* written, int written_all,
                              const int32_t* room, int room_all, int sm_count, cudaStream_t stream) {
    const size_t smem = meta_smem(c);
    cudaError_t e = cudaSuccess;
    if (smem > 47 * 1024)  // (and some static shared memory)
        e = cudaFuncSetAttribute(fork_meta_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    const ForkArgs a{parents, written, room, written_all, room_all};
    e = launch_after(fork_meta_kernel, c.B, kMetaThreads, smem, stream, c, a);
    if (e != cudaSuccess) return e;
    const int plan_blocks = c.B * c.groups;
    // Without parents every beam is its own first child: nothing is copied.
    const int64_t parts = parents ? static_cast<int64_t>(c.B) * c.K * c.L * 2 * c.H / (kCopyThreads / 32) : 0;
    const unsigned blocks = plan_blocks + (parts > 0 || parents ? copy_blocks(parts, sm_count) : 0);
    return launch_after(cache_finish_kernel, blocks, kCopyThreads, plan_smem(), stream, c, plan_blocks);
}

cudaError_t launch_cache_commit(const CacheView& c, const int32_t* path, int path_stride, const int32_t* counts,
                                int room_all, int sm_count, cudaStream_t stream) {
    // Two rounds of a CTA's threads, or so many CTAs that all SMs have some.
    const int64_t slots = static_cast<int64_t>(c.B) * c.K, items = static_cast<int64_t>(c.L) * 2 * c.H * (c.D * c.elem / 16);
    int64_t parts = (items + 2 * kCopyThreads - 1) / (2 * kCopyThreads);
    const int64_t cap = slots * 2 > sm_count * 8 ? 2 : sm_count * 8 / slots;
    if (parts > cap) parts = cap;
    const cudaError_t e = launch_after(commit_move_kernel, static_cast<unsigned>(slots * parts), kCopyThreads, 0, stream, c,
                                       path, path_stride, counts, static_cast<int>(parts));
    if (e != cudaSuccess) return e;
    return launch_cache_fork(c, nullptr, c.accepted, 0, nullptr, room_all, sm_count, stream);
}

cudaError_t launch_cache_compact(const CacheView& c, int sm_count, cudaStream_t stream) {
    const cudaError_t e = launch_after(compact_meta_kernel, 1, 1024, 0, stream, c);
    if (e != cudaSuccess) return e;
    const int64_t most = static_cast<int64_t>(c.P) * c.L * 2 * c.H * c.page * c.D * c.elem / 16 / (kCopyThreads * 4);
    return launch_after(compact_move_kernel, copy_blocks(most, sm_count), kCopyThreads, 0, stream, c);
}

cudaError_t launch_cache_refresh(const CacheView& c, int dtype, int values, int sm_count, cudaStream_t stream) {
    cudaError_t e = cudaMemsetAsync(c.references, 0, static_cast<size_t>(c.P) * 4, stream);
    if (e != cudaSuccess) return e;
    const int64_t entries = static_cast<int64_t>(c.B) * c.K * c.M;
    refresh_count_kernel<<<copy_blocks((entries + 255) / 256, sm_count), 256, 0, stream>>>(c);
    refresh_plan_kernel<<<c.B * c.groups, kCopyThreads, plan_smem(), stream>>>(c);
    if (values != 0) {
        e = cudaMemsetAsync(c.words + kWordOdd, 0, 4, stream);
        if (e != cudaSuccess) return e;
        const uint32_t exponent = dtype == DBS_CUDA_DTYPE_F16 ? 0x7c00u : 0x7f80u;
        const uint32_t lo = dtype == DBS_CUDA_DTYPE_F32 ? exponent << 16 : exponent;
        refresh_values_kernel<<<sm_count * 8, 256, 0, stream>>>(c, lo, exponent << 16, values == DBS_CUDA_CACHE_VALUES_IF_SET);
        e = cudaMemcpyAsync(c.status + 1, c.words + kWordOdd, 4, cudaMemcpyDeviceToDevice, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaGetLastError();
}

}  // namespace dbsb
