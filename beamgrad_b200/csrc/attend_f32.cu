// SPDX-License-Identifier: MIT
//
// Attention over the paged cache in float32, on the multiply-add pipe: the tensor cores would round
// the operands to 11 bits.
//
// Blocks of 16, 32 or 64 query rows by tiles of 64 positions (32 for heads above 128), copied by
// cp.async, the next tile while this one is worked on. Scores run on register tiles of 4 x 4 (of
// float4 along the head), outputs on 1, 2 or 4 rows by a float4: laid over a warp so that the eight
// shared-memory reads of 16 bytes for 64 multiply-adds take 8 (12) passes of the banks: rows are
// padded by 16 bytes, and rows of one read lie next to each other. At 32 rows of 128 the multiply-adds
// take 4096 cycles a tile and SM, at 16 rows the bytes bound it (2800 cycles). 64 rows have 16 warps,
// which hide each other's reads (165 rows over 14421: 331 us, with blocks of 32 and 8 warps 373; with
// the join as it is now 318); with fewer rows 8 warps of larger tiles do better (32 rows over 16000: 184 us
// against 214, now 179: 39 % of the multiply-add pipe).
#include "attend.cuh"

namespace dbsb {

namespace {

constexpr int threads_of(int rows) { return rows > 32 ? 512 : 256; }

template <int DP, int ROWS>
struct Shape {
    static constexpr int kRows = ROWS, kThreads = threads_of(ROWS), kWarps = kThreads / 32;
    static constexpr int kKeys = DP > 128 ? 32 : 64;
    static constexpr int kPitch = DP + 4;              // floats of a staged row
    static constexpr int kStage = 2 * kKeys * kPitch;  // floats: keys, values
    // Scores: a warp has 16 rows by 32 positions of one part of the head.
    static constexpr int kRowWarps = kRows / 16, kKeyWarps = kKeys / 32;
    static constexpr int kSplit = kWarps / (kRowWarps * kKeyWarps);
    static constexpr int kScorePitch = kKeys + 4;
    static constexpr int kScores = kRows * kScorePitch;
    // Output: half the warps by 2; a thread has kOwn rows and, of every 32 groups of four columns, one.
    static constexpr int kOwn = kRows / kWarps;
    static constexpr int kCols = DP / 128;
    static constexpr int kBytes = (2 * kStage + kSplit * kScores + kRows * kPitch) * 4;
    static constexpr int kOut = kRows * (DP + 2);
    static constexpr bool kMany = kRows == 64 || (DP > 128 && kRows == 32);  // the most that a block has
};

struct Control {
    int sums[35];
    WorkSplit split;
    CacheUnit unit[2][4];
    int64_t row_at[2][64];  // of the tile's positions: the row's element among the pages of a layer's keys
    int64_t query_at[64];
    float factor[64], top[64], sum[64];
    int last;
};

__device__ __forceinline__ void copy16(float* to, const float* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_address(to)), "l"(from) : "memory");
}

template <int DP, int ROWS>
__global__ void __launch_bounds__(threads_of(ROWS), 1)
attend_f32_kernel(const __grid_constant__ CacheView c, const __grid_constant__ AttendParams a) {
    using S = Shape<DP, ROWS>;
    constexpr int kThreads = S::kThreads;
    extern __shared__ __align__(16) float smem[];
    __shared__ Control ctl;
    float* stages = smem;
    float* scores = stages + 2 * S::kStage;          // [kSplit][kRows][kScorePitch]; the weights in the first
    float* query = scores + S::kSplit * S::kScores;  // [kRows][kPitch]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile_units = S::kKeys >> c.page_log2 > 0 ? S::kKeys >> c.page_log2 : 1;
    const int page_tiles = c.page > S::kKeys ? c.page / S::kKeys : 1;  // tiles of a page (64 by tiles of 32)

    // This kernel may run while the new tokens are still being written. Plan, lengths, queries and complete
    // pages were there before that began; the first copy from a page that is not complete waits for it.
    if (a.k == nullptr) grid_wait();
    grid_release();
    // (No tile more a CTA for whole segments: 32 drafted tokens over 2000 took 174 us for 157.)
    const WorkSplit work = split_work<S::kRows, S::kMany>(c, a, tile_units, 1, 0, ctl.sums, &ctl.split, blockIdx.x, gridDim.x);
    bool waited = a.k == nullptr, odd = false, odd_known = false;  // odd: a value that is not finite was met, now or before
    int group = work.group;
    int64_t base = work.base;
    const float scale = a.scale * kLog2e;
    const int vecs = c.D / 4;
    // Scores: a thread has rows 4 apart and positions 8 apart.
    const int part = warp / (S::kRowWarps * S::kKeyWarps);
    const int s_row = warp % S::kRowWarps * 16 + (lane >> 3), s_key = warp / S::kRowWarps % S::kKeyWarps * 32 + (lane & 7);
    // Weights: kPerRow threads a row. Output: rows 2 apart.
    constexpr int kPerRow = kThreads / S::kRows, kEach = S::kKeys / kPerRow, kOwn = S::kOwn;
    const int w_row = tid / kPerRow, w_key = tid % kPerRow;
    const int o_row = warp % (S::kWarps / 2) * 2 * kOwn + (lane >> 4), o_col = warp / (S::kWarps / 2) * 16 + (lane & 15);
    constexpr int kColStep = 32;
    const int64_t kind_step = static_cast<int64_t>(c.P) * c.H * c.page * c.D;
    const float* pages = static_cast<const float*>(c.pages) + static_cast<int64_t>(a.layer) * 2 * kind_step;

    for (int64_t cur = work.lo; cur < work.hi;) {
        const Piece p = piece_at<S::kRows, S::kMany>(c, a, work, cur, group, base, tile_units);
        const int n_tiles = (p.t1 - p.t0) * page_tiles;
        cur += p.t1 - p.t0;
        const int b = p.group / c.groups, beam0 = (p.group - b * c.groups) * kGroupBeams;
        const int row0 = p.block * S::kRows;
        const int rows = p.rows - row0 < S::kRows ? p.rows - row0 : S::kRows;
        const CacheUnit* units = c.units + static_cast<int64_t>(p.group) * c.unit_cap;
        __syncthreads();
        if (tid < rows) {
            const RowId id = row_id(a, row0 + tid);
            ctl.query_at[tid] = b * a.qs[0] + (beam0 + id.beam) * a.qs[1] + id.token * a.qs[2] + (p.head * a.G + id.head) * a.qs[3];
        }
        __syncthreads();
        for (int i = tid; i < S::kRows * (DP / 4); i += kThreads) {
            const int r = i / (DP / 4), v = i % (DP / 4);
            float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < rows && v < vecs) q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + ctl.query_at[r]) + v);
            *reinterpret_cast<float4*>(query + r * S::kPitch + v * 4) = q;
        }
        SeenTiles seen = seen_tiles<S::kRows>(c, a, p, tile_units, page_tiles);
        // Where the rows of tile t lie: kKeys positions of its units' pages; past the last unit page 0,
        // whatever finite values lie there meet weights of zero.
        auto find = [&](int t, int slot) {
            if (tid >= S::kKeys || t >= n_tiles) return;
            const int first = (p.t0 + t / page_tiles) * tile_units, offset = t % page_tiles * S::kKeys;
            const int unit = first + (tid >> c.page_log2);
            int4 v = make_int4(0, 0, 0, -1);  // no beam holds it
            if (unit < p.units) v = __ldg(reinterpret_cast<const int4*>(units + unit));
            ctl.row_at[slot][tid] = (((static_cast<int64_t>(v.x) * c.H + p.head) << c.page_log2) + ((tid + offset) & (c.page - 1))) * c.D;
            if ((tid & (c.page - 1)) == 0)
                ctl.unit[slot][tid >> c.page_log2] = CacheUnit{v.x, v.y + offset, static_cast<uint32_t>(v.z), v.w};
        };
        auto fetch = [&](int slot) {
            constexpr int kChunks = DP / 4, kAtOnce = kThreads / kChunks;
            float* stage = stages + slot * S::kStage;
            const int v = tid % kChunks, first = tid / kChunks;
            for (int i = 0; !waited && i < tile_units; ++i) {
                if (ctl.unit[slot][i].limit < 0) continue;
                grid_wait();
                waited = true;
            }
            if (v < vecs) {
#pragma unroll
                for (int j = 0; j < S::kKeys / kAtOnce; ++j) {
                    const int key = first + j * kAtOnce;
                    const float* from = pages + ctl.row_at[slot][key] + v * 4;
                    copy16(stage + key * S::kPitch + v * 4, from);
                    copy16(stage + (S::kKeys + key) * S::kPitch + v * 4, from + kind_step);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // The row that this thread weighs.
        RowId id{0, 0, 0};
        if (w_row < rows) id = row_id(a, row0 + w_row);
        const int64_t bk = static_cast<int64_t>(b) * a.beams + beam0 + id.beam;
        const int count = w_row < rows ? new_count(a, bk) : 0;
        const bool live = w_row < rows && id.token < count;
        const uint32_t bit = live ? 1u << id.beam : 0u;
        const uint8_t* fresh = a.mask ? a.mask + (bk * a.N + id.token) * a.N : nullptr;
        float top = -INFINITY, sum = 0.0f;
        float4 acc[S::kCols][kOwn];
#pragma unroll
        for (int j = 0; j < S::kCols; ++j)
#pragma unroll
            for (int r = 0; r < kOwn; ++r) acc[j][r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

        // (5 x 17 beams of 62 tokens over 72: 974 us with every tile for every block, so 184.)
        int now_t = seen.next(0), next_t = seen.next(now_t + 1);
        find(now_t, 0);
        __syncthreads();
        if (now_t < n_tiles) fetch(0);
        find(next_t, 1);
        __syncthreads();
        for (int slot = 0; now_t < n_tiles; slot ^= 1) {
            if (next_t < n_tiles) {
                fetch(slot ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncthreads();
            const float* keys = stages + slot * S::kStage;
            const float* values = keys + S::kKeys * S::kPitch;
            {
                float s[4][4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[r][k] = 0.0f;
#pragma unroll 4
                for (int v = part; v < vecs; v += S::kSplit) {
                    float4 q[4], x[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) q[r] = *reinterpret_cast<const float4*>(query + (s_row + 4 * r) * S::kPitch + v * 4);
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const float4*>(keys + (s_key + 8 * k) * S::kPitch + v * 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            s[r][k] = fmaf(q[r].w, x[k].w, fmaf(q[r].z, x[k].z, fmaf(q[r].y, x[k].y, fmaf(q[r].x, x[k].x, s[r][k]))));
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int k = 0; k < 4; ++k) scores[part * S::kScores + (s_row + 4 * r) * S::kScorePitch + s_key + 8 * k] = s[r][k];
            }
            __syncthreads();
            {
                float x[kEach];
                float now = -INFINITY;
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int key = w_key + kPerRow * e;
                    float v = scores[w_row * S::kScorePitch + key];
#pragma unroll
                    for (int i = 1; i < S::kSplit; ++i) v += scores[i * S::kScores + w_row * S::kScorePitch + key];
                    const CacheUnit u = ctl.unit[slot][key >> c.page_log2];
                    bool sees = (u.mask & bit) != 0;
                    const int j = u.start + (key & (c.page - 1)) - u.limit;
                    if (sees && u.limit >= 0 && j >= 0) sees = j < count && (fresh ? fresh[j] != 0 : j <= id.token);
                    x[e] = sees ? v * scale : -INFINITY;
                    now = fmaxf(now, x[e]);
                }
#pragma unroll
                for (int m = kPerRow / 2; m > 0; m >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, m));
                now = fmaxf(now, top);
                const float ref = now == -INFINITY ? 0.0f : now;
                const float keep = exp2_fast(top - ref);
                top = now;
                sum *= keep;
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const float w = exp2_fast(x[e] - ref);
                    sum += w;
                    scores[w_row * S::kScorePitch + w_key + kPerRow * e] = w;
                }
                if (w_key == 0) ctl.factor[w_row] = keep;
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kOwn; ++r) {
                const float f = ctl.factor[o_row + 2 * r];
#pragma unroll
                for (int j = 0; j < S::kCols; ++j) acc[j][r].x *= f, acc[j][r].y *= f, acc[j][r].z *= f, acc[j][r].w *= f;
            }
#pragma unroll
            for (int j = 0; j < S::kCols; ++j) {
                const int col = o_col + kColStep * j;
                if (col >= vecs) break;
#pragma unroll 4
                for (int k = 0; k < S::kKeys; k += 4) {
                    float4 w[kOwn], x[4];
#pragma unroll
                    for (int r = 0; r < kOwn; ++r) w[r] = *reinterpret_cast<const float4*>(scores + (o_row + 2 * r) * S::kScorePitch + k);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(values + (k + i) * S::kPitch + col * 4);
#pragma unroll
                    for (int r = 0; r < kOwn; ++r) {
                        const float y[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            acc[j][r].x = fmaf(y[i], x[i].x, acc[j][r].x), acc[j][r].y = fmaf(y[i], x[i].y, acc[j][r].y);
                            acc[j][r].z = fmaf(y[i], x[i].z, acc[j][r].z), acc[j][r].w = fmaf(y[i], x[i].w, acc[j][r].w);
                        }
                    }
                }
            }
            now_t = next_t;
            next_t = seen.next(now_t + 1);
            find(next_t, slot);  // (this tile's places and units were last read before the last barrier but one)
            __syncthreads();
        }
        if (!odd_known) {
            grid_wait();
            odd = __ldcg(c.status + 1) != 0;
            odd_known = true;
        }
        if (odd) break;
        // To the output, or to this CTA's part of a divided segment.
#pragma unroll
        for (int m = kPerRow / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        if (w_key == 0) {
            ctl.top[w_row] = top;
            ctl.sum[w_row] = sum;
        }
        __syncthreads();
        const bool whole = p.t0 == 0 && p.t1 == p.tiles;
        float* parts = static_cast<float*>(a.workspace) + DBS_CUDA_CACHE_WORKSPACE_ZEROED / 4;
        int32_t* counters = static_cast<int32_t*>(a.workspace);
        float* out_part = parts + static_cast<int64_t>(2 * blockIdx.x + (p.t0 == 0)) * S::kOut;
#pragma unroll
        for (int r = 0; r < kOwn; ++r) {
            if (o_row + 2 * r >= rows) break;
            const RowId rid = row_id(a, row0 + o_row + 2 * r);
            const int64_t rbk = static_cast<int64_t>(b) * a.beams + beam0 + rid.beam;
            const int64_t place = (rbk * a.N + rid.token) * a.Hq + p.head * a.G + rid.head;
            const bool shown = rid.token < new_count(a, rbk);
            const float m = ctl.top[o_row + 2 * r], l = ctl.sum[o_row + 2 * r];
            const float inverse = l > 0.0f ? 1.0f / l : l;
#pragma unroll
            for (int j = 0; j < S::kCols; ++j) {
                const int col = o_col + kColStep * j;
                if (col >= vecs) break;
                const float4 o = acc[j][r];
                if (!whole) {
                    *reinterpret_cast<float4*>(out_part + (col * S::kRows + o_row + 2 * r) * 4) = o;
                } else {
                    reinterpret_cast<float4*>(static_cast<float*>(a.out) + place * c.D)[col] =
                        shown ? make_float4(o.x * inverse, o.y * inverse, o.z * inverse, o.w * inverse)
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
            if (o_col == 0) {
                if (!whole) {
                    out_part[S::kRows * DP + o_row + 2 * r] = m;
                    out_part[S::kRows * DP + S::kRows + o_row + 2 * r] = l;
                } else if (a.lse != nullptr) {
                    a.lse[place] = shown && l != 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
                }
            }
        }
        if (whole) continue;
        __syncthreads();
        const Span span = span_of(work, p);
        if (tid == 0) {
            __threadfence();  // of all the threads' stores, which the barrier put before this
            const int before = atomicAdd(counters + span.c0, 1);
            ctl.last = before == span.c1 - span.c0;
            if (ctl.last) counters[span.c0] = 0;
        }
        __syncthreads();
        if (!ctl.last) continue;
        __threadfence();
        join_parts<float, S::kRows, DP, kThreads>(c, a, p, span, b, beam0, row0, rows, parts, smem, tid);
    }
    if (!odd_known) {  // (a CTA without tiles)
        grid_wait();
        odd = __ldcg(c.status + 1) != 0;
    }
    // Weights of zero would not keep such a value out of the sums. All CTAs see that.
    if (odd) {
        __syncthreads();
        attend_all_rows<float>(c, a, smem, warp, kThreads / 32);
    }
}

// Floats of the largest partial result.
constexpr int kMostOut = Shape<128, 64>::kOut > Shape<256, 32>::kOut ? Shape<128, 64>::kOut : Shape<256, 32>::kOut;

template <int DP, int ROWS>
cudaError_t launch_shape(const CacheView& c, const AttendParams& a, int sm_count, cudaStream_t stream) {
    using S = Shape<DP, ROWS>;
    static_assert(S::kBytes <= 224 * 1024 && join_scratch(ROWS) <= S::kBytes && S::kOut <= kMostOut);
    auto* kernel = attend_f32_kernel<DP, ROWS>;
    static std::atomic<uint64_t> ready{0};  // a bit a device
    const cudaError_t e = allow_shared(kernel, S::kBytes, ready);
    if (e != cudaSuccess) return e;
    return launch_after(kernel, sm_count, S::kThreads, S::kBytes, stream, c, a);
}

template <int DP>
cudaError_t launch_width(const CacheView& c, const AttendParams& a, int sm_count, cudaStream_t stream) {
    const int rows = attend_f32_shape(c, a).rows;
    if (rows == 16) return launch_shape<DP, 16>(c, a, sm_count, stream);
    if constexpr (DP <= 128)
        if (rows == 64) return launch_shape<DP, 64>(c, a, sm_count, stream);
    return launch_shape<DP, 32>(c, a, sm_count, stream);
}

}  // namespace

// As many rows as a group has, up to 64 (32 for heads above 128, which leave no room for more). Rows past the
// group's cost multiply-adds with zeros.
BlockShape attend_f32_shape(const CacheView& c, const AttendParams& a) {
    const int64_t rows = group_rows(a);
    if (c.D > 128) return {rows <= 16 ? 16 : 32, Shape<256, 32>::kKeys};
    return {rows <= 16 ? 16 : (rows <= 32 ? 32 : 64), Shape<128, 64>::kKeys};
}

int64_t attend_f32_workspace(const CacheView&, const AttendParams&, int sm_count) {
    // A counter for each CTA first, then two partial results for each.
    return DBS_CUDA_CACHE_WORKSPACE_ZEROED + static_cast<int64_t>(2) * sm_count * kMostOut * 4;
}

cudaError_t launch_attend_f32(const CacheView& c, const AttendParams& a, int sm_count, cudaStream_t stream) {
    if (c.D <= 128) return launch_width<128>(c, a, sm_count, stream);
    return launch_width<256>(c, a, sm_count, stream);
}

}  // namespace dbsb
