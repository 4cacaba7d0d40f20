// SPDX-License-Identifier: MIT
//
// Attention over the paged cache for float16 and bfloat16 heads of 136 to 256, on mma.sync: 128 rows
// of such an output do not leave tensor memory room for two streams of scores (attend_tc.cu). Made for
// groups of few rows, where the bytes decide (16 sequences of 8 beams over 2000, 4 query heads on 8 key
// heads of 256, bfloat16: 81 us, the bytes take 41); one of many rows reads every tile again for each 32 of
// them, from L2 (256 rows over 4000, 16 sequences of 4 key heads: 341 us for 43 us of bytes).
//
// Bound by the bytes of keys and values: each is read once for all rows of a group of beams, and
// every SM reads an equal share (attend.cuh). A producer warp copies tiles of 64 positions
// through a ring of stages by TMA; eight warps compute, each on 16 positions of a tile and all
// rows: with positions instead of rows divided among the warps, a key or value is taken from
// shared memory once, by one warp, and no warp waits for another inside the loop. Each warp keeps
// the running maximum, sum and output of its positions (in 32 bits); the warps are joined once, at
// the end of a segment.
//
// Scores are taken in base 2: scale * log2(e) is applied to the 32-bit product. Weights are
// rounded to the input type for the second product, as the values are; their sum is taken before. In float16
// they are 2^15 at the most instead of 1 (kLift), since below 2^-14 its steps are no longer relative; the
// statistics carry that.
#include "attend.cuh"

namespace dbsb {

namespace {

constexpr int DP = 256;  // the head, padded
constexpr int kTileKeys = 64;
constexpr int kComputeWarps = 8;
constexpr int kComputeThreads = kComputeWarps * 32;
constexpr int kThreads = kComputeThreads + 128;  // and the producer's warpgroup, of which one warp works
constexpr int kMaxStages = 8;
template <class T> constexpr float kLift = std::is_same_v<T, __half> ? 15.0f : 0.0f;  // log2 of the largest weight

template <int WR>
struct Shape {
    static constexpr int kRows = 16 * WR;
    static constexpr int kBlocks = DP / 64;
    static constexpr int kHalf = kBlocks * kTileKeys * 128;  // bytes of a tile's keys
    static constexpr int kStages = 128 * 1024 / (2 * kHalf);
    static constexpr int kQuery = kRows * DP * 2;
    static constexpr int kJoin = 4 * 16 * DP * 4;
    static_assert(join_scratch(kRows) <= kJoin);
    static constexpr int kOut = kRows * (DP + 2);  // floats of a partial result
    static constexpr int kBytes = 1024 + kStages * 2 * kHalf + kQuery + kJoin;
};

// 16-byte chunk c of row r in a 128-byte-wide swizzled block.
__device__ __forceinline__ uint32_t swizzled(int r, int c) {
    return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <class T> __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct Control {
    uint64_t full[kMaxStages], empty[kMaxStages];
    CacheUnit unit[kMaxStages][4];
    int sums[35];
    WorkSplit split;
    float top[kComputeWarps][16], sum[kComputeWarps][16];  // each compute warp's row statistics
    float row_top[32], row_sum[32];
    int last;
    int64_t query_at[32];
};

// WR = 1: the two halves of the compute warps take alternate tiles; 2: they take halves of the rows
// and every tile.
template <class T, int WR>
__global__ void __launch_bounds__(kThreads, 1)
attend_mma_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CacheView c,
                  const __grid_constant__ AttendParams a) {
    using S = Shape<WR>;
    constexpr int kSteps = DP / 16, kHalfRows = 16;
    extern __shared__ uint8_t raw[];
    __shared__ Control ctl;
    uint8_t* smem = raw + (1024 - (smem_address(raw) & 1023)) % 1024;
    const uint32_t stages = smem_address(smem);
    uint8_t* query = smem + S::kStages * 2 * S::kHalf;
    float* join = reinterpret_cast<float*>(query + S::kQuery);  // 4 buffers of [kHalfRows][DP]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile_units = kTileKeys >> c.page_log2;
    constexpr int blocks = S::kBlocks;  // all of them: past head_dim the copies fill in zeros

    if (tid == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            barrier_init(smem_address(&ctl.full[s]), 1);
            barrier_init(smem_address(&ctl.empty[s]), WR == 1 ? kComputeWarps / 2 : kComputeWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // The plan was complete before the new tokens' copy began; only the pages have to be waited for.
    if (a.k == nullptr) grid_wait();
    const WorkSplit work = split_work<S::kRows, (WR == 2)>(c, a, tile_units, 1, 0, ctl.sums, &ctl.split, blockIdx.x, gridDim.x);
    __syncthreads();
    grid_wait();
    grid_release();
    if (__ldcg(c.status + 1) != 0) {
        attend_all_rows<T>(c, a, reinterpret_cast<float*>(smem), warp, kThreads / 32);
        return;
    }
    int group = work.group;
    int64_t base = work.base;
    int it = 0;  // tiles so far

    // Registers: launched with 168 a thread; 2 x 128 x 232 + 128 x 40 = 384 x 168.
    if (warp >= kComputeWarps) {  // producer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp > kComputeWarps) return;
        asm volatile("fence.proxy.async;" ::: "memory");
        for (int64_t cur = work.lo; cur < work.hi;) {
            const Piece p = piece_at<S::kRows, (WR == 2)>(c, a, work, cur, group, base, tile_units);
            const CacheUnit* units = c.units + static_cast<int64_t>(p.group) * c.unit_cap;
            auto fetch = [&](int t) {
                CacheUnit u{-1, 0, 0, -1};
                const int i = t * tile_units + lane;
                if (lane < tile_units && i < p.units) {
                    const int4 v = __ldg(reinterpret_cast<const int4*>(units + i));
                    u = CacheUnit{v.x, v.y, static_cast<uint32_t>(v.z), v.w};
                }
                return u;
            };
            CacheUnit next = fetch(p.t0);
            for (int t = p.t0; t < p.t1; ++t, ++it) {
                const CacheUnit u = next;
                if (t + 1 < p.t1) next = fetch(t + 1);
                const int stage = it % S::kStages;
                const uint32_t full = smem_address(&ctl.full[stage]);
                if (it >= S::kStages) barrier_wait(smem_address(&ctl.empty[stage]), (it / S::kStages - 1) & 1, c.status);
                if (lane < tile_units) ctl.unit[stage][lane] = u;
                const int valid = __popc(__ballot_sync(0xffffffffu, u.page >= 0));
                __syncwarp();
                const int copies = valid * blocks * 2;  // units are valid from the first on
                if (lane == 0) barrier_expect(full, static_cast<uint32_t>(copies) * c.page * 128);
                __syncwarp();
                const int which = lane / (blocks * 2), part = lane - which * blocks * 2;
                const int page = __shfl_sync(0xffffffffu, u.page, which & 31);
                if (lane < copies) {
                    const int kind = part / blocks, block = part - kind * blocks;
                    const int64_t row = (((static_cast<int64_t>(a.layer) * 2 + kind) * c.P + page) * c.H + p.head) * c.page;
                    const uint32_t to = stages + stage * 2 * S::kHalf + kind * S::kHalf + block * (kTileKeys * 128) +
                                        which * c.page * 128;
                    tma_load(to, &map, block * 64, static_cast<int>(row), full);
                }
            }
            cur += p.t1 - p.t0;
        }
        // No copy may be in flight when the CTA ends, even if a wait gave up.
        for (int i = it > S::kStages ? it - S::kStages : 0; i < it; ++i)
            barrier_wait(smem_address(&ctl.full[i % S::kStages]), (i / S::kStages) & 1, c.status);
        return;
    }

    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int half = warp / (kComputeWarps / 2), quarter = warp % (kComputeWarps / 2);
    const int row_in_tile = lane >> 2, pair = lane & 3;
    const float scale = a.scale * kLog2e;
    const uint32_t query_at = smem_address(query) + (WR == 2 ? half * kHalfRows * DP * 2 : 0);
    for (int64_t cur = work.lo; cur < work.hi;) {
        const Piece p = piece_at<S::kRows, (WR == 2)>(c, a, work, cur, group, base, tile_units);
        const int b = p.group / c.groups, beam0 = (p.group - b * c.groups) * kGroupBeams;
        const int row0 = p.block * S::kRows;
        // The queries: [row][DP], 128-byte blocks swizzled by row.
        const int rows = p.rows - row0 < S::kRows ? p.rows - row0 : S::kRows;
        named_sync(1, kComputeThreads);
        if (tid < rows) {
            const RowId id = row_id(a, row0 + tid);
            ctl.query_at[tid] = b * a.qs[0] + (beam0 + id.beam) * a.qs[1] + id.token * a.qs[2] + (p.head * a.G + id.head) * a.qs[3];
        }
        named_sync(1, kComputeThreads);
        load_queries<T, S::kRows, DP, kComputeThreads>(c, a, ctl.query_at, rows, tid, [&](int r, int chunk, uint4 v) {
            *reinterpret_cast<uint4*>(query + (chunk >> 3) * (S::kRows * 128) + swizzled(r, chunk & 7)) = v;
        });
        named_sync(1, kComputeThreads);
        // Which beams the warp's rows belong to; rows past the count or the end see nothing.
        const int warp_row0 = WR == 2 ? half * kHalfRows : 0;
        uint32_t bit[2];
        uint32_t need = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = row0 + warp_row0 + row_in_tile + 8 * e;
            bit[e] = 0;
            if (r < p.rows) {
                const RowId id = row_id(a, r);
                const bool live = a.counts == nullptr || id.token < new_count(a, static_cast<int64_t>(b) * a.beams + beam0 + id.beam);
                if (live) bit[e] = 1u << id.beam;
            }
            need |= bit[e];
        }
        need = __reduce_or_sync(0xffffffffu, need);

        float top[2], sum[2], acc[kSteps * 2][4];
        top[0] = top[1] = -INFINITY;
        sum[0] = sum[1] = 0.0f;
#pragma unroll
        for (int n = 0; n < kSteps * 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
        for (int t = p.t0; t < p.t1; ++t, ++it) {
            if (WR == 1 && (it & 1) != half) continue;
            const int stage = it % S::kStages;
            barrier_wait(smem_address(&ctl.full[stage]), (it / S::kStages) & 1, c.status);
            const int key0 = quarter * 16;
            const CacheUnit u = ctl.unit[stage][key0 >> c.page_log2];
            if (u.page >= 0 && (u.mask & need) != 0) {
                const uint32_t keys = stages + stage * 2 * S::kHalf;
                float s[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    uint32_t kf[4];
                    const int row = key0 + (lane & 7) + ((lane & 16) >> 1), chunk = 2 * k + ((lane >> 3) & 1);
                    ldmatrix4(kf, keys + (chunk >> 3) * (kTileKeys * 128) + swizzled(row, chunk & 7));
                    uint32_t qf[4];
                    const int qrow = warp_row0 + (lane & 15), qchunk = 2 * k + (lane >> 4);
                    ldmatrix4(qf, smem_address(query) + (qchunk >> 3) * (S::kRows * 128) + swizzled(qrow, qchunk & 7));
                    mma<T>(s[0], qf, kf[0], kf[1]);
                    mma<T>(s[1], qf, kf[2], kf[3]);
                }
                const bool plain = u.limit < 0 && (u.mask & need) == need;
                uint32_t weights[4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] *= scale;
                if (!plain) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool holds = (bit[e] & u.mask) != 0;
                        int64_t fresh = 0;
                        int token = 0, count = 0;
                        if (holds && u.limit >= 0) {
                            const RowId id = row_id(a, row0 + warp_row0 + row_in_tile + 8 * e);
                            const int64_t bk = static_cast<int64_t>(b) * a.beams + beam0 + id.beam;
                            token = id.token;
                            count = new_count(a, bk);
                            fresh = (bk * a.N + token) * a.N;
                        }
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                bool sees = holds;
                                if (holds && u.limit >= 0) {
                                    const int pos = u.start + ((key0 + n * 8 + pair * 2 + x) & (c.page - 1));
                                    const int j = pos - u.limit;
                                    if (j >= 0) sees = j < count && (a.mask ? a.mask[fresh + j] != 0 : j <= token);
                                }
                                if (!sees) s[n][2 * e + x] = -INFINITY;
                            }
                    }
                }
                // One online-softmax step of the warp's 16 positions.
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float now = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
                    now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 1));
                    now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 2));
                    now = fmaxf(now, top[e]);
                    const float ref = now == -INFINITY ? 0.0f : now;
                    const float keep = exp2_fast(top[e] - ref);
                    if (__any_sync(0xffffffffu, now != top[e])) {
#pragma unroll
                        for (int n = 0; n < kSteps * 2; ++n) {
                            acc[n][2 * e] *= keep;
                            acc[n][2 * e + 1] *= keep;
                        }
                    }
                    top[e] = now;
                    const float low = ref - kLift<T>;
                    float w[4];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int x = 0; x < 2; ++x) w[2 * n + x] = exp2_fast(s[n][2 * e + x] - low);
                    sum[e] = sum[e] * keep + ((w[0] + w[1]) + (w[2] + w[3]));
                    weights[e] = Pack<T>::pair(w[0], w[1]);
                    weights[2 + e] = Pack<T>::pair(w[2], w[3]);
                }
#pragma unroll
                for (int n = 0; n < kSteps; ++n) {
                    uint32_t vf[4];
                    const int row = key0 + (lane & 15), chunk = 2 * n + (lane >> 4);
                    ldmatrix4_trans(vf, keys + S::kHalf + (chunk >> 3) * (kTileKeys * 128) + swizzled(row, chunk & 7));
                    mma<T>(acc[2 * n], weights, vf[0], vf[1]);
                    mma<T>(acc[2 * n + 1], weights, vf[2], vf[3]);
                }
            }
            __syncwarp();
            if (lane == 0) barrier_arrive(smem_address(&ctl.empty[stage]));
        }
        cur += p.t1 - p.t0;

        // Join the warps: the rows' maxima and sums, then the outputs at the common maximum, through
        // four buffers in two rounds (the upper warps of a half's set, then the lower ones).
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = sum[e];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (pair == 0) {
                ctl.top[warp][row_in_tile + 8 * e] = top[e];
                ctl.sum[warp][row_in_tile + 8 * e] = l;
            }
        }
        named_sync(1, kComputeThreads);
        constexpr int kSet = WR == 1 ? kComputeWarps : kComputeWarps / 2;  // warps with the same rows
        const int set0 = WR == 1 ? 0 : half * kSet, rank = warp - set0;
        if (tid < S::kRows) {
            const int r = WR == 2 ? tid % kHalfRows : tid, from = WR == 2 ? tid / kHalfRows * kSet : 0;
            float m = -INFINITY;
            for (int i = 0; i < kSet; ++i) m = fmaxf(m, ctl.top[from + i][r]);
            const float ref = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            for (int i = 0; i < kSet; ++i) l += ctl.sum[from + i][r] * exp2_fast(ctl.top[from + i][r] - ref);
            ctl.row_top[tid] = m;  // (without kLift, as the warps' own)
            ctl.row_sum[tid] = l;
        }
        named_sync(1, kComputeThreads);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float m = ctl.row_top[warp_row0 + row_in_tile + 8 * e];
            const float factor = exp2_fast(top[e] - (m == -INFINITY ? 0.0f : m));
#pragma unroll
            for (int n = 0; n < kSteps * 2; ++n) {
                acc[n][2 * e] *= factor;
                acc[n][2 * e + 1] *= factor;
            }
        }
        constexpr int kBuffers = kSet / 2;  // a set's; kBuffers * WR == 4
        float* mine = join + ((WR == 1 ? 0 : half * kBuffers) + rank % kBuffers) * (kHalfRows * DP);
        auto spot = [&](int n, int e) {
            const int r = row_in_tile + 8 * e;
            return mine + r * DP + ((n * 8 + pair * 2) ^ ((r & 7) << 3));
        };
        if (rank >= kBuffers) {
#pragma unroll
            for (int n = 0; n < kSteps * 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<float2*>(spot(n, e)) = make_float2(acc[n][2 * e], acc[n][2 * e + 1]);
        }
        named_sync(1, kComputeThreads);
        if (rank < kBuffers) {
#pragma unroll
            for (int n = 0; n < kSteps * 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float2* at = reinterpret_cast<float2*>(spot(n, e));
                    const float2 o = *at;
                    *at = make_float2(acc[n][2 * e] + o.x, acc[n][2 * e + 1] + o.y);
                }
        }
        named_sync(1, kComputeThreads);
        // Four values at a time: to the output, or to this CTA's part of a divided segment.
        const bool whole = p.t0 == 0 && p.t1 == p.tiles;
        const int vecs = c.D / 4;
        auto put = [&](int r, int vec, float4 o, float m, float l) {
            const RowId id = row_id(a, row0 + r);
            const int64_t bk = static_cast<int64_t>(b) * a.beams + beam0 + id.beam;
            const int64_t row = (bk * a.N + id.token) * a.Hq + p.head * a.G + id.head;
            const bool live = a.counts == nullptr || id.token < new_count(a, bk);
            const float inverse = live ? (l > 0.0f ? 1.0f / l : l) : 0.0f;
            uint2 packed = make_uint2(Pack<T>::pair(o.x * inverse, o.y * inverse), Pack<T>::pair(o.z * inverse, o.w * inverse));
            if (!live) packed = make_uint2(0, 0);
            reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * c.D)[vec] = packed;
            if (vec == 0 && a.lse != nullptr) a.lse[row] = live && l != 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
        };
        float* parts = static_cast<float*>(a.workspace) + DBS_CUDA_CACHE_WORKSPACE_ZEROED / 4;
        int32_t* counters = static_cast<int32_t*>(a.workspace);
        float* part = parts + static_cast<int64_t>(2 * blockIdx.x + (p.t0 == 0)) * S::kOut;
        for (int i = tid; i < rows * vecs; i += kComputeThreads) {
            const int r = i / vecs, vec = i - r * vecs;
            const int in_set = WR == 2 ? r % kHalfRows : r, buffer0 = WR == 2 ? r / kHalfRows * kBuffers : 0;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < kBuffers; ++j) {
                const float4 x = *reinterpret_cast<const float4*>(join + (buffer0 + j) * (kHalfRows * DP) + in_set * DP +
                                                                  ((vec * 4) ^ ((in_set & 7) << 3)));
                o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
            }
            const float m = ctl.row_top[r] - kLift<T>, l = ctl.row_sum[r];
            if (whole) {
                put(r, vec, o, m, l);
            } else {
                *reinterpret_cast<float4*>(part + (vec * S::kRows + r) * 4) = o;
                if (vec == 0) {
                    part[S::kRows * DP + r] = m;
                    part[S::kRows * DP + S::kRows + r] = l;
                }
            }
        }
        if (whole) continue;
        named_sync(1, kComputeThreads);
        const Span span = span_of(work, p);
        if (tid == 0) {
            __threadfence();  // of all the threads' stores, which the barrier put before this
            const int before = atomicAdd(counters + span.c0, 1);
            ctl.last = before == span.c1 - span.c0;
            if (ctl.last) counters[span.c0] = 0;
        }
        named_sync(1, kComputeThreads);
        if (!ctl.last) continue;
        __threadfence();
        join_parts<T, S::kRows, DP, kComputeThreads>(c, a, p, span, b, beam0, row0, rows, parts, join, tid);
    }
}

template <class T, int WR>
cudaError_t launch_shape(const CacheView& c, const CUtensorMap& map, const AttendParams& a, int sm_count,
                         cudaStream_t stream) {
    using S = Shape<WR>;
    static_assert(S::kOut <= Shape<2>::kOut);
    auto* kernel = attend_mma_kernel<T, WR>;
    static std::atomic<uint64_t> ready{0};  // a bit a device
    const cudaError_t e = allow_shared(kernel, S::kBytes, ready);
    if (e != cudaSuccess) return e;
    return launch_after(kernel, sm_count, kThreads, S::kBytes, stream, map, c, a);
}

template <class T>
cudaError_t launch_typed(const CacheView& c, const CUtensorMap& map, const AttendParams& a, int sm_count,
                         cudaStream_t stream) {
    if (attend_mma_shape(c, a).rows == 16) return launch_shape<T, 1>(c, map, a, sm_count, stream);
    return launch_shape<T, 2>(c, map, a, sm_count, stream);
}

}  // namespace

// 16 rows, or 32 where a group has more. Fewer rows than that cost products with zeros, not bytes.
BlockShape attend_mma_shape(const CacheView&, const AttendParams& a) { return {group_rows(a) <= 16 ? 16 : 32, kTileKeys}; }

bool page_map(const CacheView& c, int dtype, CUtensorMap* map) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(c.D), static_cast<cuuint64_t>(c.L) * 2 * c.P * c.H * c.page};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(c.D) * 2};
    const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(c.page)}, steps[2] = {1, 1};
    const auto type = dtype == DBS_CUDA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, type, 2, c.pages, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t attend_mma_workspace(const CacheView&, const AttendParams&, int sm_count) {
    // A counter for each CTA first, then two partial results for each.
    return DBS_CUDA_CACHE_WORKSPACE_ZEROED + static_cast<int64_t>(2) * sm_count * Shape<2>::kOut * 4;
}

cudaError_t launch_attend_mma(const CacheView& c, int dtype, const AttendParams& a, int sm_count, cudaStream_t stream) {
    CUtensorMap map;
    if (!page_map(c, dtype, &map)) return cudaErrorInvalidValue;
    if (dtype == DBS_CUDA_DTYPE_F16) return launch_typed<__half>(c, map, a, sm_count, stream);
    return launch_typed<__nv_bfloat16>(c, map, a, sm_count, stream);
}

}  // namespace dbsb
