// SPDX-License-Identifier: MIT
//
// Pieces that the attention kernels share: element types, the row-at-a-time form, the split of
// the work over the CTAs, and the copies and barriers of the tiled kernels.
#pragma once

#include <atomic>
#include <climits>
#include <type_traits>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cache.cuh"

namespace dbsb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <class T> struct Pack;  // 16 bytes of elements
template <> struct Pack<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ void widen(const uint4& v, float* f) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ bool finite(uint32_t w) { return (w & 0x7f800000u) != 0x7f800000u; }
};
template <> struct Pack<__half> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void widen(const uint4& v, float* f) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
    static __device__ __forceinline__ bool finite(uint32_t w) {
        return (w & 0x7c00u) != 0x7c00u && (w & 0x7c000000u) != 0x7c000000u;
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void widen(const uint4& v, float* f) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ bool finite(uint32_t w) {
        return (w & 0x7f80u) != 0x7f80u && (w & 0x7f800000u) != 0x7f800000u;
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};

// Four consecutive elements.
__device__ __forceinline__ void store4(float* to, float4 v) { *reinterpret_cast<float4*>(to) = v; }
template <class T> __device__ __forceinline__ void store4(T* to, float4 v) {
    *reinterpret_cast<uint2*>(to) = make_uint2(Pack<T>::pair(v.x, v.y), Pack<T>::pair(v.z, v.w));
}
template <class T> __device__ __forceinline__ float to_float(T x) { return static_cast<float>(x); }
template <class T> __device__ __forceinline__ T from_float(float x) { return static_cast<T>(x); }

__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}
// 2^x, within 2 ulp: the weights are sums' terms of at most 1 in magnitude.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// New tokens of (b, k): clamped into [0, N]. row: b * beams + k.
__device__ __forceinline__ int new_count(const AttendParams& a, int64_t row) {
    if (a.counts == nullptr) return a.N;
    const int n = a.counts[row];
    return n < 0 ? 0 : (n > a.N ? a.N : n);
}

// One query row by one warp: 32 positions a round, a lane each for the scores, the lanes over the
// head's elements for the values, in which a value that the row does not see takes no part. Right
// for every type and every value; the tiled kernels use it once the cache holds values that are
// not finite, because there a weight of zero would not keep them out of a product.
template <class T>
__device__ __noinline__ void attend_row(const CacheView& c, const AttendParams& a, int64_t row, float* query) {
    const int lane = threadIdx.x & 31;
    const int hq = static_cast<int>(row % a.Hq);
    const int64_t token = row / a.Hq;
    const int i = static_cast<int>(token % a.N);
    const int64_t bk = token / a.N, b = bk / a.beams, k = bk % a.beams;
    const int64_t slot = b * c.K + k;
    const int h = hq / a.G, count = new_count(a, bk), length = c.lengths[slot];
    const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + k * a.qs[1] + i * a.qs[2] + hq * a.qs[3];
    __syncwarp();
    for (int d = lane; d < c.D; d += 32) query[d] = to_float(q[d]) * a.scale;
    __syncwarp();
    constexpr int kEach = DBS_CUDA_CACHE_MAX_HEAD_DIM / 32;
    float acc[kEach] = {};
    float top = -INFINITY, total = 0.0f;
    const int64_t end = i < count ? static_cast<int64_t>(length) + count : 0;
    const uint8_t* mask = a.mask ? a.mask + (bk * a.N + i) * a.N : nullptr;
    const T* pages = static_cast<const T*>(c.pages);
    const int vecs = c.D / Pack<T>::n;
    for (int64_t base = 0; base < end; base += 32) {
        const int64_t pos = base + lane, col = pos >> c.page_log2;
        int p = -1;
        if (pos < end && col < c.M) p = c.table[slot * c.M + col];
        if (pos >= length && p >= 0) {
            const int j = static_cast<int>(pos - length);
            if (mask ? mask[j] == 0 : j > i) p = -1;
        }
        const int64_t at = p < 0 ? 0
            : (((static_cast<int64_t>(a.layer) * 2 * c.P + p) * c.H + h) * c.page + (pos & (c.page - 1))) * c.D;
        float score = -INFINITY;
        if (p >= 0) {
            float sum = 0.0f;
            for (int v = 0; v < vecs; ++v) {
                float f[Pack<T>::n];
                Pack<T>::widen(reinterpret_cast<const uint4*>(pages + at)[v], f);
#pragma unroll
                for (int e = 0; e < Pack<T>::n; ++e) sum = fmaf(query[v * Pack<T>::n + e], f[e], sum);
            }
            score = sum;
        }
        const unsigned seen = __ballot_sync(0xffffffffu, p >= 0);
        if (seen == 0) continue;
        const float now = fmaxf(top, lanes_max(score));
        // A row whose scores are all -inf so far keeps weights of zero instead of NaN.
        const float ref = now == -INFINITY ? 0.0f : now;
        const float keep = expf(top - ref);
        const float weight = p >= 0 ? expf(score - ref) : 0.0f;
        total = total * keep + lanes_sum(weight);
        top = now;
#pragma unroll
        for (int e = 0; e < kEach; ++e) acc[e] *= keep;
        for (unsigned rest = seen; rest != 0; rest &= rest - 1) {
            const int from = __ffs(rest) - 1;
            const float w = __shfl_sync(0xffffffffu, weight, from);
            const T* v = pages + __shfl_sync(0xffffffffu, at, from) + static_cast<int64_t>(c.P) * c.H * c.page * c.D;
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (lane + 32 * e < c.D) acc[e] = fmaf(w, to_float(v[lane + 32 * e]), acc[e]);
        }
    }
    T* out = static_cast<T*>(a.out) + row * c.D;
    const float inverse = total > 0.0f ? 1.0f / total : total;  // 0: nothing seen; NaN stays
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (lane + 32 * e < c.D) out[lane + 32 * e] = from_float<T>(acc[e] * inverse);
    if (a.lse != nullptr && lane == 0) a.lse[row] = total == 0.0f ? -INFINITY : top + logf(total);
}

template <class T>
__device__ __forceinline__ void attend_all_rows(const CacheView& c, const AttendParams& a, float* query, int warp,
                                                int warps) {
    const int64_t rows = static_cast<int64_t>(c.B) * a.beams * a.N * a.Hq;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * warps + warp; row < rows;
         row += static_cast<int64_t>(gridDim.x) * warps)
        attend_row<T>(c, a, row, query + warp * DBS_CUDA_CACHE_MAX_HEAD_DIM);
}

// ---------------------------------------------------------------------------
// The split of the work. A segment is one group of beams, one block of kRows query rows of it
// (rows in (beam, token, head of the key head's group) order) and one key head; its tiles are the
// group's units, a few at a time. All tiles of all segments form one line that is cut into equal
// parts, one a CTA, so that every SM reads the same amount whatever the lengths are. A segment
// that a cut divides is joined by the CTA that finishes its part last, or by a kernel of its own.
// ---------------------------------------------------------------------------
struct WorkSplit {
    int64_t total;   // tiles
    int ctas;        // CTAs that take part
    int64_t lo, hi;  // this CTA's tiles
    int group;       // block of a group that tile lo lies in
    int64_t base;    // its first tile
};

// One row block of a group. The line has the first blocks of all groups, then the second ones and so on.
struct GroupWork {
    int group, block;
    int units, tiles, rows;  // of the group
    bool there;              // the group has such a block
};

template <int kRows>
__device__ __forceinline__ int row_blocks(const CacheView& c, const AttendParams& a) {
    const int beams = a.beams < kGroupBeams ? a.beams : kGroupBeams;
    return (beams * a.N * a.G + kRows - 1) / kRows;
}

// kMany: a group may have more rows than a block.
template <int kRows, bool kMany>
__device__ __forceinline__ GroupWork group_work(const CacheView& c, const AttendParams& a, int i, int tile_units) {
    const int groups = c.B * c.groups;
    GroupWork w;
    w.block = kMany && i >= groups ? i / groups : 0;
    w.group = i - w.block * groups;
    const int first = (w.group % c.groups) * kGroupBeams;
    int beams = a.beams - first;
    beams = beams < 0 ? 0 : (beams > kGroupBeams ? kGroupBeams : beams);
    w.units = c.unit_count[w.group];
    w.tiles = (w.units + tile_units - 1) / tile_units;
    if (w.tiles < 1) w.tiles = 1;  // rows without a page are written too
    w.rows = beams * a.N * a.G;
    w.there = w.rows > w.block * kRows;
    return w;
}

// The share of CTA `cta` of `grid`. All threads of the block; sums: 35 ints, found: a WorkSplit in shared
// memory. The host has checked that the tiles of all segments are counted in 31 bits.
template <int kRows, bool kMany>
__device__ WorkSplit split_work(const CacheView& c, const AttendParams& a, int tile_units, int min_tiles, int spare, int* sums,
                                WorkSplit* found, int cta, int grid) {
    const int blocks = kMany ? row_blocks<kRows>(c, a) : 1, groups = c.B * c.groups * blocks, tid = threadIdx.x, threads = blockDim.x;
    auto tiles_of = [&](int g, int* longest) {
        *longest = 0;
        if (g >= groups) return 0;
        const GroupWork w = group_work<kRows, kMany>(c, a, g, tile_units);
        if (!w.there) return 0;
        *longest = w.tiles;
        return w.tiles * c.H;
    };
    // One round where a thread a group is enough; its count and place are kept for below.
    int total = 0, mine = 0, at = 0;
    if (tid == 0) sums[33] = sums[34] = 0;
    for (int base = 0; base < groups; base += threads) {
        int sum, s;
        mine = tiles_of(base + tid, &s);
        at = total + block_scan(mine, sums, &sum);
        total += sum;
        s = __reduce_max_sync(0xffffffffu, s);
        const int there = __popc(__ballot_sync(0xffffffffu, mine > 0));
        if ((tid & 31) == 0 && s > 0) {
            atomicMax(sums + 33, s);
            atomicAdd(sums + 34, there * c.H);
        }
    }
    __syncthreads();
    // A segment in more than 32 parts would cost more to join than its parts save: the longest one is 32
    // CTAs' work at the most (and so lies in 34 of them: kMaxParts).
    int64_t ctas = total / min_tiles;
    if (total > 0) {
        const int64_t cap = static_cast<int64_t>(total) * 32 / sums[33];
        if (ctas > cap) ctas = cap;
    }
    if (ctas > grid) ctas = grid;
    // As many CTAs a segment as a whole number, if that makes a CTA's share longer by `spare` tiles at most:
    // the shares then begin and end with segments of one length, and a second piece takes a CTA longer.
    const int64_t segments = sums[34], fit = segments > 0 ? ctas / segments * segments : 0;
    if (fit > 0 && total * (ctas - fit) <= spare * ctas * fit) ctas = fit;
    // CTAs with the same tiles for different row blocks take them at the same time, so that keys and
    // values come from memory once for all blocks (16 drafted trees, two blocks each: 1.07 GB read where the
    // second block followed the first, 0.55 GB so; 346 us and 326).
    if (kMany && blocks <= 8 && ctas >= 16 * blocks) ctas -= ctas % blocks;
    if (ctas < 1) ctas = 1;
    WorkSplit w;
    w.total = total;
    w.ctas = static_cast<int>(ctas);
    w.lo = static_cast<int64_t>(total) * cta / ctas;
    w.hi = static_cast<int64_t>(total) * (cta + 1) / ctas;
    w.group = 0;
    w.base = 0;
    if (cta >= ctas) {
        w.lo = w.hi = 0;
        return w;
    }
    if (groups <= threads) {
        if (mine > 0 && at <= w.lo && w.lo < at + mine) {
            w.group = tid;
            w.base = at;
            *found = w;
        }
    } else {
        int before = 0;
        for (int base = 0; base < groups && before <= w.lo; base += threads) {
            int sum, s;
            mine = tiles_of(base + tid, &s);
            at = before + block_scan(mine, sums, &sum);
            if (mine > 0 && at <= w.lo && w.lo < at + mine) {
                w.group = base + tid;
                w.base = at;
                *found = w;
            }
            before += sum;
        }
    }
    __syncthreads();
    w.group = found->group;
    w.base = found->base;
    return w;
}

// The CTA whose part holds tile x.
__device__ __forceinline__ int cta_of(const WorkSplit& w, int64_t x) {
    return static_cast<int>(((x + 1) * w.ctas - 1) / w.total);
}

// A CTA's share of one segment.
struct Piece {
    int group, block, head;  // block: row block
    int t0, t1;              // tiles
    int tiles, units, rows;  // of the group
    int64_t first;           // the segment's first tile on the line
};

// The CTAs that hold a divided segment's first and last tile.
struct Span {
    int c0, c1;
};
__device__ __forceinline__ Span span_of(const WorkSplit& w, const Piece& p) {
    Span s;
    s.c0 = p.t0 == 0 ? static_cast<int>(blockIdx.x) : cta_of(w, p.first);
    s.c1 = p.t1 == p.tiles ? static_cast<int>(blockIdx.x) : cta_of(w, p.first + p.tiles - 1);
    return s;
}

// The piece at tile `cur` of the line; advances group and base to it.
template <int kRows, bool kMany>
__device__ __forceinline__ Piece piece_at(const CacheView& c, const AttendParams& a, const WorkSplit& w, int64_t cur,
                                          int& group, int64_t& base, int tile_units) {
    GroupWork g = group_work<kRows, kMany>(c, a, group, tile_units);
    while (true) {
        const int64_t size = g.there ? static_cast<int64_t>(g.tiles) * c.H : 0;
        if (cur < base + size) break;
        base += size;
        g = group_work<kRows, kMany>(c, a, ++group, tile_units);
    }
    const int off = static_cast<int>(cur - base);
    Piece p;
    p.group = g.group;
    p.block = g.block;
    p.head = off / g.tiles;
    p.t0 = off - p.head * g.tiles;
    const int64_t left = w.hi - cur;
    p.t1 = left < g.tiles - p.t0 ? p.t0 + static_cast<int>(left) : g.tiles;
    p.tiles = g.tiles;
    p.units = g.units;
    p.rows = g.rows;
    p.first = base + static_cast<int64_t>(p.head) * g.tiles;
    return p;
}

// Row r of a group's block: its beam within the group, drafted token and query head.
struct RowId {
    int beam, token, head;
};
__device__ __forceinline__ RowId row_id(const AttendParams& a, int r) {
    RowId id;
    const int per = a.N * a.G;
    id.beam = r / per;
    r -= id.beam * per;
    id.token = r / a.G;
    id.head = r - id.token * a.G;
    return id;
}

// The tiles of a piece that a beam of its row block holds a page of: beams that draft many tokens fill
// blocks of their own, and the other beams' pages are nothing to those. All lanes of a warp together.
struct SeenTiles {
    const CacheUnit* units;  // the piece's first
    uint32_t beams;          // of the block; 0: all that the group has
    int count, step, parts;  // units: of the group from there on, a tile's; a unit's tiles if it fills several
    int tiles, window;       // of the piece; the first of the 32 that `bits` tells of
    uint32_t bits;

    __device__ __forceinline__ void look() {
        const int at = window + static_cast<int>(threadIdx.x & 31), unit = at / parts * step;
        bool any = false;
#pragma unroll 1
        for (int i = unit; at < tiles && i < unit + step && i < count; ++i) any |= (__ldg(&units[i].mask) & beams) != 0;
        bits = __ballot_sync(0xffffffffu, any);
    }
    // The first such tile from t on, or `tiles`; t never falls.
    __device__ __forceinline__ int next(int t) {
        if (beams == 0) return t;
        if (window >= tiles) return tiles;
        uint32_t rest = t - window < 32 ? bits & (0xffffffffu << (t - window)) : 0u;
        while (rest == 0) {
            window += 32;
            if (window >= tiles) return tiles;
            look();
            rest = bits;
        }
        return window + __ffs(rest) - 1;
    }
};
template <int kRows>
__device__ __forceinline__ SeenTiles seen_tiles(const CacheView& c, const AttendParams& a, const Piece& p, int tile_units, int parts) {
    const int row0 = p.block * kRows, rows = p.rows - row0 < kRows ? p.rows - row0 : kRows, per = a.N * a.G;
    const int first = row0 / per, beams = (row0 + rows - 1) / per - first + 1;
    SeenTiles s;
    s.units = c.units + static_cast<int64_t>(p.group) * c.unit_cap + p.t0 * tile_units;
    s.beams = beams * per == p.rows ? 0u : (beams < 32 ? (1u << beams) - 1 : 0xffffffffu) << first;
    s.count = p.units - p.t0 * tile_units;
    s.step = tile_units;
    s.parts = parts;
    s.tiles = (p.t1 - p.t0) * parts;
    s.window = 0;
    s.bits = 0;
    if (s.beams != 0) s.look();
    return s;
}

// The queries of a row block by kThreads threads, eight loads in flight each. at: the rows' places
// in q, in shared memory; put(row, chunk, value) gets 16 bytes of every row of the block, zeros past
// its end and past the head.
template <class T, int kRows, int DP, int kThreads, class Put>
__device__ __forceinline__ void load_queries(const CacheView& c, const AttendParams& a, const int64_t* at, int rows, int tid,
                                             Put&& put) {
    constexpr int kChunks = DP / 8, kStride = kThreads / kChunks, kTotal = (kRows + kStride - 1) / kStride;
    constexpr int kEach = kTotal < 8 ? kTotal : 8;
    const int chunk = tid % kChunks, first = tid / kChunks;
    const T* q = static_cast<const T*>(a.q) + chunk * 8;
#pragma unroll 1
    for (int i = 0; i < kTotal; i += kEach) {
        uint4 v[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int r = first + (i + j) * kStride;
            v[j] = make_uint4(0, 0, 0, 0);
            if (r < rows && chunk * 8 < c.D) v[j] = __ldg(reinterpret_cast<const uint4*>(q + at[r]));
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int r = first + (i + j) * kStride;
            if (r < kRows) put(r, chunk, v[j]);
        }
    }
}

// The parts of a divided segment to the output, in their order, so that the result does not depend
// on which CTA comes last: its kJoin rows from `first` on. A part: kRows x DP sums (four columns of all
// rows together), the rows' references (base 2), their weights' sums. scratch: join_scratch(kJoin) bytes
// of shared memory. All kThreads threads of named barrier 1.
//
// The last CTA joins alone, so that its latency is the call's: the parts' shares go through shared
// memory once, and the values are read in flat order, where one index gives row and place (indexes kept
// an item each cost the loop before it its registers: 64 sequences of 8 beams over 576 in 79 us for 71).
constexpr int kMaxParts = 34;  // of a segment (split_work)
constexpr int join_scratch(int rows) { return rows * (12 + 4 * kMaxParts); }

template <class T, int kRows, int DP, int kThreads, int kJoin = kRows, int kEach = 4, int kAtOnce = (kThreads > 256 ? 2 : 4)>
__device__ __forceinline__ void join_parts(const CacheView& c, const AttendParams& a, Piece p, Span span, int b,
                                           int beam0, int row0, int rows, const float* parts, void* scratch, int tid,
                                           int first = 0) {
    constexpr int kOut = kRows * (DP + 2);
    rows = rows - first < kJoin ? rows - first : kJoin;
    row0 += first;
    const int n_parts = span.c1 - span.c0 + 1;
    // A CTA's second part is the one that begins a segment.
    auto part_of = [&](int i) { return parts + static_cast<int64_t>(2 * (span.c0 + i) + (i == 0)) * kOut; };
    int64_t* places = static_cast<int64_t*>(scratch);
    float* shown_rows = reinterpret_cast<float*>(places + kJoin);  // 1; 0 for rows that are not shown
    float* factors = shown_rows + kJoin;                           // [part][row]: the part's share over the sum
    // Eight lanes a row, each for every eighth part.
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += kThreads / 8) {
        const int r = r0 + tid / 8, lane = tid % 8;
        float m = -INFINITY, l = 0.0f;
#pragma unroll 1
        for (int j0 = 0; j0 < n_parts; j0 += 32) {
            float pm[4], pl[4], now = m;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j0 + lane + 8 * k;
                const bool there = j < n_parts && r < rows;
                pm[k] = there ? __ldcg(part_of(j) + kRows * DP + first + r) : -INFINITY;
                pl[k] = there ? __ldcg(part_of(j) + kRows * DP + kRows + first + r) : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j0 + lane + 8 * k;
                if (j < n_parts && r < rows) factors[j * kJoin + r] = pm[k];
                now = fmaxf(now, pm[k]);
            }
#pragma unroll
            for (int d = 4; d > 0; d >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
            const float ref = now == -INFINITY ? 0.0f : now;
            l *= exp2_fast(m - ref);
#pragma unroll
            for (int k = 0; k < 4; ++k) l = fmaf(pl[k], exp2_fast(pm[k] - ref), l);
            m = now;
        }
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        if (r >= rows) continue;
        const float ref = m == -INFINITY ? 0.0f : m, inverse = l > 0.0f ? 1.0f / l : l;
#pragma unroll 1
        for (int j = lane; j < n_parts; j += 8) {
            float& f = factors[j * kJoin + r];  // this lane's own
            f = exp2_fast(f - ref) * inverse;
        }
        if (lane == 0) {
            const RowId id = row_id(a, row0 + r);
            const int64_t bk = static_cast<int64_t>(b) * a.beams + beam0 + id.beam;
            const bool shown = id.token < new_count(a, bk);
            const int64_t at = (bk * a.N + id.token) * a.Hq + p.head * a.G + id.head;
            places[r] = at;
            shown_rows[r] = shown ? 1.0f : 0.0f;
            if (a.lse != nullptr) a.lse[at] = shown && l != 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
        }
    }
    __syncwarp();
    asm volatile("barrier.sync 1, %0;" ::"r"(kThreads) : "memory");
    // Four values of kEach items from kAtOnce parts in flight.
    const int items = kJoin * (c.D / 4);
#pragma unroll 1
    for (int i0 = tid; i0 < items; i0 += kEach * kThreads) {
        float4 o[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) o[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (int j0 = 0; j0 < n_parts; j0 += kAtOnce) {
            float4 v[kAtOnce][kEach];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const float* x = part_of(j0 + k < n_parts ? j0 + k : j0);
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int i = i0 + e * kThreads;
                    v[k][e] = i < items && i % kJoin < rows ? __ldcg(reinterpret_cast<const float4*>(x) + i / kJoin * kRows + first + i % kJoin) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (j0 + k >= n_parts) break;
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int r = (i0 + e * kThreads) % kJoin;
                    const float f = factors[(j0 + k) * kJoin + (r < rows ? r : 0)];
                    o[e].x = fmaf(v[k][e].x, f, o[e].x), o[e].y = fmaf(v[k][e].y, f, o[e].y);
                    o[e].z = fmaf(v[k][e].z, f, o[e].z), o[e].w = fmaf(v[k][e].w, f, o[e].w);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = i0 + e * kThreads, r = i % kJoin;
            if (i >= items || r >= rows) continue;
            if (shown_rows[r] == 0.0f) o[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            store4(static_cast<T*>(a.out) + places[r] * c.D + i / kJoin * 4, o[e]);
        }
    }
}

// ---------------------------------------------------------------------------
// Barriers and copies. Every wait is bounded: it records a timeout in the cache's status word and
// goes on, so that a kernel ends whatever happens.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_address(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void barrier_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
constexpr int kWaitLimit = 1 << 20;  // tries; each may sleep for the hardware's time limit
__device__ __forceinline__ void barrier_wait_long(uint32_t bar, uint32_t parity, int32_t* status) {
    for (int i = 0; i < kWaitLimit; ++i) {
        if (barrier_try(bar, parity)) return;
        if ((i & 1023) == 1023 && (*static_cast<volatile int32_t*>(status) & DBS_CUDA_CACHE_STATUS_TIMEOUT) != 0) return;
    }
    atomicOr(status, DBS_CUDA_CACHE_STATUS_TIMEOUT);
}
__device__ __forceinline__ void barrier_wait(uint32_t bar, uint32_t parity, int32_t* status) {
    if (!barrier_try(bar, parity)) barrier_wait_long(bar, parity, status);
}
__device__ __forceinline__ void named_sync(int id, int threads) {
    asm volatile("barrier.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// Dynamic shared memory of a kernel, allowed once a device. ready: a bit for each that has it.
template <class Kernel>
cudaError_t allow_shared(Kernel* kernel, int bytes, std::atomic<uint64_t>& ready) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = uint64_t{1} << (dev & 63);
    if (dev < 64 && (ready.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(bit, std::memory_order_release);
    return e;
}

// The tensor map of the pages as [rows, head_dim], boxes of one page by 64 elements, swizzled so
// that eight rows of 128 bytes cover all banks. False: the driver refused it.
bool page_map(const CacheView& c, int dtype, CUtensorMap* map);

// Query rows of a block and positions of a tile, of the kernel that a call takes.
struct BlockShape {
    int rows, keys;
};
// Query rows of a group of beams at the most.
inline int64_t group_rows(const AttendParams& a) {
    return static_cast<int64_t>(a.beams < kGroupBeams ? a.beams : kGroupBeams) * a.N * a.G;
}
BlockShape attend_f32_shape(const CacheView& c, const AttendParams& a);
BlockShape attend_tc_shape(const CacheView& c, const AttendParams& a);
BlockShape attend_mma_shape(const CacheView& c, const AttendParams& a);

int64_t attend_f32_workspace(const CacheView& c, const AttendParams& a, int sm_count);
cudaError_t launch_attend_f32(const CacheView& c, const AttendParams& a, int sm_count, cudaStream_t stream);
int64_t attend_tc_workspace(const CacheView& c, const AttendParams& a, int sm_count);
cudaError_t launch_attend_tc(const CacheView& c, int dtype, const AttendParams& a, int sm_count, cudaStream_t stream);
int64_t attend_mma_workspace(const CacheView& c, const AttendParams& a, int sm_count);
cudaError_t launch_attend_mma(const CacheView& c, int dtype, const AttendParams& a, int sm_count, cudaStream_t stream);

}  // namespace dbsb
