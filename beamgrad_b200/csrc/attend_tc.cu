// SPDX-License-Identifier: MIT
//
// Attention of a group of beams over the paged cache on the fifth-generation tensor cores, for
// float16 and bfloat16 and heads of up to 128.
//
// 128 query rows by 128 positions at a time: S = Q K^T into tensor memory, the weights P back to
// tensor memory in the place of S, O += P V in tensor memory. One warp copies keys and values by
// TMA through a ring of slots (a slot holds 128 rows of keys or of values), one warp issues the
// products, and the others turn scores into weights. S, P and O are two streams: the products of one
// run while the other takes exponentials.
//
// NQ = 2 (more than 128 rows): each stream has query rows of its own, 256 a block, and takes every
// tile, so that keys and values cross from L2 once for 256 rows. NQ = 1: both have the same rows and
// take alternate tiles. A stream of 128 rows has two warpgroups, each for a half of the positions (four
// warps a scheduler; with two, the exponentials wait for their own latency). With at most 64 (32)
// rows these lie in tensor memory 2 (4) times and each copy weighs a half (a quarter) of the
// positions, with zeros for the others: the product costs the same, and the chain from scores to
// weights is a half (a quarter) as long. Copies and streams are joined at the end of a segment.
//
// Rescaling is put off, as has been published for attention on this architecture (the code is this
// engine's own): a row's reference for the exponentials is raised only when its maximum has grown by
// more than 2^8. Until then the weights stay below 2^8 and the sums within 32 bits, and O in tensor
// memory is left alone (in float16 all of them are 2^7 higher: kLift). Weights are rounded to the input
// type, as the values are; their sum is taken before. All statistics are 32 bits.
#include "attend.cuh"

namespace dbsb {

namespace {

constexpr int kTileKeys = 128;
constexpr int kMaxSlots = 12;
constexpr int kMinTiles = 2;     // tiles of a CTA at least: a join costs about as much as two
// A tile more for whole segments: a second piece costs a CTA more (2 x 3 beams' drafts of 18 over 1222: 34 us,
// so 30; 4 beams' drafts of 21 over 211: 32 us, so 25). Two more are too many (32 beams over 4060: 75 us, 78).
constexpr int kSpareTiles = 1;
constexpr float kRaise = 8.0f;  // log2 of the growth that a reference tolerates
// log2 of what all weights of a row are multiplied by. In float16 a weight below 2^-14 is a denormal with steps
// of 2^-24: 2^7 on top of the 2^8 that a reference tolerates uses the range up to 2^15. The statistics say so
// (a reference lower by as much), and the division at the end takes it out.
template <class T> constexpr float kLift = std::is_same_v<T, __half> ? 7.0f : 0.0f;

struct Control {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t queries, scores[2], weights[2], output[2];
    WorkSplit split;
    int sums[35];
    uint32_t tmem;
    int last;
    union {
        int64_t query_at[256];              // while queries are loaded: the rows' places
        struct {
            float top[256], sum[256];       // at the end of a segment: [copy][row]
        };
        float half[2][2][128];              // between a stream's warpgroups: [stream][half][row]
    };
};

template <int DP, int NQ, int COPIES>
struct Shape {
    static constexpr int kRows = NQ == 2 ? 256 : 128 / COPIES;
    static constexpr int kHalves = COPIES == 1 ? 2 : 1;   // warpgroups of a stream
    static constexpr int kCols = 128 / (COPIES * kHalves);  // positions of a tile that a thread weighs
    static constexpr int kSoftThreads = 256 * kHalves;
    // And the copying and the issuing warp, in a warpgroup where registers change hands.
    static constexpr int kThreads = kSoftThreads + (kHalves == 2 ? 128 : 64);
    static constexpr int kCopyWarp = kSoftThreads / 32, kIssueWarp = kCopyWarp + 1;
    static constexpr int kBlocks = DP / 64;
    static constexpr int kSlot = kTileKeys * DP * 2;
    // Divided segments are joined here, or by attend_join_kernel.
    static constexpr bool kJoined = COPIES > 1;
    // The queries; at the end of a segment copies (256 x 32 floats) and parts are joined there.
    static constexpr int kQuery = NQ * 128 * DP * 2 > 32768 ? NQ * 128 * DP * 2 : 32768;
    static_assert(!kJoined || join_scratch(kRows) <= kQuery);
    static constexpr int kFit = (227 * 1024 - static_cast<int>(sizeof(Control)) - kQuery) / kSlot;
    static constexpr int kSlots = kFit < kMaxSlots ? kFit : kMaxSlots;
    static constexpr int kOut = kRows * (DP + 2);  // floats of a partial result
    static constexpr int kBytes = kSlots * kSlot + kQuery + sizeof(Control);
};

// ---- tcgen05 ----
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// The first tile that is taken; a piece without any takes one all the same.
__device__ __forceinline__ int first_tile(SeenTiles& seen) {
    const int t = seen.next(0);
    return t < seen.tiles ? t : 0;
}

// One lane of the (converged) warp. Products are issued by the elected lane of a warp that runs its
// loop as a whole: with a loop for one lane alone, every operand of every product takes a detour to
// the warp's uniform registers (8 products took 750 cycles to issue instead of 512).
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(kind), "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(kind), "r"(static_cast<uint32_t>(add))
        : "memory");
}
#define REGS8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define REGS32(r, i) REGS8(r, i), REGS8(r, i + 8), REGS8(r, i + 16), REGS8(r, i + 24)
// 32 columns of the warp's 32 lanes, with the wait for them: a use of a register cannot move
// before it.
__device__ __forceinline__ void tmem_load(uint32_t (&r)[32], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n tcgen05.wait::ld.sync.aligned;"
        : REGS32(r, 0)
        : "r"(at)
        : "memory");
}
#undef REGS32
#undef REGS8
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Whether any thread of the named barrier says so.
__device__ __forceinline__ bool named_any(int id, int threads, bool yes) {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.red.or.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(any)
        : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(yes))
        : "memory");
    return any != 0;
}

// Shared-memory operand with 128-byte rows, swizzled: eight rows (1024 bytes) to the next eight
// rows, and `blocks` bytes between 64-element blocks of an operand that runs along the row.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t blocks) {
    return static_cast<uint64_t>((at & 0x3ffffu) >> 4) | static_cast<uint64_t>(blocks >> 4) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | uint64_t{1} << 46 | uint64_t{2} << 61;
}
// Instruction word: 32-bit sums, both operands of one 16-bit type, 128 rows, `columns` columns;
// by_row: the second operand's columns run along its rows (values: positions by elements).
template <class T>
__device__ __forceinline__ constexpr uint32_t product_kind(int columns, bool by_row) {
    constexpr uint32_t type = sizeof(T) == 2 && std::is_same_v<T, __nv_bfloat16> ? 1 : 0;
    return 1u << 4 | type << 7 | type << 10 | (by_row ? 1u << 16 : 0u) | static_cast<uint32_t>(columns / 8) << 17 | 8u << 24;
}

// ---- exponentials ----
// Pairs of 32-bit numbers, one instruction for both.
using Pair = uint64_t;
__device__ __forceinline__ Pair pair_of(float x, float y) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
    return p;
}
__device__ __forceinline__ void unpair(Pair p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ Pair pair_fma(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair pair_add(Pair a, Pair b) {
    Pair d;
    asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <class T, int DP, int NQ, int COPIES, bool SKIP>
__global__ void __launch_bounds__(Shape<DP, NQ, COPIES>::kThreads, 1)
attend_tc_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CacheView c,
                 const __grid_constant__ AttendParams a) {
    using S = Shape<DP, NQ, COPIES>;
    constexpr int kHalves = S::kHalves, kSoftThreads = S::kSoftThreads;
    constexpr int kCopyWarp = S::kCopyWarp, kIssueWarp = S::kIssueWarp;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* query = smem + S::kSlots * S::kSlot;
    Control& ctl = *reinterpret_cast<Control*>(query + S::kQuery);
    const uint32_t slots = smem_address(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile_units = kTileKeys >> c.page_log2;

    if (tid == 0) {
        for (int s = 0; s < S::kSlots; ++s) {
            barrier_init(smem_address(&ctl.full[s]), 1);
            barrier_init(smem_address(&ctl.empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrier_init(smem_address(&ctl.scores[i]), 1);
            barrier_init(smem_address(&ctl.weights[i]), 4 * kHalves);
            barrier_init(smem_address(&ctl.output[i]), 1);
        }
        barrier_init(smem_address(&ctl.queries), kSoftThreads / 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // This kernel may run while the new tokens are still being written. Plan, lengths, queries and
    // complete pages were there before that began; the copying warp waits for it at the first page
    // that is not complete, the others before they look whether a value was not finite.
    if (a.k == nullptr) grid_wait();
    grid_release();
    const WorkSplit work = split_work<S::kRows, (NQ == 2)>(c, a, tile_units, kMinTiles, kSpareTiles, ctl.sums, &ctl.split, blockIdx.x, gridDim.x);
    if (work.lo >= work.hi) {
        grid_wait();
        if (__ldcg(c.status + 1) != 0 && warp < kSoftThreads / 32)
            attend_all_rows<T>(c, a, reinterpret_cast<float*>(smem), warp, kSoftThreads / 32);
        return;
    }
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_address(&ctl.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl.tmem;  // S of the streams, then O: 128 columns each
    int group = work.group;
    int64_t base = work.base;

    // Registers: 640 threads are launched with 96 each, 512 x 104 + 128 x 64 (320 have 168 each, which
    // is enough for all roles).
    if (warp >= kCopyWarp) {
        if constexpr (kHalves == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp > kIssueWarp) return;
        int used = 0;  // slots so far: K0 V0 K1 V1 ...
        if (warp == kCopyWarp) {
            bool waited = false;
            for (int64_t cur = work.lo; cur < work.hi;) {
                const Piece p = piece_at<S::kRows, (NQ == 2)>(c, a, work, cur, group, base, tile_units);
                const CacheUnit* units = c.units + static_cast<int64_t>(p.group) * c.unit_cap;
                const int n_tiles = p.t1 - p.t0;
                // The page of this lane's copy; past the last unit, page 0: whatever finite values lie
                // there meet weights of zero.
                const int which = lane / S::kBlocks, block = lane % S::kBlocks;
                auto unit_of = [&](int t) {
                    const int i = (p.t0 + t) * tile_units + which;
                    return t < n_tiles && which < tile_units && i < p.units ? __ldg(reinterpret_cast<const int4*>(units + i))
                                                                            : make_int4(0, 0, 0, -1);
                };
                int t = 0, after = 1;
                SeenTiles seen;
                if constexpr (SKIP) {
                    seen = seen_tiles<S::kRows>(c, a, p, tile_units, 1);
                    t = first_tile(seen);
                    after = seen.next(t + 1);
                }
                int4 next = unit_of(t);
#pragma unroll 1
                while (t < n_tiles) {
                    const int page = next.x;
                    if (!waited && __any_sync(0xffffffffu, next.w >= 0)) {
                        grid_wait();
                        asm volatile("fence.proxy.async;" ::: "memory");
                        waited = true;
                    }
                    next = unit_of(after);
                    t = after++;
                    if constexpr (SKIP) after = seen.next(after);
#pragma unroll 1
                    for (int kind = 0; kind < 2; ++kind, ++used) {
                        const int slot = used % S::kSlots;
                        const uint32_t full = smem_address(&ctl.full[slot]);
                        if (used >= S::kSlots)
                            barrier_wait(smem_address(&ctl.empty[slot]), (used / S::kSlots - 1) & 1, c.status);
                        if (lane == 0) barrier_expect(full, S::kSlot);
                        __syncwarp();
                        if (which < tile_units) {
                            const int64_t row = (((static_cast<int64_t>(a.layer) * 2 + kind) * c.P + page) * c.H + p.head) * c.page;
                            tma_load(slots + slot * S::kSlot + block * (kTileKeys * 128) + which * c.page * 128, &map, block * 64,
                                     static_cast<int>(row), full);
                        }
                    }
                }
                cur += n_tiles;
            }
            // No copy may be in flight when the CTA ends, even if a wait gave up.
            for (int i = used > S::kSlots ? used - S::kSlots : 0; i < used; ++i)
                barrier_wait(smem_address(&ctl.full[i % S::kSlots]), (i / S::kSlots) & 1, c.status);
        } else {
            constexpr uint32_t kScores = product_kind<T>(kTileKeys, false), kValues = product_kind<T>(DP, true);
            uint32_t query_phase = 0, weight_phase = 0;  // a bit a stream
            auto wait_slot = [&](int i) {
                barrier_wait(smem_address(&ctl.full[i % S::kSlots]), (i / S::kSlots) & 1, c.status);
                fence_after();
            };
            for (int64_t cur = work.lo; cur < work.hi;) {
                const Piece p = piece_at<S::kRows, (NQ == 2)>(c, a, work, cur, group, base, tile_units);
                int n = p.t1 - p.t0;
                cur += n;
                if constexpr (SKIP) {
                    SeenTiles seen = seen_tiles<S::kRows>(c, a, p, tile_units, 1);
                    if (seen.beams != 0) {
                        n = 0;
                        for (int t = first_tile(seen); t < seen.tiles; t = seen.next(t + 1)) ++n;
                    }
                }
                barrier_wait(smem_address(&ctl.queries), query_phase, c.status);
                query_phase ^= 1;
                fence_after();
                // Jobs: a stream and a tile. Two streams on every tile, or one stream a tile, in turn or
                // always the first.
                const int per_tile = NQ == 2 && p.rows - p.block * S::kRows > 128 ? 2 : 1;
                const int jobs = n * per_tile, streams = NQ == 1 ? 2 : per_tile;
                auto scores = [&](int j) {
                    const int stream = streams == 2 ? j & 1 : 0, slot = used + 2 * (per_tile == 2 ? j >> 1 : j);
                    if (per_tile == 1 || stream == 0) wait_slot(slot);
                    const uint64_t q = operand(smem_address(query) + (NQ == 2 ? stream * 128 * DP * 2 : 0), 16);
                    const uint64_t k = operand(slots + slot % S::kSlots * S::kSlot, 16);
                    if (elected()) {
#pragma unroll
                        for (int s = 0; s < DP / 16; ++s) {
                            const uint64_t at = ((s >> 2) * (128 * 128) + (s & 3) * 32) >> 4;
                            product_ss(tmem + stream * 128, q + at, k + at, kScores, s > 0);
                        }
                        commit(smem_address(&ctl.scores[stream]));
                        if (per_tile == 1 || stream == 1) commit(smem_address(&ctl.empty[slot % S::kSlots]));
                    }
                    __syncwarp();
                };
                scores(0);
                if (streams == 2 && jobs > 1) scores(1);
#pragma unroll 1
                for (int j = 0; j < jobs; ++j) {
                    const int stream = streams == 2 ? j & 1 : 0, slot = used + 2 * (per_tile == 2 ? j >> 1 : j) + 1;
                    if (per_tile == 1 || stream == 0) wait_slot(slot);
                    barrier_wait(smem_address(&ctl.weights[stream]), weight_phase >> stream & 1, c.status);
                    weight_phase ^= 1u << stream;
                    fence_after();
                    const bool add = j >= streams;  // the stream's first job begins the sum
                    const uint64_t v = operand(slots + slot % S::kSlots * S::kSlot, kTileKeys * 128);
                    if (elected()) {
                        // The weights of kCols positions lie at the front of those positions' scores.
#pragma unroll
                        for (int s = 0; s < kTileKeys / 16; ++s)
                            product_ts(tmem + 256 + stream * 128,
                                       tmem + stream * 128 + s * 16 / S::kCols * S::kCols + s * 16 % S::kCols / 2,
                                       v + s * ((16 * 128) >> 4), kValues, add || s > 0);
                        if (per_tile == 1 || stream == 1) commit(smem_address(&ctl.empty[slot % S::kSlots]));
                        if (j + streams >= jobs) commit(smem_address(&ctl.output[stream]));
                    }
                    __syncwarp();
                    if (j + streams < jobs) scores(j + streams);
                }
                used += 2 * n;
            }
            named_sync(2, kSoftThreads + 32);  // every read of tensor memory is over
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        }
        return;
    }

    // Scores to weights.
    if constexpr (kHalves == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int stream = warp / (4 * kHalves), half = kHalves == 2 ? (warp >> 2) & 1 : 0, row = tid & 127;  // of the stream's 128
    const int my_row = NQ == 2 ? stream * 128 + row : row % S::kRows, copy = NQ == 2 ? 0 : row / S::kRows;
    const int col0 = (kHalves == 2 ? half : copy) * S::kCols;  // the first position of a tile that the thread weighs
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + stream * 128 + col0, o_at = tmem + lanes + 256 + stream * 128;
    const uint32_t scores_bar = smem_address(&ctl.scores[stream]), weights_bar = smem_address(&ctl.weights[stream]);
    // Not 0, which would make a masked score's -inf a NaN.
    const float scale = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale turns the queries' signs
    uint32_t score_phase = 0, output_phase = 0;
    bool odd = false, odd_known = false;  // whether a value that is not finite was met, in this call or before
    // The next segment's place, and with few rows its queries, are fetched before this one's output.
    constexpr int kChunks8 = DP / 8, kAhead = COPIES > 1 ? S::kRows * kChunks8 / kSoftThreads : 1;
    uint4 ahead[kAhead];
    auto fetch_ahead = [&](const Piece& p) {
        if constexpr (COPIES > 1) {
            const int b = p.group / c.groups, beam0 = (p.group - b * c.groups) * kGroupBeams, chunk = tid % kChunks8;
            const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + beam0 * a.qs[1] + p.head * a.G * a.qs[3] + chunk * 8;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int r = p.block * S::kRows + tid / kChunks8 + k * (kSoftThreads / kChunks8);
                ahead[k] = make_uint4(0, 0, 0, 0);
                if (r < p.rows && chunk * 8 < c.D) {
                    const RowId id = row_id(a, r);
                    ahead[k] = __ldg(reinterpret_cast<const uint4*>(q + id.beam * a.qs[1] + id.token * a.qs[2] + id.head * a.qs[3]));
                }
            }
        }
    };
    auto put_query = [&](int r, int chunk, uint4 v) {
        v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
#pragma unroll
        for (int i = 0; i < (NQ == 2 ? 1 : COPIES); ++i) {
            const int in = (r & 127) + i * S::kRows;
            *reinterpret_cast<uint4*>(query + (r >> 7) * (128 * DP * 2) + (chunk >> 3) * (128 * 128) + in * 128 +
                                      (((chunk & 7) ^ (in & 7)) << 4)) = v;
        }
    };
    Piece p = piece_at<S::kRows, (NQ == 2)>(c, a, work, work.lo, group, base, tile_units), next_piece = p;
    fetch_ahead(p);
    for (int64_t cur = work.lo; cur < work.hi; p = next_piece) {
        const int n_tiles = p.t1 - p.t0;
        cur += n_tiles;
        const int b = p.group / c.groups, beam0 = (p.group - b * c.groups) * kGroupBeams;
        const int row0 = p.block * S::kRows;
        const int rows = p.rows - row0 < S::kRows ? p.rows - row0 : S::kRows;
        const bool mine = my_row < rows;
        RowId id{0, 0, 0};
        if (mine) id = row_id(a, row0 + my_row);
        // Both streams are done with the last segment's products, and so with its queries.
        named_sync(1, kSoftThreads);
        if constexpr (COPIES > 1) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) put_query(tid / kChunks8 + k * (kSoftThreads / kChunks8), tid % kChunks8, ahead[k]);
        } else {
            if (half == 0 && (NQ == 2 || stream == 0))
                ctl.query_at[my_row] = b * a.qs[0] + (beam0 + id.beam) * a.qs[1] + id.token * a.qs[2] + (p.head * a.G + id.head) * a.qs[3];
            named_sync(1, kSoftThreads);
            load_queries<T, S::kRows, DP, kSoftThreads>(c, a, ctl.query_at, rows, tid, put_query);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(smem_address(&ctl.queries));

        const int64_t bk = static_cast<int64_t>(b) * a.beams + beam0 + id.beam;
        const int count = mine ? new_count(a, bk) : 0;
        const bool live = mine && id.token < count;
        const uint32_t bit = live ? 1u << id.beam : 0u;
        const uint32_t need = __reduce_or_sync(0xffffffffu, bit);
        const uint8_t* fresh = a.mask ? a.mask + (bk * a.N + id.token) * a.N : nullptr;
        const CacheUnit* units = c.units + static_cast<int64_t>(p.group) * c.unit_cap;

        float top = -INFINITY, sum = 0.0f;  // the reference (a score) and the weights' sum
        const bool active = NQ == 1 || rows > stream * 128;
        SeenTiles seen;
        int first = NQ == 2 ? 0 : stream;
        if constexpr (SKIP) {
            seen = seen_tiles<S::kRows>(c, a, p, tile_units, 1);
            first = first_tile(seen);
        }
        bool began = false;
        if (active) {
            // Tiles from the first on whose units are all complete and held by every row of the warp.
            int plain_tiles = 0;
            {
                const int from = p.t0 * tile_units, to = p.t1 * tile_units < p.units ? p.t1 * tile_units : p.units;
                int leading = 0;
#pragma unroll 1
                for (int i = from; i < to && leading == i - from; i += 128) {
                    int4 v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[k] = i + 32 * k + lane < to ? __ldg(reinterpret_cast<const int4*>(units + i + 32 * k + lane)) : make_int4(0, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool whole = i + 32 * k + lane < to && v[k].w < 0 && (static_cast<uint32_t>(v[k].z) & need) == need;
                        const uint32_t gaps = ~__ballot_sync(0xffffffffu, whole);
                        if (leading == i - from + 32 * k) leading += gaps == 0 ? 32 : __ffs(gaps) - 1;
                    }
                }
                plain_tiles = leading / tile_units;
            }
            // A lane each; `other`: the unit has no position among the warp's.
            const bool other = (lane << c.page_log2) >= col0 + S::kCols || ((lane + 1) << c.page_log2) <= col0;
            auto unit_of = [&](int t) {
                CacheUnit u{-1, 0, 0, -1};
                const int i = (p.t0 + t) * tile_units + lane;
                if (t < n_tiles && lane < tile_units && i < p.units) {
                    const int4 v = __ldg(reinterpret_cast<const int4*>(units + i));
                    u = CacheUnit{v.x, v.y, static_cast<uint32_t>(v.z), v.w};
                }
                return u;
            };
#pragma unroll 1
            for (int t = first; t < n_tiles; t = SKIP ? seen.next(t + 1) : t + (NQ == 2 ? 1 : 2)) {
                CacheUnit u{-1, 0, 0, -1};
                bool none = need == 0, plain = true;
                if (t >= plain_tiles) {
                    u = unit_of(t);
                    none = __all_sync(0xffffffffu, other || (u.mask & need) == 0);
                    plain = __all_sync(0xffffffffu, other || (u.limit < 0 && (u.mask & need) == need));
                }
                barrier_wait(scores_bar, score_phase, c.status);
                score_phase ^= 1;
                fence_after();
                constexpr int kChunks = S::kCols / 32;
                uint32_t s[32], sees[kChunks];
                float peak = -INFINITY;
                if (!none) {
                    // The row's maximum. A NaN among the scores stays in it.
#pragma unroll
                    for (int i = 0; i < kChunks; ++i) {
                        tmem_load(s, s_at + 32 * i);
                        if (!plain) {
                            sees[i] = 0;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {  // 16 positions lie in one unit
                                const int col = col0 + 32 * i + 16 * h, from = col >> c.page_log2;
                                const uint32_t holders = __shfl_sync(0xffffffffu, u.mask, from);
                                const int limit = __shfl_sync(0xffffffffu, u.limit, from);
                                const int start = __shfl_sync(0xffffffffu, u.start, from) + (col & (c.page - 1));
                                const bool holds = (holders & bit) != 0;
                                uint32_t bits = holds ? 0xffffu : 0u;
                                if (limit >= 0) {
                                    // The holder's committed tokens end in this page: of the new ones behind them
                                    // a chain shows the first, a mask those that it names.
                                    const int old = limit - start;
                                    const int upto = old + (fresh ? 0 : (id.token < count ? id.token + 1 : count));
                                    if (upto < 16) bits &= upto > 0 ? (1u << upto) - 1 : 0u;
                                    if (fresh != nullptr && holds && old < 16 && old + count > 0) {
#pragma unroll
                                        for (int e = 0; e < 16; ++e)
                                            if (e >= old && e - old < count) bits |= (fresh[e - old] != 0 ? 1u : 0u) << e;
                                    }
                                }
                                sees[i] |= bits << (16 * h);
                            }
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if ((sees[i] >> e & 1) == 0) s[e] = 0xff800000u;
                        }
                        float most[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) most[e] = __uint_as_float(s[e]);
#pragma unroll
                        for (int e = 4; e + 1 < 32; e += 2)
                            most[(e >> 1) & 3] = max3(most[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                        peak = max3(peak, max3(most[0], most[1], most[2]), most[3]);
                    }
                }
                // Whether the row's reference is to be raised, and for the halves of a stream to what.
                bool raise_it = peak != -INFINITY && !((peak - top) * scale <= kRaise);
                bool any_raised;
                if constexpr (kHalves == 2) {
                    any_raised = named_any(3 + stream, 256, raise_it);
                    if (any_raised) {
                        ctl.half[stream][half][row] = peak;
                        named_sync(3 + stream, 256);
                        const float its = ctl.half[stream][half ^ 1][row];
                        peak = max3(peak, its, its);
                        raise_it = peak != -INFINITY && !((peak - top) * scale <= kRaise);
                        named_sync(3 + stream, 256);
                    }
                } else {
                    any_raised = __any_sync(0xffffffffu, raise_it);
                }
                if (any_raised) {
                    float keep = 1.0f;
                    if (raise_it) {
                        keep = exp2_fast((top - peak) * scale);
                        top = peak;
                        sum *= keep;
                    }
                    // (The products so far are done: these scores were issued behind them.)
#pragma unroll 1
                    for (int i = half * (DP / 32 / kHalves); began && i < (half + 1) * (DP / 32 / kHalves); ++i) {
                        uint32_t o[32];
                        tmem_load(o, o_at + 32 * i);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_store(o_at + 32 * i, o);
                    }
                }
                // Nothing seen yet: any reference gives weights of 0. A maximum that is inf or NaN gives NaN.
                const float ref = top == -INFINITY ? 0.0f : (top < INFINITY ? top * scale : NAN);
                const float lift = kLift<T> - ref;
                const Pair scale2 = pair_of(scale, scale), ref2 = pair_of(lift, lift);
                Pair part[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    uint32_t w[16];
                    if (none) {
                        // No row of the warp sees any of it.
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = 0;
                    } else {
                        if (kChunks > 1) {
                            tmem_load(s, s_at + 32 * i);
                            if (!plain) {
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if ((sees[i] >> e & 1) == 0) s[e] = 0xff800000u;
                            }
                        }
                        // In stages: a result is not used before its latency is over. (With a quarter of the
                        // exponentials by a polynomial on the multiply-add pipe, 16 drafted trees took 317 us for
                        // 309, 32 wide beams 73.7 us for 70.1.)
                        Pair x[16];
                        float u[16], v[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            x[e] = pair_fma(pair_of(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), scale2, ref2);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            unpair(x[e], u[e], v[e]);
                            u[e] = exp2_fast(u[e]);
                            v[e] = exp2_fast(v[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            part[e & 1] = pair_add(part[e & 1], pair_of(u[e], v[e]));
                            w[e] = Pack<T>::pair(u[e], v[e]);
                        }
                    }
                    tmem_store(s_at + 16 * i, w);
                }
                if constexpr (COPIES > 1) {  // the weights of the other copies' positions
                    const uint32_t zero[16] = {};
#pragma unroll 1
                    for (int g = 0; g < COPIES; ++g) {
                        if (g == copy) continue;
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) tmem_store(tmem + lanes + stream * 128 + g * S::kCols + 16 * i, zero);
                    }
                }
                float x0, x1;
                unpair(pair_add(part[0], part[1]), x0, x1);
                sum += x0 + x1;
                tmem_stored();
                began = true;
                fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(weights_bar);
            }
        }
        if (cur < work.hi) {
            next_piece = piece_at<S::kRows, (NQ == 2)>(c, a, work, cur, group, base, tile_units);
            fetch_ahead(next_piece);
        }
        if (!odd_known) {
            grid_wait();
            odd = __ldcg(c.status + 1) != 0;
            odd_known = true;
        }
        if (began) {
            barrier_wait(smem_address(&ctl.output[stream]), output_phase, c.status);
            output_phase ^= 1;
            fence_after();
        }
        // Weights of zero did not keep a value that is not finite out of the products. All CTAs see that
        // and leave these outputs alone.
        if (odd) continue;

        // To the output, or to this CTA's part of a divided segment (of which four columns of all rows lie
        // together).
        const bool whole = p.t0 == 0 && p.t1 == p.tiles;
        float* parts = static_cast<float*>(a.workspace) + DBS_CUDA_CACHE_WORKSPACE_ZEROED / 4;
        [[maybe_unused]] int32_t* counters = static_cast<int32_t*>(a.workspace);
        float* part = parts + static_cast<int64_t>(2 * blockIdx.x + (p.t0 == 0)) * S::kOut;
        float m = top == -INFINITY ? top : top * scale - kLift<T>, l = sum;  // base-2 reference, sum
        const bool holds_rows = (my_row & ~31) < rows && (NQ == 1 || began);  // of the warp
        if constexpr (kHalves == 2) {
            named_sync(1, kSoftThreads);  // (query_at shares the space)
            ctl.half[stream][half][row] = l;
            named_sync(1, kSoftThreads);
            l += ctl.half[stream][half ^ 1][row];
        }
        // NQ = 1: the row's 2 * COPIES results, stream by stream. A warpgroup of either stream reads the
        // outputs of both, for 32 columns of its own at a time.
        constexpr int kParts = NQ == 2 ? 1 : 2 * COPIES;
        const int streams = n_tiles > 1 ? 2 : 1;  // a segment of one tile has no second stream
        auto row_stats = [&](int r, float* ref, float* total) {
            float top_all = -INFINITY, l_all = 0.0f;
#pragma unroll
            for (int i = 0; i < kParts; ++i) top_all = fmaxf(top_all, ctl.top[i * S::kRows + r]);
            *ref = top_all == -INFINITY ? 0.0f : top_all;
#pragma unroll
            for (int i = 0; i < kParts; ++i) l_all = fmaf(ctl.sum[i * S::kRows + r], exp2_fast(ctl.top[i * S::kRows + r] - *ref), l_all);
            *total = l_all;
            return top_all;
        };
        float factor0 = 1.0f, factor1 = 0.0f;
        if constexpr (NQ == 1) {
            if constexpr (COPIES == 1) named_sync(1, kSoftThreads);  // (half shares the space)
            ctl.top[(stream * COPIES + copy) * S::kRows + my_row] = m;
            ctl.sum[(stream * COPIES + copy) * S::kRows + my_row] = l;
            fence_before();
            named_sync(1, kSoftThreads);
            fence_after();
            float ref;
            m = row_stats(my_row, &ref, &l);
            factor0 = exp2_fast(ctl.top[copy * S::kRows + my_row] - ref);
            factor1 = exp2_fast(ctl.top[(COPIES + copy) * S::kRows + my_row] - ref);
        }
        const uint32_t from = NQ == 2 ? o_at : tmem + lanes + 256;
        auto columns = [&](uint32_t (&o)[32], int i) {
            tmem_load(o, from + 32 * i);
            if constexpr (NQ == 1) {
                uint32_t x[32];
                if (streams > 1) {
                    tmem_load(x, from + 128 + 32 * i);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = 0;
                }
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    o[e] = __float_as_uint(fmaf(__uint_as_float(o[e]), factor0, __uint_as_float(x[e]) * factor1));
            }
        };
        const int64_t place = (bk * a.N + id.token) * a.Hq + p.head * a.G + id.head;
        const float inverse = l > 0.0f ? 1.0f / l : l;
        const int groups = NQ == 2 ? kHalves : 2 * kHalves, my_group = NQ == 2 ? half : stream * kHalves + half;
        if constexpr (COPIES == 1) {
            T* out = static_cast<T*>(a.out) + place * c.D;
#pragma unroll 1
            for (int i = my_group; i < DP / 32; i += groups) {
                uint32_t o[32];
                if (holds_rows) columns(o, i);
                if (!mine) continue;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (i * 32 + e * 8 >= c.D) break;
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (live) {
                            auto y = [&](int x) { return __uint_as_float(o[8 * e + x]) * inverse; };
                            v = make_uint4(Pack<T>::pair(y(0), y(1)), Pack<T>::pair(y(2), y(3)), Pack<T>::pair(y(4), y(5)),
                                           Pack<T>::pair(y(6), y(7)));
                        }
                        reinterpret_cast<uint4*>(out)[i * 4 + e] = v;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        *reinterpret_cast<uint4*>(part + ((i * 8 + e) * S::kRows + my_row) * 4) =
                            make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
            }
        } else {
            // The copies, through shared memory: a warpgroup's [copy][row][8], swizzled.
            constexpr int kEach = S::kRows / 16;  // rows that a thread puts together, four columns of each
            const int t = tid & 127, vec = t & 7;
            int64_t to[kEach];
            float scales[kEach];  // -1: rows that are not shown
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const int r = (t >> 3) + 16 * k;
                if (r >= rows) break;
                const RowId rid = row_id(a, row0 + r);
                const int64_t rbk = static_cast<int64_t>(b) * a.beams + beam0 + rid.beam;
                to[k] = ((rbk * a.N + rid.token) * a.Hq + p.head * a.G + rid.head) * c.D + vec * 4;
                float unused, l_row;
                row_stats(r, &unused, &l_row);
                scales[k] = rid.token < new_count(a, rbk) ? (l_row > 0.0f ? 1.0f / l_row : l_row) : -1.0f;
            }
            float4* stage = reinterpret_cast<float4*>(query) + stream * 1024;
#pragma unroll 1
            for (int i = my_group; i < DP / 32; i += groups) {
                if (holds_rows) {
                    uint32_t o[32];
                    columns(o, i);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        stage[row * 8 + (e ^ (row & 7))] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                                                        __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
                }
                named_sync(3 + stream, 128);
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const int r = (t >> 3) + 16 * k;
                    if (r >= rows) break;
                    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int j = 0; j < COPIES; ++j) {
                        const float4 x = stage[(j * S::kRows + r) * 8 + (vec ^ (r & 7))];
                        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
                    }
                    if (i * 32 + vec * 4 >= c.D) continue;
                    if (whole) {
                        const float f = scales[k];
                        uint2 v = make_uint2(Pack<T>::pair(o.x * f, o.y * f), Pack<T>::pair(o.z * f, o.w * f));
                        if (f == -1.0f) v = make_uint2(0, 0);
                        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + to[k] + i * 32) = v;
                    } else {
                        *reinterpret_cast<float4*>(part + ((i * 8 + vec) * S::kRows + r) * 4) = o;
                    }
                }
                named_sync(3 + stream, 128);
            }
        }
        if (mine && half == 0 && copy == 0 && (NQ == 2 || stream == 0)) {
            if (whole) {
                if (a.lse != nullptr) a.lse[place] = live && l != 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
            } else {
                part[S::kRows * DP + my_row] = m;
                part[S::kRows * DP + S::kRows + my_row] = l;
            }
        }
        if constexpr (S::kJoined) {
            if (whole) continue;
            named_sync(1, kSoftThreads);
            const Span span = span_of(work, p);
            if (tid == 0) {
                __threadfence();  // of all the threads' stores, which the barrier put before this
                const int before = atomicAdd(counters + span.c0, 1);
                ctl.last = before == span.c1 - span.c0;
                if (ctl.last) counters[span.c0] = 0;
            }
            named_sync(1, kSoftThreads);
            if (!ctl.last) continue;
            __threadfence();
            join_parts<T, S::kRows, DP, kSoftThreads>(c, a, p, span, b, beam0, row0, rows, parts, query, tid);
        }
    }
    fence_before();
    named_sync(2, kSoftThreads + 32);
    if (odd) attend_all_rows<T>(c, a, reinterpret_cast<float*>(query), warp, kSoftThreads / 32);
}

// Joins the divided segments of blocks of 128 rows and more, an eighth of a block a CTA, and a segment by
// the CTAs numbered after the one that has its first tile. The last of a segment's CTAs alone would read
// parts of 64 or 128 KB: 8 sequences of 32 beams over 4060 took 88 us, 6 beams' drafts of 18 over 1222
// 41.5 us; with this kernel 74 and 34 (84 and 36 with four CTAs a segment). Smaller blocks' parts are
// joined within less time than a kernel takes to start.
constexpr int kJoinThreads = 256, kJoinCtas = 8;  // of a segment

template <class T, int kRows, int DP>
__global__ void __launch_bounds__(kJoinThreads, 4)
attend_join_kernel(const __grid_constant__ CacheView c, const __grid_constant__ AttendParams a, int ctas) {
    constexpr int kJoin = kRows / kJoinCtas;
    __shared__ __align__(16) uint8_t scratch[join_scratch(kJoin)];
    __shared__ int sums[35];
    __shared__ WorkSplit found;
    grid_release();
    const int cta = blockIdx.x / kJoinCtas, first = blockIdx.x % kJoinCtas * kJoin, tile_units = kTileKeys >> c.page_log2;
    const WorkSplit work = split_work<kRows, (kRows > 128)>(c, a, tile_units, kMinTiles, kSpareTiles, sums, &found, cta, ctas);
    Piece p{};
    bool divided = false;  // a segment begins among this CTA's tiles and ends past them
    if (work.lo < work.hi) {
        int group = work.group;
        int64_t base = work.base;
        p = piece_at<kRows, (kRows > 128)>(c, a, work, work.hi - 1, group, base, tile_units);
        divided = p.first >= work.lo && p.first + p.tiles > work.hi;
    }
    const int row0 = p.block * kRows, rows = p.rows - row0 < kRows ? p.rows - row0 : kRows;
    // Those with nothing to do make room; the first one stays, so that this grid ends after the attention.
    divided = divided && first < rows;
    if (!divided && blockIdx.x != 0) return;
    grid_wait();
    // (After a value that was not finite the outputs are complete.)
    if (!divided || __ldcg(c.status + 1) != 0) return;
    const Span span{cta, cta_of(work, p.first + p.tiles - 1)};
    const int b = p.group / c.groups, beam0 = (p.group - b * c.groups) * kGroupBeams;
    join_parts<T, kRows, DP, kJoinThreads, kJoin, 2, 4>(c, a, p, span, b, beam0, row0, rows,
                                                        static_cast<const float*>(a.workspace) + DBS_CUDA_CACHE_WORKSPACE_ZEROED / 4, scratch, threadIdx.x, first);
}

template <class T, int DP, int NQ, int COPIES, bool SKIP>
cudaError_t launch_shape(const CacheView& c, const CUtensorMap& map, const AttendParams& a, int sm_count,
                         cudaStream_t stream) {
    using S = Shape<DP, NQ, COPIES>;
    static_assert(S::kBytes <= 227 * 1024 && S::kSlots >= 4 && S::kOut <= Shape<128, 2, 1>::kOut);
    auto* kernel = attend_tc_kernel<T, DP, NQ, COPIES, SKIP>;
    static std::atomic<uint64_t> ready{0};  // a bit a device
    cudaError_t e = allow_shared(kernel, S::kBytes, ready);
    if (e == cudaSuccess) e = launch_after(kernel, sm_count, S::kThreads, S::kBytes, stream, map, c, a);
    if constexpr (!S::kJoined) {
        if (e == cudaSuccess) e = launch_after(attend_join_kernel<T, S::kRows, DP>, kJoinCtas * sm_count, kJoinThreads, 0, stream, c, a, sm_count);
    }
    return e;
}

template <class T, int DP>
cudaError_t launch_width(const CacheView& c, const CUtensorMap& map, const AttendParams& a, int sm_count,
                         cudaStream_t stream) {
    const int rows = attend_tc_shape(c, a).rows;
    if (rows == 32) return launch_shape<T, DP, 1, 4, false>(c, map, a, sm_count, stream);
    if (rows == 64) return launch_shape<T, DP, 1, 2, false>(c, map, a, sm_count, stream);
    if (rows == 128) return launch_shape<T, DP, 1, 1, false>(c, map, a, sm_count, stream);
    // Several blocks of several beams: a block passes over the tiles of which its beams hold nothing (17 beams
    // of 62 tokens over 72: 92 us, so 81, and 79 with the exponentials as they are now). Where every block has
    // all beams that costs registers for nothing (16 drafted trees: 347 us, so 360).
    if (group_rows(a) > 256 && a.beams > 1) return launch_shape<T, DP, 2, 1, true>(c, map, a, sm_count, stream);
    return launch_shape<T, DP, 2, 1, false>(c, map, a, sm_count, stream);
}

template <class T>
cudaError_t launch_typed(const CacheView& c, const CUtensorMap& map, const AttendParams& a, int sm_count,
                         cudaStream_t stream) {
    return c.D <= 64 ? launch_width<T, 64>(c, map, a, sm_count, stream) : launch_width<T, 128>(c, map, a, sm_count, stream);
}

}  // namespace

BlockShape attend_tc_shape(const CacheView&, const AttendParams& a) {
    const int64_t rows = group_rows(a);
    return {rows <= 32 ? 32 : (rows <= 64 ? 64 : (rows <= 128 ? 128 : 256)), kTileKeys};
}

int64_t attend_tc_workspace(const CacheView&, const AttendParams&, int sm_count) {
    // A counter for each CTA first, then two partial results for each.
    return DBS_CUDA_CACHE_WORKSPACE_ZEROED + static_cast<int64_t>(2) * sm_count * Shape<128, 2, 1>::kOut * 4;
}

cudaError_t launch_attend_tc(const CacheView& c, int dtype, const AttendParams& a, int sm_count, cudaStream_t stream) {
    CUtensorMap map;
    if (!page_map(c, dtype, &map)) return cudaErrorInvalidValue;
    if (dtype == DBS_CUDA_DTYPE_F16) return launch_typed<__half>(c, map, a, sm_count, stream);
    return launch_typed<__nv_bfloat16>(c, map, a, sm_count, stream);
}

}  // namespace dbsb
