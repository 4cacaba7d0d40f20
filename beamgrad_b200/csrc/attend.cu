// SPDX-License-Identifier: MIT
//
// Attention over the paged beam cache, and the write of the new tokens before it
// (include/dbs_cuda_cache.h gives the definition).
#include "attend.cuh"

namespace dbsb {

namespace {

constexpr int kAppendThreads = 256;

// Keys and values of the new tokens into their pages, 16 bytes a thread. A value that is not
// finite raises the cache's second status word: the attention then keeps masked values out of its
// sums element by element, where otherwise a weight of zero is enough.
template <class T>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ CacheView c, const __grid_constant__ AttendParams a) {
    grid_wait();
    grid_release();
    const int vecs = c.D / Pack<T>::n;
    const int64_t items = static_cast<int64_t>(c.B) * a.beams * a.N * c.H * vecs;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x; i < items;
         i += static_cast<int64_t>(gridDim.x) * kAppendThreads) {
        const int vec = static_cast<int>(i % vecs);
        int64_t rest = i / vecs;
        const int h = static_cast<int>(rest % c.H);
        rest /= c.H;
        const int j = static_cast<int>(rest % a.N);
        const int64_t bk = rest / a.N;
        const int64_t b = bk / a.beams, k = bk % a.beams;
        // The rows are on their way while their place is looked up.
        const T* ks = static_cast<const T*>(a.k) + b * a.ks[0] + k * a.ks[1] + j * a.ks[2] + h * a.ks[3];
        const T* vs = static_cast<const T*>(a.v) + b * a.vs[0] + k * a.vs[1] + j * a.vs[2] + h * a.vs[3];
        const uint4 kx = __ldg(reinterpret_cast<const uint4*>(ks) + vec), vx = __ldg(reinterpret_cast<const uint4*>(vs) + vec);
        const int64_t slot = b * c.K + k, pos = static_cast<int64_t>(c.lengths[slot]) + j, col = pos >> c.page_log2;
        if (j >= new_count(a, bk)) continue;
        if (col >= c.M) {
            atomicOr(c.status, DBS_CUDA_CACHE_STATUS_CAPACITY);
            continue;
        }
        const int p = c.table[slot * c.M + col];
        if (p < 0) continue;
        const int64_t block = static_cast<int64_t>(a.layer) * 2 * c.P + p;
        const int64_t row = pos & (c.page - 1);
        uint4* pages = static_cast<uint4*>(c.pages);
        pages[((block * c.H + h) * c.page + row) * vecs + vec] = kx;
        pages[(((block + c.P) * c.H + h) * c.page + row) * vecs + vec] = vx;
        if (!(Pack<T>::finite(vx.x) && Pack<T>::finite(vx.y) && Pack<T>::finite(vx.z) && Pack<T>::finite(vx.w)))
            c.status[1] = 1;
    }
}

template <class T>
cudaError_t launch_append(const CacheView& c, const AttendParams& a, int sm_count, cudaStream_t stream) {
    if (a.k == nullptr) return cudaSuccess;
    const int64_t items = static_cast<int64_t>(c.B) * a.beams * a.N * c.H * (c.D / Pack<T>::n);
    const int64_t want = (items + kAppendThreads - 1) / kAppendThreads, cap = 8 * sm_count;
    return launch_after(append_kernel<T>, static_cast<unsigned>(want < cap ? want : cap), kAppendThreads, 0, stream, c, a);
}

}  // namespace

bool attend_counts_tiles(const CacheView& c, const AttendParams& a) {
    const BlockShape shape = c.elem == 4 ? attend_f32_shape(c, a) : (c.D <= 128 ? attend_tc_shape(c, a) : attend_mma_shape(c, a));
    const int tile_units = shape.keys > c.page ? shape.keys / c.page : 1;
    const int64_t blocks = (group_rows(a) + shape.rows - 1) / shape.rows, tiles = (c.unit_cap + tile_units - 1) / tile_units;
    return static_cast<double>(tiles) * blocks * c.H * c.B * c.groups < INT_MAX;
}

int64_t attend_workspace(const CacheView& c, const AttendParams& a, int sm_count) {
    if (c.elem == 4) return attend_f32_workspace(c, a, sm_count);
    return c.D <= 128 ? attend_tc_workspace(c, a, sm_count) : attend_mma_workspace(c, a, sm_count);
}

cudaError_t launch_attend(const CacheView& c, int dtype, const AttendParams& a, int sm_count, cudaStream_t stream) {
    const cudaError_t e = dtype == DBS_CUDA_DTYPE_F32 ? launch_append<float>(c, a, sm_count, stream)
                          : dtype == DBS_CUDA_DTYPE_F16 ? launch_append<__half>(c, a, sm_count, stream)
                                                        : launch_append<__nv_bfloat16>(c, a, sm_count, stream);
    if (e != cudaSuccess) return e;
    if (dtype == DBS_CUDA_DTYPE_F32) return launch_attend_f32(c, a, sm_count, stream);
    return c.D <= 128 ? launch_attend_tc(c, dtype, a, sm_count, stream) : launch_attend_mma(c, dtype, a, sm_count, stream);
}

}  // namespace dbsb
