// SPDX-License-Identifier: MIT
//
// C ABI of the paged beam cache (include/dbs_cuda_cache.h): argument checks and launches.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <limits>

#include "cache.cuh"

namespace dbsb {
namespace {

constexpr int64_t kMaxElements = int64_t{1} << 46;

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int elem_bytes(int code) {
    if (code == DBS_CUDA_DTYPE_F32) return 4;
    return code == DBS_CUDA_DTYPE_F16 || code == DBS_CUDA_DTYPE_BF16 ? 2 : 0;
}

int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    static int known[64] = {};  // a device's count never changes: a racing store writes the same
    if (dev < 64 && known[dev] > 0) return known[dev];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
    if (dev < 64) known[dev] = n;
    return n;
}

// Sizes that the kernels take. Slots, table entries and units are counted in 31 bits, pages of a
// layer and kind too.
bool valid_sizes(const DBSCudaCache* c) {
    if (c == nullptr || c->reserved0 != 0) return false;
    for (int32_t n : {c->batch_size, c->beam_size, c->max_pages, c->num_pages, c->num_layers, c->num_heads, c->head_dim})
        if (n < 1) return false;
    if (c->beam_size > DBS_CUDA_MAX_BEAM || c->head_dim > DBS_CUDA_CACHE_MAX_HEAD_DIM || c->head_dim % 8 != 0) return false;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64) return false;
    if (elem_bytes(c->data_type) == 0) return false;
    const int64_t int_max = std::numeric_limits<int32_t>::max();
    if (static_cast<int64_t>(c->max_pages) * c->page_size > int_max / 2) return false;
    if (static_cast<int64_t>(c->batch_size) * c->beam_size > int_max / c->max_pages) return false;
    if (c->num_heads > 65536 || c->num_layers > 65536) return false;
    const double rows = 2.0 * c->num_layers * c->num_pages * c->num_heads * c->page_size;
    return rows < int_max && rows * c->head_dim < static_cast<double>(kMaxElements);
}

CacheView view_of(const DBSCudaCache& c) {
    CacheView v = {};
    v.B = c.batch_size, v.K = c.beam_size, v.M = c.max_pages, v.P = c.num_pages;
    v.L = c.num_layers, v.H = c.num_heads, v.D = c.head_dim, v.page = c.page_size;
    v.page_log2 = c.page_size == 16 ? 4 : (c.page_size == 32 ? 5 : 6);
    v.elem = elem_bytes(c.data_type);
    v.groups = (c.beam_size + kGroupBeams - 1) / kGroupBeams;
    v.unit_cap = (c.beam_size < kGroupBeams ? c.beam_size : kGroupBeams) * c.max_pages;
    v.pages = c.pages;
    v.table = c.table;
    v.lengths = c.lengths;
    v.references = c.references;
    v.status = c.status;
    return v;
}

// The view of a cache whose arrays are in place; false: refused.
bool open(const DBSCudaCache* c, CacheView& v) {
    if (!valid_sizes(c)) return false;
    for (const void* p : {static_cast<const void*>(c->table), static_cast<const void*>(c->lengths),
                          static_cast<const void*>(c->status)})
        if (p == nullptr || !aligned(p, 4)) return false;
    if (!c->pages || !aligned(c->pages, 16) || !c->references || !aligned(c->references, 16)) return false;
    if (!c->plan || !aligned(c->plan, 256)) return false;
    v = view_of(*c);
    return cache_plan_layout(v, c->plan) <= c->plan_bytes;
}

int finish(cudaError_t e, cudaStream_t stream) {
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return DBS_CUDA_STATUS_LAUNCH_FAILED;
    }
    bool sync = dbs_cuda_get_synchronization() != 0;
    for (const char* name : {"DBS_CUDA_SYNC_CHECK", "DBS_CUDA_DEBUG_SYNC"}) {
        const char* value = std::getenv(name);
        sync = sync || (value != nullptr && value[0] == '1');
    }
    if (sync && cudaStreamSynchronize(stream) != cudaSuccess) return DBS_CUDA_STATUS_LAUNCH_FAILED;
    return DBS_CUDA_STATUS_OK;
}

bool params_of(const CacheView& v, const DBSCudaAttendArgs* a, AttendParams& p) {
    if (a == nullptr || a->reserved0 != 0 || a->layer < 0 || a->layer >= v.L) return false;
    if (a->beams < 1 || a->beams > v.K || a->new_tokens < 1 || a->new_tokens > 65536) return false;
    if (a->query_heads < 1 || a->query_heads % v.H != 0 || !std::isfinite(a->scale)) return false;
    const int64_t int_max = std::numeric_limits<int32_t>::max();
    const int64_t tokens = static_cast<int64_t>(v.B) * a->beams * a->new_tokens;
    if (tokens > int_max / a->query_heads) return false;
    if (a->mask != nullptr && tokens > (int64_t{1} << 46) / a->new_tokens) return false;
    p = AttendParams{};
    p.layer = a->layer, p.beams = a->beams, p.N = a->new_tokens, p.Hq = a->query_heads, p.G = a->query_heads / v.H;
    p.scale = a->scale;
    return attend_counts_tiles(v, p);
}

}  // namespace
}  // namespace dbsb

using namespace dbsb;

extern "C" {

DBS_CUDA_EXPORT int64_t dbs_cuda_cache_plan_bytes(const DBSCudaCache* cache) {
    if (!valid_sizes(cache)) return -1;
    CacheView v = view_of(*cache);
    return cache_plan_layout(v, nullptr);
}

DBS_CUDA_EXPORT int dbs_cuda_cache_refresh(const DBSCudaCache* cache, int values, void* stream_ptr) {
    CacheView v;
    if (!open(cache, v) || values < 0 || values > DBS_CUDA_CACHE_VALUES_IF_SET) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    return finish(launch_cache_refresh(v, cache->data_type, values, sm_count(), stream), stream);
}

DBS_CUDA_EXPORT int dbs_cuda_cache_fork(const DBSCudaCache* cache, const int32_t* parents, const int32_t* written,
                                        int32_t written_all, const int32_t* room, int32_t room_all, void* stream_ptr) {
    CacheView v;
    if (!open(cache, v) || written_all < 0 || room_all < 0) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    if (!aligned(parents, 4) || !aligned(written, 4) || !aligned(room, 4)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    return finish(launch_cache_fork(v, parents, written, written_all, room, room_all, sm_count(), stream), stream);
}

DBS_CUDA_EXPORT int dbs_cuda_cache_commit(const DBSCudaCache* cache, const int32_t* path, int32_t path_stride,
                                          const int32_t* counts, int32_t room_all, void* stream_ptr) {
    CacheView v;
    if (!open(cache, v) || !path || path_stride < 1 || !counts || room_all < 0) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    if (!aligned(path, 4) || !aligned(counts, 4)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    return finish(launch_cache_commit(v, path, path_stride, counts, room_all, sm_count(), stream), stream);
}

DBS_CUDA_EXPORT int dbs_cuda_cache_compact(const DBSCudaCache* cache, void* stream_ptr) {
    CacheView v;
    if (!open(cache, v)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    return finish(launch_cache_compact(v, sm_count(), stream), stream);
}

DBS_CUDA_EXPORT int64_t dbs_cuda_cache_attend_workspace_size(const DBSCudaCache* cache, const DBSCudaAttendArgs* args) {
    if (!valid_sizes(cache)) return -1;
    const CacheView v = view_of(*cache);
    AttendParams p;
    if (!params_of(v, args, p)) return -1;
    return attend_workspace(v, p, sm_count());
}

DBS_CUDA_EXPORT int dbs_cuda_cache_attend(const DBSCudaCache* cache, const DBSCudaAttendArgs* args, void* stream_ptr) {
    CacheView v;
    AttendParams p;
    if (!open(cache, v) || !params_of(v, args, p)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const DBSCudaAttendArgs& a = *args;
    if (!a.q || !aligned(a.q, 16) || !a.out || !aligned(a.out, 16)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    if ((a.k == nullptr) != (a.v == nullptr) || !aligned(a.k, 16) || !aligned(a.v, 16)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    if (!aligned(a.counts, 4) || !aligned(a.lse, 4)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const int step = 16 / v.elem;  // rows of q, k and v are read 16 bytes at a time
    for (int i = 0; i < 4; ++i) {
        p.qs[i] = a.q_strides[i], p.ks[i] = a.k_strides[i], p.vs[i] = a.v_strides[i];
        if (p.qs[i] % step != 0 || (a.k && (p.ks[i] % step != 0 || p.vs[i] % step != 0))) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    }
    if (!a.workspace || !aligned(a.workspace, 256) || a.workspace_bytes < attend_workspace(v, p, sm_count()))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    p.q = a.q, p.k = a.k, p.v = a.v, p.mask = a.mask, p.counts = a.counts, p.out = a.out, p.lse = a.lse;
    p.workspace = a.workspace, p.workspace_bytes = a.workspace_bytes;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    return finish(launch_attend(v, cache->data_type, p, sm_count(), stream), stream);
}

}  // extern "C"
