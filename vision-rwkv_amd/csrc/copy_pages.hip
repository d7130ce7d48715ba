// Pages of a pool copied by a list of (from, to), every page as it was before the call (gfx950): forks, moves over pages that move as well, cleared pages.
// Bound by the pages' bytes.  An entry whose source no other entry overwrites and whose target no other reads goes by itself ("free"); the others
// ("tied") go strip by strip: a workgroup reads its strip of all their sources into the LDS before it writes one of their targets, so the strips need
// nothing of each other and no page is copied twice.
#include "vrwkv_common.h"
#include <algorithm>

namespace vrwkv {
namespace {

constexpr int THREADS = 256, MAX_LIST = 4096, TIED_BYTES = 96 * 1024, STRIP = 16 * 1024, TIED_THREADS = 512;
enum { SKIP = 0, FREE = 1, TIED = 2 };

struct PageParams {
    char* pool;
    const char* source;
    const void *from, *to;
    int* plan;
    long long stride, source_stride, bytes;
    int from64, to64, M, P, source_P, same;
};
__device__ __forceinline__ long long index_at(const void* p, int wide, int i) {
    return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// A wave for each entry.
__global__ __launch_bounds__(THREADS) void plan_kernel(const PageParams p) {
    const int i = blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= p.M) return;
    const long long from = index_at(p.from, p.from64, i), to = index_at(p.to, p.to64, i);
    bool good = to >= 0 && to < p.P && from >= -1 && from < p.source_P && !(p.same && from == to);
    bool later = false, tied = false;
    for (int j = lane; j < p.M; j += 64) {
        const long long f = index_at(p.from, p.from64, j), t = index_at(p.to, p.to64, j);
        later |= j > i && t == to && f >= -1 && f < p.source_P;
        tied |= p.same && j != i && (f == to || (t == from && from >= 0));
    }
    good = good && !__any(later);
    tied = __any(tied);
    if (lane == 0) p.plan[i] = good ? (tied ? TIED : FREE) : SKIP;
}

// U: 16, 4, 2 or 1 bytes at a time
template <typename U>
__global__ __launch_bounds__(THREADS) void free_kernel(const PageParams p, int strips) {
    const int i = blockIdx.x / strips, s = blockIdx.x % strips;
    if (p.plan[i] != FREE) return;
    const long long from = index_at(p.from, p.from64, i), to = index_at(p.to, p.to64, i);
    const long long units = p.bytes / sizeof(U), u0 = (long long)s * (STRIP / sizeof(U)) + threadIdx.x;
    const U* src = reinterpret_cast<const U*>(p.source + (from < 0 ? 0 : from) * p.source_stride);
    U* dst = reinterpret_cast<U*>(p.pool + to * p.stride);
    constexpr int N = 4;
    for (int k = 0; k < (int)(STRIP / sizeof(U)); k += N * THREADS) {
        U t[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const long long u = u0 + k + e * THREADS;
            t[e] = U{};
            if (from >= 0 && u < units) t[e] = src[u];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const long long u = u0 + k + e * THREADS;
            if (u < units) dst[u] = t[e];
        }
    }
}

template <typename U>
__global__ __launch_bounds__(TIED_THREADS) void tied_kernel(const PageParams p) {
    __shared__ int list[MAX_LIST];                        // tied entries
    __shared__ U data[TIED_BYTES / sizeof(U)];
    __shared__ int count;
    const int tid = threadIdx.x;
    if (tid == 0) count = 0;
    __syncthreads();
    for (int i = tid; i < p.M; i += TIED_THREADS)
        if (p.plan[i] == TIED) list[atomicAdd(&count, 1)] = i;    // (in any order: targets differ)
    __syncthreads();
    const int m = count;
    if (m == 0) return;
    const long long units = p.bytes / sizeof(U);
    // units of a page that a strip holds: as many as the LDS has room for, a power of two up to 1 KB
    int width = 1;
    while (2 * width * m <= (int)(TIED_BYTES / sizeof(U)) && 2 * width * (int)sizeof(U) <= 1024) width *= 2;
    const long long strips = (units + width - 1) / width;
    for (long long s = blockIdx.x; s < strips; s += gridDim.x) {
        for (int e = tid; e < m * width; e += TIED_THREADS) {
            const int i = list[e / width];
            const long long from = index_at(p.from, p.from64, i), u = s * width + e % width;
            data[e] = from >= 0 && u < units ? reinterpret_cast<const U*>(p.source + from * p.source_stride)[u] : U{};
        }
        __syncthreads();
        for (int e = tid; e < m * width; e += TIED_THREADS) {
            const int i = list[e / width];
            const long long to = index_at(p.to, p.to64, i), u = s * width + e % width;
            if (u < units) reinterpret_cast<U*>(p.pool + to * p.stride)[u] = data[e];
        }
        __syncthreads();
    }
}

template <typename U>
void launch_copies(const PageParams& p, hipStream_t st) {
    const int strips = (int)((p.bytes + STRIP - 1) / STRIP);
    hipLaunchKernelGGL((free_kernel<U>), dim3((unsigned)((long long)p.M * strips)), dim3(THREADS), 0, st, p, strips);
    if (p.same && p.M > 1) hipLaunchKernelGGL((tied_kernel<U>), dim3(device_cus()), dim3(TIED_THREADS), 0, st, p);
}

}  // namespace
}  // namespace vrwkv

using namespace vrwkv;

extern "C" size_t vrwkv_copy_pages_workspace_bytes(int M) { return M > 0 ? (size_t)M * sizeof(int) : 0; }

extern "C" int vrwkv_copy_pages(void* pool, long long stride, int P, const void* source, long long source_stride, int source_P, long long page_bytes,
                                const void* from, int from64, const void* to, int to64, int M, void* workspace, size_t workspace_bytes, void* hip_stream) {
    const char* who = "vrwkv_copy_pages";
    if (!pool || !source || !from || !to) { set_error("%s: null pointer", who); return VRWKV_INVALID_ARG; }
    if (M <= 0 || P <= 0 || source_P < 0 || page_bytes <= 0) { set_error("%s: sizes must be positive", who); return VRWKV_INVALID_ARG; }
    if (M > MAX_LIST) { set_error("%s: %d entries, at most %d", who, M, MAX_LIST); return VRWKV_UNSUPPORTED_SHAPE; }
    if (stride < page_bytes || source_stride < page_bytes) { set_error("%s: pages overlap", who); return VRWKV_INVALID_ARG; }
    if (((page_bytes + STRIP - 1) / STRIP) * M >= 1LL << 24) { set_error("%s: too many bytes", who); return VRWKV_UNSUPPORTED_SHAPE; }
    if (((size_t)from & (from64 ? 7 : 3)) || ((size_t)to & (to64 ? 7 : 3))) { set_error("%s: an index is not aligned to its elements", who); return VRWKV_INVALID_ARG; }
    if (!workspace || workspace_bytes < vrwkv_copy_pages_workspace_bytes(M)) { set_error("%s: workspace of %zu bytes, %zu needed", who, workspace ? workspace_bytes : 0, vrwkv_copy_pages_workspace_bytes(M)); return VRWKV_WORKSPACE_TOO_SMALL; }
    if ((size_t)workspace & 3) { set_error("%s: workspace must be 4-byte aligned", who); return VRWKV_INVALID_ARG; }
    const char *a = static_cast<const char*>(pool), *b = static_cast<const char*>(source);
    const bool same = a == b && stride == source_stride;
    const long long a_end = (P - 1) * stride + page_bytes, b_end = source_P ? (source_P - 1) * source_stride + page_bytes : 0;
    if (!same && a < b + b_end && b < a + a_end) { set_error("%s: the source overlaps the pool", who); return VRWKV_INVALID_ARG; }
    PageParams p{static_cast<char*>(pool), b, from, to, static_cast<int*>(workspace), stride, source_stride, page_bytes, from64, to64, M, P, source_P, same};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    hipLaunchKernelGGL(plan_kernel, dim3((M + THREADS / 64 - 1) / (THREADS / 64)), dim3(THREADS), 0, st, p);
    const size_t bits = (size_t)pool | (size_t)source | (size_t)stride | (size_t)source_stride | (size_t)page_bytes;
    if (!(bits & 15)) launch_copies<uint4>(p, st);
    else if (!(bits & 3)) launch_copies<unsigned>(p, st);
    else if (!(bits & 1)) launch_copies<unsigned short>(p, st);
    else launch_copies<unsigned char>(p, st);
    return check_launch(who);
}
