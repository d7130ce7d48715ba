// Pages of a pool copied by a list of (from, to), every page as it was before the call (gfx950): forks, moves over pages that move as well, cleared pages.
// Bound by the pages' bytes.  An entry whose source no other entry overwrites and whose target no other reads goes by itself ("free"); the others
// ("tied") go strip by strip: a workgroup reads its strip of all their sources into registers before it writes one of their targets, so the strips need
// nothing of each other and no page is copied twice.  Two workgroups a compute unit: one reads while the other writes.  (Strips through the LDS, one
// workgroup: 103 us for 690 of 1024 pages of 196 KB; so 74.)
#include "vrwkv_common.h"
#include <algorithm>

namespace vrwkv {
namespace {

constexpr int THREADS = 512, MAX_LIST = 4096, SMALL_LIST = 256;
enum { SKIP = 0, FREE = 1, TIED = 2 };

struct PageParams {
    char* pool;
    const char* source;
    const void *from, *to;
    int* plan;                                            // what each entry is; null: lists of up to SMALL_LIST entries, which every workgroup looks through
    long long stride, source_stride, bytes;
    int from64, to64, M, P, source_P, same;
    int strips, held, free_blocks;                        // strips of a page that goes by itself; units that a thread takes of one
};
__device__ __forceinline__ long long index_at(const void* p, int wide, int i) {
    return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}
__device__ __forceinline__ bool entry_good(const PageParams& p, long long from, long long to) {
    return to >= 0 && to < p.P && from >= -1 && from < p.source_P && !(p.same && from == to);
}
// What entry j makes of entry i: 1: i does not count, 2: i is tied.
__device__ __forceinline__ int entry_flags(const PageParams& p, int i, long long from, long long to, int j, long long f, long long t) {
    const bool later = j > i && t == to && f >= -1 && f < p.source_P, tied = p.same && j != i && (f == to || (t == from && from >= 0));
    return (later ? 1 : 0) | (tied ? 2 : 0);
}
__device__ __forceinline__ int entry_kind(bool good, int flags) { return !good || (flags & 1) ? SKIP : flags & 2 ? TIED : FREE; }

// A workgroup for each entry.
__global__ __launch_bounds__(256) void plan_kernel(const PageParams p) {
    const int i = blockIdx.x;
    const long long from = index_at(p.from, p.from64, i), to = index_at(p.to, p.to64, i);
    int flags = 0;
    for (int j = threadIdx.x; j < p.M; j += 256) flags |= entry_flags(p, i, from, to, j, index_at(p.from, p.from64, j), index_at(p.to, p.to64, j));
    const int f1 = __syncthreads_or(flags & 1), f2 = __syncthreads_or(flags & 2);
    if (threadIdx.x == 0) p.plan[i] = entry_kind(entry_good(p, from, to), (f1 ? 1 : 0) | (f2 ? 2 : 0));
}

// U: 16, 4, 2 or 1 bytes at a time.  HELD: units that a thread holds: the more, the wider the strips (690 pages of 196 KB: 92 us with 16, strips of 128 bytes; 74 with 24 and
// strips of 256; 174 with 48 and 512, one workgroup a compute unit), the fewer, the sooner a short list's few strips are begun.
template <typename U, int HELD>
__global__ __launch_bounds__(THREADS, HELD <= 16 ? 4 : 2) void copy_kernel(const PageParams p) {
    __shared__ int sfrom[MAX_LIST], sto[MAX_LIST];        // tied entries
    __shared__ long long lfrom[SMALL_LIST], lto[SMALL_LIST];
    __shared__ int count;
    const int tid = threadIdx.x;
    const long long units = p.bytes / (long long)sizeof(U);
    U t[HELD];

    if ((int)blockIdx.x < p.free_blocks) {
        const int i = blockIdx.x / p.strips, s = blockIdx.x % p.strips;
        const long long from = index_at(p.from, p.from64, i), to = index_at(p.to, p.to64, i);
        int kind;
        if (p.plan) kind = p.plan[i];
        else {
            const int flags = tid < p.M ? entry_flags(p, i, from, to, tid, index_at(p.from, p.from64, tid), index_at(p.to, p.to64, tid)) : 0;
            const int f1 = __syncthreads_or(flags & 1), f2 = __syncthreads_or(flags & 2);
            kind = entry_kind(entry_good(p, from, to), (f1 ? 1 : 0) | (f2 ? 2 : 0));
        }
        if (kind != FREE) return;
        const U* src = reinterpret_cast<const U*>(p.source + (from < 0 ? 0 : from) * p.source_stride);
        U* dst = reinterpret_cast<U*>(p.pool + to * p.stride);
        const long long u0 = (long long)s * p.held * THREADS + tid;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            t[k] = U{};
            if (k < p.held && from >= 0 && u0 + k * THREADS < units) t[k] = src[u0 + k * THREADS];
        }
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (k < p.held && u0 + k * THREADS < units) dst[u0 + k * THREADS] = t[k];
        return;
    }

    // ---- tied entries, in any order: their targets differ
    if (tid == 0) count = 0;
    if (!p.plan && tid < p.M) {
        lfrom[tid] = index_at(p.from, p.from64, tid);
        lto[tid] = index_at(p.to, p.to64, tid);
    }
    __syncthreads();
    if (p.plan) {
        for (int i = tid; i < p.M; i += THREADS)
            if (p.plan[i] == TIED) {
                const int e = atomicAdd(&count, 1);
                sfrom[e] = (int)index_at(p.from, p.from64, i);
                sto[e] = (int)index_at(p.to, p.to64, i);
            }
    } else if (tid < p.M) {
        const long long from = lfrom[tid], to = lto[tid];
        int flags = 0;
        for (int j = 0; j < p.M; ++j) flags |= entry_flags(p, tid, from, to, j, lfrom[j], lto[j]);
        if (entry_kind(entry_good(p, from, to), flags) == TIED) {
            const int e = atomicAdd(&count, 1);
            sfrom[e] = (int)from;
            sto[e] = (int)to;
        }
    }
    __syncthreads();
    const int m = count;
    if (m == 0) return;
    // units of a page that a strip holds: as many as the threads have room for, a power of two up to 1 KB
    int shift = 0;
    while ((2 << shift) * m <= HELD * THREADS && (2 << shift) * (int)sizeof(U) <= 1024) ++shift;
    const int all = m << shift, mask = (1 << shift) - 1;
    const long long strips = (units + mask) >> shift;
    for (long long s = blockIdx.x - p.free_blocks; s < strips; s += gridDim.x - p.free_blocks) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            const int e = tid + k * THREADS;
            const long long u = (s << shift) + (e & mask);
            t[k] = U{};
            if (e < all && u < units) {
                const int from = sfrom[e >> shift];
                if (from >= 0) t[k] = reinterpret_cast<const U*>(p.source + from * p.source_stride)[u];
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every source of this strip has been read ...
        __syncthreads();                                   // ... by every wave, before one of its targets is written
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            const int e = tid + k * THREADS;
            const long long u = (s << shift) + (e & mask);
            if (e < all && u < units) reinterpret_cast<U*>(p.pool + sto[e >> shift] * p.stride)[u] = t[k];
        }
    }
}

template <typename U>
void launch_copies(PageParams p, hipStream_t st) {
    const long long units = p.bytes / (long long)sizeof(U);
    const int held = p.M > SMALL_LIST ? 24 : 16;
    p.held = 16;
    while (p.held > 1 && p.M * ((units + (long long)p.held * THREADS - 1) / (p.held * THREADS)) < 2048) p.held /= 2;
    p.strips = (int)((units + (long long)p.held * THREADS - 1) / (p.held * THREADS));
    p.free_blocks = p.M * p.strips;
    // (as many as there are strips if every entry is tied)
    long long width = 1;
    while (2 * width * p.M <= held * THREADS && 2 * width * (int)sizeof(U) <= 1024) width *= 2;
    const int tied_blocks = p.same && p.M > 1 ? (int)std::min<long long>(2 * device_cus(), (units + width - 1) / width) : 0;
    const dim3 grid(p.free_blocks + tied_blocks), block(THREADS);
    if (held == 24) hipLaunchKernelGGL((copy_kernel<U, 24>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((copy_kernel<U, 16>), grid, block, 0, st, p);
}

}  // namespace
}  // namespace vrwkv

using namespace vrwkv;

extern "C" size_t vrwkv_copy_pages_workspace_bytes(int M) { return M > SMALL_LIST ? (size_t)M * sizeof(int) : 0; }

extern "C" int vrwkv_copy_pages(void* pool, long long stride, int P, const void* source, long long source_stride, int source_P, long long page_bytes,
                                const void* from, int from64, const void* to, int to64, int M, void* workspace, size_t workspace_bytes, void* hip_stream) {
    const char* who = "vrwkv_copy_pages";
    if (!pool || !source || !from || !to) { set_error("%s: null pointer", who); return VRWKV_INVALID_ARG; }
    if (M <= 0 || P <= 0 || source_P < 0 || page_bytes <= 0) { set_error("%s: sizes must be positive", who); return VRWKV_INVALID_ARG; }
    if (M > MAX_LIST) { set_error("%s: %d entries, at most %d", who, M, MAX_LIST); return VRWKV_UNSUPPORTED_SHAPE; }
    if (stride < page_bytes || source_stride < page_bytes) { set_error("%s: pages overlap", who); return VRWKV_INVALID_ARG; }
    if (((size_t)from & (from64 ? 7 : 3)) || ((size_t)to & (to64 ? 7 : 3))) { set_error("%s: an index is not aligned to its elements", who); return VRWKV_INVALID_ARG; }
    if (M > SMALL_LIST && (!workspace || workspace_bytes < vrwkv_copy_pages_workspace_bytes(M))) { set_error("%s: workspace of %zu bytes, %zu needed", who, workspace ? workspace_bytes : 0, vrwkv_copy_pages_workspace_bytes(M)); return VRWKV_WORKSPACE_TOO_SMALL; }
    if (M > SMALL_LIST && ((size_t)workspace & 3)) { set_error("%s: workspace must be 4-byte aligned", who); return VRWKV_INVALID_ARG; }
    const char *a = static_cast<const char*>(pool), *b = static_cast<const char*>(source);
    if (source_P == 1) source_stride = stride;            // (one page has no distance to a next one: it takes the other's)
    else if (P == 1) stride = source_stride;
    const bool same = a == b && stride == source_stride;
    const long long a_end = (P - 1) * stride + page_bytes, b_end = source_P ? (source_P - 1) * source_stride + page_bytes : 0;
    // (pages of the same stride that lie in each other's gaps, as those of two layers in one pool, are apart as well)
    const long long shift = ((b - a) % stride + stride) % stride;
    const bool gaps = stride == source_stride && shift >= page_bytes && shift + page_bytes <= stride;
    if (!same && !gaps && a < b + b_end && b < a + a_end) { set_error("%s: the source overlaps the pool", who); return VRWKV_INVALID_ARG; }
    PageParams p{static_cast<char*>(pool), b, from, to, M > SMALL_LIST ? static_cast<int*>(workspace) : nullptr, stride, source_stride, page_bytes, from64, to64, M, P, source_P, same, 0, 0, 0};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const size_t bits = (size_t)pool | (size_t)source | (size_t)stride | (size_t)source_stride | (size_t)page_bytes;
    const int unit = !(bits & 15) ? 16 : !(bits & 3) ? 4 : !(bits & 1) ? 2 : 1;
    // (a launch has less than 2^32 threads, of 16 units each)
    if (page_bytes / unit >= 1LL << 35 || page_bytes / unit * M >= 1LL << 35) { set_error("%s: too many bytes", who); return VRWKV_UNSUPPORTED_SHAPE; }
    if (p.plan) hipLaunchKernelGGL(plan_kernel, dim3(M), dim3(256), 0, st, p);
    if (unit == 16) launch_copies<uint4>(p, st);
    else if (unit == 4) launch_copies<unsigned>(p, st);
    else if (unit == 2) launch_copies<unsigned short>(p, st);
    else launch_copies<unsigned char>(p, st);
    return check_launch(who);
}
