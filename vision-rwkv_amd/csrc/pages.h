#pragma once
#include "vrwkv_common.h"

namespace vrwkv {

// The pages of a pool that a step's rows name (NULL: row n has page n).
struct Slots {
    const void* p;
    int is64, rows, pages;
    __device__ __forceinline__ long long at(int n) const { return !p ? n : is64 ? static_cast<const long long*>(p)[n] : (long long)static_cast<const int*>(p)[n]; }
    __device__ __forceinline__ bool has(long long slot) const { return slot >= 0 && slot < pages; }
    // Rows of one page are tokens behind each other: the workgroup of the first takes them all.  Of the rows n0 .. n0 + R - 1: `skipped`, a bit for each that is not the first of its
    // page, and `shared`, for each that has others behind it (nearly always neither).  For all threads of a workgroup together.
    template <int R>
    __device__ __forceinline__ void find_others(int n0, const long long (&slot)[R], unsigned& skipped, unsigned& shared) const {
        skipped = shared = 0;
        if (!p) return;
        __shared__ unsigned found[2];
        unsigned front = 0, back = 0;
        for (int i = threadIdx.x; i < rows; i += blockDim.x) {
            const long long s = at(i);
            if (!has(s)) continue;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (s == slot[r] && i != n0 + r) (i < n0 + r ? front : back) |= 1u << r;
        }
        if (!__syncthreads_or(front | back)) return;
        if (threadIdx.x < 2) found[threadIdx.x] = 0;
        __syncthreads();
        if (front) atomicOr(&found[0], front);             // (bits: the order does not matter)
        if (back) atomicOr(&found[1], back);
        __syncthreads();
        skipped = found[0], shared = found[1];
    }
    __device__ __forceinline__ int behind(int after, long long slot) const {
        __shared__ int found;
        if (threadIdx.x == 0) found = rows;
        __syncthreads();
        for (int i = after + 1 + threadIdx.x; i < rows; i += blockDim.x)
            if (at(i) == slot) {
                atomicMin(&found, i);                      // (whole numbers: the order does not matter)
                break;
            }
        __syncthreads();
        const int n = found;
        __syncthreads();
        return n;
    }
};

}  // namespace vrwkv
