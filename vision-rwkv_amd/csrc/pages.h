#pragma once
#include "vrwkv_common.h"

namespace vrwkv {

// The pages of a pool that a step's rows name (NULL: row n has page n).
struct Slots {
    const void* p;
    int is64, rows, pages;
    __device__ __forceinline__ long long at(int n) const { return !p ? n : is64 ? static_cast<const long long*>(p)[n] : (long long)static_cast<const int*>(p)[n]; }
    __device__ __forceinline__ bool has(long long slot) const { return slot >= 0 && slot < pages; }
    // Rows of one page are tokens behind each other: the workgroup of the first takes them all.  Whether row n0's is the first; next: the row behind it, `rows` if
    // there is none, as nearly always.  For all threads of a workgroup together.
    __device__ __forceinline__ bool first_of_page(int n0, long long slot, int& next) const {
        next = rows;
        if (!p || !has(slot)) return true;
        int others = 0;                                    // 1: a row in front, 2: one behind
        for (int i = threadIdx.x; i < rows; i += blockDim.x)
            if (i != n0 && at(i) == slot) others |= i < n0 ? 1 : 2;
        if (!__syncthreads_or(others)) return true;
        if (__syncthreads_or(others & 1)) return false;
        next = behind(n0, slot);
        return true;
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
