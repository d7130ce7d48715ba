#pragma once
#include "vrwkv_common.h"

namespace vrwkv {

// Values exchanged between the lanes of a group of P = 2, 4, 8 or 16 neighbours, in registers.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_ROW_BROADCAST = 0x150;                  // + a lane of the row of sixteen

// x of lane Q of the group
template <int P, int Q>
__device__ __forceinline__ float from_lane(float x) {
    if constexpr (P == 2) return dpp<Q | Q << 2 | (2 + Q) << 4 | (2 + Q) << 6>(x);
    else if constexpr (P == 4) return dpp<Q * 0x55>(x);
    else if constexpr (P == 8) {
        const int low = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), DPP_ROW_BROADCAST + Q, 0xf, 0xf, true);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(low, __builtin_bit_cast(int, x), DPP_ROW_BROADCAST + 8 + Q, 0xf, 0xc, false));
    } else return dpp<DPP_ROW_BROADCAST + Q>(x);
}
// x of a lane whose bit M differs (and, for 4 and 8, the bits below as well)
template <int M>
__device__ __forceinline__ float across(float x) {
    if constexpr (M == 1) return dpp<0xB1>(x);            // quad_perm [1,0,3,2]
    else if constexpr (M == 2) return dpp<0x4E>(x);       // quad_perm [2,3,0,1]
    else if constexpr (M == 4) return dpp<0x141>(x);      // row_half_mirror
    else return dpp<0x140>(x);                            // row_mirror
}
// v[i * P + q] of every lane, summed over the group's lanes and left in lane q as v[i]: at each step a lane keeps one half of its sums and gets the other lanes'
// parts of it, so that P sums cost 3 (P - 1) instructions and not P log2(P).
template <int P, int COUNT, int M = P / 2>
__device__ __forceinline__ void sum_to_lanes(float (&v)[COUNT], int p) {
    if constexpr (M >= 1) {
        const bool up = p & M;
#pragma unroll
        for (int i = 0; i < COUNT / P; ++i)
#pragma unroll
            for (int q = 0; q < M; ++q) {
                const float a = v[i * P + q], b = v[i * P + q + M];
                v[i * P + q] = (up ? b : a) + across<M>(up ? a : b);
            }
        sum_to_lanes<P, COUNT, M / 2>(v, p);
    }
}

}  // namespace vrwkv
