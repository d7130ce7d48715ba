// One more token for each of N sequences whose states are pages of a pool: S = exp(g) S + k v^T in place, y = scale S^T q (gfx950).
// Bound by the pages, read and written once, past the caches' favour (512 sequences of 12 heads, 201 MB: 43 us where three pools take turns, 4 more without; pools that the
// last-level cache holds from step to step lose by it, 88 us for 81 with one pool of 201 MB): a workgroup holds 64 columns of one head's state in registers (four rows of sixty-four columns a wave
// instruction, 16 bytes a lane; sixteen rows a workgroup), with every load of the page on its way before the first is used.
// A slot that several rows name takes their tokens in the rows' order: the first row's workgroup goes through the others, which do nothing.
#include "vrwkv_common.h"
#include <algorithm>

namespace vrwkv {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int THREADS = 256, COLS = 64;

struct StepParams {
    const void *q, *k, *v, *g, *slots;
    void* y;
    float* pool;
    long long q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, g_sn, g_sh, page;
    int slots64, g_dtype, N, P, H, share_q, share_k, share_v, Dk, Dv, vec;
    float scale;
};
__device__ __forceinline__ long long slot_of(const StepParams& p, int n) {
    if (!p.slots) return n;
    return p.slots64 ? static_cast<const long long*>(p.slots)[n] : (long long)static_cast<const int*>(p.slots)[n];
}

constexpr int GRID_Y = 32768;
__device__ __forceinline__ float gate_at(const StepParams& p, long long i) {
    return p.g_dtype == VRWKV_F32 ? static_cast<const float*>(p.g)[i] : p.g_dtype == VRWKV_BF16 ? to_f32(static_cast<const __hip_bfloat16*>(p.g)[i]) : to_f32(static_cast<const __half*>(p.g)[i]);
}

// NX: sixteenths of the rows of a state
template <typename IO, int NX>
__global__ __launch_bounds__(THREADS) void step_kernel(const StepParams p) {
    __shared__ f32x4 red[4][16];
    __shared__ int found[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, cg = tid & 15, rg = tid >> 4;
    const int two = p.Dv > COLS ? 1 : 0;                  // tiles of a head next to each other
    const int z = blockIdx.x & two, h = blockIdx.x >> two, n0 = blockIdx.y + GRID_Y * blockIdx.z;
    if (n0 >= p.N) return;
    const int d = z * COLS + 4 * cg;
    const long long slot = slot_of(p, n0);
    const bool known = slot >= 0 && slot < p.P;

    float* const page = p.pool + (known ? slot : 0) * p.page + (long long)h * p.Dk * p.Dv;
    f32x4 S[NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) {
        const int x = rg + 16 * i;
        S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (known && x < p.Dk) {
            const float* r = page + (long long)x * p.Dv + d;
            if (p.vec && d < p.Dv) S[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(r));
            else
                for (int c = 0; c < 4; ++c)
                    if (d + c < p.Dv) S[i][c] = r[c];
        }
    }
    // a token's numbers: fetched with the page, before anything is waited for
    float kk[NX], qq[NX], dec;
    f32x4 vv;
    const auto token = [&](int n) {
        const IO* q = static_cast<const IO*>(p.q) + n * p.q_sn + (h / p.share_q) * p.q_sh;
        const IO* k = static_cast<const IO*>(p.k) + n * p.k_sn + (h / p.share_k) * p.k_sh;
        const IO* v = static_cast<const IO*>(p.v) + n * p.v_sn + (h / p.share_v) * p.v_sh;
        dec = gate_at(p, n * p.g_sn + h * p.g_sh);
#pragma unroll
        for (int c = 0; c < 4; ++c) vv[c] = d + c < p.Dv ? to_f32(v[d + c]) : 0.f;
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const int x = rg + 16 * i;
            kk[i] = x < p.Dk ? to_f32(k[x]) : 0.f;
            qq[i] = x < p.Dk ? to_f32(q[x]) : 0.f;
        }
    };
    token(n0);
    // the next row behind `after` with this slot, N if none
    const auto next_row = [&](int after) {
        int best = p.N;
        for (int i = after + 1 + tid; i < p.N; i += THREADS)
            if (slot_of(p, i) == slot) { best = i; break; }
#pragma unroll
        for (int o = 32; o; o >>= 1) best = min(best, __shfl_xor(best, o));
        __syncthreads();
        if (lane == 0) found[wave] = best;
        __syncthreads();
        return min(min(found[0], found[1]), min(found[2], found[3]));
    };
    int n = n0, next = p.N;
    if (known && p.slots) {
        int others = 0;                                   // rows with the same slot, which are few if any: 1 in front of this one, 2 behind
        for (int i = tid; i < p.N; i += THREADS)
            if (i != n0 && slot_of(p, i) == slot) others |= i < n0 ? 1 : 2;
        if (__syncthreads_or(others)) {
            if (__syncthreads_or(others & 1)) return;
            next = next_row(n0);
        }
    }
    for (;;) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        const float e = expf(dec);
        if (known) {
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                const bool there = rg + 16 * i < p.Dk;    // (a row that is not: its zeros would be NaN beside an infinity of v)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    S[i][c] = there ? fmaf(S[i][c], e, kk[i] * vv[c]) : 0.f;
                    y[c] = fmaf(qq[i], S[i][c], y[c]);
                }
            }
        }
        if (next >= p.N && known) {
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                const int x = rg + 16 * i;
                if (x < p.Dk) {
                    float* r = page + (long long)x * p.Dv + d;
                    if (p.vec && d < p.Dv) __builtin_nontemporal_store(S[i], reinterpret_cast<f32x4*>(r));
                    else
                        for (int c = 0; c < 4; ++c)
                            if (d + c < p.Dv) r[c] = S[i][c];
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            y[c] += __shfl_xor(y[c], 16);
            y[c] += __shfl_xor(y[c], 32);
        }
        if (lane < 16) red[wave][lane] = y;
        __syncthreads();
        if (tid < COLS && z * COLS + tid < p.Dv) {
            const int c = tid & 3, l = tid >> 2;
            float s = p.scale * ((red[0][l][c] + red[1][l][c]) + (red[2][l][c] + red[3][l][c]));
            if (!known) s = slot == -1 ? 0.f : __builtin_nanf("");
            static_cast<IO*>(p.y)[((long long)n * p.H + h) * p.Dv + z * COLS + tid] = from_f32<IO>(s);
        }
        if (next >= p.N) break;
        n = next;
        next = next_row(n);
        token(n);
        __syncthreads();
    }
}

template <typename IO>
int launch_step(const StepParams& p, hipStream_t st) {
    const dim3 grid((unsigned)(p.H * (p.Dv > COLS ? 2 : 1)), (unsigned)std::min(p.N, GRID_Y), (unsigned)((p.N + GRID_Y - 1) / GRID_Y)), block(THREADS);
    if (p.Dk <= 64) hipLaunchKernelGGL((step_kernel<IO, 4>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((step_kernel<IO, 8>), grid, block, 0, st, p);
    return check_launch("vrwkv_decay_step");
}

}  // namespace
}  // namespace vrwkv

using namespace vrwkv;

extern "C" int vrwkv_decay_step(const vrwkv_decay_step_args* args, void* hip_stream) {
    const char* who = "vrwkv_decay_step";
    if (!args || !args->q || !args->k || !args->v || !args->g || !args->y || !args->pool) { set_error("%s: null pointer", who); return VRWKV_INVALID_ARG; }
    const vrwkv_decay_step_args& a = *args;
    if (a.N <= 0 || a.P <= 0 || a.H <= 0 || a.Hq <= 0 || a.Hk <= 0 || a.Hv <= 0) { set_error("%s: N, P and the numbers of heads must be positive", who); return VRWKV_INVALID_ARG; }
    if (a.dtype < VRWKV_F32 || a.dtype > VRWKV_F16 || a.g_dtype < VRWKV_F32 || a.g_dtype > VRWKV_F16) { set_error("%s: dtype must be fp32, bf16 or fp16", who); return VRWKV_UNSUPPORTED_DTYPE; }
    if (a.H % a.Hq || a.H % a.Hk || a.H % a.Hv) { set_error("%s: H (%d) must be a multiple of the heads of q, k and v (%d, %d, %d)", who, a.H, a.Hq, a.Hk, a.Hv); return VRWKV_UNSUPPORTED_SHAPE; }
    if (a.Dk < 1 || a.Dk > 128 || a.Dv < 1 || a.Dv > 128) { set_error("%s: head sizes (%d, %d) must be 1 to 128", who, a.Dk, a.Dv); return VRWKV_UNSUPPORTED_SHAPE; }
    if (!a.slots && a.N > a.P) { set_error("%s: %d rows without slots, and %d pages", who, a.N, a.P); return VRWKV_INVALID_ARG; }
    if (a.page_stride < (long long)a.H * a.Dk * a.Dv) { set_error("%s: pages overlap", who); return VRWKV_INVALID_ARG; }
    if ((long long)a.N * a.H * 2 >= 1LL << 24) { set_error("%s: too many rows and heads", who); return VRWKV_UNSUPPORTED_SHAPE; }
    const size_t e = a.dtype == VRWKV_F32 ? 4 : 2, ge = a.g_dtype == VRWKV_F32 ? 4 : 2;
    if ((((size_t)a.q | (size_t)a.k | (size_t)a.v | (size_t)a.y) & (e - 1)) || ((size_t)a.g & (ge - 1)) || ((size_t)a.pool & 3) || (a.slots && ((size_t)a.slots & (a.slots64 ? 7 : 3)))) {
        set_error("%s: a tensor is not aligned to its elements", who);
        return VRWKV_INVALID_ARG;
    }
    StepParams p{a.q, a.k, a.v, a.g, a.slots, a.y, a.pool, a.q_stride[0], a.q_stride[1], a.k_stride[0], a.k_stride[1], a.v_stride[0], a.v_stride[1],
                 a.g_stride[0], a.g_stride[1], a.page_stride, a.slots64, a.g_dtype, a.N, a.P, a.H, a.H / a.Hq, a.H / a.Hk, a.H / a.Hv, a.Dk, a.Dv,
                 ((size_t)a.pool & 15) == 0 && a.Dv % 4 == 0 && a.page_stride % 4 == 0, a.scale};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (a.dtype == VRWKV_F32) return launch_step<float>(p, st);
    if (a.dtype == VRWKV_BF16) return launch_step<__hip_bfloat16>(p, st);
    return launch_step<__half>(p, st);
}
