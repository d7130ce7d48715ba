// The short causal convolution of each channel over the tokens (gfx950): what its forward, its gradients and its form for single tokens share.
//
//     p_t = sum_j w_j x_{t - (K-1) + j} + b        y_t = silu(p_t) or p_t        g_t = gy_t silu'(p_t)
//     dx_t = sum_j w_j g_{t + (K-1) - j}           dw_j = sum_t g_t x_{t - (K-1) + j}          db = sum_t g_t
//
// Bound by the memory: each row is read once and written once.  A lane holds VEC channels and goes along a run of tokens with the last K - 1 rows in registers, the next rows on their
// way; the K - 1 rows in front of a run are read again (from L2).  64 x 196 tokens of 1536 channels in bf16: forward 19.6 us (3.9 TB/s), gradients 37 (3.1); from
// five taps on, whose weights are read one at a time, 43 (5), 56 (6) and 65 (8), and a call of the gradients 79 to 93 for 53.  A sequence's first state stands for K - 1 tokens in front of it, in both directions.
#pragma once
#include "sequences.h"
#include <algorithm>

namespace vrwkv {
namespace conv {
namespace {

constexpr int THREADS = 256;

struct Params {
    const void *x, *state, *gy, *glast;
    ParamVec w, bias;
    Sequences seq;
    void *y, *last, *dx, *dstate;
    float* part;                                           // (parts, K + 1, E): sums of dw and db
    long long x_b, x_t, g_b, g_t;
    int N, rows, T, E, K, silu, run, runs;                 // run: tokens of a run; runs: of a batch row
    bool weights_aligned;                                  // a lane's weights and biases at multiples of theirs in size
};

__device__ __forceinline__ float silu_of(float p) { return p * fast_rcp(1.f + fast_exp2(-LOG2E * p)); }
__device__ __forceinline__ float silu_slope(float p) {
    const float s = fast_rcp(1.f + fast_exp2(-LOG2E * p));
    return s * fmaf(p, 1.f - s, 1.f);
}

// VEC channels of a row, packed and wide
template <typename IO, int VEC> using Packed = typename RawVec<sizeof(IO) * VEC>::type;
template <int VEC> struct Wide { float v[VEC]; };

// The channels of a lane: their weights, and rows of tensors.  KT: taps that registers are there for, K or 8 for all K from 5.
template <typename IO, int VEC, int KT>
struct Lane {
    const Params& p;
    int c;
    bool there;
    Wide<VEC> w[KT], bias;
    __device__ __forceinline__ Lane(const Params& p_, int vec) : p(p_) {
        there = vec * VEC < p.E;
        c = there ? vec * VEC : 0;
    }
    __device__ __forceinline__ void read_weights() {
        if (KT < 8 && p.weights_aligned) {
            if (p.w.dtype == VRWKV_F32) read_params<float>();
            else if (p.w.dtype == VRWKV_BF16) read_params<__hip_bfloat16>();
            else read_params<__half>();
            return;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
#pragma unroll
            for (int j = 0; j < KT; ++j) w[j].v[i] = used(j) ? p.w.value(p.w.fetch((c + i) * p.K + j - (KT - p.K))) : 0.f;
            bias.v[i] = p.bias.p ? p.bias.value(p.bias.fetch(c + i)) : 0.f;
        }
    }
    // VEC numbers of a parameter next to each other
    template <typename T>
    static __device__ __forceinline__ void read_vec(const void* t, int at, float* v) {
        constexpr int ONE = sizeof(T) * VEC > 16 ? VEC / 2 : VEC;
#pragma unroll
        for (int i = 0; i < VEC; i += ONE) {
            float x[ONE];
            load_vec<T, ONE>(static_cast<const T*>(t) + at + i, x);
#pragma unroll
            for (int k = 0; k < ONE; ++k) v[i + k] = x[k];
        }
    }
    template <typename T>
    __device__ __forceinline__ void read_params() {        // the weights of VEC channels lie next to each other
        float all[VEC * KT];
#pragma unroll
        for (int j = 0; j < KT; ++j) read_vec<T>(p.w.p, c * KT + j * VEC, all + j * VEC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            bias.v[i] = 0.f;
#pragma unroll
            for (int j = 0; j < KT; ++j) w[j].v[i] = all[i * KT + j];
        }
        if (p.bias.p) read_vec<T>(p.bias.p, c, bias.v);
    }
    __device__ __forceinline__ bool used(int j) const { return KT < 8 || j >= KT - p.K; }   // (a weight of zero would make an infinite row NaN)
    __device__ __forceinline__ Packed<IO, VEC> packed(const void* t, long long at) const { return load_packed<IO, VEC>(static_cast<const IO*>(t) + at + c); }
    __device__ __forceinline__ Wide<VEC> row(const void* t, long long at) const {
        Wide<VEC> r;
        load_vec<IO, VEC>(static_cast<const IO*>(t) + at + c, r.v);
        return r;
    }
    __device__ __forceinline__ void store(void* t, long long at, const Wide<VEC>& r) const {
        if (there) store_vec<IO, VEC>(static_cast<IO*>(t) + at + c, r.v);
    }
    // token t of the sequence n that begins at `begin`, in front of it its first state
    __device__ __forceinline__ Wide<VEC> token(int n, int b, int t, int begin) const {
        if (t >= begin) return row(p.x, b * p.x_b + t * p.x_t);
        if (p.state && t >= begin - (p.K - 1)) return row(p.state, ((long long)n * (p.K - 1) + t - begin + p.K - 1) * p.E);
        return Wide<VEC>{};
    }
    __device__ __forceinline__ Wide<VEC> pre(const Wide<VEC> (&x)[KT]) const {
        Wide<VEC> s = bias;
#pragma unroll
        for (int j = 0; j < KT; ++j)
            if (used(j))
#pragma unroll
                for (int i = 0; i < VEC; ++i) s.v[i] = fmaf(w[j].v[i], x[j].v[i], s.v[i]);
        return s;
    }
};
// The run of tokens of batch row b that a wave takes: [t0, t1), of them [from, to) in sequences.
struct Run {
    int b, t0, t1, from, to;
    Walk w;
    __device__ __forceinline__ Run(const Params& p, int run) {
        b = run / p.runs;
        t0 = run % p.runs * p.run;
        t1 = min(p.T, t0 + p.run);
    }
    __device__ __forceinline__ void find(const Params& p, int lane) {
        p.seq.inside(t0, t1, from, to);
        w.find(p.seq, b, from, lane);
    }
};

// ---- launches --------------------------------------------------------------------------------------------------------

struct Plan { int run, runs, rows, waves; };              // waves: of a row's channels

// Channels that a lane takes: of `most` bytes where all rows of all tensors lie at multiples of it, pairs of 16-bit ones at multiples of 4, else one.
int vec_of(int dtype, int E, int most, size_t bits, const long long* strides, int n) {
    const int e = dtype == VRWKV_F32 ? 4 : 2;
    for (int i = 0; i < n; ++i) bits |= (size_t)strides[i] * e;
    bits |= (size_t)E * e;
    return bits % most == 0 ? most / e : e == 2 && bits % 4 == 0 ? 2 : 1;
}

bool weights_fit(const void* w, const void* b, int dtype, int vec) {
    const size_t n = std::min(16, vec * (dtype == VRWKV_F32 ? 4 : 2));
    return (((size_t)w | (size_t)b) & (n - 1)) == 0;
}

template <typename F>
int with_taps(int K, F&& f) {
    if (K == 2) return f(std::integral_constant<int, 2>());
    if (K == 3) return f(std::integral_constant<int, 3>());
    if (K == 4) return f(std::integral_constant<int, 4>());
    return f(std::integral_constant<int, 8>());
}
// f with the element type and the channels of a lane: sixteen bytes of fp32, VEC16 of 16 bits, or two or one of those
template <int VEC16, typename F>
int with_types(int dtype, int vec, F&& f) {
    const auto half = [&](auto io) {
        if (vec == VEC16) return f(io, std::integral_constant<int, VEC16>());
        return vec == 2 ? f(io, std::integral_constant<int, 2>()) : f(io, std::integral_constant<int, 1>());
    };
    if (dtype == VRWKV_F32) return vec == 4 ? f(float(), std::integral_constant<int, 4>()) : f(float(), std::integral_constant<int, 1>());
    if (dtype == VRWKV_BF16) return half(__hip_bfloat16());
    return half(__half());
}

bool typed(int d) { return d >= VRWKV_F32 && d <= VRWKV_F16; }
bool aligned(const void* p, int dtype) { return ((size_t)p & (dtype == VRWKV_F32 ? 3 : 1)) == 0; }

int check(const char* who, const vrwkv_conv_args* args, bool backward) {
    if (!args || !args->x || !args->weight || (!backward && !args->y) || (backward && (!args->gy || !args->dx || !args->dweight))) { set_error("%s: null pointer", who); return VRWKV_INVALID_ARG; }
    const vrwkv_conv_args& a = *args;
    if (a.N <= 0 || a.T <= 0 || a.E <= 0) { set_error("%s: N, T and E must be positive", who); return VRWKV_INVALID_ARG; }
    if (!typed(a.dtype) || !typed(a.param_dtype)) { set_error("%s: dtype must be fp32, bf16 or fp16", who); return VRWKV_UNSUPPORTED_DTYPE; }
    if (a.K < 2 || a.K > 8) { set_error("%s: 2 to 8 taps (%d)", who, a.K); return VRWKV_UNSUPPORTED_SHAPE; }
    if (a.x_stride[1] < 0 || a.x_stride[1] >= 1 << 22 || (backward && (a.gy_stride[1] < 0 || a.gy_stride[1] >= 1 << 22))) {
        set_error("%s: tokens must be less than 2^22 elements apart", who);
        return VRWKV_UNSUPPORTED_SHAPE;
    }
    if (a.T >= 1 << 30 || a.N >= 1 << 30 || a.E > (1 << 22) - WAVE || (!a.offsets && (long long)a.N * ((a.T + 7) / 8) >= 1LL << 30)) { set_error("%s: too many tokens, sequences or channels", who); return VRWKV_UNSUPPORTED_SHAPE; }
    bool fits = aligned(a.x, a.dtype) && aligned(a.state, a.dtype) && aligned(a.y, a.dtype) && aligned(a.last, a.dtype) && aligned(a.weight, a.param_dtype) && aligned(a.bias, a.param_dtype) &&
                (!a.offsets || ((size_t)a.offsets & (a.offsets64 ? 7 : 3)) == 0);
    if (backward)
        fits = fits && aligned(a.gy, a.dtype) && aligned(a.glast, a.dtype) && aligned(a.dx, a.dtype) && aligned(a.dstate, a.dtype) && aligned(a.dweight, a.param_dtype) &&
               aligned(a.dbias, a.param_dtype) && ((size_t)a.workspace & 15) == 0;
    if (!fits) { set_error("%s: a tensor is not aligned to its elements, or the workspace to 16 bytes", who); return VRWKV_INVALID_ARG; }
    return VRWKV_OK;
}

Params params_of(const vrwkv_conv_args& a, const Plan& pl, int vec) {
    Params p{};
    p.weights_aligned = weights_fit(a.weight, a.bias, a.param_dtype, vec);
    p.x = a.x, p.state = a.state, p.gy = a.gy, p.glast = a.glast;
    p.w = ParamVec(a.weight, a.param_dtype, 1.f), p.bias = ParamVec(a.bias, a.param_dtype, 1.f);
    p.seq = Sequences{a.offsets, a.offsets64, a.N, a.T};
    p.y = a.y, p.last = a.last, p.dx = a.dx, p.dstate = a.dstate;
    p.x_b = a.x_stride[0], p.x_t = a.x_stride[1], p.g_b = a.gy_stride[0], p.g_t = a.gy_stride[1];
    p.N = a.N, p.rows = pl.rows, p.T = a.T, p.E = a.E, p.K = a.K, p.silu = a.silu, p.run = pl.run, p.runs = pl.runs;
    return p;
}

}  // namespace
}  // namespace conv
}  // namespace vrwkv
