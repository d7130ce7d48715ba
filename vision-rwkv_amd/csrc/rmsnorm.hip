// The root-mean-square norm of rows of C channels with the residual's addition, its output in 8 bits with a scale for each row, and its gradients (gfx950).
//
//     r = x + residual (rounded to the residual's type)        s = 1 / sqrt(mean(r^2) + eps)        n = s r        y = n w
//     dr = s (g - n mean(g n)) + gr with g = gy w              dw = sum_rows gy n
//
// Bound by the memory: a row is read once, held in registers by one wave or four, and written once.  Rows whose width or place does not allow 16-byte vectors, or that are too
// wide for the registers (from 8193 channels of 16 bits and 4097 of 32), are read a second time (from the caches) one element a lane: 1176 rows of 16384 in bf16 72 us for 19 of as many bytes in
// narrower rows, in 8 bits 107 for 23, back 105 for 45; 18871 of 1021 59, 85 and 76.  12544 rows of 768 in bf16: with a bf16 residual and e4m3 out 16 us (4.2 TB/s), with an fp32 residual 24
// (4.8) and back 31 (5.0) and 4 for the weight's sums.
#include "wave_sum.h"
#include <algorithm>

namespace vrwkv {
namespace rmsnorm {
namespace {

constexpr int THREADS = 256;

struct Params {
    const void *x, *residual, *gy, *gsum;
    ParamVec w;
    void *y, *sum, *dx, *dresidual;
    float *scale, *part, *stat;                            // part: (workgroups, C) sums of dw; stat: s of each row
    long long rows, x_r, res_r, gy_r, gsum_r;
    int C, out_kind;
    float eps;
    bool weights_aligned;                                  // at a multiple of a vector's size
};

// The value that the four waves of a workgroup, or one wave, agree on.
template <int WAVES, bool MAX>
__device__ __forceinline__ float agreed(float v, float* red) {
    if (MAX) {
        // (a NaN wins: fmax would drop it)
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const float u = __shfl_xor(v, o);
            v = u != u || u > v ? u : v;
        }
    } else v = wave_sum(v);
    if (WAVES == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    if (!MAX) return (red[0] + red[1]) + (red[2] + red[3]);
    v = red[0];
#pragma unroll
    for (int k = 1; k < 4; ++k) v = red[k] != red[k] || red[k] > v ? red[k] : v;
    return v;
}
__device__ __forceinline__ float larger(float m, float v) {
    const float a = fabsf(v);
    return a != a || a > m ? a : m;
}
// 1 / sqrt to one unit in the last place: the approximation, which takes subnormal numbers for zeros (hence the powers of two), and one Newton step (an infinite or zero argument stays what the
// approximation makes of it)
__device__ __forceinline__ float inverse_root(float v) {
    const bool small = v < 0x1p-100f;
    const float x = small ? v * 0x1p96f : v, s = __builtin_amdgcn_rsqf(x), t = s * fmaf(-0.5f * x, s * s, 1.5f);
    return (fabsf(t) < 1e38f ? t : s) * (small ? 0x1p48f : 1.f);
}

__device__ __forceinline__ float top_of(int kind) { return kind == VRWKV_Y_INT8 ? 127.f : 448.f; }
// What a row's results are divided by: 1 / scale and -scale (0 where the scale is infinite: nothing is left over from a product with that).
struct Divisor { float inverse, minus; };
// four results of a row in 8 bits.  The quotient by the scale is rounded once: the product with the rounded 1 / scale is off by up to one and a half units, which puts a quotient on the border of two
// numbers (of a bf16 row and weight one in three thousand is) on the wrong side of it; what is left of v after the product, times 1 / scale, is what it lacks.
__device__ __forceinline__ unsigned packed8(const float* v, Divisor by, float top, int kind) {
    float q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        q[k] = v[k] * by.inverse;
        q[k] = fmaf(fmaf(q[k], by.minus, v[k]), by.inverse, q[k]);
        q[k] = q[k] > top ? top : q[k] < -top ? -top : q[k];   // (a NaN stays one)
    }
    if (kind == VRWKV_Y_E4M3) {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], r, true);
    }
    unsigned r = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) r |= ((unsigned)(int)(q[k] == q[k] ? rintf(q[k]) : 0.f) & 0xffu) << (8 * k);
    return r;
}
// the row's scale and what its results are divided by
__device__ __forceinline__ float scale_of(float most, float top, Divisor& by) {
    float s = most / top;
    s = s < 1.1754943508222875e-38f ? 1.1754943508222875e-38f : s;
    by.inverse = 1.f / s;
    by.minus = fabsf(s) < __builtin_inff() ? -s : 0.f;
    return s;
}

// VEC elements of a row: one or two 16-byte vectors, or one element
template <typename T, int VEC>
__device__ __forceinline__ void read(const void* t, long long at, float (&v)[VEC]) {
    constexpr int ONE = sizeof(T) * VEC > 16 ? VEC / 2 : VEC;
#pragma unroll
    for (int i = 0; i < VEC; i += ONE) {
        float x[ONE];
        load_vec<T, ONE>(static_cast<const T*>(t) + at + i, x);
#pragma unroll
        for (int k = 0; k < ONE; ++k) v[i + k] = x[k];
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void write(void* t, long long at, const float (&v)[VEC]) {
    constexpr int ONE = sizeof(T) * VEC > 16 ? VEC / 2 : VEC;
#pragma unroll
    for (int i = 0; i < VEC; i += ONE) {
        float x[ONE];
#pragma unroll
        for (int k = 0; k < ONE; ++k) x[k] = v[i + k];
        store_vec<T, ONE>(static_cast<T*>(t) + at + i, x);
    }
}
// the weights of VEC channels
template <int VEC>
__device__ __forceinline__ void weights(const Params& p, int c, float (&w)[VEC]) {
    if (VEC > 1 && p.weights_aligned) {
        if (p.w.dtype == VRWKV_F32) read<float, VEC>(p.w.p, c, w);
        else if (p.w.dtype == VRWKV_BF16) read<__hip_bfloat16, VEC>(p.w.p, c, w);
        else read<__half, VEC>(p.w.p, c, w);
    } else
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[k] = p.w.value(p.w.fetch(c + k));
}
// VEC elements of a row of x and residual, added and rounded
template <typename IO, typename RES, int VEC>
__device__ __forceinline__ void sum_of(const Params& p, long long row, int c, float (&r)[VEC]) {
    if (p.x) read<IO, VEC>(p.x, row * p.x_r + c, r);
    if (p.residual) {
        float t[VEC];
        read<RES, VEC>(p.residual, row * p.res_r + c, t);
#pragma unroll
        for (int k = 0; k < VEC; ++k) r[k] = to_f32(from_f32<RES>(r[k] + t[k]));
    }
}
template <typename IO, int VEC>
__device__ __forceinline__ void put_row(const Params& p, long long row, int c, const float (&y)[VEC], Divisor by) {
    if (p.out_kind == VRWKV_Y_SAME) {
        write<IO, VEC>(p.y, row * p.C + c, y);
        return;
    }
    unsigned char* to = static_cast<unsigned char*>(p.y) + row * p.C + c;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int k = 0; k < VEC; k += 4) reinterpret_cast<unsigned*>(to)[k / 4] = packed8(&y[k], by, top_of(p.out_kind), p.out_kind);
    } else {
        const float v[4] = {y[0], 0.f, 0.f, 0.f};
        *to = (unsigned char)packed8(v, by, top_of(p.out_kind), p.out_kind);
    }
}

// Workgroups in two dimensions: a launch's first has room for 2^24 of 256 threads.
constexpr int GRID_X = 1 << 22;
__device__ __forceinline__ long long group() { return (long long)blockIdx.y * GRID_X + blockIdx.x; }
dim3 grid_of(long long groups) { return dim3((unsigned)std::min<long long>(groups, GRID_X), (unsigned)((groups + GRID_X - 1) / GRID_X)); }

// A row in the registers of WAVES waves, NV vectors a lane.
template <typename IO, typename RES, int VEC, int NV, int WAVES>
__global__ __launch_bounds__(THREADS) void forward_kernel(const Params p) {
    __shared__ float red[4];
    const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const long long row = WAVES == 1 ? group() * 4 + (threadIdx.x >> 6) : group();
    if (row >= p.rows) return;
    float r[NV][VEC], w[NV][VEC], s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WAVES + lane) * VEC;
#pragma unroll
        for (int k = 0; k < VEC; ++k) r[i][k] = w[i][k] = 0.f;
        if (c < p.C) {
            weights<VEC>(p, c, w[i]);
            sum_of<IO, RES, VEC>(p, row, c, r[i]);
            if (p.sum) write<RES, VEC>(p.sum, row * p.C + c, r[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) s = fmaf(r[i][k], r[i][k], s);
    s = inverse_root(agreed<WAVES, false>(s, red) / (float)p.C + p.eps);
    float most = 0.f;
    Divisor by{};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WAVES + lane) * VEC;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            r[i][k] = r[i][k] * s * w[i][k];
            most = larger(most, r[i][k]);
        }
    }
    if (p.out_kind != VRWKV_Y_SAME) {
        const float v = scale_of(agreed<WAVES, true>(most, red), top_of(p.out_kind), by);
        if (lane == 0) p.scale[row] = v;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WAVES + lane) * VEC;
        if (c < p.C) put_row<IO, VEC>(p, row, c, r[i], by);
    }
}

// Any row: a workgroup each, read again for each of its passes.
template <typename IO, typename RES>
__global__ __launch_bounds__(THREADS) void forward_any_kernel(const Params p) {
    __shared__ float red[4];
    const long long row = group();
    if (row >= p.rows) return;
    float s = 0.f, r[1];
    for (int c = threadIdx.x; c < p.C; c += THREADS) {
        sum_of<IO, RES, 1>(p, row, c, r);
        if (p.sum) write<RES, 1>(p.sum, row * p.C + c, r);
        s = fmaf(r[0], r[0], s);
    }
    s = inverse_root(agreed<4, false>(s, red) / (float)p.C + p.eps);
    float most = 0.f;
    Divisor by{};
    const auto value = [&](int c) {
        sum_of<IO, RES, 1>(p, row, c, r);
        return r[0] * s * p.w.value(p.w.fetch(c));
    };
    if (p.out_kind != VRWKV_Y_SAME) {
        for (int c = threadIdx.x; c < p.C; c += THREADS) most = larger(most, value(c));
        const float v = scale_of(agreed<4, true>(most, red), top_of(p.out_kind), by);
        if (threadIdx.x == 0) p.scale[row] = v;
    }
    for (int c = threadIdx.x; c < p.C; c += THREADS) {
        const float y[1] = {value(c)};
        put_row<IO, 1>(p, row, c, y, by);
    }
}

// gsum and the two gradients of a vector of a row; r is the forward's sum, of the residual's type (or x)
template <typename IO, typename RES, int VEC>
__device__ __forceinline__ void put_gradients(const Params& p, long long row, int c, float (&d)[VEC]) {
    if (p.gsum) {
        float t[VEC];
        read<RES, VEC>(p.gsum, row * p.gsum_r + c, t);
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[k] += t[k];
    }
    if (p.dx) write<IO, VEC>(p.dx, row * p.C + c, d);
    if (p.dresidual) write<RES, VEC>(p.dresidual, row * p.C + c, d);
}
template <typename IO, typename RES, int VEC>
__device__ __forceinline__ void saved_of(const Params& p, long long row, int c, float (&r)[VEC]) {
    read<RES, VEC>(p.sum, row * p.x_r + c, r);
}

// Rows in turn, their sums for dw in registers until the end.
template <typename IO, typename RES, int VEC, int NV, int WAVES>
__global__ __launch_bounds__(THREADS) void backward_kernel(const Params p) {
    __shared__ float red[4], sums[WAVES == 1 ? 4 : 1][64 * VEC];
    const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
    const long long first = WAVES == 1 ? (long long)blockIdx.x * 4 + wave : blockIdx.x, step = WAVES == 1 ? gridDim.x * 4LL : gridDim.x;
    float dw[NV][VEC], w[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WAVES + lane) * VEC;
#pragma unroll
        for (int k = 0; k < VEC; ++k) dw[i][k] = w[i][k] = 0.f;
        if (c < p.C) weights<VEC>(p, c, w[i]);
    }
    for (long long row = first; row < p.rows; row += step) {
        float r[NV][VEC], g[NV][VEC], s = 0.f, m = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * WAVES + lane) * VEC;
#pragma unroll
            for (int k = 0; k < VEC; ++k) r[i][k] = g[i][k] = 0.f;
            if (c < p.C) {
                saved_of<IO, RES, VEC>(p, row, c, r[i]);
                read<IO, VEC>(p.gy, row * p.gy_r + c, g[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                s = fmaf(r[i][k], r[i][k], s);
                m = fmaf(g[i][k] * w[i][k], r[i][k], m);
            }
        s = inverse_root(agreed<WAVES, false>(s, red) / (float)p.C + p.eps);
        m = agreed<WAVES, false>(m, red) / (float)p.C * s;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * WAVES + lane) * VEC;
            float d[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float n = r[i][k] * s;
                dw[i][k] = fmaf(g[i][k], n, dw[i][k]);
                d[k] = s * fmaf(-n, m, g[i][k] * w[i][k]);
            }
            if (c < p.C) put_gradients<IO, RES, VEC>(p, row, c, d);
        }
    }
    if (!p.part) return;
    float* const out = p.part + (long long)blockIdx.x * p.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WAVES + lane) * VEC;
        if (WAVES > 1) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (c < p.C) out[c + k] = dw[i][k];
        } else {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VEC; ++k) sums[wave][lane * VEC + k] = dw[i][k];
            __syncthreads();
            for (int j = threadIdx.x; j < 64 * VEC; j += THREADS)
                if (i * 64 * VEC + j < p.C) out[i * 64 * VEC + j] = (sums[0][j] + sums[1][j]) + (sums[2][j] + sums[3][j]);
        }
    }
}

// Any row: dx, and s of each row for the next kernel.
template <typename IO, typename RES>
__global__ __launch_bounds__(THREADS) void backward_any_kernel(const Params p) {
    __shared__ float red[4];
    const long long row = group();
    if (row >= p.rows) return;
    float s = 0.f, m = 0.f, r[1];
    const IO* gy = static_cast<const IO*>(p.gy) + row * p.gy_r;
    for (int c = threadIdx.x; c < p.C; c += THREADS) {
        saved_of<IO, RES, 1>(p, row, c, r);
        s = fmaf(r[0], r[0], s);
        m = fmaf(to_f32(gy[c]) * p.w.value(p.w.fetch(c)), r[0], m);
    }
    s = inverse_root(agreed<4, false>(s, red) / (float)p.C + p.eps);
    m = agreed<4, false>(m, red) / (float)p.C * s;
    if (threadIdx.x == 0) p.stat[row] = s;
    for (int c = threadIdx.x; c < p.C; c += THREADS) {
        saved_of<IO, RES, 1>(p, row, c, r);
        float d[1] = {s * fmaf(-r[0] * s, m, to_f32(gy[c]) * p.w.value(p.w.fetch(c)))};
        put_gradients<IO, RES, 1>(p, row, c, d);
    }
}
// Parts of dw: a column a thread, rows blockIdx.y, + gridDim.y, ..
template <typename IO, typename RES>
__global__ __launch_bounds__(THREADS) void weight_any_kernel(const Params p) {
    const int c = blockIdx.x * THREADS + threadIdx.x;
    if (c >= p.C) return;
    float v = 0.f, r[1];
#pragma unroll 4
    for (long long row = blockIdx.y; row < p.rows; row += gridDim.y) {
        saved_of<IO, RES, 1>(p, row, c, r);
        v = fmaf(to_f32(static_cast<const IO*>(p.gy)[row * p.gy_r + c]), r[0] * p.stat[row], v);
    }
    p.part[(long long)blockIdx.y * p.C + c] = v;
}

// ---- launches --------------------------------------------------------------------------------------------------------

// Vectors of a lane and waves of a row; 0 where rows are taken element by element.  One wave holds rows of up to two vectors a lane, which saves the waves' agreement in 8 bits (12544 x 768
// 15.6 us for 23.3); wider ones are four waves' (12544 x 1536 forward 44 for 49, back 61 for 70, in 8 bits 33 for 38).
struct Plan { int nv, waves, parts; };
bool typed(int d) { return d >= VRWKV_F32 && d <= VRWKV_F16; }
size_t size_of(int d) { return d == VRWKV_F32 ? 4 : 2; }

// (element sizes of a vector follow x's type: eight elements of 16 bits, four of fp32)
Plan plan_of(const vrwkv_rmsnorm_args& a, bool backward) {
    const int vec = a.dtype == VRWKV_F32 ? 4 : 8, vectors = a.C / vec;
    const size_t e = size_of(a.dtype), re = size_of(a.residual_dtype);
    // every row of every tensor at a multiple of a vector (8 bits: of four bytes)
    bool fits = a.C % vec == 0 && a.C <= 64 * 4 * vec * 4;
    const auto rows_at = [&](const void* p, long long stride, size_t size) { fits = fits && (!p || (((size_t)p | (size_t)(stride * (long long)size)) & (vec * size - 1 < 15 ? vec * size - 1 : 15)) == 0); };
    if (backward) {
        rows_at(a.sum, a.x_stride, re), rows_at(a.gy, a.gy_stride, e), rows_at(a.gsum, a.gsum_stride, re), rows_at(a.dx, a.C, e), rows_at(a.dresidual, a.C, re);
    } else {
        rows_at(a.x, a.x_stride, e), rows_at(a.residual, a.residual_stride, re), rows_at(a.sum, a.C, re);
        if (a.out_kind == VRWKV_Y_SAME) rows_at(a.y, a.C, e);
        else fits = fits && ((size_t)a.y & 3) == 0;
    }
    Plan p{0, 4, 0};
    if (fits) {
        p.waves = vectors <= 128 ? 1 : 4;
        const int nv = (vectors + 64 * p.waves - 1) / (64 * p.waves);
        p.nv = nv <= 1 ? 1 : nv <= 2 ? 2 : 4;
    }
    const long long groups = p.nv && p.waves == 1 ? (a.rows + 3) / 4 : a.rows;
    p.parts = (int)std::min<long long>(groups, p.nv ? 4LL * device_cus() : 256);
    return p;
}
bool weights_fit(const vrwkv_rmsnorm_args& a) { return ((size_t)a.weight & (std::min<size_t>(16, (a.dtype == VRWKV_F32 ? 4 : 8) * size_of(a.weight_dtype)) - 1)) == 0; }
size_t backward_bytes(const vrwkv_rmsnorm_args& a, const Plan& p) { return ((size_t)p.parts * a.C * 4 + 15) / 16 * 16 + (p.nv ? 0 : (size_t)a.rows * 4); }

template <typename F>
int with_types(int dtype, int residual_dtype, F&& f) {
    const auto pair = [&](auto io) { return residual_dtype == VRWKV_F32 ? f(io, float()) : f(io, io); };
    if (dtype == VRWKV_F32) return f(float(), float());
    if (dtype == VRWKV_BF16) return pair(__hip_bfloat16());
    return pair(__half());
}
template <typename F>
void with_plan(const Plan& p, F&& f) {
    const auto waves = [&](auto nv) {
        if (p.waves == 1) f(nv, std::integral_constant<int, 1>());
        else f(nv, std::integral_constant<int, 4>());
    };
    if (p.nv == 1) waves(std::integral_constant<int, 1>());
    else if (p.nv == 2) waves(std::integral_constant<int, 2>());
    else f(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());   // (no row of one wave takes so many)
}

int check(const char* who, const vrwkv_rmsnorm_args* args, bool backward) {
    if (!args || !args->weight || (!backward && (!args->x || !args->y || (args->out_kind != VRWKV_Y_SAME && !args->scale))) || (backward && (!args->sum || !args->gy || (!args->dx && !args->dresidual && !args->dweight)))) {
        set_error("%s: null pointer", who);
        return VRWKV_INVALID_ARG;
    }
    const vrwkv_rmsnorm_args& a = *args;
    if (a.rows <= 0 || a.C <= 0) { set_error("%s: rows and C must be positive", who); return VRWKV_INVALID_ARG; }
    if (!typed(a.dtype) || !typed(a.weight_dtype) || (a.residual_dtype != a.dtype && a.residual_dtype != VRWKV_F32)) {
        set_error("%s: dtype must be fp32, bf16 or fp16, the residual's that or fp32", who);
        return VRWKV_UNSUPPORTED_DTYPE;
    }
    if (a.out_kind < VRWKV_Y_SAME || a.out_kind > VRWKV_Y_INT8) { set_error("%s: unknown kind of output %d", who, a.out_kind); return VRWKV_INVALID_ARG; }
    if (a.rows >= 1LL << 31) { set_error("%s: 2^31 rows or more", who); return VRWKV_UNSUPPORTED_SHAPE; }
    // (a thread's next channel has to stay within an int; the launch that ends the sums of dweight has room for 2^27 columns)
    const int most = backward && a.dweight ? (1 << 27) - 32 : 0x7fffffff - 255;
    if (a.C > most) { set_error("%s: more than %d channels", who, most); return VRWKV_UNSUPPORTED_SHAPE; }
    const size_t e = size_of(a.dtype) - 1, re = size_of(a.residual_dtype) - 1, we = size_of(a.weight_dtype) - 1;
    if ((((size_t)a.x | (size_t)a.gy | (size_t)a.dx) & e) || (((size_t)a.residual | (size_t)a.sum | (size_t)a.gsum | (size_t)a.dresidual) & re) || (((size_t)a.weight | (size_t)a.dweight) & we) ||
        (a.out_kind == VRWKV_Y_SAME && ((size_t)a.y & e)) || ((size_t)a.scale & 3) || ((size_t)a.workspace & 15)) {
        set_error("%s: a tensor is not aligned to its elements, or the workspace to 16 bytes", who);
        return VRWKV_INVALID_ARG;
    }
    return VRWKV_OK;
}

}  // namespace
}  // namespace rmsnorm
}  // namespace vrwkv

using namespace vrwkv;
using namespace vrwkv::rmsnorm;

extern "C" int vrwkv_rmsnorm(const vrwkv_rmsnorm_args* args, void* hip_stream) {
    const char* who = "vrwkv_rmsnorm";
    if (const int rc = check(who, args, false)) return rc;
    const vrwkv_rmsnorm_args& a = *args;
    Params p{};
    p.x = a.x, p.residual = a.residual, p.w = ParamVec(a.weight, a.weight_dtype, 1.f), p.y = a.y, p.sum = a.sum, p.scale = a.scale;
    p.rows = a.rows, p.x_r = a.x_stride, p.res_r = a.residual_stride, p.C = a.C, p.out_kind = a.out_kind, p.eps = a.eps;
    p.weights_aligned = weights_fit(a);
    const Plan pl = plan_of(a, false);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    return with_types(a.dtype, a.residual_dtype, [&](auto io, auto res) {
        using IO = decltype(io);
        using RES = decltype(res);
        constexpr int VEC = 16 / sizeof(IO);
        if (!pl.nv) hipLaunchKernelGGL((forward_any_kernel<IO, RES>), grid_of(a.rows), dim3(THREADS), 0, st, p);
        else
            with_plan(pl, [&](auto nv, auto waves) {
                constexpr int NV = decltype(nv)::value, WAVES = decltype(waves)::value;
                hipLaunchKernelGGL((forward_kernel<IO, RES, VEC, NV, WAVES>), grid_of(WAVES == 1 ? (a.rows + 3) / 4 : a.rows), dim3(THREADS), 0, st, p);
            });
        return check_launch(who);
    });
}

extern "C" size_t vrwkv_rmsnorm_bwd_workspace_bytes(const vrwkv_rmsnorm_args* args) {
    return args && args->rows > 0 && args->C > 0 ? backward_bytes(*args, plan_of(*args, true)) : 0;
}

extern "C" int vrwkv_rmsnorm_bwd(const vrwkv_rmsnorm_args* args, void* hip_stream) {
    const char* who = "vrwkv_rmsnorm_bwd";
    if (const int rc = check(who, args, true)) return rc;
    const vrwkv_rmsnorm_args& a = *args;
    const Plan pl = plan_of(a, true);
    const size_t need = backward_bytes(a, pl);
    if (!a.workspace || a.workspace_bytes < need) { set_error("%s: workspace of %zu bytes, %zu needed", who, a.workspace ? a.workspace_bytes : (size_t)0, need); return VRWKV_WORKSPACE_TOO_SMALL; }
    Params p{};
    p.sum = a.sum, p.w = ParamVec(a.weight, a.weight_dtype, 1.f), p.gy = a.gy, p.gsum = a.gsum, p.dx = a.dx, p.dresidual = a.dresidual;
    p.rows = a.rows, p.x_r = a.x_stride, p.gy_r = a.gy_stride, p.gsum_r = a.gsum_stride, p.C = a.C, p.eps = a.eps;
    p.weights_aligned = weights_fit(a);
    p.part = a.dweight ? static_cast<float*>(a.workspace) : nullptr;
    p.stat = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + ((size_t)pl.parts * a.C * 4 + 15) / 16 * 16);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int rc = with_types(a.dtype, a.residual_dtype, [&](auto io, auto res) {
        using IO = decltype(io);
        using RES = decltype(res);
        constexpr int VEC = 16 / sizeof(IO);
        if (pl.nv)
            with_plan(pl, [&](auto nv, auto waves) {
                constexpr int NV = decltype(nv)::value, WAVES = decltype(waves)::value;
                hipLaunchKernelGGL((backward_kernel<IO, RES, VEC, NV, WAVES>), dim3(pl.parts), dim3(THREADS), 0, st, p);
            });
        else {
            hipLaunchKernelGGL((backward_any_kernel<IO, RES>), grid_of(a.rows), dim3(THREADS), 0, st, p);
            if (p.part) hipLaunchKernelGGL((weight_any_kernel<IO, RES>), dim3((a.C + THREADS - 1) / THREADS, pl.parts), dim3(THREADS), 0, st, p);
        }
        return check_launch(who);
    });
    if (rc != VRWKV_OK || !p.part) return rc;
    launch_batch_sum(p.part, SumOut(a.dweight, a.weight_dtype), nullptr, SumOut(nullptr), pl.parts, a.C, st);
    return check_launch(who);
}
