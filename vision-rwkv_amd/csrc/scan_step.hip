// One more token for each of N sequences whose states are pages of a pool: h = exp(dt A) h + dt u B, y = (C h + D u) silu(z), h written back (gfx950).
// Bound by the pages, read and written once: P lanes hold four states each of NC channels, 16 bytes a lane and channel.  A workgroup takes its channels of R rows, one after the other, with the
// next row's page on its way: A, as large as a page, comes from L2 once for the R.  Two channels and four rows where that leaves four workgroups a compute unit, else one and one.
// 512 rows of 1536 x 16 states, 101 MB: 23.5 us (4.5 TB/s) where the last-level cache holds the pools (three of 63 MB in turn), 31 to 35 where it does not (eight); with loads and stores past the
// caches 32 in both.  One channel and one row: 42.  One row alone: 3.9.
#include "scan.h"
#include "pages.h"
#include <algorithm>

namespace vrwkv {
namespace scan {
namespace {

constexpr int GRID_Y = 32768;

struct StepParams {
    const void *u, *delta, *B, *C, *z;
    const float* A;
    ParamVec D, bias;
    Slots slots;
    float* pool;
    void* y;
    long long u_n, d_n, z_n, B_n, B_g, C_n, C_g, page;
    int E, S, G, softplus, blocks;
};

// VEC: states and A are read and written 16 bytes at a time
template <typename IO, int P, int NC, int R, bool VEC>
__global__ __launch_bounds__(THREADS) void step_kernel(const StepParams p) {
    const int tid = threadIdx.x, q = tid % P, of_group = p.E / p.G, g = blockIdx.x / p.blocks, n0 = (blockIdx.y + GRID_Y * blockIdx.z) * R;
    if (n0 >= p.slots.rows) return;
    int e[NC];
    bool there[NC];
    f32x4 a[NC], h[NC], ahead[NC];
    float bias[NC], skip[NC];
    const auto row_of = [&](const float* t, f32x4& x) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = 4 * q + k < p.S ? t[k] : 0.f;
    };
    long long slot[R];
#pragma unroll
    for (int r = 0; r < R; ++r) slot[r] = n0 + r < p.slots.rows ? p.slots.at(n0 + r) : -2;
    const auto page_of = [&](long long s) { return p.pool + s * p.page; };
    const auto fetch = [&](long long s) {
        const bool known = p.slots.has(s);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            ahead[c] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (!known || !there[c]) continue;
            const float* t = page_of(s) + (long long)e[c] * p.S + 4 * q;
            if (VEC) ahead[c] = *reinterpret_cast<const f32x4*>(t);
            else row_of(t, ahead[c]);
        }
    };
    IO u[NC], d[NC], z[NC], Bt[4], Ct[4];                  // the next row's token
    const auto token = [&](int n) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u[c] = static_cast<const IO*>(p.u)[n * p.u_n + e[c]];
            d[c] = static_cast<const IO*>(p.delta)[n * p.d_n + e[c]];
            if (p.z) z[c] = static_cast<const IO*>(p.z)[n * p.z_n + e[c]];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = min(4 * q + k, p.S - 1);
            Bt[k] = static_cast<const IO*>(p.B)[n * p.B_n + g * p.B_g + s];
            Ct[k] = static_cast<const IO*>(p.C)[n * p.C_n + g * p.C_g + s];
        }
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int i = ((blockIdx.x % p.blocks) * NC + c) * (THREADS / P) + tid / P;
        there[c] = i < of_group;
        e[c] = g * of_group + min(i, of_group - 1);
    }
    fetch(slot[0]);
    token(n0);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (VEC) a[c] = *reinterpret_cast<const f32x4*>(p.A + (long long)e[c] * p.S + 4 * q);
        else row_of(p.A + (long long)e[c] * p.S + 4 * q, a[c]);
        a[c] *= LOG2E;
        bias[c] = p.bias.p ? p.bias.value(p.bias.fetch(e[c])) : 0.f;
        skip[c] = p.D.p ? p.D.value(p.D.fetch(e[c])) : 0.f;
    }
    unsigned skipped, shared;
    p.slots.find_others<R>(n0, slot, skipped, shared);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (n0 + r >= p.slots.rows) return;
        const bool known = p.slots.has(slot[r]);
        const bool mine = !(skipped >> r & 1);
#pragma unroll
        for (int c = 0; c < NC; ++c) h[c] = ahead[c];
        if (R > 1 && r + 1 < R) fetch(slot[r + 1 < R ? r + 1 : 0]);
        int n = n0 + r, next = mine && (shared >> r & 1) ? p.slots.behind(n, slot[r]) : p.slots.rows;
        bool again = mine;
        // (a row's own token has been read; the next row's is read while it is worked on, and once more behind rows of the same page)
        while (again) {
            float y[NC], Bf[4], Cf[4], uf[NC], df[NC], zf[NC];
#pragma unroll
            for (int k = 0; k < 4; ++k) Bf[k] = to_f32(Bt[k]), Cf[k] = to_f32(Ct[k]);
#pragma unroll
            for (int c = 0; c < NC; ++c) uf[c] = to_f32(u[c]), df[c] = to_f32(d[c]), zf[c] = p.z ? to_f32(z[c]) : 0.f;
            if (next < p.slots.rows) token(next);
            else if (R > 1 && r + 1 < R) token(min(n0 + r + 1, p.slots.rows - 1));
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float raw = df[c] + bias[c], dt = p.softplus ? softplus(raw) : raw, x = dt * uf[c];
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool pad = !VEC && 4 * q + k >= p.S;
                    h[c][k] = pad ? 0.f : fmaf(fast_exp2(dt * a[c][k]), h[c][k], x * Bf[k]);
                    s = pad ? s : fmaf(Cf[k], h[c][k], s);
                }
                if (P > 1) s += across<1>(s);
                if (P > 2) s += across<2>(s);
                if (P > 4) s += across<4>(s);
                if (P > 8) s += across<8>(s);
                y[c] = fmaf(skip[c], uf[c], s);
                if (p.z) y[c] *= zf[c] * sigmoid(zf[c]);
                if (!known) y[c] = slot[r] == -1 ? 0.f : __builtin_nanf("");
            }
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (there[c] && q == 0) static_cast<IO*>(p.y)[(long long)n * p.E + e[c]] = from_f32<IO>(y[c]);
            again = next < p.slots.rows;
            if (again) {
                n = next;
                next = p.slots.behind(n, slot[r]);
            }
        }
        if (!mine && R > 1 && r + 1 < R) token(min(n0 + r + 1, p.slots.rows - 1));
        if (!known || !mine) continue;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (!there[c]) continue;
            float* to = page_of(slot[r]) + (long long)e[c] * p.S + 4 * q;
            if (VEC) *reinterpret_cast<f32x4*>(to) = h[c];
            else
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (4 * q + k < p.S) to[k] = h[c][k];
        }
    }
}

template <typename IO, int P, int NC, int R>
int launch(StepParams& p, bool vec, hipStream_t st) {
    const int each = THREADS / P * NC, groups = (p.slots.rows + R - 1) / R;
    p.blocks = (p.E / p.G + each - 1) / each;
    const dim3 grid((unsigned)(p.G * p.blocks), (unsigned)std::min(groups, GRID_Y), (unsigned)((groups + GRID_Y - 1) / GRID_Y)), block(THREADS);
    if (vec && p.S == 4 * P) hipLaunchKernelGGL((step_kernel<IO, P, NC, R, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((step_kernel<IO, P, NC, R, false>), grid, block, 0, st, p);
    return check_launch("vrwkv_scan_step");
}
template <typename IO, int P>
int launch(StepParams& p, bool vec, hipStream_t st) {
    const long long workgroups = (long long)p.G * ((p.E / p.G + THREADS / P - 1) / (THREADS / P)) * p.slots.rows;
    return workgroups >= 8LL * 4 * device_cus() ? launch<IO, P, 2, 4>(p, vec, st) : launch<IO, P, 1, 1>(p, vec, st);
}
template <typename IO>
int launch(StepParams& p, bool vec, hipStream_t st) {
    if (p.S <= 4) return launch<IO, 1>(p, vec, st);
    if (p.S <= 8) return launch<IO, 2>(p, vec, st);
    if (p.S <= 16) return launch<IO, 4>(p, vec, st);
    if (p.S <= 32) return launch<IO, 8>(p, vec, st);
    return launch<IO, 16>(p, vec, st);
}

}  // namespace
}  // namespace scan
}  // namespace vrwkv

using namespace vrwkv;

extern "C" int vrwkv_scan_step(const vrwkv_scan_step_args* args, void* hip_stream) {
    const char* who = "vrwkv_scan_step";
    if (!args || !args->u || !args->delta || !args->A || !args->B || !args->C || !args->pool || !args->y) { set_error("%s: null pointer", who); return VRWKV_INVALID_ARG; }
    const vrwkv_scan_step_args& a = *args;
    if (a.N <= 0 || a.P <= 0 || a.E <= 0 || a.G <= 0) { set_error("%s: N, P, E and G must be positive", who); return VRWKV_INVALID_ARG; }
    if (a.dtype < VRWKV_F32 || a.dtype > VRWKV_F16 || a.D_dtype < VRWKV_F32 || a.D_dtype > VRWKV_F16 || a.bias_dtype < VRWKV_F32 || a.bias_dtype > VRWKV_F16) {
        set_error("%s: dtype must be fp32, bf16 or fp16", who);
        return VRWKV_UNSUPPORTED_DTYPE;
    }
    if (a.S < 1 || a.S > 64 || a.E % a.G || a.E > 1 << 22) { set_error("%s: 1 to 64 states (%d), E (%d, at most 2^22) a multiple of G (%d)", who, a.S, a.E, a.G); return VRWKV_UNSUPPORTED_SHAPE; }
    if (a.N >= 1 << 30) { set_error("%s: 2^30 rows or more", who); return VRWKV_UNSUPPORTED_SHAPE; }
    if (!a.slots && a.N > a.P) { set_error("%s: %d rows without slots, and %d pages", who, a.N, a.P); return VRWKV_INVALID_ARG; }
    if (a.page_stride < (long long)a.E * a.S) { set_error("%s: pages overlap", who); return VRWKV_INVALID_ARG; }
    const size_t w = a.dtype == VRWKV_F32 ? 3 : 1;
    if ((((size_t)a.u | (size_t)a.delta | (size_t)a.B | (size_t)a.C | (size_t)a.z | (size_t)a.y) & w) || (((size_t)a.pool | (size_t)a.A) & 3) ||
        ((size_t)a.D & (a.D_dtype == VRWKV_F32 ? 3 : 1)) || ((size_t)a.delta_bias & (a.bias_dtype == VRWKV_F32 ? 3 : 1)) || (a.slots && ((size_t)a.slots & (a.slots64 ? 7 : 3)))) {
        set_error("%s: a tensor is not aligned to its elements", who);
        return VRWKV_INVALID_ARG;
    }
    scan::StepParams p{a.u, a.delta, a.B, a.C, a.z, a.A, ParamVec(a.D, a.D_dtype, 1.f), ParamVec(a.delta_bias, a.bias_dtype, 1.f), Slots{a.slots, a.slots64, a.N, a.P}, a.pool, a.y,
                       a.u_stride, a.delta_stride, a.z_stride, a.B_stride[0], a.B_stride[1], a.C_stride[0], a.C_stride[1], a.page_stride, a.E, a.S, a.G, a.softplus, 0};
    const bool vec = (((size_t)a.pool | (size_t)a.A) & 15) == 0 && a.page_stride % 4 == 0;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (a.dtype == VRWKV_F32) return scan::launch<float>(p, vec, st);
    if (a.dtype == VRWKV_BF16) return scan::launch<__hip_bfloat16>(p, vec, st);
    return scan::launch<__half>(p, vec, st);
}
