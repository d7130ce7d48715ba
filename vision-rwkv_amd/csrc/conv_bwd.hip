// The gradients of the short causal convolution (conv.h).
#include "conv.h"

namespace vrwkv {
namespace conv {
namespace {

constexpr int AHEAD = 4;                                  // (eight rows of two tensors ahead: 49 us for 37 at 64 x 196 x 1536 bf16, for want of registers)
// Runs parts apart, one after the other: their sums for dw and db stay in registers until the end.
template <typename IO, int VEC, int KT>
__global__ __launch_bounds__(THREADS) void backward_kernel(const Params p, int run_blocks) {
    __shared__ float red[THREADS / WAVE][WAVE * VEC];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x >= run_blocks) {                   // sequences without a token hand the last states' gradients on
        if (blockIdx.y) return;
        const long long page = (long long)(p.K - 1) * p.E;
        for (int n = blockIdx.x - run_blocks; n < p.N; n += gridDim.x - run_blocks)
            if (p.seq.at(n + 1) <= p.seq.at(n))
                for (long long i = threadIdx.x; i < page; i += THREADS) static_cast<IO*>(p.dstate)[n * page + i] = p.glast ? static_cast<const IO*>(p.glast)[n * page + i] : from_f32<IO>(0.f);
        return;
    }
    Lane<IO, VEC, KT> my(p, blockIdx.y * WAVE + lane);
    my.read_weights();
    Wide<VEC> dw[KT], db{};
#pragma unroll
    for (int j = 0; j < KT; ++j) dw[j] = Wide<VEC>{};
    for (int number = blockIdx.x * (THREADS / WAVE) + wave; number < p.rows * p.runs; number += run_blocks * (THREADS / WAVE)) {
        Run r(p, __builtin_amdgcn_readfirstlane(number));
        const int stop = min(p.T, r.t1 + p.K - 1);         // the gradients of a run's tokens come from up to K - 1 tokens behind it
        Packed<IO, VEC> ahead_x[AHEAD], ahead_g[AHEAD];
        const auto fetch = [&](int t) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int at = min(t + i, stop - 1);
                ahead_x[i] = my.packed(p.x, r.b * p.x_b + at * p.x_t);
                ahead_g[i] = my.packed(p.gy, r.b * p.g_b + at * p.g_t);
            }
        };
        fetch(r.t0);
        r.find(p, lane);
        const int to = p.seq.offsets ? min(stop, p.seq.at(p.N)) : stop;
        Wide<VEC> x[KT], acc[KT];                          // acc[d]: what has come to token t - d
#pragma unroll
        for (int j = 0; j < KT; ++j) acc[j] = x[j] = Wide<VEC>{};
#pragma unroll
        for (int j = 0; j < KT - 1; ++j)
            if (r.w.begin < r.t0 && my.used(j)) x[j + 1] = my.token(r.w.n, r.b, r.t0 - (KT - 1) + j, r.w.begin);
        // token t of the sequence, or of its first state, is complete (of offsets that do not ascend a sequence may begin behind the token it is looked up for: nothing in front of its state is written)
        const auto done = [&](int t, Wide<VEC> v, int tail) {
            if (tail >= 0 && p.glast) {
                const Wide<VEC> g = my.row(p.glast, ((long long)r.w.n * (p.K - 1) + tail) * p.E);
#pragma unroll
                for (int k = 0; k < VEC; ++k) v.v[k] += g.v[k];
            }
            if (t >= r.w.begin) {
                if (t >= r.t0 && t < r.t1) my.store(p.dx, ((long long)r.b * p.T + t) * p.E, v);
            } else if (p.dstate && t >= r.w.begin - (p.K - 1) && r.w.begin >= r.t0 && r.w.begin < r.t1) my.store(p.dstate, ((long long)r.w.n * (p.K - 1) + t - r.w.begin + p.K - 1) * p.E, v);
        };
        bool over = false;
        for (int t = r.t0; t < stop && !over; t += AHEAD) {
            Packed<IO, VEC> now_x[AHEAD], now_g[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) now_x[i] = ahead_x[i], now_g[i] = ahead_g[i];
            if (t + AHEAD < stop) fetch(t + AHEAD);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int ti = t + i;
                if (over || ti >= stop) break;
                if (ti < r.from || ti >= to) {
                    if (ti < r.t1) my.store(p.dx, ((long long)r.b * p.T + ti) * p.E, Wide<VEC>{});
                    else over = true;
                    continue;
                }
                if (ti == r.w.begin) {
                    if (ti >= r.t1) { over = true; break; }
#pragma unroll
                    for (int j = 0; j < KT - 1; ++j) x[j + 1] = my.used(j) ? my.token(r.w.n, r.b, r.w.begin - (KT - 1) + j, r.w.begin) : Wide<VEC>{};
#pragma unroll
                    for (int j = 0; j < KT; ++j) acc[j] = Wide<VEC>{};
                }
#pragma unroll
                for (int j = 0; j < KT - 1; ++j) x[j] = x[j + 1];
                widen_packed<IO, VEC>(now_x[i], x[KT - 1].v);
                Wide<VEC> g;
                widen_packed<IO, VEC>(now_g[i], g.v);
                if (p.silu) {
                    const Wide<VEC> s = my.pre(x);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) g.v[k] *= silu_slope(s.v[k]);
                }
                if (ti < r.t1) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        db.v[k] += g.v[k];
#pragma unroll
                        for (int j = 0; j < KT; ++j)
                            if (my.used(j)) dw[j].v[k] = fmaf(g.v[k], x[j].v[k], dw[j].v[k]);
                    }
                }
#pragma unroll
                for (int d = KT - 1; d >= 0; --d)
                    if (my.used(KT - 1 - d))
#pragma unroll
                        for (int k = 0; k < VEC; ++k) acc[d].v[k] = fmaf(my.w[KT - 1 - d].v[k], g.v[k], d ? acc[d - 1].v[k] : 0.f);
                if (KT < 8) done(ti - (KT - 1), acc[KT - 1], -1);
                else
#pragma unroll
                    for (int d = 4; d < KT; ++d)
                        if (d == p.K - 1) done(ti - d, acc[d], -1);
                if (ti == r.w.end - 1) {
#pragma unroll
                    for (int d = KT - 2; d >= 0; --d)
                        if (d <= p.K - 2) done(ti - d, acc[d], p.K - 2 - d);
                    r.w.next(p.seq);
                    if (ti + 1 >= r.t1) over = true;
                }
            }
        }
    }
    float* const out = p.part + (long long)blockIdx.x * (p.K + 1) * p.E;
    const int first = blockIdx.y * WAVE * VEC;
    const auto leave = [&](const Wide<VEC>& v, int row) {  // the waves' sums, one row at a time
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) red[wave][lane * VEC + k] = v.v[k];
        __syncthreads();
        for (int i = threadIdx.x; i < WAVE * VEC; i += THREADS)
            if (first + i < p.E) out[(long long)row * p.E + first + i] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
    };
#pragma unroll
    for (int j = 0; j < KT; ++j)
        if (my.used(j)) leave(dw[j], j - (KT - p.K));
    leave(db, p.K);
}

// dweight (E, K) and dbias (E) from the parts: 64 channels and four slices of the parts a workgroup, one tap or the bias each.
__global__ __launch_bounds__(THREADS) void finish_kernel(const float* part, void* dw, void* db, int parts, int E, int K, int dtype) {
    __shared__ float red[THREADS / WAVE][WAVE];
    const int c = blockIdx.x * WAVE + (threadIdx.x & 63), j = blockIdx.y, slice = threadIdx.x >> 6;
    float v = 0.f;
    if (c < E)
#pragma unroll 8
        for (int k = slice; k < parts; k += THREADS / WAVE) v += part[((long long)k * (K + 1) + j) * E + c];
    red[slice][threadIdx.x & 63] = v;
    __syncthreads();
    if (slice || c >= E) return;
    v = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    void* to = j < K ? dw : db;
    const long long i = j < K ? (long long)c * K + j : c;
    if (!to) return;
    if (dtype == VRWKV_F32) static_cast<float*>(to)[i] = v;
    else if (dtype == VRWKV_BF16) static_cast<__hip_bfloat16*>(to)[i] = from_f32<__hip_bfloat16>(v);
    else static_cast<__half*>(to)[i] = from_f32<__half>(v);
}

constexpr int BACKWARD_VEC = 4;                            // channels of 16 bits a lane: weights, sums and rows of K taps for eight would take 340 registers
int backward_vec(const vrwkv_conv_args& a) {
    const long long strides[] = {a.offsets ? 0 : a.x_stride[0], a.x_stride[1], a.offsets ? 0 : a.gy_stride[0], a.gy_stride[1]};
    return vec_of(a.dtype, a.E, a.dtype == VRWKV_F32 ? 16 : 2 * BACKWARD_VEC, (size_t)a.x | (size_t)a.gy | (size_t)a.dx | (size_t)a.state | (size_t)a.dstate | (size_t)a.glast, strides, 4);
}

// As many runs as there are waves at once, three for each of the chip's vector units, of 8 tokens at least; a wave takes several where there are more rows than that.
// 64 x 196 and 8 x 2048 tokens of 1536 channels in bf16: 37 and 45 us; with a third more waves than fit 44 and 53, with twice as many 46 and 53.
int waves_at_once(const Plan& p) { return std::max(1, 12 * device_cus() / p.waves); }
Plan plan_of(const vrwkv_conv_args& a, int vec) {
    Plan p;
    p.rows = a.offsets ? 1 : a.N;
    p.waves = (a.E + WAVE * vec - 1) / (WAVE * vec);
    const int pieces = std::max(1, std::min(waves_at_once(p) / p.rows, a.T / 8));
    p.run = (a.T + pieces - 1) / pieces;
    p.runs = (a.T + p.run - 1) / p.run;
    return p;
}
int parts_of(const Plan& p) { return (int)((std::min<long long>(waves_at_once(p), (long long)p.rows * p.runs) + THREADS / WAVE - 1) / (THREADS / WAVE)); }


}  // namespace
}  // namespace conv
}  // namespace vrwkv

using namespace vrwkv;
using namespace vrwkv::conv;

extern "C" size_t vrwkv_conv_bwd_workspace_bytes(const vrwkv_conv_args* args) {
    if (!args || args->N <= 0 || args->T <= 0 || args->E <= 0 || args->K < 2 || args->K > 8) return 0;
    const Plan p = plan_of(*args, backward_vec(*args));
    return (size_t)parts_of(p) * (args->K + 1) * args->E * 4;
}

extern "C" int vrwkv_conv_bwd(const vrwkv_conv_args* args, void* hip_stream) {
    const char* who = "vrwkv_conv_bwd";
    if (const int rc = check(who, args, true)) return rc;
    const vrwkv_conv_args& a = *args;
    const int vec = backward_vec(a);
    const Plan pl = plan_of(a, vec);
    const int parts = parts_of(pl);
    const size_t need = (size_t)parts * (a.K + 1) * a.E * 4;
    if (!a.workspace || a.workspace_bytes < need) { set_error("%s: workspace of %zu bytes, %zu needed", who, a.workspace ? a.workspace_bytes : (size_t)0, need); return VRWKV_WORKSPACE_TOO_SMALL; }
    Params p = params_of(a, pl, vec);
    p.part = static_cast<float*>(a.workspace);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int extra = a.offsets && a.dstate ? std::min(a.N, 64) : 0;
    const auto launched = [&](auto io, auto v) {
        using IO = decltype(io);
        constexpr int VEC = decltype(v)::value;
        return with_taps(a.K, [&](auto k) {
            constexpr int KT = decltype(k)::value;
            hipLaunchKernelGGL((backward_kernel<IO, VEC, KT>), dim3(parts + extra, pl.waves), dim3(THREADS), 0, st, p, parts);
            return check_launch(who);
        });
    };
    const int rc = with_types<BACKWARD_VEC>(a.dtype, vec, launched);
    if (rc != VRWKV_OK) return rc;
    hipLaunchKernelGGL(finish_kernel, dim3((a.E + WAVE - 1) / WAVE, a.K + 1), dim3(THREADS), 0, st, p.part, a.dweight, a.dbias, parts, a.E, a.K, a.param_dtype);
    return check_launch(who);
}
