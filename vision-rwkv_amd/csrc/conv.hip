// The short causal convolution (conv.h): whole sequences, and one more token of each of N.
#include "conv.h"
#include "pages.h"

namespace vrwkv {
namespace conv {
namespace {

constexpr int AHEAD = 8;
// Runs of 8 tokens, longer ones (up to 64) once there are four waves for each of the chip's vector units.  64 x 196 x 1536 bf16: 19.6 us with 8, 21.8 with 16, 30 with 32.
Plan plan_of(const vrwkv_conv_args& a, int vec) {
    Plan p;
    p.rows = a.offsets ? 1 : a.N;
    p.waves = (a.E + WAVE * vec - 1) / (WAVE * vec);
    const long long run = (long long)p.rows * a.T * p.waves / (16LL * device_cus());
    p.run = (int)std::max(8LL, std::min(64LL, run / AHEAD * AHEAD));
    p.runs = (a.T + p.run - 1) / p.run;
    return p;
}

// What is behind the last token of each sequence: element i of (N, K - 1, E).
template <typename IO>
__device__ __forceinline__ void last_states(const Params& p, long long first, long long step) {
    const long long all = (long long)p.N * (p.K - 1) * p.E;
    for (long long i = first; i < all; i += step) {
        const int c = (int)(i % p.E), k = (int)(i / p.E % (p.K - 1)), n = (int)(i / p.E / (p.K - 1));
        const int begin = p.seq.offsets ? p.seq.of_lane(n) : 0, end = p.seq.offsets ? max(begin, p.seq.of_lane(n + 1)) : p.T, t = end - (p.K - 1) + k;
        IO v = from_f32<IO>(0.f);
        if (t >= begin) v = static_cast<const IO*>(p.x)[(p.seq.offsets ? 0 : n * p.x_b) + t * p.x_t + c];
        else if (p.state) v = static_cast<const IO*>(p.state)[((long long)n * (p.K - 1) + t - begin + p.K - 1) * p.E + c];
        static_cast<IO*>(p.last)[i] = v;
    }
}

// Waves of a workgroup take runs next to each other.  The last `extra` workgroups write the states.  Workgroups go on in z where x ends: a launch's dimension has room for 2^24 of 256 threads.
constexpr int GRID_X = 1 << 22;
template <typename IO, int VEC, int KT>
__global__ __launch_bounds__(THREADS) void forward_kernel(const Params p, int run_blocks, int extra) {
    const int lane = threadIdx.x & 63, block = blockIdx.z * GRID_X + blockIdx.x;
    if (block >= run_blocks) {
        if (blockIdx.y == 0 && block < run_blocks + extra) last_states<IO>(p, (long long)(block - run_blocks) * THREADS + threadIdx.x, (long long)extra * THREADS);
        return;
    }
    const int number = block * (THREADS / WAVE) + (threadIdx.x >> 6);
    if (number >= p.rows * p.runs) return;
    Run r(p, __builtin_amdgcn_readfirstlane(number));
    Lane<IO, VEC, KT> my(p, blockIdx.y * WAVE + lane);
    Packed<IO, VEC> ahead[AHEAD], front[KT - 1];
    const auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ahead[i] = my.packed(p.x, r.b * p.x_b + min(t + i, r.t1 - 1) * p.x_t);
    };
    // all rows, and the weights, before it is known what sequences there are
#pragma unroll
    for (int j = 0; j < KT - 1; ++j)
        if (my.used(j)) front[j] = my.packed(p.x, r.b * p.x_b + max(r.t0 - (KT - 1) + j, 0) * p.x_t);
    fetch(r.t0);
    my.read_weights();
    r.find(p, lane);
    Wide<VEC> x[KT];                                       // x[j]: token t - (KT - 1) + j
#pragma unroll
    for (int j = 0; j < KT - 1; ++j) {
        x[j + 1] = Wide<VEC>{};
        const int t = r.t0 - (KT - 1) + j;
        if (!my.used(j) || r.w.begin >= r.t0) continue;
        if (t >= r.w.begin) widen_packed<IO, VEC>(front[j], x[j + 1].v);
        else x[j + 1] = my.token(r.w.n, r.b, t, r.w.begin);
    }
    for (int t = r.t0; t < r.t1; t += AHEAD) {
        Packed<IO, VEC> now[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) now[i] = ahead[i];
        if (t + AHEAD < r.t1) fetch(t + AHEAD);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (t + i >= r.t1) break;
            const long long out = ((long long)r.b * p.T + t + i) * p.E;
            if (t + i < r.from || t + i >= r.to) {
                my.store(p.y, out, Wide<VEC>{});
                continue;
            }
            if (t + i == r.w.begin) {
#pragma unroll
                for (int j = 0; j < KT - 1; ++j) x[j + 1] = my.used(j) ? my.token(r.w.n, r.b, r.w.begin - (KT - 1) + j, r.w.begin) : Wide<VEC>{};
            }
#pragma unroll
            for (int j = 0; j < KT - 1; ++j) x[j] = x[j + 1];
            widen_packed<IO, VEC>(now[i], x[KT - 1].v);
            Wide<VEC> y = my.pre(x);
            if (p.silu)
#pragma unroll
                for (int k = 0; k < VEC; ++k) y.v[k] = silu_of(y.v[k]);
            my.store(p.y, out, y);
            if (t + i == r.w.end - 1) r.w.next(p.seq);
        }
    }
}

constexpr int GRID_Y = 32768;
struct StepParams {
    Params f;
    Slots slots;
    void* pool;
    long long page, x_n;
};
template <typename IO, int VEC, int KT>
__global__ __launch_bounds__(THREADS) void step_kernel(const StepParams sp) {
    const Params& p = sp.f;
    const int n0 = blockIdx.y + GRID_Y * blockIdx.z;
    if (n0 >= sp.slots.rows) return;
    const long long slot = sp.slots.at(n0);
    const bool known = sp.slots.has(slot);
    IO* const page = static_cast<IO*>(sp.pool) + (known ? slot : 0) * sp.page;
    Lane<IO, VEC, KT> my(p, blockIdx.x * THREADS + threadIdx.x);
    my.read_weights();
    Wide<VEC> x[KT];
    Wide<VEC> now = my.row(p.x, n0 * sp.x_n);
#pragma unroll
    for (int j = 0; j < KT - 1; ++j) x[j + 1] = known && my.used(j) && my.there ? my.row(page, (long long)(j - (KT - p.K)) * p.E) : Wide<VEC>{};
    const long long slots[1] = {slot};
    unsigned skipped, shared;
    sp.slots.find_others<1>(n0, slots, skipped, shared);
    if (skipped) return;
    int next = shared ? sp.slots.behind(n0, slot) : sp.slots.rows;
    for (int n = n0;;) {
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) x[j] = x[j + 1];
        x[KT - 1] = now;
        Wide<VEC> y = my.pre(x);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if (p.silu) y.v[k] = silu_of(y.v[k]);
            if (!known) y.v[k] = slot == -1 ? 0.f : __builtin_nanf("");
        }
        my.store(p.y, (long long)n * p.E, y);
        if (next >= sp.slots.rows) break;
        n = next;
        next = sp.slots.behind(n, slot);
        now = my.row(p.x, n * sp.x_n);
    }
    if (!known) return;
#pragma unroll
    for (int j = 1; j < KT; ++j)
        if (my.used(j - 1)) my.store(page, (long long)(j - 1 - (KT - p.K)) * p.E, x[j]);
}

}  // namespace
}  // namespace conv
}  // namespace vrwkv

using namespace vrwkv;
using namespace vrwkv::conv;

extern "C" int vrwkv_conv_fwd(const vrwkv_conv_args* args, void* hip_stream) {
    const char* who = "vrwkv_conv_fwd";
    if (const int rc = check(who, args, false)) return rc;
    const vrwkv_conv_args& a = *args;
    const long long strides[] = {a.offsets ? 0 : a.x_stride[0], a.x_stride[1]};
    const int vec = vec_of(a.dtype, a.E, 16, (size_t)a.x | (size_t)a.y | (size_t)a.state, strides, 2);
    const Plan pl = plan_of(a, vec);
    const Params p = params_of(a, pl, vec);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int blocks = (int)(((long long)pl.rows * pl.runs + THREADS / WAVE - 1) / (THREADS / WAVE));
    const int extra = a.last ? (int)std::min<long long>(4LL * device_cus(), ((long long)a.N * (a.K - 1) * a.E + THREADS - 1) / THREADS) : 0;
    return with_types<8>(a.dtype, vec, [&](auto io, auto v) {
        using IO = decltype(io);
        constexpr int VEC = decltype(v)::value;
        return with_taps(a.K, [&](auto k) {
            constexpr int KT = decltype(k)::value;
            hipLaunchKernelGGL((forward_kernel<IO, VEC, KT>), dim3(std::min(blocks + extra, GRID_X), pl.waves, (blocks + extra + GRID_X - 1) / GRID_X), dim3(THREADS), 0, st, p, blocks, extra);
            return check_launch(who);
        });
    });
}

extern "C" int vrwkv_conv_step(const vrwkv_conv_step_args* args, void* hip_stream) {
    const char* who = "vrwkv_conv_step";
    if (!args || !args->x || !args->weight || !args->pool || !args->y) { set_error("%s: null pointer", who); return VRWKV_INVALID_ARG; }
    const vrwkv_conv_step_args& a = *args;
    if (a.N <= 0 || a.P <= 0 || a.E <= 0) { set_error("%s: N, P and E must be positive", who); return VRWKV_INVALID_ARG; }
    if (!typed(a.dtype) || !typed(a.param_dtype)) { set_error("%s: dtype must be fp32, bf16 or fp16", who); return VRWKV_UNSUPPORTED_DTYPE; }
    if (a.K < 2 || a.K > 8 || a.E > 1 << 22) { set_error("%s: 2 to 8 taps (%d), and at most 2^22 channels", who, a.K); return VRWKV_UNSUPPORTED_SHAPE; }
    if (a.N >= 1 << 30) { set_error("%s: 2^30 rows or more", who); return VRWKV_UNSUPPORTED_SHAPE; }
    if (!a.slots && a.N > a.P) { set_error("%s: %d rows without slots, and %d pages", who, a.N, a.P); return VRWKV_INVALID_ARG; }
    if (a.page_stride < (long long)(a.K - 1) * a.E) { set_error("%s: pages overlap", who); return VRWKV_INVALID_ARG; }
    if (!aligned(a.x, a.dtype) || !aligned(a.y, a.dtype) || !aligned(a.pool, a.dtype) || !aligned(a.weight, a.param_dtype) || !aligned(a.bias, a.param_dtype) ||
        (a.slots && ((size_t)a.slots & (a.slots64 ? 7 : 3)))) {
        set_error("%s: a tensor is not aligned to its elements", who);
        return VRWKV_INVALID_ARG;
    }
    StepParams sp{};
    sp.f.x = a.x, sp.f.y = a.y, sp.f.w = ParamVec(a.weight, a.param_dtype, 1.f), sp.f.bias = ParamVec(a.bias, a.param_dtype, 1.f);
    sp.f.E = a.E, sp.f.K = a.K, sp.f.silu = a.silu;
    sp.slots = Slots{a.slots, a.slots64, a.N, a.P}, sp.pool = a.pool, sp.page = a.page_stride, sp.x_n = a.x_stride;
    const long long strides[] = {a.x_stride, a.page_stride};
    const int vec = vec_of(a.dtype, a.E, 16, (size_t)a.x | (size_t)a.y | (size_t)a.pool, strides, 2);
    sp.f.weights_aligned = weights_fit(a.weight, a.bias, a.param_dtype, vec);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const dim3 grid((a.E / vec + THREADS - 1) / THREADS, std::min(a.N, GRID_Y), (a.N + GRID_Y - 1) / GRID_Y);
    return with_types<8>(a.dtype, vec, [&](auto io, auto v) {
        using IO = decltype(io);
        constexpr int VEC = decltype(v)::value;
        return with_taps(a.K, [&](auto k) {
            constexpr int KT = decltype(k)::value;
            hipLaunchKernelGGL((step_kernel<IO, VEC, KT>), grid, dim3(THREADS), 0, st, sp);
            return check_launch(who);
        });
    });
}
