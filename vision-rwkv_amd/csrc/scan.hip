// vrwkv_scan_fwd and vrwkv_scan_bwd: checks, cuts and the sums that end a backward pass (the kernels: scan.h, scan_short.h, scan_bwd.h).
#include "scan_bwd.h"
#include "scan_short.h"
#include <algorithm>
#include <cstdint>

namespace vrwkv {
namespace scan {

// Instantiated in scan_{f32,bf16,f16}.hip and scan_bwd_{f32,bf16,f16}.hip.
extern template int launch_forward<float>(const Params&, hipStream_t);
extern template int launch_forward<__hip_bfloat16>(const Params&, hipStream_t);
extern template int launch_forward<__half>(const Params&, hipStream_t);
extern template int launch_short<float>(const Params&, int, hipStream_t);
extern template int launch_backward<float>(const BackParams&, int, hipStream_t);
extern template int launch_short<__hip_bfloat16>(const Params&, int, hipStream_t);
extern template int launch_backward<__hip_bfloat16>(const BackParams&, int, hipStream_t);
extern template int launch_short<__half>(const Params&, int, hipStream_t);
extern template int launch_backward<__half>(const BackParams&, int, hipStream_t);

namespace {

struct Plan {
    int P, rows, blocks, L, nseg, parts;                  // parts: workgroups that the rows of the batch are dealt out to, in a backward
    size_t states;                                        // floats of one state for all channels, filled up to four a lane
};
// (one lane for up to four states would have all of sixteen tokens' numbers in its registers: forward 89 us for 78, with gradients 562 for 331 at 64 x 196 x 1536 bf16)
int lanes_of(int S) { return S <= 8 ? 2 : S <= 16 ? 4 : S <= 32 ? 8 : 16; }

// Few sequences are cut into segments, which costs a pass over them in front of the one with the results: enough pieces for four waves on each of the chip's vector units, none
// shorter than 32 tokens, no more than 64 (a segment goes through those in front of it).  2 x 4150 tokens of 768 channels, bf16 forward: 690 us whole, 157 in 8, 84 in 43; 8 x 196 of
// 1536, which have half as many waves without it, 36.8 whole and 35.9 in 7.
Plan plan_of(const vrwkv_scan_args& a) {
    Plan p;
    p.P = lanes_of(a.S);
    p.rows = a.offsets ? 1 : a.N;
    p.blocks = (a.E / a.G + THREADS / p.P - 1) / (THREADS / p.P);
    p.states = (size_t)a.E * 4 * p.P;
    const long long groups = (long long)p.rows * a.G * p.blocks, wanted = 4LL * device_cus();
    long long n = option(OPT_SCAN_SEGMENTS);
    if (!n) n = 2 * groups > wanted ? 1 : std::min<long long>((wanted + groups - 1) / groups, a.T / 32);
    n = std::max(1LL, std::min(64LL, n));
    p.L = (int)((a.T + n - 1) / n + BATCH - 1) / BATCH * BATCH;
    p.nseg = (a.T + p.L - 1) / p.L;
    p.parts = (int)std::max(1LL, std::min<long long>(p.rows, 8LL * device_cus() / std::max(1LL, (long long)a.G * p.blocks * p.nseg)));
    return p;
}

// Whether a forward goes through scan_short.h: one workgroup a compute unit, and four rounds of its waves over the tokens.  bf16, 16 states, that kernel against the segments': 196 tokens of
// 384 channels 7.9 us for 16.3, 1024 of 384 23 for 27; beyond it 196 of 1536 (384 workgroups) 13.6 for 15.2, 1024 of 1536 45 for 32, 4 x 196 of 1536 39 for 24, 4150 of 384 80 for 51.
bool is_short(const vrwkv_scan_args& a) {
    const long long groups = (long long)(a.offsets ? 1 : a.N) * a.G * ((a.E / a.G + SHORT_CHANNELS - 1) / SHORT_CHANNELS);
    return !option(OPT_SCAN_SEGMENTS) && groups <= device_cus() && a.T <= 4 * BATCH * short_waves(a.S);
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }
size_t chunks_of(const vrwkv_scan_args& a) { return ((size_t)a.T + BATCH - 1) / BATCH; }
size_t segment_bytes(const vrwkv_scan_args& a, const Plan& p) { return p.nseg > 1 ? up16((size_t)p.rows * p.nseg * p.states * 4) + up16((size_t)p.rows * p.nseg * a.E * 4) : 0; }
size_t forward_bytes(const vrwkv_scan_args& a, const Plan& p) { return is_short(a) ? 0 : segment_bytes(a, p); }
size_t part_bc_floats(const vrwkv_scan_args& a, const Plan& p) { return (size_t)p.blocks * p.rows * a.T * a.G * 8 * p.P; }
size_t backward_bytes(const vrwkv_scan_args& a, const Plan& p) {
    const size_t parts = (size_t)p.parts * p.nseg;
    return segment_bytes(a, p) + up16(part_bc_floats(a, p) * 4) + up16(parts * p.states * 4) + 2 * up16(parts * a.E * 4);
}

bool typed(int d) { return d >= VRWKV_F32 && d <= VRWKV_F16; }
bool aligned(const void* p, int dtype) { return ((size_t)p & (dtype == VRWKV_F32 ? 3 : 1)) == 0; }

int check(const char* who, const vrwkv_scan_args* args, bool backward) {
    if (!args) { set_error("%s: null pointer", who); return VRWKV_INVALID_ARG; }
    const vrwkv_scan_args& a = *args;
    if (!a.u || !a.delta || !a.A || !a.B || !a.C || (!backward && !a.y) || (backward && (!a.gy || !a.kept || !a.du || !a.ddelta || !a.dA || !a.dB || !a.dC || (a.z && !a.dz)))) {
        set_error("%s: null pointer", who);
        return VRWKV_INVALID_ARG;
    }
    if (a.N <= 0 || a.T <= 0 || a.E <= 0 || a.G <= 0) { set_error("%s: N, T, E and G must be positive", who); return VRWKV_INVALID_ARG; }
    if (!typed(a.dtype) || !typed(a.D_dtype) || !typed(a.bias_dtype)) { set_error("%s: dtype must be fp32, bf16 or fp16", who); return VRWKV_UNSUPPORTED_DTYPE; }
    if (a.S < 1 || a.S > 64 || a.E % a.G || a.E > 1 << 22 || a.G > 1 << 16) { set_error("%s: 1 to 64 states (%d), E (%d, at most 2^22) a multiple of G (%d, at most 2^16)", who, a.S, a.E, a.G); return VRWKV_UNSUPPORTED_SHAPE; }
    const long long strides[] = {a.u_stride[1], a.delta_stride[1], a.z_stride[1], backward ? a.gy_stride[1] : 0, a.B_stride[1], a.C_stride[1]};
    for (long long s : strides)
        if (s < 0 || s >= 1LL << 22) { set_error("%s: tokens must be less than 2^22 elements apart", who); return VRWKV_UNSUPPORTED_SHAPE; }
    const Plan p = plan_of(a);
    if (a.T >= 1 << 30 || a.N >= 1 << 30 || p.rows > 65535 || (long long)a.G * p.blocks >= 1 << 24) { set_error("%s: at most 65535 rows of less than 2^30 tokens, less than 2^30 sequences", who); return VRWKV_UNSUPPORTED_SHAPE; }
    bool fits = aligned(a.u, a.dtype) && aligned(a.delta, a.dtype) && aligned(a.B, a.dtype) && aligned(a.C, a.dtype) && aligned(a.z, a.dtype) && aligned(a.D, a.D_dtype) &&
                aligned(a.delta_bias, a.bias_dtype) && (((size_t)a.A | (size_t)a.state | (size_t)a.last) & 3) == 0 && (((size_t)a.kept | (size_t)a.workspace) & 15) == 0 &&
                (!a.offsets || ((size_t)a.offsets & (a.offsets64 ? 7 : 3)) == 0);
    if (!backward) fits = fits && aligned(a.y, a.dtype);
    else
        fits = fits && aligned(a.gy, a.dtype) && aligned(a.du, a.dtype) && aligned(a.ddelta, a.dtype) && aligned(a.dz, a.dtype) && aligned(a.dB, a.dtype) && aligned(a.dC, a.dtype) &&
               aligned(a.dD, a.D_dtype) && aligned(a.dbias, a.bias_dtype) && (((size_t)a.dA | (size_t)a.dstate | (size_t)a.glast) & 3) == 0;
    if (!fits) { set_error("%s: a tensor is not aligned to its elements, kept or the workspace to 16 bytes", who); return VRWKV_INVALID_ARG; }
    const size_t need = backward ? backward_bytes(a, p) : forward_bytes(a, p);
    if (need && (!a.workspace || a.workspace_bytes < need)) { set_error("%s: workspace of %zu bytes, %zu needed", who, a.workspace ? a.workspace_bytes : (size_t)0, need); return VRWKV_WORKSPACE_TOO_SMALL; }
    return VRWKV_OK;
}

Params params_of(const vrwkv_scan_args& a, const Plan& pl) {
    Params p{};
    p.u = a.u, p.delta = a.delta, p.B = a.B, p.C = a.C, p.z = a.z, p.A = a.A, p.state = a.state;
    p.D = ParamVec(a.D, a.D_dtype, 1.f), p.bias = ParamVec(a.delta_bias, a.bias_dtype, 1.f);
    p.seq = Sequences{a.offsets, a.offsets64, a.N, a.T};
    p.y = a.y, p.last = a.last, p.kept = a.kept;
    p.u_b = a.u_stride[0], p.u_t = a.u_stride[1], p.d_b = a.delta_stride[0], p.d_t = a.delta_stride[1], p.z_b = a.z_stride[0], p.z_t = a.z_stride[1];
    p.B_b = a.B_stride[0], p.B_t = a.B_stride[1], p.B_g = a.B_stride[2], p.C_b = a.C_stride[0], p.C_t = a.C_stride[1], p.C_g = a.C_stride[2];
    p.N = a.N, p.rows = pl.rows, p.T = a.T, p.E = a.E, p.S = a.S, p.G = a.G, p.softplus = a.softplus, p.L = pl.L, p.nseg = pl.nseg, p.blocks = pl.blocks;
    char* ws = static_cast<char*>(a.workspace);
    if (pl.nseg > 1) {
        p.seg_h = reinterpret_cast<float*>(ws);
        p.seg_dt = reinterpret_cast<float*>(ws + up16((size_t)pl.rows * pl.nseg * pl.states * 4));
    }
    return p;
}

struct Finish {
    const float *part_bc, *part_A, *part_D, *part_bias;
    void *dB, *dC, *dD, *dbias;
    float* dA;
    long long tokens;                                     // of all rows
    int parts, blocks, E, S, G, W, dtype, D_dtype, bias_dtype, column_blocks;   // W: floats of a filled-up row of states
};
__device__ __forceinline__ void put(void* to, long long i, int dtype, float v) {
    if (dtype == VRWKV_F32) static_cast<float*>(to)[i] = v;
    else if (dtype == VRWKV_BF16) static_cast<__hip_bfloat16*>(to)[i] = from_f32<__hip_bfloat16>(v);
    else static_cast<__half*>(to)[i] = from_f32<__half>(v);
}
// What workgroups have left of sums: over parts for A, D and the bias, 64 columns and four slices of the parts a workgroup; over channels for B and C.  Fixed orders.
__global__ __launch_bounds__(THREADS) void finish_kernel(const Finish f) {
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < f.column_blocks) {
        __shared__ float red[4][64];
        const long long i = (long long)blockIdx.x * 64 + (tid & 63), A = (long long)f.E * f.W;
        const float* src = nullptr;
        long long step = 0;
        if (i < A) src = f.part_A + i, step = A;
        else if (i < A + f.E) src = f.part_D + (i - A), step = f.E;
        else if (i < A + 2 * f.E) src = f.part_bias + (i - A - f.E), step = f.E;
        float v = 0.f;
        if (src)
#pragma unroll 8
            for (int k = tid >> 6; k < f.parts; k += 4) v += src[k * step];
        red[tid >> 6][tid & 63] = v;
        __syncthreads();
        if (tid >= 64 || !src) return;
        v = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
        if (i < A) {
            const int n = (int)(i % f.W);
            if (n < f.S) f.dA[i / f.W * f.S + n] = v;
        } else if (i < A + f.E) {
            if (f.dD) put(f.dD, i - A, f.D_dtype, v);
        } else if (f.dbias) put(f.dbias, i - A - f.E, f.bias_dtype, v);
        return;
    }
    const long long all = f.tokens * f.G * 2 * f.W;
    for (long long i = (long long)(blockIdx.x - f.column_blocks) * THREADS + tid; i < all; i += (long long)(gridDim.x - f.column_blocks) * THREADS) {
        float v = 0.f;
#pragma unroll 8
        for (int k = 0; k < f.blocks; ++k) v += f.part_bc[k * all + i];
        const int n = (int)(i % f.W), which = (int)(i / f.W % 2);
        if (n < f.S) put(which ? f.dC : f.dB, i / (2 * f.W) * f.S + n, f.dtype, v);
    }
}

}  // namespace
}  // namespace scan
}  // namespace vrwkv

using namespace vrwkv;
using namespace vrwkv::scan;

static bool scan_sizes(const vrwkv_scan_args* a) { return a && a->N > 0 && a->T > 0 && a->E > 0 && a->G > 0 && a->S >= 1 && a->S <= 64; }

extern "C" size_t vrwkv_scan_kept_bytes(const vrwkv_scan_args* args) {
    if (!scan_sizes(args)) return 0;
    const Plan p = plan_of(*args);
    return (size_t)p.rows * chunks_of(*args) * p.states * 4;
}
extern "C" size_t vrwkv_scan_fwd_workspace_bytes(const vrwkv_scan_args* args) { return scan_sizes(args) ? forward_bytes(*args, plan_of(*args)) : 0; }
extern "C" size_t vrwkv_scan_bwd_workspace_bytes(const vrwkv_scan_args* args) { return scan_sizes(args) ? backward_bytes(*args, plan_of(*args)) : 0; }

extern "C" int vrwkv_scan_fwd(const vrwkv_scan_args* args, void* hip_stream) {
    if (const int rc = check("vrwkv_scan_fwd", args, false)) return rc;
    const Plan pl = plan_of(*args);
    Params p = params_of(*args, pl);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (is_short(*args)) {
        p.blocks = (args->E / args->G + SHORT_CHANNELS - 1) / SHORT_CHANNELS;
        if (args->dtype == VRWKV_F32) return launch_short<float>(p, 4 * pl.P, st);
        if (args->dtype == VRWKV_BF16) return launch_short<__hip_bfloat16>(p, 4 * pl.P, st);
        return launch_short<__half>(p, 4 * pl.P, st);
    }
    if (args->dtype == VRWKV_F32) return launch_forward<float>(p, st);
    if (args->dtype == VRWKV_BF16) return launch_forward<__hip_bfloat16>(p, st);
    return launch_forward<__half>(p, st);
}

extern "C" int vrwkv_scan_bwd(const vrwkv_scan_args* args, void* hip_stream) {
    if (const int rc = check("vrwkv_scan_bwd", args, true)) return rc;
    const vrwkv_scan_args& a = *args;
    const Plan pl = plan_of(a);
    BackParams bp{};
    bp.f = params_of(a, pl);
    bp.gy = a.gy, bp.glast = a.glast, bp.du = a.du, bp.dd = a.ddelta, bp.dz = a.dz, bp.dstate = a.dstate, bp.gy_b = a.gy_stride[0], bp.gy_t = a.gy_stride[1];
    bp.seg_r = bp.f.seg_h;
    const size_t parts = (size_t)pl.parts * pl.nseg;
    char* ws = static_cast<char*>(a.workspace) + segment_bytes(a, pl);
    const auto take = [&](size_t floats) {
        float* at = reinterpret_cast<float*>(ws);
        ws += up16(floats * 4);
        return at;
    };
    bp.part_bc = take(part_bc_floats(a, pl));
    bp.part_A = take(parts * pl.states);
    bp.part_D = take(parts * a.E);
    bp.part_bias = take(parts * a.E);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int rc = a.dtype == VRWKV_F32 ? launch_backward<float>(bp, pl.parts, st) : a.dtype == VRWKV_BF16 ? launch_backward<__hip_bfloat16>(bp, pl.parts, st) : launch_backward<__half>(bp, pl.parts, st);
    if (rc != VRWKV_OK) return rc;
    Finish f{bp.part_bc, bp.part_A, bp.part_D, bp.part_bias, a.dB, a.dC, a.dD, a.dbias, a.dA, (long long)pl.rows * a.T, (int)parts, pl.blocks, a.E, a.S, a.G, 4 * pl.P, a.dtype, a.D_dtype, a.bias_dtype, 0};
    const long long columns = (long long)a.E * (4 * pl.P + 2), sums = f.tokens * a.G * 8 * pl.P;
    f.column_blocks = (int)((columns + 63) / 64);
    hipLaunchKernelGGL(finish_kernel, dim3((unsigned)(f.column_blocks + std::min<long long>((sums + THREADS - 1) / THREADS, 1 << 20))), dim3(THREADS), 0, st, f);
    return check_launch("vrwkv_scan_bwd");
}
