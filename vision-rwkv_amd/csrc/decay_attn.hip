// Host side of the attention with a decay for each head (decay_attn.h), and the passes around its kernel: the states in front of the segments, and the
// sums that gradients of shared heads and of the decays leave to the end.
#include "decay_bwd.h"
#include <algorithm>
#include <cstdint>

namespace vrwkv {
namespace decay {
namespace {

// The state in front of each segment from the segments' own ones: a lane carries four numbers, of XS rows of fragments, along the sequence.
// Grid (DX / 16 / XS * N * H * tiles, 1, roles).  Several segments' states are on their way at a time: one by one they were 0.35 us each.
template <int DX, int XS>
__global__ __launch_bounds__(THREADS) void segments_kernel(const Params p) {
    constexpr int XG = DX / 16 / XS, U = XS == 1 ? 8 : 4;
    touch(p);
    const Role& r = p.role[blockIdx.z];
    int id = blockIdx.x / XG;
    const int z = id % r.tiles;
    id /= r.tiles;
    const int h = id % p.H, n = id / p.H;
    const Place w = sequence_place(p, n, 64);
    const int x0 = blockIdx.x % XG * XS, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int count = segment_count(p, w.len);
    if (count == 1) return;                               // (starts from what it is given)
    f32x4 carry[XS];
#pragma unroll
    for (int x = 0; x < XS; ++x) carry[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r.init) {
        const StatePage s(r.init + ((long long)n * p.H + h) * ((long long)r.dx * r.dz), r.sx, r.sz, r.dx, r.dz, 16 * x0 + 4 * (lane >> 4), z * TZ + 16 * wave + (lane & 15));
#pragma unroll
        for (int x = 0; x < XS; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) carry[x][i] = s.load(16 * x + i);
    }
    const int lead = segment_page(p, n, w.first, 0), step = p.by_start ? 2 : 1, rest = segment_page(p, n, w.first, 1) - step;
    const auto at = [&](int i) {                          // the i-th on the way
        const int j = r.reverse ? count - 1 - i : i;
        return (long long)(j == 0 ? lead : rest + step * j) * p.H + h;
    };
    const long long in_tile = ((long long)x0 * 4 + wave) * 64 * 4 + lane * 4;
    for (int i0 = 0; i0 < count; i0 += U) {
        f32x4 own[U][XS];
        float d[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u + 1 < count) {                     // (the last one on the way has not been made)
#pragma unroll
                for (int x = 0; x < XS; ++x) own[u][x] = *reinterpret_cast<const f32x4*>(r.seg + (at(i0 + u) * r.tiles + z) * (DX * TZ) + in_tile + x * 1024);
                d[u] = r.seg_decay[at(i0 + u)];
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u < count)
#pragma unroll
                for (int x = 0; x < XS; ++x) {
                    if (i0 + u > 0) *reinterpret_cast<f32x4*>(r.seg + (at(i0 + u) * r.tiles + z) * (DX * TZ) + in_tile + x * 1024) = carry[x];
                    if (i0 + u + 1 < count)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            // (a decay of +0 is too small for fp32, and an infinity stays one; one of -0 forgets, and makes NaN of it)
                            const bool stays = __builtin_bit_cast(unsigned, d[u]) == 0u && fabsf(carry[x][c]) == __builtin_inff();
                            carry[x][c] = fmaf(carry[x][c], stays ? 1.f : d[u], own[u][x][c]);
                        }
                }
    }
}

// out (rows, heads, D) = the sums of part (parts, rows, heads * share, D) over the parts and the heads that share one, rounded once
struct Sum {
    const float* part;
    void* out;
    long long count, apart;                               // results, or fours of them; numbers from part to part
    int D, share, parts, fours;
};
struct Sums {
    Sum s[3];
    const float* decay_part;                              // dg (rows, H) = the sums of (tiles, rows, H), of which each has decay_count numbers; or
    const double* decay_sums;                             // dg (H) = the sums of (segments and tiles, H), in 64 bits: a workgroup for each head
    void* dg;
    long long decay_count, decay_n;
    int n, g_dtype, tiles, H;                             // sums of s
};
__device__ __forceinline__ void put_decay(const Sums& all, long long i, float x) {
    if (all.g_dtype == VRWKV_F32) static_cast<float*>(all.dg)[i] = x;
    else if (all.g_dtype == VRWKV_BF16) static_cast<__hip_bfloat16*>(all.dg)[i] = from_f32<__hip_bfloat16>(x);
    else static_cast<__half*>(all.dg)[i] = from_f32<__half>(x);
}
// All that a call adds up, in one launch: y 0 .. n - 1 the gradients of s, y = n those of the decays.
template <typename IO>
__global__ __launch_bounds__(THREADS) void sums_kernel(const Sums all) {
    const long long first = (long long)blockIdx.x * THREADS + threadIdx.x, step = (long long)gridDim.x * THREADS;
    if ((int)blockIdx.y < all.n) {
        const Sum t = all.s[blockIdx.y];
        if (t.fours) {
            const int D4 = t.D / 4;
            for (long long i = first; i < t.count; i += step) {
                const float* q = t.part + i / D4 * t.share * t.D + i % D4 * 4;
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
                for (int p = 0; p < t.parts; ++p)
                    for (int j = 0; j < t.share; ++j) {
                        const f32x4 x = *reinterpret_cast<const f32x4*>(q + p * t.apart + j * t.D);
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[c] += x[c];
                    }
                IO o[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) o[c] = from_f32<IO>(s[c]);
                __builtin_memcpy(static_cast<IO*>(t.out) + 4 * i, o, sizeof(o));
            }
            return;
        }
        for (long long i = first; i < t.count; i += step) {
            const float* q = t.part + i / t.D * t.share * t.D + i % t.D;
            float s = 0.f;
            for (int p = 0; p < t.parts; ++p)
                for (int j = 0; j < t.share; ++j) s += q[p * t.apart + j * t.D];
            static_cast<IO*>(t.out)[i] = from_f32<IO>(s);
        }
    } else if (all.decay_part) {
        for (long long i = first; i < all.decay_count; i += step) {
            float s = all.decay_part[i];
            for (int t = 1; t < all.tiles; ++t) s += all.decay_part[t * all.decay_count + i];
            put_decay(all, i, s);
        }
    } else {
        __shared__ double red[THREADS / 64];
        for (int h = blockIdx.x; h < all.H; h += gridDim.x) {
            double s = 0.;
            for (long long i = threadIdx.x; i < all.decay_n; i += THREADS) s += all.decay_sums[i * all.H + h];
#pragma unroll
            for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
            __syncthreads();                               // (the head in front has been read)
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
            __syncthreads();
            if (threadIdx.x == 0) put_decay(all, h, (float)((red[0] + red[1]) + (red[2] + red[3])));
        }
    }
}

size_t elem(int dtype) { return dtype == VRWKV_F32 ? 4 : 2; }
int pad_dx(int d) { return d <= 64 ? 64 : 128; }
int tiles_of(int d) { return (d + TZ - 1) / TZ; }
int chunk_of(int dtype) { return dtype == VRWKV_F32 ? 32 : 64; }   // of the gradients' pass

// workgroups of a launch of outputs that the chip holds at once
int slots(int dtype, int dx, bool backward) {
    const int per_cu = backward ? 1 : dtype == VRWKV_F32 && dx == 128 ? 1 : 2;
    return per_cu * device_cus();
}
// Tokens of a segment.  Rows of a batch: calls of fewer sequences and heads than fill the chip are cut, into that number of pieces, up to 64 a row, whose estimated time is least: a round
// lasts as long as its longest piece's chunks and two or three more for its start; pieces cost another pass over their rows for their states,
// half as long, and one over the states.  The numbers are fitted to the measurements below, on one card, and to no others.  (Gradients of 48 sequences of 577 tokens in tiles of 64 of 80 channels, fp16: 1 piece 130 us, 2 pieces 109, 3 119, 5 105; of 24 of 4150,
// fp32: 8 pieces 215, 10 189, 11 222, 22 202.  Outputs of the latter: 10 pieces 60, 13 63, 17 55, 22 57; of 48
// of 16384, fp16: 8 pieces 219, 10 189, 11 206, 16 182, 20 194, 32 190.  Taken with intermediate operands of two terms, which made 16-bit calls some 10 % shorter.)
int segment_len(const vrwkv_decay_args& a, int dx, int tiles, int roles, bool backward) {
    const long long wgs = (long long)a.H * tiles * roles, room = slots(a.dtype, dx, backward);
    if (!a.offsets) {
        const int chunks = (a.T + 63) / 64;
        int best = 1;
        double least = 1e30;
        for (int pieces = 1; pieces <= std::min(chunks / 2, 64) || pieces == 1; ++pieces) {
            const int len = (chunks + pieces - 1) / pieces, n = (chunks + len - 1) / len;
            const auto rounds = [&](long long slots) { return (double)((wgs * a.N * n + slots - 1) / slots); };
            double cost;
            if (backward) {                               // (the passes over states hold three workgroups a compute unit, and take 0.43 of the gradients' time; one of them without a cut)
                const double states = 0.43 * rounds(3LL * device_cus()) * (len + 2.7);
                cost = rounds(room) * (len + 2.7) + (n == 1 ? states : 2 * states + 0.9);
            } else {                                      // (a second workgroup makes a compute unit's round 1.3 to 1.55 times as long; the rounds of more overlap)
                const double load = (double)(wgs * a.N * n) / device_cus();
                const double once = (room == device_cus() ? rounds(room) : load <= 1 ? 1 : load <= 2 ? 1 + 0.28 * load : 1.75 + 0.6 * (load - 2)) * (len + 2);
                cost = n == 1 ? once : 1.5 * once + 3 + n / 16.0;
            }
            if (cost < least) { least = cost; best = len; }
        }
        return best * 64;
    }
    // Packed: the host does not know the lengths, and some sequence may be as long as all of them together: as many pieces of all tokens as fill the chip twice, of 256 tokens
    // at least (that is a plain quotient: no estimate can be made of lengths that are not known, and rows that would stay whole in a batch are cut here).
    return (int)std::max<long long>(256, (long long)a.T * wgs / (2 * room) / 64 * 64);
}
bool cut(const vrwkv_decay_args& a, int seg_len) { return a.T > seg_len; }
long long segment_total(const vrwkv_decay_args& a, int seg_len) {
    return a.offsets ? (long long)a.T / seg_len + a.N : (long long)a.N * ((a.T + seg_len - 1) / seg_len);
}
// pages of states: the segments' or, of many packed sequences, by where segments start (segment_page)
bool by_start(const vrwkv_decay_args& a, int seg_len) { return a.offsets && a.N > a.T / seg_len + 2; }
long long page_total(const vrwkv_decay_args& a, int seg_len) { return by_start(a, seg_len) ? 2 * ((long long)a.T / seg_len + 1) : segment_total(a, seg_len); }
long long chunk_total(const vrwkv_decay_args& a, int L) { return a.offsets ? (long long)a.T / L + a.N : (long long)a.N * ((a.T + L - 1) / L); }
long long rows_of(const vrwkv_decay_args& a) { return a.offsets ? a.T : (long long)a.N * a.T; }

// Workspace pieces, one behind the other on 256 bytes; with base null only their sum.
struct Pieces {
    char* base;
    size_t used = 0;
    template <typename T> T* take(size_t n) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used = (used + n * sizeof(T) + 255) & ~(size_t)255;
        return p;
    }
};

int check_common(const vrwkv_decay_args* a, const char* who) {
    if (!a) { set_error("%s: null args", who); return VRWKV_INVALID_ARG; }
    if (a->N <= 0 || a->T <= 0 || a->H <= 0 || a->Hq <= 0 || a->Hk <= 0 || a->Hv <= 0) { set_error("%s: N, T and the numbers of heads must be positive", who); return VRWKV_INVALID_ARG; }
    if (a->dtype < VRWKV_F32 || a->dtype > VRWKV_F16 || a->g_dtype < VRWKV_F32 || a->g_dtype > VRWKV_F16) { set_error("%s: dtype must be fp32, bf16 or fp16", who); return VRWKV_UNSUPPORTED_DTYPE; }
    if (a->H % a->Hq || a->H % a->Hk || a->H % a->Hv) { set_error("%s: H (%d) must be a multiple of the heads of q, k and v (%d, %d, %d)", who, a->H, a->Hq, a->Hk, a->Hv); return VRWKV_UNSUPPORTED_SHAPE; }
    if (a->Dk < 1 || a->Dk > 128 || a->Dv < 1 || a->Dv > 128) { set_error("%s: head sizes (%d, %d) must be 1 to 128", who, a->Dk, a->Dv); return VRWKV_UNSUPPORTED_SHAPE; }
    if (chunk_total(*a, 32) >= 1LL << 30 || (chunk_total(*a, 64) + a->N) * a->H >= 1LL << 24 || (long long)a->N * a->H * 32 >= 1LL << 24) { set_error("%s: too many tokens and heads", who); return VRWKV_UNSUPPORTED_SHAPE; }
    return VRWKV_OK;
}
int check_tensors(const vrwkv_decay_args& a, const char* who) {
    if (!a.q || !a.k || !a.v || !a.g) { set_error("%s: null q, k, v or g", who); return VRWKV_INVALID_ARG; }
    const size_t m = elem(a.dtype) - 1;
    for (const void* p : {a.q, a.k, a.v, (const void*)a.y, a.gy, (const void*)a.dq, (const void*)a.dk, (const void*)a.dv})
        if ((size_t)p & m) { set_error("%s: a tensor is not aligned to its elements", who); return VRWKV_INVALID_ARG; }
    // (offsets inside a chunk's rows are 32 bits)
    for (const long long st : {a.q_stride[1], a.k_stride[1], a.v_stride[1], a.gy ? a.gy_stride[1] : 0, a.g_stride[1], (long long)a.H * std::max(a.Dk, a.Dv)})
        if (st < 0 || st >= 1 << 22) { set_error("%s: tokens %lld elements apart, at most 2^22", who, st); return VRWKV_UNSUPPORTED_SHAPE; }
    for (const void* p : {a.g, (const void*)a.dg})
        if ((size_t)p & (elem(a.g_dtype) - 1)) { set_error("%s: g is not aligned to its elements", who); return VRWKV_INVALID_ARG; }
    for (const void* p : {(const void*)a.state, (const void*)a.last, (const void*)a.glast, (const void*)a.dstate})
        if ((size_t)p & 3) { set_error("%s: a state is not aligned to its elements", who); return VRWKV_INVALID_ARG; }
    if (a.offsets && ((size_t)a.offsets & (a.offsets64 ? 7 : 3))) { set_error("%s: offsets are not aligned to their elements", who); return VRWKV_INVALID_ARG; }
    return VRWKV_OK;
}
View view(const void* p, const long long (&s)[3], int heads, const vrwkv_decay_args& a) { return View{p, s[0], s[1], s[2], a.H / heads}; }
OutView out_view(void* p, int D, const vrwkv_decay_args& a, bool f32) {
    const long long st = (long long)a.H * D;
    return OutView{p, st * a.T, st, D, f32};
}
// Whether rows may be read, or results written, in 16-byte pieces.
bool in_pieces(const View& v, int d, int dtype) {
    const long long per16 = 16 / (long long)elem(dtype);
    return !v.p || (((size_t)v.p & 15) == 0 && v.sb % per16 == 0 && v.st % per16 == 0 && v.sh % per16 == 0 && d % 8 == 0);
}
bool in_pieces(const OutView& v, int d) { return ((size_t)v.p & 15) == 0 && d % 8 == 0; }
template <typename P>
P common(const vrwkv_decay_args& a, int seg_len) {
    P p{};
    p.offsets = a.offsets;
    p.off64 = a.offsets64;
    p.g = a.g;
    p.g_sb = a.g_stride[0];
    p.g_st = a.g_stride[1];
    p.g_sh = a.g_stride[2];
    p.g_dtype = a.g_dtype;
    p.rows = rows_of(a);
    p.N = a.N;
    p.T = a.T;
    p.H = a.H;
    p.seg_len = seg_len;
    p.nseg = a.offsets ? 0 : (a.T + seg_len - 1) / seg_len;
    p.segs = (int)segment_total(a, seg_len);
    p.by_start = by_start(a, seg_len);
    p.scale = a.scale;
    return p;
}
int launch(const Params& p, int dtype, int dx, int mode, hipStream_t st) {
    bool vec = true;
    for (int i = 0; i < p.n_roles; ++i) {
        const Role& r = p.role[i];
        vec = vec && in_pieces(r.a, r.dx, dtype) && in_pieces(r.b, r.dx, dtype) && in_pieces(r.c, r.dz, dtype) && in_pieces(r.o, r.dz);
    }
    if (dtype == VRWKV_F32) return launch_decay<float>(p, dx, mode, vec, st);
    if (dtype == VRWKV_BF16) return launch_decay<__hip_bfloat16>(p, dx, mode, vec, st);
    return launch_decay<__half>(p, dx, mode, vec, st);
}
// The segments' own states and the states in front of them, for the roles of p.
int launch_segments(const Params& p, int dtype, int dx, hipStream_t st) {
    const int s = launch(p, dtype, dx, STATES, st);
    if (s != VRWKV_OK) return s;
    // (many sequences, most of them not cut: a quarter of the workgroups, 48 packed prompts of 16 heads 10.2 to 8.1 us; few long ones: all that there may be)
    const long long sequences = (long long)p.N * p.H * p.role[0].tiles;
    const int wide = sequences * (dx / 16) > 2048 ? 4 : 1;
    const dim3 grid((unsigned)(dx / 16 / wide * sequences), 1, p.n_roles), block(THREADS);
    if (dx == 64 && wide == 1) hipLaunchKernelGGL((segments_kernel<64, 1>), grid, block, 0, st, p);
    else if (dx == 64) hipLaunchKernelGGL((segments_kernel<64, 4>), grid, block, 0, st, p);
    else if (wide == 1) hipLaunchKernelGGL((segments_kernel<128, 1>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((segments_kernel<128, 4>), grid, block, 0, st, p);
    return check_launch("decay_attention (segments)");
}
void take_segments(Role& r, Pieces& ws, const vrwkv_decay_args& a, long long pages, int dx) {
    r.seg = ws.take<float>((size_t)pages * a.H * r.tiles * dx * TZ);
    r.seg_decay = ws.take<float>((size_t)pages * a.H);
}

struct FwdPlan {
    int dx, seg_len;
    Role role{};
    FwdPlan(const vrwkv_decay_args& a, Pieces& ws) {
        dx = pad_dx(a.Dk);
        role.dx = a.Dk;
        role.dz = a.Dv;
        role.tiles = tiles_of(a.Dv);
        seg_len = segment_len(a, dx, role.tiles, 1, false);
        if (cut(a, seg_len)) take_segments(role, ws, a, page_total(a, seg_len), dx);
    }
};
// A pass that keeps the states in front of the chunks, and one for all gradients (decay_bwd.h); tiles of 64 channels of larger heads, and heads that share a row of q, k or v, leave
// parts that are added up behind.
struct BwdPlan {
    int dxv, tk, tv, seg_len;
    Role r{}, s{};                                        // R back along the tokens; S along them
    float *fq = nullptr, *fk = nullptr, *fv = nullptr, *fg = nullptr;   // parts
    double* sums = nullptr;                               // of decays that all tokens share
    BwdPlan(const vrwkv_decay_args& a, Pieces& ws) {
        dxv = pad_dx(a.Dv);
        tk = tiles_of(a.Dk);
        tv = tiles_of(a.Dv);
        r.dx = s.dx = a.Dv;
        r.dz = s.dz = a.Dk;
        r.tiles = s.tiles = tk;
        r.reverse = 1;
        seg_len = segment_len(a, dxv, tk * tv, 1, true);
        const long long segs = segment_total(a, seg_len), rows = rows_of(a);
        if (cut(a, seg_len)) {
            take_segments(r, ws, a, page_total(a, seg_len), dxv);
            take_segments(s, ws, a, page_total(a, seg_len), dxv);
        }
        if (a.dq && (a.Hq < a.H || tv > 1)) fq = ws.take<float>((size_t)rows * a.H * a.Dk * tv);
        if (a.dk && (a.Hk < a.H || tv > 1)) fk = ws.take<float>((size_t)rows * a.H * a.Dk * tv);
        if (a.dv && (a.Hv < a.H || tk > 1)) fv = ws.take<float>((size_t)rows * a.H * a.Dv * tk);
        s.anchors = ws.take<float>((size_t)chunk_total(a, chunk_of(a.dtype)) * a.H * tk * dxv * TZ);
        if (a.dg && a.g_per_head) sums = ws.take<double>((size_t)segs * tk * tv * a.H);
        else if (a.dg && (tk * tv > 1 || a.g_dtype != VRWKV_F32)) fg = ws.take<float>((size_t)rows * a.H * tk * tv);
    }
};
// A launch has less than 2^32 threads.
int check_grid(const vrwkv_decay_args& a, int seg_len, int tiles, int threads, const char* who) {
    if (std::max(segment_total(a, seg_len) * threads, (long long)a.N * 8 * THREADS) * a.H * tiles < 1LL << 32) return VRWKV_OK;
    set_error("%s: too many sequences and heads", who);
    return VRWKV_UNSUPPORTED_SHAPE;
}
int check_workspace(const vrwkv_decay_args& a, size_t need, const char* who) {
    if (need && (!a.workspace || a.workspace_bytes < need)) { set_error("%s: workspace of %zu bytes, %zu needed", who, a.workspace ? a.workspace_bytes : 0, need); return VRWKV_WORKSPACE_TOO_SMALL; }
    if (need && ((size_t)a.workspace & 15)) { set_error("%s: workspace must be 16-byte aligned", who); return VRWKV_INVALID_ARG; }
    return VRWKV_OK;
}

}  // namespace
}  // namespace decay
}  // namespace vrwkv

using namespace vrwkv;
using namespace vrwkv::decay;

extern "C" size_t vrwkv_decay_fwd_workspace_bytes(const vrwkv_decay_args* args) {
    if (check_common(args, "vrwkv_decay_fwd") != VRWKV_OK) return 0;
    Pieces ws{nullptr};
    FwdPlan plan(*args, ws);
    return ws.used;
}

extern "C" int vrwkv_decay_fwd(const vrwkv_decay_args* args, void* hip_stream) {
    const char* who = "vrwkv_decay_fwd";
    int s = check_common(args, who);
    if (s == VRWKV_OK) s = check_tensors(*args, who);
    if (s != VRWKV_OK) return s;
    const vrwkv_decay_args& a = *args;
    if (!a.y) { set_error("%s: null y", who); return VRWKV_INVALID_ARG; }
    Pieces size{nullptr};
    FwdPlan sized(a, size);
    if ((s = check_grid(a, sized.seg_len, sized.role.tiles, OUT_THREADS, who)) != VRWKV_OK || (s = check_workspace(a, size.used, who)) != VRWKV_OK) return s;
    Pieces ws{static_cast<char*>(a.workspace)};
    FwdPlan plan(a, ws);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    Params p = common<Params>(a, plan.seg_len);
    p.n_roles = 1;
    Role& r = p.role[0] = plan.role;
    r.a = view(a.q, a.q_stride, a.Hq, a);
    r.b = view(a.k, a.k_stride, a.Hk, a);
    r.c = view(a.v, a.v_stride, a.Hv, a);
    r.o = out_view(a.y, a.Dv, a, false);
    r.init = a.state;
    r.last = a.last;
    r.sx = a.Dv;
    r.sz = 1;
    r.s_upd = 1.f;
    if (r.seg && (s = launch_segments(p, a.dtype, plan.dx, st)) != VRWKV_OK) return s;
    return launch(p, a.dtype, plan.dx, PLAIN, st);
}

extern "C" size_t vrwkv_decay_bwd_workspace_bytes(const vrwkv_decay_args* args) {
    if (check_common(args, "vrwkv_decay_bwd") != VRWKV_OK) return 0;
    Pieces ws{nullptr};
    BwdPlan plan(*args, ws);
    return ws.used;
}

extern "C" int vrwkv_decay_bwd(const vrwkv_decay_args* args, void* hip_stream) {
    const char* who = "vrwkv_decay_bwd";
    int s = check_common(args, who);
    if (s == VRWKV_OK) s = check_tensors(*args, who);
    if (s != VRWKV_OK) return s;
    const vrwkv_decay_args& a = *args;
    if (!a.gy) { set_error("%s: null gy", who); return VRWKV_INVALID_ARG; }
    Pieces size{nullptr};
    BwdPlan sized(a, size);
    if ((s = check_grid(a, sized.seg_len, sized.tk * sized.tv, BWD_THREADS, who)) != VRWKV_OK || (s = check_workspace(a, size.used, who)) != VRWKV_OK) return s;
    Pieces ws{static_cast<char*>(a.workspace)};
    BwdPlan b(a, ws);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const View q = view(a.q, a.q_stride, a.Hq, a), k = view(a.k, a.k_stride, a.Hk, a), v = view(a.v, a.v_stride, a.Hv, a), gy = view(a.gy, a.gy_stride, a.H, a);
    Params p = common<Params>(a, b.seg_len);
    for (Role* r : {&b.r, &b.s}) {
        r->b = r == &b.r ? gy : v;
        r->c = r == &b.r ? q : k;
        r->init = r == &b.r ? a.glast : a.state;
        r->sx = 1;                                        // rows of v's channels, columns of k's
        r->sz = a.Dv;
        r->s_upd = r == &b.r ? a.scale : 1.f;
    }
    if (b.r.seg) {
        p.n_roles = 2;
        p.role[0] = b.r;
        p.role[1] = b.s;
        if ((s = launch_segments(p, a.dtype, b.dxv, st)) != VRWKV_OK) return s;
    }
    p.n_roles = 1;
    p.role[0] = b.s;
    if ((a.state || a.T > chunk_of(a.dtype)) && (s = launch(p, a.dtype, b.dxv, CHUNKS, st)) != VRWKV_OK) return s;
    BwdParams t = common<BwdParams>(a, b.seg_len);
    t.in[0] = q;
    t.in[1] = k;
    t.in[2] = v;
    t.gy = gy;
    t.out[0] = out_view(b.fq ? b.fq : a.dq, a.Dk, a, b.fq != nullptr);
    t.out[1] = out_view(b.fk ? b.fk : a.dk, a.Dk, a, b.fk != nullptr);
    t.out[2] = out_view(b.fv ? b.fv : a.dv, a.Dv, a, b.fv != nullptr);
    t.dg = b.sums ? nullptr : b.fg ? b.fg : static_cast<float*>(a.dg);
    t.dg_sums = b.sums;
    t.chunks = b.s.anchors;
    t.seg = b.r.seg;
    t.seg_front = b.s.seg;
    t.state = a.state;
    t.glast = a.glast;
    t.dstate = a.dstate;
    t.Dk = a.Dk;
    t.Dv = a.Dv;
    t.tk = b.tk;
    t.tv = b.tv;
    const bool vec = in_pieces(q, a.Dk, a.dtype) && in_pieces(k, a.Dk, a.dtype) && in_pieces(v, a.Dv, a.dtype) && in_pieces(gy, a.Dv, a.dtype) && in_pieces(t.out[0], a.Dk) && in_pieces(t.out[1], a.Dk) &&
                     in_pieces(t.out[2], a.Dv);
    s = a.dtype == VRWKV_F32 ? launch_decay_bwd<float>(t, vec, st) : a.dtype == VRWKV_BF16 ? launch_decay_bwd<__hip_bfloat16>(t, vec, st) : launch_decay_bwd<__half>(t, vec, st);
    if (s != VRWKV_OK) return s;
    Sums sums{};
    long long most = 1;
    const auto add = [&](const float* part, void* out, int heads, int D, int parts) {
        if (!part) return;
        const long long rows = rows_of(a);
        const bool fours = D % 4 == 0 && ((size_t)out & 15) == 0;
        const long long count = rows * heads * D / (fours ? 4 : 1);
        sums.s[sums.n++] = Sum{part, out, count, rows * a.H * D, D, a.H / heads, parts, fours};
        most = std::max(most, count);
    };
    add(b.fq, a.dq, a.Hq, a.Dk, b.tv);
    add(b.fk, a.dk, a.Hk, a.Dk, b.tv);
    add(b.fv, a.dv, a.Hv, a.Dv, b.tk);
    const bool decays = b.sums || b.fg;
    if (decays) {
        sums.decay_part = b.fg;
        sums.decay_sums = b.sums;
        sums.dg = a.dg;
        sums.decay_count = rows_of(a) * a.H;
        sums.decay_n = segment_total(a, b.seg_len) * b.tk * b.tv;
        sums.g_dtype = a.g_dtype;
        sums.tiles = b.tk * b.tv;
        sums.H = a.H;
        most = std::max(most, b.fg ? sums.decay_count : (long long)a.H * THREADS);
    }
    if (sums.n || decays) {
        const dim3 grid((unsigned)std::min<long long>((most + THREADS - 1) / THREADS, 8192), sums.n + (decays ? 1 : 0));
        if (a.dtype == VRWKV_F32) hipLaunchKernelGGL((sums_kernel<float>), grid, dim3(THREADS), 0, st, sums);
        else if (a.dtype == VRWKV_BF16) hipLaunchKernelGGL((sums_kernel<__hip_bfloat16>), grid, dim3(THREADS), 0, st, sums);
        else hipLaunchKernelGGL((sums_kernel<__half>), grid, dim3(THREADS), 0, st, sums);
    }
    return check_launch(who);
}
