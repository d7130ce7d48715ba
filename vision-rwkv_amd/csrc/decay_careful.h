// The recurrence token by token in fp32, for the workgroups whose results are not all finite (gfx950).
// The chunks' products meet what the definition never multiplies: a masked zero times an infinity behind it, the terms of an operand that is infinite (or,
// finite, above bf16's largest number) against each other.  All of that ends in a result that is not finite, so results tell, for one instruction each; the workgroup
// then makes its segment's results again as they are defined: a token's infinities and NaN reach those behind it, and no other.
// Segments start from states that are right in the same sense: their own ones are made here too where they are not finite, and the scan over them keeps an
// infinity that a product of decays too small for fp32 multiplies.
// The state lies in the LDS, one index along the lanes, the other, over which a result sums, by waves; eight tokens at a time are staged as fp32, and a thread takes
// a number of the state through all eight.  0.26 us a token of a segment: one sequence of 16 384 tokens with a NaN 46 us to 0.27 ms, 64 x 196 x 12 heads
// with one in every row 28 to 180 us.
#pragma once

namespace vrwkv {
namespace decay {

constexpr int CAREFUL_TOKENS = 8;
constexpr float LOWEST_DECAY = -103.98f;                  // below it an exponential is zero in fp32
template <int DX>
struct CarefulTokens {
    float b[DX][CAREFUL_TOKENS], c[CAREFUL_TOKENS][64], e[CAREFUL_TOKENS];
};
template <int DX>
struct CarefulLds : CarefulTokens<DX> {
    float st[DX][64], a[DX][CAREFUL_TOKENS];
    float part[CAREFUL_TOKENS][8][64];                    // of results, by waves
};
// A head's rows of one sequence, from channel d on; they have dim.
template <typename IO>
struct CarefulRows {
    const IO* p;
    long long st;
    int count;
    __device__ __forceinline__ CarefulRows(const View& v, int base, int first, int head, int d, int dim)
        : p(static_cast<const IO*>(v.p) + base * v.sb + (long long)first * v.st + (head / v.share) * v.sh + d), st(v.st), count(dim - d) {}
    __device__ __forceinline__ float at(int token, int d, bool there) const { return there && d < count ? to_f32(p[token * st + d]) : 0.f; }
};
// Where a state's number lies that the matrix instructions' accumulators hold, rows contracted.
__device__ __forceinline__ int careful_place(int row, int column) { return (((row >> 4) * 4 + (column >> 4)) * 64 + ((row >> 2) & 3) * 16 + (column & 15)) * 4 + (row & 3); }

// Every number of a state (rows, 64) by the first WAVES waves: f(row, lane); wave w has the rows DX / WAVES w and those behind.
template <int DX, int WAVES = 8, typename F>
__device__ __forceinline__ void careful_each(int rows, const F& f) {
    const int lane = threadIdx.x & 63, first = DX / WAVES * (int)(threadIdx.x >> 6), end = min(rows, first + DX / WAVES);
    if (threadIdx.x < 64 * WAVES)
#pragma unroll 1
        for (int row = first; row < end; ++row) f(row, lane);
}

// n tokens staged, the first of them in memory t0, in their order or (rev) the last one first: rows of b and c, and the decays on the way: a token's own or (rev) that of the
// one behind it.  A place without a token keeps a state: decay 1, and zeros.
template <int DX, typename IO>
__device__ __forceinline__ void careful_stage(CarefulTokens<DX>& m, const Gates& gates, const CarefulRows<IO>& b, const CarefulRows<IO>& c, float c_scale, int t0, int n, int len, bool rev) {
    const int tid = threadIdx.x;
#pragma unroll 1
    for (int x = tid; x < CAREFUL_TOKENS * DX; x += blockDim.x) {
        const int i = x / DX, d = x % DX;
        m.b[d][i] = b.at(t0 + (rev ? n - 1 - i : i), d, i < n);
    }
#pragma unroll 1
    for (int x = tid; x < CAREFUL_TOKENS * 64; x += blockDim.x) {
        const int i = x >> 6;
        m.c[i][x & 63] = c_scale * c.at(t0 + (rev ? n - 1 - i : i), x & 63, i < n);
    }
    if (tid < CAREFUL_TOKENS) {
        const int t = rev ? n - tid : tid;
        const bool there = tid < n && t0 + t < len;
        const float g = gates.widen(gates.fetch(t0, t, there));
        m.e[tid] = there ? expf(g) : 1.f;
    }
}

// st = exp(g) st + b c c_scale for the tokens from .. to - 1 of a sequence of len, or (rev) back along them with the decay of the token behind; out(token, lane, sum of a a_scale st).
// Called by all threads.
template <int DX, typename IO, typename F>
__device__ __forceinline__ void careful_scan(CarefulLds<DX>& m, const Gates& gates, const CarefulRows<IO>& a, const CarefulRows<IO>& b, const CarefulRows<IO>& c, float a_scale, float c_scale, int from, int to, int len,
                                             bool rev, const F& out) {
    const int tid = threadIdx.x, wave = tid >> 6, rows = min(DX, b.count);
#pragma unroll 1
    for (int i0 = 0, n; i0 < to - from; i0 += n) {
        n = min(CAREFUL_TOKENS, to - from - i0);
        const int t0 = rev ? to - i0 - n : from + i0;      // the first of them in memory
        __syncthreads();                                   // (what was staged before has been read)
        careful_stage(m, gates, b, c, c_scale, t0, n, len, rev);
#pragma unroll 1
        for (int x = tid; x < CAREFUL_TOKENS * DX; x += blockDim.x) {
            const int i = x / DX, d = x % DX;
            m.a[d][i] = a_scale * a.at(t0 + (rev ? n - 1 - i : i), d, i < n);
        }
        __syncthreads();
        float e[CAREFUL_TOKENS], x[CAREFUL_TOKENS], y[CAREFUL_TOKENS];
#pragma unroll
        for (int i = 0; i < CAREFUL_TOKENS; ++i) {
            e[i] = m.e[i];
            x[i] = m.c[i][tid & 63];
            y[i] = 0.f;
        }
        careful_each<DX>(rows, [&](int row, int lane) {
            float s = m.st[row][lane];
#pragma unroll
            for (int i = 0; i < CAREFUL_TOKENS; ++i) {
                s = fmaf(s, e[i], m.b[row][i] * x[i]);
                y[i] = fmaf(m.a[row][i], s, y[i]);
            }
            m.st[row][lane] = s;
        });
        if (wave < 8)
#pragma unroll
            for (int i = 0; i < CAREFUL_TOKENS; ++i) m.part[i][wave][tid & 63] = y[i];
        __syncthreads();
        if (wave < n) {
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) sum += m.part[wave][r][tid & 63];
            out(t0 + (rev ? n - 1 - wave : wave), tid & 63, sum);
        }
    }
}
// A segment's own state, in its place (four waves).  It starts from nothing: the first token's decay is that of what is in front, and only the segment's.
template <typename IO, int DX>
__device__ __forceinline__ void careful_segment(CarefulTokens<DX>& m, const Call& p, const Role& r, const Place& w, int z, int h) {
    Gates gates;
    gates.open(p, w.base, w.first, h);
    const CarefulRows<IO> b(r.b, w.base, w.first, h, 0, r.dx), c(r.c, w.base, w.first, h, z * TZ, r.dz);
    float* const seg = r.seg + (((long long)w.page * p.H + h) * r.tiles + z) * (DX * TZ);
#pragma unroll 1
    for (int i0 = 0, n; i0 < w.s1 - w.s0; i0 += n) {
        n = min(CAREFUL_TOKENS, w.s1 - w.s0 - i0);
        __syncthreads();                                   // (what was staged before has been read)
        careful_stage(m, gates, b, c, r.s_upd, r.reverse ? w.s1 - i0 - n : w.s0 + i0, n, w.len, r.reverse);
        __syncthreads();
        careful_each<DX, THREADS / 64>(r.dx, [&](int row, int lane) {
            float s = i0 ? seg[careful_place(row, lane)] : 0.f;
#pragma unroll
            for (int i = 0; i < CAREFUL_TOKENS; ++i) s = fmaf(s, i0 + i ? m.e[i] : 1.f, m.b[row][i] * m.c[i][lane]);
            seg[careful_place(row, lane)] = s;
        });
    }
}

// Whether a workgroup has work here, and where its kernel's arguments (one struct) are, to be read again: kept in registers from the kernel's start they would spill in its chunks.
struct Careful {
    int wanted;
    unsigned args[2];
};
__device__ __forceinline__ void careful_begin(Careful& c) {
    const unsigned long long at = (unsigned long long)__builtin_amdgcn_kernarg_segment_ptr();   // (in the kernel's own body: null in a function that is called)
    if (threadIdx.x == 0) {
        c.wanted = 0;
        c.args[0] = (unsigned)at;
        c.args[1] = (unsigned)(at >> 32);
    }
}
template <typename P>
__device__ __forceinline__ P arguments_again(const Careful& c) {
    static_assert(sizeof(P) % 4 == 0 && std::is_trivially_copyable<P>::value, "");
    const unsigned lo = uniform(c.args[0]), hi = uniform(c.args[1]);
    const auto* words = (const __attribute__((address_space(4))) unsigned*)((unsigned long long)hi << 32 | lo);
    unsigned w[sizeof(P) / 4];
#pragma unroll
    for (unsigned i = 0; i < sizeof(P) / 4; ++i) w[i] = words[i];
    P p;
    __builtin_memcpy(&p, w, sizeof(P));
    return p;
}

// A segment's outputs and, where it is the last, the state behind it.
template <typename IO, int DX, int L>
__device__ __forceinline__ void careful_outputs(const Careful& careful, CarefulLds<DX>& m, int* offs) {
    const Params p = arguments_again<Params>(careful);
    const Role& r = p.role[0];
    const int z = blockIdx.x & (r.tiles - 1), h = blockIdx.x >> (r.tiles - 1), gid = grid_segment();
    const Place w = find_place<OUT_THREADS>(p, gid, L, offs);
    const long long page = ((long long)w.n * p.H + h) * ((long long)r.dx * r.dz);
    Gates gates;
    gates.open(p, w.base, w.first, h);
    const CarefulRows<IO> q(r.a, w.base, w.first, h, 0, r.dx), k(r.b, w.base, w.first, h, 0, r.dx), v(r.c, w.base, w.first, h, z * TZ, r.dz);
    const float* const seg = w.is_first ? nullptr : r.seg + (((long long)w.page * p.H + h) * r.tiles + z) * (DX * TZ);
    careful_each<DX>(r.dx, [&](int row, int lane) {
        const int column = z * TZ + lane;
        m.st[row][lane] = seg ? seg[careful_place(row, lane)] : r.init && column < r.dz ? r.init[page + row * r.sx + column * r.sz] : 0.f;
    });
    careful_scan(m, gates, q, k, v, p.scale, 1.f, w.s0, w.s1, w.len, false, [&](int token, int lane, float y) {
        const int column = z * TZ + lane;
        if (column < r.dz) static_cast<IO*>(r.o.p)[w.base * r.o.sb + (long long)(w.first + token) * r.o.st + h * r.o.sh + column] = from_f32<IO>(y);
    });
    if (r.last && w.is_last)
        careful_each<DX>(r.dx, [&](int row, int lane) {
            const int column = z * TZ + lane;
            if (column < r.dz) r.last[page + row * r.sx + column * r.sz] = m.st[row][lane];
        });
}

}  // namespace decay
}  // namespace vrwkv
