// The selective state space scan (gfx950): h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t^T, y_t = (C_t h_t + D u_t) silu(z_t).
//
// Every channel e and state s has a decay of its own at every token, exp(dt[t,e] A[e,s]): there is no product of matrices in it, and what bounds it is one exponential (at a quarter of the
// vector rate) and four vector operations for each token, channel and state.  P lanes hold one channel, four states each; sixteen tokens are taken at a time.  What
// belongs to a token and channel alone (step size, softplus, gate, rounding) is computed by one lane of the P for every P-th token, and handed to
// the others in registers; sums over states go the same way back.  B and C of sixteen tokens lie in LDS in fp32, for the 256 / P channels of a workgroup.
//
// 64 x 196 tokens of 1536 channels with 16 states, bf16: 108 us, 220 cycles a token and wave, of which its 36 instructions take 196 (a vector operation between exponentials 4.5 cycles, an
// exponential 8.3); the bytes alone 30.  4, 8, 32 and 64 states: 79, 76, 165 and 290.
#pragma once
#include "lanes.h"
#include "sequences.h"
#include <utility>

namespace vrwkv {
namespace scan {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int THREADS = 256, BATCH = 16;

struct Params {
    const void *u, *delta, *B, *C, *z;
    const float *A, *state;
    ParamVec D, bias;
    Sequences seq;                                         // .offsets null: one sequence a row
    void* y;
    float *last, *kept;                                    // kept: the states in front of every sixteenth token, (batch, chunks, E, 4 P)
    float *seg_h, *seg_dt;                                 // of each segment: its last states from zeros, (batch, segments, E, 4 P), and its sum of step sizes
    long long u_b, u_t, d_b, d_t, z_b, z_t, B_b, B_t, B_g, C_b, C_t, C_g;
    int N, rows, T, E, S, G, softplus, L, nseg, blocks;    // rows: of the batch; L: tokens of a segment; blocks: workgroups of a group's channels
};

// A kernel's arguments, read where they are asked for: kept in scalar registers they run over into lanes of vector registers, and come back from there one instruction a word.
#define SCAN_CONSTANT __attribute__((opencl_constant))
template <typename T>
__device__ __forceinline__ const SCAN_CONSTANT T& arguments() {
    unsigned none = 0;
    asm volatile("" : "+s"(none));                         // (else all that is read through it is kept after all)
    return *reinterpret_cast<const SCAN_CONSTANT T*>(reinterpret_cast<unsigned long long>(__builtin_amdgcn_kernarg_segment_ptr()) + none);
}
__device__ __forceinline__ Sequences sequences_of(const SCAN_CONSTANT Sequences& s) { return Sequences{s.offsets, s.is64, s.N, s.T}; }

// log(1 + q) for q in 0 .. 1 as 2 atanh(q / (2 + q)): an odd series in s = q / (2 + q) <= 1/3, cut to five terms by a Chebyshev fit (8e-9 relative).  (1 + q rounded first
// would cost 6e-8 / q: step sizes of a thousandth would be off by 6e-5.)
__device__ __forceinline__ float log1p_unit(float q) {
    const float s = q * fast_rcp(2.f + q), w = s * s;
    return s * fmaf(fmaf(fmaf(fmaf(0.2817465662956238f, w, 0.2796141803264618f), w, 0.40024852752685547f), w, 0.6666631698608398f), w, 2.f);
}
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1p_unit(fast_exp2(-LOG2E * fabsf(x))); }
__device__ __forceinline__ float sigmoid(float x) { return fast_rcp(1.f + fast_exp2(-LOG2E * x)); }

// h behind tokens whose step sizes add up to `dt`, A in powers of two: as a fraction and an exponent, so that neither an h of zero meets an overflow nor an infinite one an underflow
__device__ __forceinline__ float decayed(float h, float dt, float a2) {
    const float x = dt * a2, n = floorf(x);
    if (!(fabsf(x) < 1e8f)) return h * fast_exp2(x);
    return __builtin_ldexpf(h * fast_exp2(x - n), (int)fmaxf(fminf(n, 1000.f), -1000.f));
}

// What a workgroup's lane works on.
template <int P>
struct Place {
    static constexpr int CHANNELS = THREADS / P;
    int lane, p, g, e;                                     // lane of the wave, of the channel; the channel's group and its number
    bool there;
    __device__ __forceinline__ Place(int E, int G, int blocks) {
        const int tid = threadIdx.x, of_group = E / G;
        lane = tid & 63;
        p = tid % P;
        g = blockIdx.x / blocks;
        const int c = (blockIdx.x % blocks) * CHANNELS + tid / P;
        there = c < of_group;
        e = g * of_group + min(c, of_group - 1);
    }
};

// A tensor's row as all lanes of a wave see it, and a lane's place in it in bytes: an address in scalar registers and 32 bits of a vector register, not 64 for each of a lane's tokens.
template <typename T>
__device__ __forceinline__ T& at_row(const T* row, unsigned bytes) {
    asm volatile("" : "+v"(bytes));                        // (else the compiler keeps their sums, from iteration to iteration)
    return *const_cast<T*>(reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + bytes));
}

// What a lane has of sixteen tokens: its channel of every P-th.
template <typename IO, int P>
struct Rows {
    static constexpr int OWN = BATCH / P;
    IO u[OWN], d[OWN], z[OWN], g[OWN];
    // tokens row + q, row + q + P, .. of a tensor whose batch row begins at `base`; behind `end` the last in front of it once more
    __device__ __forceinline__ void fetch(IO (&to)[OWN], const void* t, long long base, long long stride, int row, int end, int q, int e) const {
        const IO* x = static_cast<const IO*>(t) + base + row * stride;
        if (row + BATCH <= end) {
            asm volatile("" : "+v"(q));                    // (nothing of this is kept for other rows)
            const unsigned place = (q * (unsigned)stride + e) * sizeof(IO);
            int step = P * (int)stride;                    // (its multiples are not kept either: scalar registers run out)
            asm volatile("" : "+s"(step));
#pragma unroll
            for (int i = 0; i < OWN; ++i, x += step) to[i] = at_row(x, place);
        } else {
            asm volatile("" : "+v"(q));
#pragma unroll
            for (int i = 0; i < OWN; ++i) to[i] = at_row(x, (min(q + i * P, end - 1 - row) * (unsigned)stride + e) * sizeof(IO));
        }
    }
};

// B and C of sixteen tokens on their way to LDS, first all of B: a wave's are of one of them.
template <typename IO, int P, int WHICH>
struct Stage {
    static constexpr int ONE = BATCH * 4 * P, VALUES = ONE * WHICH, EACH = (VALUES + THREADS - 1) / THREADS;
    IO raw[EACH];
    template <typename Args>
    __device__ __forceinline__ void fetch(const Args& p, long long b, int g, int row, int from, int to) {
        const int first = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63);
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const bool isC = first + k * THREADS >= ONE;
            const int i = threadIdx.x + k * THREADS, t = i % ONE / (4 * P), n = i % (4 * P);
            const IO* x = isC ? static_cast<const IO*>(p.C) + b * p.C_b + row * p.C_t + g * p.C_g : static_cast<const IO*>(p.B) + b * p.B_b + row * p.B_t + g * p.B_g;
            raw[k] = from_f32<IO>(0.f);
            if (i < VALUES && row + t >= from && row + t < to && n < p.S) raw[k] = at_row(x, (t * (unsigned)(isC ? p.C_t : p.B_t) + n) * sizeof(IO));
        }
    }
    __device__ __forceinline__ void put(float* to) const {
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int i = threadIdx.x + k * THREADS;
            if (i < VALUES) to[i % ONE / (4 * P) * WHICH * 4 * P + i / ONE * 4 * P + i % (4 * P)] = to_f32(raw[k]);
        }
    }
};

// B and C of two tokens after the other two.  NEXT: read from LDS while the two in front are worked on (with two to five waves a vector unit nothing else hides the way from there).
template <int P, int WHICH, bool NEXT>
struct Pairs {
    f32x4 B[2], C[2], B_next[2], C_next[2];
    __device__ __forceinline__ void read(const float* bc, int pair, int p) {
        const f32x4* x = reinterpret_cast<const f32x4*>(bc);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            B_next[t] = x[(2 * pair + t) * WHICH * P + p];
            if (WHICH == 2) C_next[t] = x[(2 * pair + t) * WHICH * P + P + p];
        }
    }
    // `pair` is worked on now; `then` (if there is one) is the next
    __device__ __forceinline__ void start(const float* bc, int pair, int p) {
        if (NEXT) read(bc, pair, p);
    }
    __device__ __forceinline__ void advance(const float* bc, int pair, int then, int p) {
        if (!NEXT) read(bc, pair, p);
#pragma unroll
        for (int t = 0; t < 2; ++t) B[t] = B_next[t], C[t] = C_next[t];
        if (NEXT && then >= 0 && then < BATCH / 2) read(bc, then, p);
        if (NEXT) __builtin_amdgcn_sched_barrier(0);
    }
};

template <int... I, typename F>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, F&& f) { (f(std::integral_constant<int, I>()), ...); }

// EMIT: the outputs of a segment from the states in front of it; without, its last states from zeros (or from its sequence's first states) and its sum of step sizes.
// FULL: S is 4 P, so that no state is there to fill up.
template <typename IO, int P, bool FULL, bool EMIT>
__global__ __launch_bounds__(THREADS, P >= 4 ? 4 : 2) void scan_kernel(const Params p) {
    constexpr int OWN = BATCH / P, WHICH = EMIT ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float bc[2][BATCH * WHICH * 4 * P];
    const Place<P> at(p.E, p.G, p.blocks);
    const int s = blockIdx.y, b = blockIdx.z, e = at.e;
    int r0 = s * p.L;
    const int r1 = min(p.T, r0 + p.L);
    int from, to;                                          // the tokens that belong to a sequence
    p.seq.inside(r0, r1, from, to);
    Walk w;
    if (!EMIT) {                                           // only of the sequence that goes on behind the segment
        w.find(p.seq, b, max(from, r1 - 1), at.lane);
        if (w.begin >= r1 || w.end <= r1) return;
        if (w.begin >= r0) {
            r0 += (w.begin - r0) / BATCH * BATCH;
            from = w.begin;
        }
    } else w.find(p.seq, b, from, at.lane);
    float a2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    bool pad[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        pad[k] = !FULL && 4 * at.p + k >= p.S;
        a2[k] = pad[k] ? 0.f : p.A[(long long)e * p.S + 4 * at.p + k] * LOG2E;
    }
    const float bias = p.bias.p ? p.bias.value(p.bias.fetch(e)) : 0.f, skip = EMIT && p.D.p ? p.D.value(p.D.fetch(e)) : 0.f;
    const auto first_state = [&](int n) {
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = p.state && !pad[k] ? p.state[((long long)n * p.E + e) * p.S + 4 * at.p + k] : 0.f;
    };
    const auto last_state = [&](int n) {
        if (!EMIT || !p.last || !at.there) return;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (!pad[k]) p.last[((long long)n * p.E + e) * p.S + 4 * at.p + k] = h[k];
    };
    if (EMIT && w.begin < r0) {                            // from the segment that the sequence begins in
        int k = w.begin / p.L;
        const float* at_h = p.seg_h + ((long long)b * p.nseg * p.E + e) * 4 * P + 4 * at.p;
        const float* at_dt = p.seg_dt + (long long)b * p.nseg * p.E + e;
        const f32x4 h0 = *reinterpret_cast<const f32x4*>(at_h + (long long)k * p.E * 4 * P);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = h0[i];
#pragma unroll 4
        for (++k; k < s; ++k) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(at_h + (long long)k * p.E * 4 * P);
            const float dt = at_dt[(long long)k * p.E];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = decayed(h[i], dt, a2[i]) + x[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = pad[i] ? 0.f : h[i];   // (an infinite step size makes what is not there NaN)
    }

    Rows<IO, P> raw;
    const auto fetch = [&](Rows<IO, P>& x, int row) {
        const auto& p = arguments<Params>();
        x.fetch(x.u, p.u, b * p.u_b, p.u_t, row, r1, at.p, e);
        x.fetch(x.d, p.delta, b * p.d_b, p.d_t, row, r1, at.p, e);
        if (EMIT && p.z) x.fetch(x.z, p.z, b * p.z_b, p.z_t, row, r1, at.p, e);
    };
    Stage<IO, P, WHICH> stage;
    fetch(raw, r0);
    stage.fetch(p, b, at.g, r0, from, to);
    stage.put(bc[0]);
    lds_barrier();
    float total = 0.f;
    int buf = 0;
    for (int row = r0; row < r1; row += BATCH, buf ^= 1) {
        const bool more = row + BATCH < r1;
        const auto& p = arguments<Params>();
        if (more) stage.fetch(p, b, at.g, row + BATCH, from, to);
        if (EMIT && p.kept && at.there)
            at_row(reinterpret_cast<const f32x4*>(p.kept) + ((long long)b * ((p.T + BATCH - 1) / BATCH) + row / BATCH) * p.E * P, (unsigned)(e * P + at.p) * 16u) = f32x4{h[0], h[1], h[2], h[3]};
        const IO* const out = static_cast<const IO*>(p.y) + ((long long)b * p.T + row) * p.E;
        const unsigned place = (at.p * (unsigned)p.E + e) * sizeof(IO);
        const int width = p.E;
        // tokens [first, behind) of the sixteen, all of one sequence; PART: not all sixteen.  P at a time: each lane's own, then the states of all, then each lane's own again
        const auto piece = [&](auto part_, int first, int behind) {
            constexpr bool PART = decltype(part_)::value;
            Pairs<P, WHICH, false> pairs;
            pairs.start(bc[buf], 0, at.p);
            each(std::make_integer_sequence<int, OWN>(), [&](auto i_) {
                constexpr int i = decltype(i_)::value;
                const float raw_d = to_f32(raw.d[i]) + bias, u = to_f32(raw.u[i]), dt = p.softplus ? softplus(raw_d) : raw_d, x = dt * u;
                const int mine = row + at.p + i * P;
                float y[P];
                each(std::make_integer_sequence<int, P>(), [&](auto q_) {
                    constexpr int q = decltype(q_)::value, j = i * P + q;
                    y[q] = 0.f;
                    if (j % 2 == 0) pairs.advance(bc[buf], j / 2, j / 2 + 1, at.p);
                    if (PART && (row + j < first || row + j >= behind)) return;
                    const float d = from_lane<P, q>(dt), v = from_lane<P, q>(x);
                    const f32x4 Bt = pairs.B[j % 2], Ct = pairs.C[j % 2];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        h[k] = fmaf(fast_exp2(d * a2[k]), h[k], v * Bt[k]);
                        if (!FULL && pad[k]) h[k] = 0.f;   // (an infinite v would make it NaN)
                    }
                    if (EMIT) {
                        y[q] = fmaf(Ct[3], h[3], fmaf(Ct[2], h[2], fmaf(Ct[1], h[1], Ct[0] * h[0])));
                    }
                });
                // (a segment's sum of step sizes is only read where one sequence goes through all of it: no token of such a one is left out)
                if (!EMIT) total += !PART || mine < r1 ? dt : 0.f;
                if (EMIT) {
                    sum_to_lanes<P, P>(y, at.p);
                    float v = fmaf(skip, u, y[0]);
                    if (p.z) {
                        const float z = to_f32(raw.z[i]);
                        v *= z * sigmoid(z);
                    }
                    if (at.there && (!PART || (mine >= first && mine < behind))) at_row(out + (long long)i * P * width, place) = from_f32<IO>(v);
                }
                if (!EMIT) asm volatile("" : "+v"(h[0]), "+v"(h[1]), "+v"(h[2]), "+v"(h[3]));   // (else the compiler puts the states off)
            });
        };
        if (EMIT && (row < from || row + BATCH > to)) {
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const int t = row + at.p + i * P;
                if (at.there && t < r1 && (t < from || t >= to)) at_row(out + (long long)i * P * width, place) = from_f32<IO>(0.f);
            }
        }
        for (;;) {                                         // one sequence after the other
            const int first = max(max(row, from), w.begin), behind = min(min(row + BATCH, to), w.end);
            if (first >= behind) break;
            if (first == w.begin) first_state(w.n);
            if (behind - first == BATCH) piece(std::false_type(), first, behind);
            else piece(std::true_type(), first, behind);
            if (behind < w.end) break;
            last_state(w.n);
            w.next(sequences_of(p.seq));
        }
        if (more) {
            fetch(raw, row + BATCH);
            stage.put(bc[buf ^ 1]);
            lds_barrier();
        }
    }
    if (EMIT) {
        if (p.seq.offsets && p.last)                       // sequences without a token keep their states
            for (int n0 = s; n0 < p.N; n0 += p.nseg * 64) {
                const int mine = n0 + at.lane * p.nseg;
                unsigned long long empty = __ballot(mine < p.N && p.seq.of_lane(min(mine, p.N - 1) + 1) <= p.seq.of_lane(min(mine, p.N - 1)));
                for (; empty; empty &= empty - 1) {
                    const int m = n0 + (__ffsll((long long)empty) - 1) * p.nseg;
                    first_state(m);
                    last_state(m);
                }
            }
    } else if (at.there) {
        const long long place = (long long)b * p.nseg + s;
        *reinterpret_cast<f32x4*>(p.seg_h + (place * p.E + e) * 4 * P + 4 * at.p) = f32x4{h[0], h[1], h[2], h[3]};
        float v[P];
#pragma unroll
        for (int q = 0; q < P; ++q) v[q] = total;
        sum_to_lanes<P, P>(v, at.p);
        if (at.p == 0) p.seg_dt[place * p.E + e] = v[0];
    }
}

// Runs f with the number of lanes a channel of S states takes, and whether it fills them.
template <typename F>
int with_lanes(int S, F&& f) {
    const auto full = [&](auto P) { return S == 4 * decltype(P)::value ? f(P, std::true_type()) : f(P, std::false_type()); };
    if (S <= 8) return full(std::integral_constant<int, 2>());
    if (S <= 16) return full(std::integral_constant<int, 4>());
    if (S <= 32) return full(std::integral_constant<int, 8>());
    return full(std::integral_constant<int, 16>());
}

template <typename IO>
int launch_forward(const Params& p, hipStream_t st) {
    return with_lanes(p.S, [&](auto P_, auto full) {
        constexpr int P = decltype(P_)::value;
        constexpr bool FULL = decltype(full)::value;
        const dim3 block(THREADS);
        if (p.nseg > 1) hipLaunchKernelGGL((scan_kernel<IO, P, FULL, false>), dim3(p.G * p.blocks, p.nseg - 1, p.rows), block, 0, st, p);
        hipLaunchKernelGGL((scan_kernel<IO, P, FULL, true>), dim3(p.G * p.blocks, p.nseg, p.rows), block, 0, st, p);
        return check_launch("vrwkv_scan_fwd");
    });
}

}  // namespace scan
}  // namespace vrwkv
