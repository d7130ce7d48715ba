// Gradients of the selective state space scan (gfx950).  With R_t the gradient of h_t, g_t = gy_t silu(z_t) and e_t = exp(dt_t A):
//
//     R_t = g_t C_t + e_{t+1} R_{t+1}        dC_t = sum_channels g_t h_t        dB_t = sum_channels R_t dt_t u_t        dA = sum_t dt_t e_t R_t h_{t-1}
//     ddt_t = sum_states (e_t R_t h_{t-1} A + R_t u_t B_t)        du_t = dt_t sum_states R_t B_t + D g_t        dz_t = gy_t (C_t h_t + D u_t) silu'(z_t)
//
// Sixteen tokens at a time, the last first: their states again from the one that the forward has kept in front of them, in registers, then back along them.  P lanes hold one channel,
// four states each, as in the forward.  dB and dC add up channels, which lie in other lanes: the sums of two tokens go through the wave in halves
// (two instructions for a sum of 64 / P lanes), then through LDS over the waves, and over workgroups by the launch that ends the pass.
//
// 64 x 196 tokens of 1536 channels with 16 states, bf16: 323 us with the sums that end the pass (9 of them), 640 cycles a token and wave.  Its 110 instructions account for about 510 of these; what is
// left is waiting that the two waves a vector unit, for which there are registers, do not hide.  Three waves, with states held of eight tokens at a time and the eight in front of them gone through twice,
// took as long as two (366 and 370 before the decays were kept in LDS), four 465.  4, 8, 32 and 64 states: 245, 238, 643 and 1382 (up to 8 states the registers overflow by nine; from 17 on the sums over
// channels that go through memory grow with the square of the states).
#pragma once
#include "scan.h"

namespace vrwkv {
namespace scan {

struct BackParams {
    Params f;
    const void* gy;
    const float* glast;
    void *du, *dd, *dz;
    float *dstate, *seg_r;                                 // seg_r: like seg_h, the gradient that a segment hands to the token in front of it
    float *part_bc, *part_A, *part_D, *part_bias;          // (blocks, tokens, G, 2, 4 P); (parts, E, 4 P); (parts, E)
    long long gy_b, gy_t;
};

// Sums over the lanes of a wave that differ above the channel's P: of v[0 .. 64 / P) of all channels, one is left in each lane of v[0], the one that sum_of_lane says.  At each step
// a lane keeps one half of its sums and gets the other lanes' parts of it.  Lanes of a row of sixteen first, in additions that read one lane and write another (4.4 cycles each,
// measured; two make a pair of sums), then rows, whose swap takes 10.
// Written out: the instruction's bank mask picks the half.  Two wait states in front of and behind reads across lanes; a sum is written before the last of the other operands is read, so that none of
// them may share a register with it, whatever values are known to be equal.
template <int HALF>
__device__ __forceinline__ void fold8(float* v) {
    if constexpr (HALF == 8)
        asm("s_nop 1\n"
#define FOLD(a, b) "v_add_f32_dpp %" #a ", %" #a ", %" #a " row_ror:8 row_mask:0xf bank_mask:0x3\n v_add_f32_dpp %" #a ", %" #b ", %" #b " row_ror:8 row_mask:0xf bank_mask:0xc\n"
            FOLD(0, 8) FOLD(1, 9) FOLD(2, 10) FOLD(3, 11) FOLD(4, 12) FOLD(5, 13) FOLD(6, 14) FOLD(7, 15) "s_nop 1"
            : "+&v"(v[0]), "+&v"(v[1]), "+&v"(v[2]), "+&v"(v[3]), "+&v"(v[4]), "+&v"(v[5]), "+&v"(v[6]), "+&v"(v[7])
            : "v"(v[8]), "v"(v[9]), "v"(v[10]), "v"(v[11]), "v"(v[12]), "v"(v[13]), "v"(v[14]), "v"(v[15]));
    else
#pragma unroll
        for (int i = 0; i < HALF; i += 4)
            asm("s_nop 1\n" FOLD(0, 4) FOLD(1, 5) FOLD(2, 6) FOLD(3, 7) "s_nop 1"
#undef FOLD
                : "+&v"(v[i]), "+&v"(v[i + 1]), "+&v"(v[i + 2]), "+&v"(v[i + 3])
                : "v"(v[i + HALF]), "v"(v[i + HALF + 1]), "v"(v[i + HALF + 2]), "v"(v[i + HALF + 3]));
}
template <int HALF>
__device__ __forceinline__ void fold4(float* v) {
#pragma unroll
    for (int i = 0; i < HALF; i += 4)
        asm("s_nop 1\n"
#define FOLD(a, b) "v_add_f32_dpp %" #a ", %" #a ", %" #a " row_shl:4 row_mask:0xf bank_mask:0x5\n v_add_f32_dpp %" #a ", %" #b ", %" #b " row_shr:4 row_mask:0xf bank_mask:0xa\n"
            FOLD(0, 4) FOLD(1, 5) FOLD(2, 6) FOLD(3, 7) "s_nop 1"
#undef FOLD
            : "+&v"(v[i]), "+&v"(v[i + 1]), "+&v"(v[i + 2]), "+&v"(v[i + 3])
            : "v"(v[i + HALF]), "v"(v[i + HALF + 1]), "v"(v[i + HALF + 2]), "v"(v[i + HALF + 3]));
}
template <int HALF, bool ROWS>
__device__ __forceinline__ void fold_rows(float* v) {
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
        const auto x = __builtin_bit_cast(unsigned, v[i]), y = __builtin_bit_cast(unsigned, v[i + HALF]);
        // (the elements are copied first: a bit cast of one as it stands takes the vector's first)
        const auto r = [&] {
            if constexpr (ROWS) return __builtin_amdgcn_permlane32_swap(x, y, false, false);
            else return __builtin_amdgcn_permlane16_swap(x, y, false, false);
        }();
        const unsigned low = r[0], high = r[1];
        v[i] = __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
    }
}
template <int P>
__device__ __forceinline__ void sum_over_channels(float (&v)[64 / P], int lane) {
    constexpr int N = 64 / P;
    if constexpr (P <= 4) {
        fold8<N / 2>(v);
        fold4<N / 4>(v);
        fold_rows<N / 8, true>(v);
        fold_rows<N / 16, false>(v);
        if constexpr (P == 2) {
            const float a = v[0] + across<2>(v[0]), b = v[1] + across<2>(v[1]);
            v[0] = lane & 2 ? b : a;
        }
    } else if constexpr (P == 8) {
        fold8<4>(v);
        fold_rows<2, true>(v);
        fold_rows<1, false>(v);
    } else {
        fold_rows<2, true>(v);
        fold_rows<1, false>(v);
    }
}
template <int P>
__device__ __forceinline__ int sum_of_lane(int lane) {
    const int rows = (lane >> 5 & 1) * 2 + (lane >> 4 & 1);  // the lanes' bits in the order of the steps
    if constexpr (P == 16) return rows;
    else if constexpr (P == 8) return (lane >> 3 & 1) * 4 + rows;
    else return ((lane >> 3 & 1) * 8 + (lane >> 2 & 1) * 4 + rows) * (4 / P) + (P == 4 ? 0 : lane >> 1 & 1);
}

// The gradient that each segment behind the first hands on, from zeros behind it (or from its sequence's end), and its sum of step sizes.
template <typename IO, int P, bool FULL>
__global__ __launch_bounds__(THREADS) void back_segments_kernel(const BackParams bp) {
    const Params& p = bp.f;
    constexpr int OWN = BATCH / P;
    __shared__ __attribute__((aligned(16))) float bc[2][BATCH * 2 * 4 * P];
    const Place<P> at(p.E, p.G, p.blocks);
    const int s = blockIdx.y + 1, b = blockIdx.z, r0 = s * p.L, r1 = min(p.T, r0 + p.L), e = at.e;
    int from, to;
    p.seq.inside(r0, r1, from, to);
    Walk w;
    w.find(p.seq, b, max(from, to - 1), at.lane);
    float a2[4], R[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) a2[k] = !FULL && 4 * at.p + k >= p.S ? 0.f : p.A[(long long)e * p.S + 4 * at.p + k] * LOG2E;
    const float bias = p.bias.p ? p.bias.value(p.bias.fetch(e)) : 0.f;
    Rows<IO, P> raw, ahead;
    const auto fetch = [&](Rows<IO, P>& x, int row) {
        x.fetch(x.d, p.delta, b * p.d_b, p.d_t, row, r1, at.p, e);
        x.fetch(x.g, bp.gy, b * bp.gy_b, bp.gy_t, row, r1, at.p, e);
        if (p.z) x.fetch(x.z, p.z, b * p.z_b, p.z_t, row, r1, at.p, e);
    };
    Stage<IO, P, 2> stage;
    const int last = r0 + (r1 - 1 - r0) / BATCH * BATCH;
    fetch(raw, last);
    stage.fetch(p, b, at.g, last, from, to);
    stage.put(bc[0]);
    lds_barrier();
    float total = 0.f;
    int buf = 0;
    for (int row = last; row >= r0; row -= BATCH, buf ^= 1) {
        const bool more = row > r0;
        if (more) {
            fetch(ahead, row - BATCH);
            stage.fetch(p, b, at.g, row - BATCH, from, to);
        }
        float dt[OWN], g[OWN];
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            const float d = to_f32(raw.d[i]) + bias;
            dt[i] = p.softplus ? softplus(d) : d;
            g[i] = to_f32(raw.g[i]);
            if (p.z) {
                const float z = to_f32(raw.z[i]);
                g[i] *= z * sigmoid(z);
            }
            total += row + at.p + i * P < r1 ? dt[i] : 0.f;
        }
        const auto piece = [&](auto part_, int first, int behind) {
            constexpr bool PART = decltype(part_)::value;
            each(std::make_integer_sequence<int, BATCH>(), [&](auto j_) {
                constexpr int j = BATCH - 1 - decltype(j_)::value;
                if (PART && (row + j < first || row + j >= behind)) return;
                const float d = from_lane<P, j % P>(dt[j / P]), v = from_lane<P, j % P>(g[j / P]);
                const f32x4 Ct = *reinterpret_cast<const f32x4*>(&bc[buf][j * 8 * P + 4 * P + 4 * at.p]);
#pragma unroll
                for (int k = 0; k < 4; ++k) R[k] = !FULL && 4 * at.p + k >= p.S ? 0.f : fast_exp2(d * a2[k]) * fmaf(Ct[k], v, R[k]);
            });
        };
        if (row >= from && row + BATCH <= to && w.within(row, BATCH)) piece(std::false_type(), 0, 0);
        else
            for (;;) {                                     // one sequence in front of the other
                const int first = max(max(row, from), w.begin), behind = min(min(row + BATCH, to), w.end);
                if (first >= behind) break;
                if (behind == w.end) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) R[k] = bp.glast && (FULL || 4 * at.p + k < p.S) ? bp.glast[((long long)w.n * p.E + e) * p.S + 4 * at.p + k] : 0.f;
                }
                piece(std::true_type(), first, behind);
                if (first > w.begin) break;
#pragma unroll
                for (int k = 0; k < 4; ++k) R[k] = 0.f;
                w.previous(p.seq);
            }
        if (more) {
            stage.put(bc[buf ^ 1]);
            raw = ahead;
            lds_barrier();
        }
    }
    if (!at.there) return;
    const long long place = (long long)b * p.nseg + s;
    *reinterpret_cast<f32x4*>(bp.seg_r + (place * p.E + e) * 4 * P + 4 * at.p) = f32x4{R[0], R[1], R[2], R[3]};
    float v[P];
#pragma unroll
    for (int q = 0; q < P; ++q) v[q] = total;
    sum_to_lanes<P, P>(v, at.p);
    if (at.p == 0) p.seg_dt[place * p.E + e] = v[0];
}

template <typename IO, int P, bool FULL>
__global__ __launch_bounds__(THREADS, 2) void back_kernel(const BackParams bp) {
    const Params& p = bp.f;
    constexpr int OWN = BATCH / P, COUNT = 64 / P, ROW = 8 * P, SUMS = BATCH * ROW, WAVES = THREADS / WAVE;
    constexpr bool KEEP = P <= 4;                          // (two workgroups a compute unit with 76 KB each; more lanes a channel have more sums in LDS: no room)
    __shared__ __attribute__((aligned(16))) float bc[2 * SUMS];   // the second half: zeros
    __shared__ float red[WAVES][SUMS];
    __shared__ f32x4 decays[KEEP ? BATCH : 1][THREADS];    // of the sixteen tokens, from the way along them for the way back
    const Place<P> at(p.E, p.G, p.blocks);
    const int s = blockIdx.y, r0 = s * p.L, r1 = min(p.T, r0 + p.L), e = at.e, wave = threadIdx.x >> 6;
    const long long part = (long long)blockIdx.z * p.nseg + s;
    int from, to;
    p.seq.inside(r0, r1, from, to);
    float a2[4], dA[4] = {0.f, 0.f, 0.f, 0.f}, dD = 0.f, dbias = 0.f;
    bool pad[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        pad[k] = !FULL && 4 * at.p + k >= p.S;
        a2[k] = pad[k] || !at.there ? 0.f : p.A[(long long)e * p.S + 4 * at.p + k] * LOG2E;
    }
    // A lane whose channel is not there adds exact zeros to dB and dC, whatever the channel holds that it reads in place of its own: no step, no states, B and C from the zeros.
    for (int i = threadIdx.x; i < SUMS; i += THREADS) bc[SUMS + i] = 0.f;
    const int row_bc = at.p + (at.there ? 0 : SUMS / 4);
    const float bias = p.bias.p ? p.bias.value(p.bias.fetch(e)) : 0.f, skip = p.D.p ? p.D.value(p.D.fetch(e)) : 0.f;
    const auto state_of = [&](const float* t, int n, float (&h)[4]) {
        const auto& p = arguments<BackParams>().f;
        int e = at.e;
        asm volatile("" : "+v"(e));                        // (no address of this is kept)
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = t && !pad[k] && at.there ? t[((long long)n * p.E + e) * p.S + 4 * at.p + k] : 0.f;
    };
    const auto first_gradient = [&](int n, const float (&h)[4]) {
        const auto& bp = arguments<BackParams>();
        const auto& p = bp.f;
        if (!bp.dstate || !at.there) return;
        int e = at.e;
        asm volatile("" : "+v"(e));
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (!pad[k]) bp.dstate[((long long)n * p.E + e) * p.S + 4 * at.p + k] = h[k];
    };
    const int last = r0 + (r1 - 1 - r0) / BATCH * BATCH, chunks = (p.T + BATCH - 1) / BATCH;
    // where a lane leaves the sum that it is left with: of token sum / 8 of a group (all of one where P is 16), B's or C's, state 4 p + sum % 4
    const int sum = sum_of_lane<P>(at.lane), leave = P == 16 ? 4 * at.p + sum : sum / 8 * ROW + sum / 4 % 2 * 4 * P + 4 * at.p + sum % 4;

    for (int b = blockIdx.z; b < p.rows; b += gridDim.z) {
        Walk w;
        w.find(p.seq, b, max(from, to - 1), at.lane);
        float R[4] = {0.f, 0.f, 0.f, 0.f};
        if (w.end > r1 && w.begin < r1) {                  // on from the segment that the sequence ends in
            int k = (w.end - 1) / p.L;
            const float* at_r = bp.seg_r + ((long long)b * p.nseg * p.E + e) * 4 * P + 4 * at.p;
            const float* at_dt = p.seg_dt + (long long)b * p.nseg * p.E + e;
            const f32x4 x0 = *reinterpret_cast<const f32x4*>(at_r + (long long)k * p.E * 4 * P);
#pragma unroll
            for (int i = 0; i < 4; ++i) R[i] = x0[i];
#pragma unroll 4
            for (--k; k > s; --k) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(at_r + (long long)k * p.E * 4 * P);
                const float dt = at_dt[(long long)k * p.E];
#pragma unroll
                for (int i = 0; i < 4; ++i) R[i] = decayed(R[i], dt, a2[i]) + x[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) R[i] = pad[i] || !at.there ? 0.f : R[i];   // (an infinite step size makes what is not there NaN)
        }
        // sixteen tokens' rows and their first state: asked for while the sums of those behind them are added up
        Rows<IO, P> raw;
        f32x4 kept;
        Stage<IO, P, 2> stage;
        const auto fetch = [&](int row) {
            const auto& bp = arguments<BackParams>();
            const auto& p = bp.f;
            raw.fetch(raw.u, p.u, b * p.u_b, p.u_t, row, r1, at.p, e);
            raw.fetch(raw.d, p.delta, b * p.d_b, p.d_t, row, r1, at.p, e);
            raw.fetch(raw.g, bp.gy, b * bp.gy_b, bp.gy_t, row, r1, at.p, e);
            if (p.z) raw.fetch(raw.z, p.z, b * p.z_b, p.z_t, row, r1, at.p, e);
            kept = at_row(reinterpret_cast<const f32x4*>(p.kept) + ((long long)b * chunks + row / BATCH) * p.E * P, (unsigned)(e * P + at.p) * 16u);
            stage.fetch(p, b, at.g, row, from, to);
        };
        fetch(last);
        stage.put(bc);
        lds_barrier();
        const float* const part_row = bp.part_bc + (((long long)(blockIdx.x % p.blocks) * p.rows + b) * p.T * p.G + at.g) * ROW;
        for (int row = last; row >= r0; row -= BATCH) {
            const bool more = row > r0;
            const auto& bp = arguments<BackParams>();
            const auto& p = bp.f;
            // a lane's own tokens: step size and its slope, u, g, and gy silu'(z)
            float dt[OWN], bend[OWN], u[OWN], g[OWN], gz[OWN];
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const float d = to_f32(raw.d[i]) + bias;
                dt[i] = !at.there ? 0.f : p.softplus ? softplus(d) : d;
                bend[i] = p.softplus ? sigmoid(d) : 1.f;
                u[i] = at.there ? to_f32(raw.u[i]) : 0.f;
                g[i] = at.there ? to_f32(raw.g[i]) : 0.f;
                if (p.z) {
                    const float z = to_f32(raw.z[i]), sg = sigmoid(z);
                    gz[i] = g[i] * (sg * fmaf(z, 1.f - sg, 1.f));
                    if (at.there) g[i] *= z * sg;
                }
            }
            const long long out = ((long long)b * p.T + row) * p.E;
            const unsigned place = (at.p * (unsigned)p.E + e) * sizeof(IO);
            const int width = p.E;
            const auto put = [&](void* t, int token, float v) { at_row(static_cast<const IO*>(t) + out + (long long)token * width, place) = from_f32<IO>(v); };
            // tokens [first, behind) of the sixteen, all of one sequence, from the state h in front of them; PART: not all sixteen
            const auto piece = [&](auto part_, int first, int behind, const float (&h)[4]) {
                constexpr bool PART = decltype(part_)::value;
                const int low = first - row, count = behind - first;
                const auto outside = [&](int j) { return PART && (unsigned)(j - low) >= (unsigned)count; };
                int lane_token = at.p, lane_sum = sum;
                if (PART) asm volatile("" : "+v"(lane_token), "+v"(lane_sum));   // (nothing of this is kept for other rows)
                float hs[BATCH + 1][4];                    // hs[j]: the state in front of token j
#pragma unroll
                for (int k = 0; k < 4; ++k) hs[0][k] = h[k];
                Pairs<P, 2, !PART> pairs;
                pairs.start(bc, 0, row_bc);
                each(std::make_integer_sequence<int, OWN>(), [&](auto i_) {
                    constexpr int i = decltype(i_)::value;
                    float y[P];
                    each(std::make_integer_sequence<int, P>(), [&](auto q_) {
                        constexpr int q = decltype(q_)::value, j = i * P + q;
                        y[q] = 0.f;
                        if (j % 2 == 0) pairs.advance(bc, j / 2, j / 2 + 1, row_bc);
#pragma unroll
                        for (int k = 0; k < 4; ++k) hs[j + 1][k] = hs[j][k];
                        if (outside(j)) return;
                        const float d = from_lane<P, q>(dt[i]), v = from_lane<P, q>(dt[i] * u[i]);
                        const f32x4 Bt = pairs.B[j % 2], Ct = pairs.C[j % 2];
                        f32x4 decay;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            decay[k] = fast_exp2(d * a2[k]);
                            hs[j + 1][k] = fmaf(decay[k], hs[j][k], v * Bt[k]);
                            if (!FULL && pad[k]) hs[j + 1][k] = 0.f;
                        }
                        if (KEEP) decays[j][threadIdx.x] = decay;
                        y[q] = fmaf(Ct[3], hs[j + 1][3], fmaf(Ct[2], hs[j + 1][2], fmaf(Ct[1], hs[j + 1][1], Ct[0] * hs[j + 1][0])));
                        asm volatile("" : "+v"(y[q]));     // (else it is made where z is looked at, from what had to wait in registers)
                    });
                    if (p.z) {
                        sum_to_lanes<P, P>(y, at.p);
                        if (at.there && !outside(lane_token + i * P)) put(bp.dz, i * P, gz[i] * fmaf(skip, u[i], y[0]));
                    }
                });
                // (B and C are read again, and the exponentials come from LDS: kept, they would fill three times as many registers as the states)
                int again = row_bc;
                asm volatile("" : "+v"(again));
#pragma unroll
                for (int i = 0; i < OWN; ++i) asm volatile("" : "+v"(dt[i]));
                pairs.start(bc, BATCH / 2 - 1, again);
                float along_B[P], along_A[P], sums[COUNT];
                f32x4 decay[2], decay_next[2];             // of two tokens, as B and C
                if (KEEP) decay_next[0] = decays[BATCH - 2][threadIdx.x], decay_next[1] = decays[BATCH - 1][threadIdx.x];
                each(std::make_integer_sequence<int, BATCH>(), [&](auto j_) {
                    constexpr int j = BATCH - 1 - decltype(j_)::value;
                    along_A[j % P] = along_B[j % P] = 0.f;
                    if (j % 2 == 1) {
                        if (KEEP) {
                            decay[0] = decay_next[0], decay[1] = decay_next[1];
                            if (j > 1) decay_next[0] = decays[j > 1 ? j - 3 : 0][threadIdx.x], decay_next[1] = decays[j > 1 ? j - 2 : 0][threadIdx.x];
                        }
                        pairs.advance(bc, j / 2, j / 2 - 1, again);
                    }
                    float dB[4] = {0.f, 0.f, 0.f, 0.f}, dC[4] = {0.f, 0.f, 0.f, 0.f};
                    if (!outside(j)) {
                        const float d = from_lane<P, j % P>(dt[j / P]), v = from_lane<P, j % P>(dt[j / P] * u[j / P]), gj = from_lane<P, j % P>(g[j / P]);
                        const f32x4 Bt = pairs.B[j % 2], Ct = pairs.C[j % 2];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float r = !FULL && pad[k] ? 0.f : fmaf(Ct[k], gj, R[k]);   // (an infinite gj would make it NaN, and with it what is summed over states)
                            dB[k] = r * v;
                            dC[k] = gj * hs[j + 1][k];
                            along_B[j % P] = fmaf(r, Bt[k], along_B[j % P]);
                            R[k] = (KEEP ? decay[j % 2][k] : fast_exp2(d * a2[k])) * r;
                            if (!FULL && pad[k]) R[k] = 0.f;
                            const float q = R[k] * hs[j][k];
                            along_A[j % P] = fmaf(q, a2[k], along_A[j % P]);
                            dA[k] = fmaf(q, d, dA[k]);
                        }
                    }
                    if constexpr (P == 16) {
                        sum_over_channels<P>(dB, at.lane);
                        sum_over_channels<P>(dC, at.lane);
                        if (!outside(j)) {
                            red[wave][j * ROW + leave] = dB[0];
                            red[wave][j * ROW + 4 * P + leave] = dC[0];
                        }
                    } else {
                        constexpr int GROUP = COUNT / 8;   // tokens whose sums go through the wave together
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            sums[j % GROUP * 8 + k] = dB[k];
                            sums[j % GROUP * 8 + 4 + k] = dC[k];
                        }
                        if constexpr (j % GROUP == 0) {
                            sum_over_channels<P>(sums, at.lane);
                            if (!outside(j + lane_sum / 8)) red[wave][j * ROW + leave] = sums[0];
                        }
                    }
                    // (else the compiler puts the additions to dA off to the end of the sixteen tokens, with all that they add up)
                    if (j % 2 == 0) asm volatile("" : "+v"(dA[0]), "+v"(dA[1]), "+v"(dA[2]), "+v"(dA[3]));
                    if constexpr (j % P == 0) {
                        constexpr int i = j / P;
                        sum_to_lanes<P, P>(along_A, at.p);
                        sum_to_lanes<P, P>(along_B, at.p);
                        const float a = fmaf(along_A[0], 1.f / LOG2E, u[i] * along_B[0]) * bend[i];
                        if (!outside(lane_token + j)) {
                            dD = fmaf(g[i], u[i], dD);
                            dbias += a;
                            if (at.there) {
                                put(bp.du, j, fmaf(dt[i], along_B[0], skip * g[i]));
                                put(bp.dd, j, a);
                            }
                        }
                    }
                });
            };
            if (row < from || row + BATCH > to) {
#pragma unroll
                for (int i = 0; i < OWN; ++i) {
                    const int t = row + at.p + i * P;
                    if (at.there && t < r1 && (t < from || t >= to)) {
                        put(bp.du, i * P, 0.f);
                        put(bp.dd, i * P, 0.f);
                        if (p.z) put(bp.dz, i * P, 0.f);
                    }
                }
            }
            for (;;) {                                     // one sequence in front of the other
                const int first = max(max(row, from), w.begin), behind = min(min(row + BATCH, to), w.end);
                if (first >= behind) break;
                float h[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) h[k] = at.there ? kept[k] : 0.f;
                if (behind == w.end) state_of(bp.glast, w.n, R);
                if (first == w.begin) state_of(p.state, w.n, h);
                if (behind - first == BATCH) piece(std::false_type(), first, behind, h);
                else piece(std::true_type(), first, behind, h);
                if (first > w.begin) break;
                first_gradient(w.n, R);
#pragma unroll
                for (int k = 0; k < 4; ++k) R[k] = 0.f;
                w.previous(sequences_of(p.seq));
            }
            if (more) fetch(row - BATCH);
            lds_barrier();
            for (int i = threadIdx.x; i < SUMS; i += THREADS) {
                const int t = row + i / ROW;
                float v = 0.f;
#pragma unroll
                for (int q = 0; q < WAVES; ++q) v += red[q][i];
                if (t < r1) at_row(part_row + (long long)row * p.G * ROW, (i / ROW * (unsigned)p.G * ROW + i % ROW) * 4u) = t >= from && t < to ? v : 0.f;
            }
            if (more) stage.put(bc);
            lds_barrier();
        }
    }
    if (p.seq.offsets && bp.dstate)                        // sequences without a token hand the last states' gradients on
        for (int n0 = s; n0 < p.N; n0 += p.nseg * 64) {
            const int mine = n0 + at.lane * p.nseg;
            unsigned long long empty = __ballot(mine < p.N && p.seq.of_lane(min(mine, p.N - 1) + 1) <= p.seq.of_lane(min(mine, p.N - 1)));
            for (; empty; empty &= empty - 1) {
                const int m = n0 + (__ffsll((long long)empty) - 1) * p.nseg;
                float h[4];
                state_of(bp.glast, m, h);
                first_gradient(m, h);
            }
        }
    float v[P], x[P];
#pragma unroll
    for (int q = 0; q < P; ++q) v[q] = dD, x[q] = dbias;
    sum_to_lanes<P, P>(v, at.p);
    sum_to_lanes<P, P>(x, at.p);
    if (!at.there) return;
    *reinterpret_cast<f32x4*>(bp.part_A + (part * p.E + e) * 4 * P + 4 * at.p) = f32x4{dA[0], dA[1], dA[2], dA[3]};
    if (at.p == 0) {
        bp.part_D[part * p.E + e] = v[0];
        bp.part_bias[part * p.E + e] = x[0];
    }
}

template <typename IO>
int launch_backward(const BackParams& bp, int parts, hipStream_t st) {
    const Params& p = bp.f;
    return with_lanes(p.S, [&](auto P_, auto full) {
        constexpr int P = decltype(P_)::value;
        constexpr bool FULL = decltype(full)::value;
        const dim3 block(THREADS);
        if (p.nseg > 1) hipLaunchKernelGGL((back_segments_kernel<IO, P, FULL>), dim3(p.G * p.blocks, p.nseg - 1, p.rows), block, 0, st, bp);
        hipLaunchKernelGGL((back_kernel<IO, P, FULL>), dim3(p.G * p.blocks, p.nseg, parts), block, 0, st, bp);
        return check_launch("vrwkv_scan_bwd");
    });
}

}  // namespace scan
}  // namespace vrwkv
