// The scan over few tokens of few channels (gfx950): selective_scan's forward where one workgroup a compute unit holds it, in one launch.
//
// What bounds such a call is the way from one token to the next and the launches, not the chip: time is cut inside a workgroup, a wave has sixteen tokens of four channels and the waves
// beside it the tokens behind.  Sixteen lanes hold one channel: lane p has token p of the sixteen for what belongs to a token alone, and states p, p + 16, .. for the rest.  A wave goes through
// its tokens from zeros, with every decay and product kept in registers; then the waves exchange their last states and sums of step sizes, each works out the states in front of its own
// tokens, and goes through them once more with what it kept: no exponential is made twice.  196 tokens of 384 channels with 16 states in bf16: 7.9 us (a launch of a few instructions: about 4).
#pragma once
#include "scan.h"

namespace vrwkv {
namespace scan {

constexpr int SHORT_P = 16, SHORT_CHANNELS = WAVE / SHORT_P;
constexpr int short_waves(int S) { return S <= 16 ? 16 : 8; }   // (the decays and products of more states fill the registers)

// NS: states a lane; W: the most waves; FULL: S is 16 NS
template <typename IO, int NS, int W, bool FULL>
__global__ __launch_bounds__(W * WAVE) void short_kernel(const Params p, const int width) {
    constexpr int P = SHORT_P;
    __shared__ float bc[W][2][BATCH][P * NS];              // B and C of a wave's tokens
    __shared__ float ends[2][W][NS][WAVE], times[2][W][WAVE], carry[2][NS][WAVE];
    __shared__ int cuts[2][W];                             // whether a sequence begins among a wave's tokens
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, q = lane % P, of_group = p.E / p.G;
    const int g = blockIdx.x / p.blocks, c = (blockIdx.x % p.blocks) * SHORT_CHANNELS + lane / P, e = g * of_group + min(c, of_group - 1), b = blockIdx.y;
    const bool there = c < of_group;
    int from, to;
    p.seq.inside(0, p.T, from, to);
    float a2[NS];
    bool pad[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        pad[k] = !FULL && q + P * k >= p.S;
        a2[k] = pad[k] ? 0.f : p.A[(long long)e * p.S + q + P * k] * LOG2E;
    }
    const float bias = p.bias.p ? p.bias.value(p.bias.fetch(e)) : 0.f, skip = p.D.p ? p.D.value(p.D.fetch(e)) : 0.f;
    const auto first_state = [&](int n, int k) { return p.state && !pad[k] ? p.state[((long long)n * p.E + e) * p.S + q + P * k] : 0.f; };
    int buf = 0;
    for (int row0 = 0; row0 < p.T; row0 += waves * BATCH, buf ^= 1) {
        const auto& p = arguments<Params>();
        const int row = row0 + wave * BATCH, read = min(row, p.T - 1), behind_read = p.T - 1 - read;
        // everything that is read, before the first of it is needed
        const auto own = [&](const void* x, long long base, long long stride) {
            return to_f32(at_row(static_cast<const IO*>(x) + base + read * stride, (min(q, behind_read) * (unsigned)stride + e) * sizeof(IO)));
        };
        float z = 0.f;
        const float u = own(p.u, b * p.u_b, p.u_t), raw = own(p.delta, b * p.d_b, p.d_t) + bias;
        if (p.z) z = own(p.z, b * p.z_b, p.z_t);
        IO raw_B[4 * NS], raw_C[4 * NS];                   // lane l: token l / 16 + 4 i, its states
        const IO* const B = static_cast<const IO*>(p.B) + b * p.B_b + read * p.B_t + g * p.B_g;
        const IO* const C = static_cast<const IO*>(p.C) + b * p.C_b + read * p.C_t + g * p.C_g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const unsigned j = min(lane / P + 4 * i, behind_read), n = pad[k] ? 0 : q + P * k;
                raw_B[i * NS + k] = at_row(B, (j * (unsigned)p.B_t + n) * sizeof(IO));
                raw_C[i * NS + k] = at_row(C, (j * (unsigned)p.C_t + n) * sizeof(IO));
            }
        Walk w;
        w.find(sequences_of(p.seq), b, max(read, from), lane);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                bc[wave][0][lane / P + 4 * i][q + P * k] = to_f32(raw_B[i * NS + k]);
                bc[wave][1][lane / P + 4 * i][q + P * k] = to_f32(raw_C[i * NS + k]);
            }
        __builtin_amdgcn_wave_barrier();
        // the sequences of the wave's tokens one after the other: h = the first states and begins() where one begins, f(whether not all tokens, first, behind), ends(n) where it ends
        float h[NS];
        const auto sequences = [&](Walk at, auto&& begins, auto&& f, auto&& ends) {
            for (;;) {
                const int first = max(max(row, from), at.begin), behind = min(min(row + BATCH, to), at.end);
                if (first >= behind) break;
                if (first == at.begin) {
#pragma unroll
                    for (int k = 0; k < NS; ++k) h[k] = first_state(at.n, k);
                    begins();
                }
                if (behind - first == BATCH) f(std::false_type(), first, behind);
                else f(std::true_type(), first, behind);
                if (behind < at.end) break;
                ends(at.n);
                at.next(sequences_of(p.seq));
            }
        };
        const float dt = p.softplus ? softplus(raw) : raw, x = dt * u;
        float decay[BATCH][NS], in[BATCH][NS], total = 0.f;
        bool cut = false;
#pragma unroll
        for (int k = 0; k < NS; ++k) h[k] = 0.f;
        sequences(w, [&] { cut = true; }, [&](auto part, int first, int behind) {
            each(std::make_integer_sequence<int, BATCH>(), [&](auto j_) {
                constexpr int j = decltype(j_)::value;
                if (decltype(part)::value && (row + j < first || row + j >= behind)) return;
                const float d = from_lane<P, j>(dt), v = from_lane<P, j>(x);
                total += d;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    decay[j][k] = fast_exp2(d * a2[k]);
                    in[j][k] = v * bc[wave][0][j][q + P * k];
                    if (!FULL && pad[k]) in[j][k] = 0.f;   // (an infinite v would make it NaN)
                    h[k] = fmaf(decay[j][k], h[k], in[j][k]);
                }
            });
        }, [](int) {});
#pragma unroll
        for (int k = 0; k < NS; ++k) ends[buf][wave][k][lane] = h[k];
        times[buf][wave][lane] = total;
        if (lane == 0) cuts[buf][wave] = cut;
        lds_barrier();
        // the states in front of these tokens: what the waves in front have left, back to the last that a sequence begins in
        const unsigned long long anew = __ballot(lane < wave && cuts[buf][lane < wave ? lane : 0]);
        float time = 0.f;
        const auto add = [&](int k, float x) {
            const float power = time * a2[k];
            h[k] += __all(fabsf(power) < 100.f) ? x * fast_exp2(power) : decayed(x, time, a2[k]);
        };
#pragma unroll
        for (int k = 0; k < NS; ++k) h[k] = 0.f;
        const int back = anew ? 63 - __builtin_clzll(anew) : 0;
        for (int i = wave - 1; i >= back; --i) {
#pragma unroll
            for (int k = 0; k < NS; ++k) add(k, ends[buf][i][k][lane]);
            time += times[buf][i][lane];
        }
        if (row0 && !anew) {
#pragma unroll
            for (int k = 0; k < NS; ++k) add(k, carry[buf][k][lane]);
        }
#pragma unroll
        for (int k = 0; k < NS; ++k) h[k] = pad[k] ? 0.f : h[k];   // (an infinite step size makes what is not there NaN)
        float y[P];
#pragma unroll
        for (int j = 0; j < P; ++j) y[j] = 0.f;
        if (p.kept && there && row < p.T) {
            float* const to_kept = p.kept + (((long long)b * ((p.T + BATCH - 1) / BATCH) + row / BATCH) * p.E + e) * width;
#pragma unroll
            for (int k = 0; k < NS; ++k)
                if (q + P * k < width) to_kept[q + P * k] = h[k];
        }
        sequences(w, [] {}, [&](auto part, int first, int behind) {
            each(std::make_integer_sequence<int, BATCH>(), [&](auto j_) {
                constexpr int j = decltype(j_)::value;
                if (decltype(part)::value && (row + j < first || row + j >= behind)) return;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    h[k] = fmaf(decay[j][k], h[k], in[j][k]);
                    const float Ct = bc[wave][1][j][q + P * k];
                    if (FULL || !pad[k]) y[j] = fmaf(Ct, h[k], y[j]);
                }
            });
        }, [&](int n) {
            if (p.last && there) {
#pragma unroll
                for (int k = 0; k < NS; ++k)
                    if (!pad[k]) p.last[((long long)n * p.E + e) * p.S + q + P * k] = h[k];
            }
        });
        if (wave == waves - 1) {
#pragma unroll
            for (int k = 0; k < NS; ++k) carry[buf ^ 1][k][lane] = h[k];
        }
        sum_to_lanes<P, P>(y, q);
        float v = fmaf(skip, u, y[0]);
        if (p.z) v *= z * sigmoid(z);
        if (there && row + q < p.T)
            at_row(static_cast<const IO*>(p.y) + ((long long)b * p.T + row) * p.E, (q * (unsigned)p.E + e) * sizeof(IO)) = from_f32<IO>(row + q >= from && row + q < to ? v : 0.f);
    }
    if (p.seq.offsets && p.last)                           // sequences without a token keep their states
        for (int n0 = wave * WAVE; n0 < p.N; n0 += waves * WAVE) {
            const int mine = n0 + lane;
            unsigned long long empty = __ballot(mine < p.N && p.seq.of_lane(min(mine, p.N - 1) + 1) <= p.seq.of_lane(min(mine, p.N - 1)));
            for (; empty; empty &= empty - 1) {
                const int n = n0 + __ffsll((long long)empty) - 1;
#pragma unroll
                for (int k = 0; k < NS; ++k)
                    if (there && !pad[k]) p.last[((long long)n * p.E + e) * p.S + q + P * k] = first_state(n, k);
            }
        }
}

template <typename IO>
int launch_short(const Params& p, int width, hipStream_t st) {
    const auto go = [&](auto NS_) {
        constexpr int NS = decltype(NS_)::value, W = short_waves(16 * NS);
        const dim3 grid(p.G * p.blocks, p.rows), block(std::min(W, (p.T + BATCH - 1) / BATCH) * WAVE);
        if (p.S == 16 * NS) hipLaunchKernelGGL((short_kernel<IO, NS, W, true>), grid, block, 0, st, p, width);
        else hipLaunchKernelGGL((short_kernel<IO, NS, W, false>), grid, block, 0, st, p, width);
        return check_launch("vrwkv_scan_fwd");
    };
    if (p.S <= 16) return go(std::integral_constant<int, 1>());
    if (p.S <= 32) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, 4>());
}

}  // namespace scan
}  // namespace vrwkv
