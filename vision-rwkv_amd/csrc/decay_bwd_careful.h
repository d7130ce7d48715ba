// Gradients token by token in fp32, for the workgroups whose results are not all finite (decay_careful.h says when and why):
//     R_t = exp(g_{t+1}) R_{t+1} + scale q_t gy_t^T,   dq_t = scale S_t gy_t,   dk_t = R_t v_t,   dv_t = R_t^T k_t,   dg_t = exp(g_t) <S_{t-1}, R_t>,   dS0 = exp(g_0) R_0
// of one tile of 64 of k's and 64 of v's channels and the tokens of one segment, from the state in front of it and the gradient behind it.  dg's states are kept
// at the front of every chunk, in the room of the states in front of the chunks, and made again from there.
// 64 x 196 tokens, 12 heads of 64, bf16, with a NaN in every row: 1.9 ms for 95 us; 2 x 4150 fp32 1.4 ms for 135.
#pragma once

namespace vrwkv {
namespace decay {

struct CarefulBwdLds {
    CarefulLds<64> scan;                                  // dq's, dk's and dv's
    float s[64][64], r[64][64];                           // [v's channel][k's]
    float k[CAREFUL_TOKENS][64], q[CAREFUL_TOKENS][64], v[64][CAREFUL_TOKENS], gy[64][CAREFUL_TOKENS];
    float e[CAREFUL_TOKENS], next[CAREFUL_TOKENS];        // exp(g) of the tokens, and of those behind them
    float part[CAREFUL_TOKENS][8];
};

template <typename IO, bool FLOW, int L, int THREADS_>
__device__ __forceinline__ void careful_gradients(const Careful& careful, CarefulBwdLds& f, int* offs) {
    CarefulLds<64>& m = f.scan;
    const BwdParams p = arguments_again<BwdParams>(careful);
    const int shift = (p.tk - 1) + (p.tv - 1), tile = blockIdx.x & ((1 << shift) - 1), h = blockIdx.x >> shift, gid = grid_segment();
    const int ik = tile & (p.tk - 1), iv = tile >> (p.tk - 1), k0 = 64 * ik, v0 = 64 * iv, nk = min(64, p.Dk - k0), nv = min(64, p.Dv - v0);
    const Place w = find_place<THREADS_>(p, gid, L, offs);
    const int nc = (w.s1 - w.s0 + L - 1) / L, tid = threadIdx.x;
    const long long page = ((long long)w.n * p.H + h) * ((long long)p.Dk * p.Dv);
    const long long tiles = p.tk * p.tv * 4096, mine = (ik * p.tv + iv) * 4096;
    float* const fronts = p.chunks + ((long long)(w.chunk0 + w.s0 / L) * p.H + h) * tiles + mine;   // of the segment's chunks; nobody else reads or writes them any more
    const long long front_step = p.H * tiles;
    const float* const front = w.is_first ? nullptr : p.seg_front + ((long long)w.page * p.H + h) * tiles + mine;
    const float* const behind = p.seg && !w.is_last ? p.seg + ((long long)w.page * p.H + h) * tiles + mine : nullptr;
    Gates gates;
    gates.open(p, w.base, w.first, h);
    const CarefulRows<IO> q(p.in[0], w.base, w.first, h, k0, p.Dk), k(p.in[1], w.base, w.first, h, k0, p.Dk), v(p.in[2], w.base, w.first, h, v0, p.Dv), gy(p.gy, w.base, w.first, h, v0, p.Dv);
    const auto put = [&](int kind, int token, int lane, float x) {
        const OutView& o = p.out[kind];
        if (!o.p || lane >= (kind == DV ? nv : nk)) return;
        const long long at = w.base * o.sb + (long long)(w.first + token) * o.st + h * o.sh + (kind == DV ? v0 : k0) + lane;
        if (o.f32) static_cast<float*>(o.p)[at + (kind == DV ? ik : iv) * p.rows * p.H * (kind == DV ? p.Dv : p.Dk)] = x;
        else static_cast<IO*>(o.p)[at] = from_f32<IO>(x);
    };
    // a page (k's channels, v's) of the call's states, as [v's][k's]; null: zeros
    const auto state_at = [&](const float* s, int row, int lane) { return s && lane < nk ? s[page + (long long)(k0 + lane) * p.Dv + v0 + row] : 0.f; };

    // ---- S: dq, and the states at the chunks' fronts
    careful_each<64>(nv, [&](int row, int lane) { m.st[row][lane] = front ? front[careful_place(row, lane)] : state_at(p.state, row, lane); });
#pragma unroll 1
    for (int c = 0; c < nc; ++c) {
        if (FLOW) careful_each<64>(nv, [&](int row, int lane) { fronts[c * front_step + careful_place(row, lane)] = m.st[row][lane]; });
        const int from = w.s0 + c * L;
        careful_scan(m, gates, gy, v, k, p.scale, 1.f, from, min(w.s1, from + L), w.len, false, [&](int token, int lane, float x) { put(DQ, token, lane, x); });
    }
    // R behind the segment, as [v's][k's]
    const auto behind_at = [&](int row, int lane) { return behind ? behind[careful_place(row, lane)] : state_at(p.glast, row, lane); };
    // ---- dg: R back along the tokens, S along them from the chunks' fronts
    if constexpr (FLOW) {
        double total = 0.;
        careful_each<64>(nv, [&](int row, int lane) { f.r[row][lane] = behind_at(row, lane); });
#pragma unroll 1
        for (int c = nc - 1; c >= 0; --c) {
            const int from = w.s0 + c * L, to = min(w.s1, from + L), blocks = (to - from + CAREFUL_TOKENS - 1) / CAREFUL_TOKENS;
#pragma unroll 1
            for (int block = blocks - 1; block >= 0; --block) {
                careful_each<64>(nv, [&](int row, int lane) { f.s[row][lane] = fronts[c * front_step + careful_place(row, lane)]; });
                float y[CAREFUL_TOKENS];
                int n = 0;
#pragma unroll 1
                for (int b = 0; b <= block; ++b) {
                    const int t0 = from + b * CAREFUL_TOKENS;
                    n = min(CAREFUL_TOKENS, to - t0);
                    __syncthreads();
#pragma unroll 1
                    for (int x = tid; x < CAREFUL_TOKENS * 64; x += THREADS_) {
                        const int i = x >> 6, d = x & 63;
                        f.k[i][d] = k.at(t0 + i, d, i < n);
                        f.v[d][i] = v.at(t0 + i, d, i < n);
                        f.q[i][d] = p.scale * q.at(t0 + i, d, i < n);
                        f.gy[d][i] = gy.at(t0 + i, d, i < n);
                    }
                    if (tid <= CAREFUL_TOKENS) {
                        const bool there = tid <= n && t0 + tid < w.len;
                        const float g = gates.widen(gates.fetch(t0, tid, there)), e = there ? expf(g) : 1.f;
                        if (tid < CAREFUL_TOKENS) f.e[tid] = tid < n ? e : 1.f;
                        if (tid > 0) f.next[tid - 1] = tid - 1 < n ? e : 1.f;
                    }
                    __syncthreads();
                    const bool last = b == block;
#pragma unroll
                    for (int i = 0; i < CAREFUL_TOKENS; ++i) y[i] = 0.f;
                    careful_each<64>(nv, [&](int row, int lane) {
                        float s = f.s[row][lane], front[CAREFUL_TOKENS];
#pragma unroll
                        for (int i = 0; i < CAREFUL_TOKENS; ++i) {
                            front[i] = s;
                            s = fmaf(s, f.e[i], f.v[row][i] * f.k[i][lane]);
                        }
                        f.s[row][lane] = s;
                        if (last) {
                            float r = f.r[row][lane];
#pragma unroll
                            for (int i = CAREFUL_TOKENS - 1; i >= 0; --i) {
                                r = fmaf(r, f.next[i], f.gy[row][i] * f.q[i][lane]);
                                if (lane < nk) y[i] = fmaf(r * f.e[i], front[i], y[i]);
                            }
                            f.r[row][lane] = r;
                        }
                    });
                }
                if (tid < 512) {
#pragma unroll
                    for (int i = 0; i < CAREFUL_TOKENS; ++i) {
                        const float sum = wave_sum(y[i]);
                        if ((tid & 63) == 0) f.part[i][tid >> 6] = sum;
                    }
                }
                __syncthreads();
                if (tid < n) {
                    double sum = 0.;
#pragma unroll
                    for (int r = 0; r < 8; ++r) sum += f.part[tid][r];
                    if (p.dg) p.dg[tile * p.rows * p.H + ((long long)w.base * p.T + w.first + from + block * CAREFUL_TOKENS + tid) * p.H + h] = (float)sum;
                    total += sum;
                }
            }
        }
        if (tid < 64 && p.dg_sums) {                       // (wave 0 has all of it)
#pragma unroll
            for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
            if (tid == 0) p.dg_sums[((long long)gid * p.tk * p.tv + tile) * p.H + h] = total;
        }
    }
    // ---- dk
    careful_each<64>(nv, [&](int row, int lane) { m.st[row][lane] = behind_at(row, lane); });
    careful_scan(m, gates, v, gy, q, 1.f, p.scale, w.s0, w.s1, w.len, true, [&](int token, int lane, float x) { put(DK, token, lane, x); });
    // ---- R the other way round, [k's][v's]: dv, and the first states' gradient
    careful_each<64>(nk, [&](int row, int lane) {
        m.st[row][lane] = behind ? behind[careful_place(lane, row)] : p.glast && lane < nv ? p.glast[page + (long long)(k0 + row) * p.Dv + v0 + lane] : 0.f;
    });
    careful_scan(m, gates, k, q, gy, 1.f, p.scale, w.s0, w.s1, w.len, true, [&](int token, int lane, float x) { put(DV, token, lane, x); });
    if (p.dstate && w.is_first) {
        const float e = expf(gates.widen(gates.fetch(0, 0, true)));
        careful_each<64>(nk, [&](int row, int lane) {
            if (lane < nv) p.dstate[page + (long long)(k0 + row) * p.Dv + v0 + lane] = m.st[row][lane] * e;
        });
    }
}

}  // namespace decay
}  // namespace vrwkv
