// Gradients of the attention with a decay for each head, all in one pass back along the chunks (gfx950).
// With S0 the state in front of a chunk (kept for every chunk by a pass of decay_attn.h), X the gradient of the state behind it, G the sums of its log
// decays, D_ts = exp(G_t - G_s) for s <= t, P = scale D (q k^T) and dP = scale D (gy v^T):
//     dq_t = sum_s dP_ts k_s + scale exp(G_t) S0 gy_t
//     dv_s = sum_t P_ts gy_t + exp(G_end - G_s) X^T k_s,       dk_s = sum_t dP_ts q_t + exp(G_end - G_s) X v_s
//     X <- exp(G_end) X + scale sum_t exp(G_t) q_t gy_t^T
//     dg_j = what crosses from tokens in front of j to j and behind: the terms P_ts (gy_t . v_s) with s < j <= t; q . (S0's part of dq) of the tokens from j on;
//            k . (X's part of dk) of those in front; exp(G_end) <S0, X>.  Sums of what crosses, so nothing cancels where little does.
// Twelve waves, three a SIMD, of three kinds: dq and dg's crossings inside the chunk (tokens t along the lanes), dk, and dv and X (tokens s along the lanes).  What
// one kind waits for the others cover: with dk, dv and X in one kind of eight waves a chunk of 64 bf16 tokens took 12 900 cycles, 60 % of them with an instruction; with
// sixteen waves the registers did not do.
// Every operand of the products is read as it lies or across its rows, so the chunk's rows are staged once (a pass each for dv, dk and dq would stage ten
// tensors for these four).  X lies in registers, rows of v's channels, and its terms in the LDS as [k's channel][v's], which both dk (rows) and dv (across) read.
// Larger heads go in tiles of 64 of k's and 64 of v's channels.  Everything is a sum over one or both kinds of tiles: dq and dk over v's, dv over k's, dg over
// all pairs; the parts are added up in fp32 behind.
// 64 x 196 tokens, 12 heads of 64, bf16: 82 us and 14.5 for the states in front (194 MB: 2.0 TB/s), the vector units busy 43 %, the matrix units 13, the LDS 31 (13 of it
// conflicts); 2 x 4150 fp32: 83 us.  A workgroup a compute unit, three a SIMD of its waves: bound by the latencies of a chunk's steps, 12 000 cycles of which no kind is idle more than
// 2500, and by 8600 at a sequence's start.
#pragma once
#include "decay_attn.h"

namespace vrwkv {
namespace decay {

constexpr int BWD_THREADS = 768;
enum Kind { DQ = 0, DK = 1, DV = 2 };

struct BwdParams : Call {
    View in[3], gy;                                       // q, k, v: what the waves of a kind stage, and
    OutView out[3];                                       // dq, dk, dv: what they make, next to each other: a kind reads its own with one load (parts lie rows * heads * channels apart)
    float* dg;                                            // [tiles][row][head]
    double* dg_sums;                                      // or, for decays that all tokens share, [segment][tiles][head]
    float* chunks;                                        // [chunk][head][tile of k][tile of v]: S0, rows of v's channels and columns of k's, as the accumulators lie
    const float *seg;                                     // [page][head][..][..]: R behind the segment, without the decay of the token behind it; null: sequences are not cut
    const float* seg_front;                               // the same: S in front of the segment
    const float *state, *glast;                           // the states in front of the first tokens; gradients of those behind the last; or null
    float* dstate;
    int Dk, Dv, tk, tv;                                   // channels; tiles of 64
};

}  // namespace decay
}  // namespace vrwkv
#include "decay_bwd_careful.h"
namespace vrwkv {
namespace decay {

template <typename IO>
struct BwdLds {
    static constexpr int L = chunk_len<IO, 64, PLAIN>, NS = in_terms<IO>, PX = 72;
    __bf16 q[NS][L][PX], k[NS][L][PX], v[NS][L][PX], gy[NS][L][PX];   // channels in the order of the state's fragments
    __bf16 x[3][64][PX];                                  // X [k's channel][v's, in that order]
    u32x4 s[3][4][2][64];                                 // S0's fragments: rows of k's channels, v's side by side
    struct Decays {
        float gh[L], gl[L], dt[L], dk[L];
        float end;
    } d[2];
    struct Flows {
        float in[2][L], out[2][L];                        // what a token receives over the chunk's front and gives over its end, by halves of the columns
        float inner[4][L], through[4];                    // what crosses it inside, by waves; what passes the chunk
    } f[2];                                               // this chunk's, and the last one's, which are summed beside this one's products
};

template <typename IO, bool FLOW, bool VEC>
__global__ __launch_bounds__(BWD_THREADS, 3) void decay_bwd_kernel(const BwdParams p) {
    using S = BwdLds<IO>;
    constexpr int L = S::L, NS = S::NS, NT = L / 16, KS = L / 32, PX = S::PX;
    constexpr int PIECES = L * 8 / 256;                   // a thread's of the tensor that its kind stages: q, k or v; the first two kinds take half of gy besides
    __shared__ S lds;
    __shared__ int offs[BWD_THREADS];
    const int tid = threadIdx.x, lane = tid & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kind = wave >> 2, w4 = wave & 3;
    touch(p);
    asm volatile("" : : "s"(p.in[0].p), "s"(p.in[1].sb), "s"(p.in[2].st), "s"(p.gy.sh), "s"(p.out[1].p), "s"(p.out[2].p), "s"(p.dg), "s"(p.tv));
    // a head's tiles next to each other: they read the same rows
    const int shift = (p.tk - 1) + (p.tv - 1), tile = blockIdx.x & ((1 << shift) - 1), h = blockIdx.x >> shift, gid = grid_segment();
    if (gid >= p.segs) return;
    const int ik = tile & (p.tk - 1), iv = tile >> (p.tk - 1), k0 = 64 * ik, v0 = 64 * iv;
    const auto out_of = [&](int kind) {
        OutView v = p.out[kind];
        if (v.p && v.f32) v.p = static_cast<float*>(v.p) + (kind == DV ? ik : iv) * p.rows * p.H * (kind == DV ? p.Dv : p.Dk);
        return v;
    };
    float* const dg_part = FLOW && p.dg ? p.dg + tile * p.rows * p.H : nullptr;
    double* const dg_sum = FLOW && p.dg_sums ? p.dg_sums + ((long long)gid * p.tk * p.tv + tile) * p.H + h : nullptr;

    const Place w = find_place<BWD_THREADS>(p, gid, L, offs);
    if (!p.nseg) {                                        // packed rows in front of the first sequence and behind the last: no gradient
        const int front = w.front, back = w.back, rows = front + max(0, p.T - back);
        for (int i = gid * 12 + wave; i < rows; i += p.segs * 12) {
            const long long row = i < front ? i : back + (i - front);
#pragma unroll
            for (int o = 0; o < 3; ++o) {
                const OutView v = out_of(o);
                const int d = (o < 2 ? k0 : v0) + lane;
                if (v.p && d < (o < 2 ? p.Dk : p.Dv)) {
                    const long long at = row * v.st + h * v.sh + d;
                    if (v.f32) static_cast<float*>(v.p)[at] = 0.f;
                    else static_cast<IO*>(v.p)[at] = from_f32<IO>(0.f);
                }
            }
            if (dg_part && lane == 0) dg_part[row * p.H + h] = 0.f;
        }
    }
    if (!w.valid) {
        if (dg_sum && tid == 0) *dg_sum = 0.;
        return;
    }
    const int nc = (w.s1 - w.s0 + L - 1) / L;
    __shared__ Careful careful;
    careful_begin(careful);
    float probe = 0.f;                                    // NaN once a result was not finite

    const int row0 = (tid & 255) >> 3, d0 = (tid & 7) * 8;
    // (half of gy: rows of even and odd blocks of 32 where a thread takes two of its own tensor, otherwise the workgroup's first and second 16)
    const int gy_row = PIECES == 2 ? row0 + 32 * kind : kind * 16 + row0;
    const bool gy_mine = kind < DV && (PIECES == 2 || row0 < 16);
    Source<IO, PIECES, 32, VEC> sa;
    Source<IO, 1, 32, VEC> sb;
    sa.open(p.in[kind], w.base, w.first, h, L, false, row0, (kind == DV ? v0 : k0) + d0, kind == DV ? p.Dv : p.Dk);
    sb.open(p.gy, w.base, w.first, h, L, false, gy_mine ? gy_row : L, v0 + d0, p.Dv);
    Gates gates;
    gates.open(p, w.base, w.first, h);
    const int tiles = p.tk * p.tv * 4096, my_tile = (ik * p.tv + iv) * 4096 + (w4 * 64 + lane) * 4;
    const float* const chunks = p.chunks + ((long long)(w.chunk0 + w.s0 / L) * p.H + h) * tiles + my_tile;
    const long long chunk_step = (long long)p.H * tiles;
    Piece<IO> ra[PIECES], rb[1];
    Gates::Raw rg{};
    constexpr int LIGHT = 4 * DK + 3;                     // the wave with the least to do: of dk, with the last tokens
    f32x4 st[4];                                          // dk: S0; dv: X.  Rows 16 x + 4 quarter + i (v's channels), column 16 w4 + col (k's)
    u32x4 held[3][2];                                     // its terms
    const auto fetch = [&](int c) {
        const int t0 = w.s0 + c * L, n = min(L, w.s1 - t0);
        sa.load(ra, t0, n, false);
        sb.load(rb, t0, n, false);
        if (wave == LIGHT) rg = gates.fetch(t0, lane, lane < n);
    };
    const auto begun = [&](int c) { return c > 0 || !w.is_first || p.state; };
    const auto fetch_state = [&](int c) {
        const bool there = begun(c);
#pragma unroll
        for (int x = 0; x < 4; ++x) st[x] = !there ? f32x4{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const f32x4*>(chunks + c * chunk_step + x * 1024);
    };
    const auto hold = [&]() {
#pragma unroll
        for (int kx = 0; kx < 2; ++kx) {
            const float x8[8] = {st[2 * kx][0], st[2 * kx][1], st[2 * kx][2], st[2 * kx][3], st[2 * kx + 1][0], st[2 * kx + 1][1], st[2 * kx + 1][2], st[2 * kx + 1][3]};
            bf16x8 t[3];
            split8<3>(x8, t);
#pragma unroll
            for (int s = 0; s < 3; ++s) held[s][kx] = __builtin_bit_cast(u32x4, t[s]);
        }
    };
    // (a kind that has no state: its registers are free while it works)
    const auto forget = [&]() {
#pragma unroll
        for (int x = 0; x < 4; ++x) st[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 3; ++s)
#pragma unroll
            for (int kx = 0; kx < 2; ++kx) held[s][kx] = u32x4{0, 0, 0, 0};
    };
    forget();
    if (nc > 0) fetch(nc - 1);

    // ---- X behind the segment
    const long long page = ((long long)w.n * p.H + h) * ((long long)p.Dk * p.Dv);
    const int zc = k0 + 16 * w4 + col;
    const bool cut = p.seg && !w.is_last;
    bool have = cut || p.glast;
    if (kind == DK) {
        if (nc > 0) fetch_state(nc - 1);
    } else if (kind == DV && cut) {
        // (R behind a segment wants the decay of the token there)
        const float d = fast_exp2(gates.widen(gates.fetch(w.s1, 0, true)) * LOG2E);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            st[x] = *reinterpret_cast<const f32x4*>(p.seg + ((long long)w.page * p.H + h) * tiles + my_tile + x * 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) st[x][i] *= d;
        }
    } else if (kind == DV && have) {
        const StatePage s(p.glast + page, 1, p.Dv, p.Dv, p.Dk, v0 + 4 * quarter, zc);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[x][i] = s.load(16 * x + i);
    }
    const int tw = w4 % NT, zt0 = w4 / NT * NT;           // this wave's tile of tokens, its first tile of channels
    Sink<IO, VEC> so;
    so.open(out_of(kind), w.base, w.first, h, 16 * tw + col, (kind == DV ? v0 : k0) + 16 * zt0 + 4 * quarter, kind == DV ? p.Dv : p.Dk);
    float* dg = dg_part ? dg_part + ((long long)w.base * p.T + w.first) * p.H + h : nullptr;
    double dg_total = 0.;                                 // (the light wave) of the segment's tokens
    int H = p.H;
    float scale = p.scale;
    keep(dg);
    keep(H);
    keep(scale);

    const auto put_decays = [&](typename S::Decays& d) { chunk_decays<L>(d, gates.widen(rg), lane, scale); };   // the light wave
    const auto put_flows = [&](const typename S::Flows& f, int t0, int n) {   // the light wave
        const int at = min(lane, L - 1);
        double in = 0., out = 0.;
        if (lane < n) {
            in = NT == 4 ? (double)f.in[0][lane] : (double)f.in[0][lane] + f.in[1][lane];
            out = NT == 4 ? (double)f.out[0][lane] : (double)f.out[0][lane] + f.out[1][lane];
        }
        const double inner = ((double)f.inner[0][at] + f.inner[1][at]) + ((double)f.inner[2][at] + f.inner[3][at]);
        const double through = ((double)f.through[0] + f.through[1]) + ((double)f.through[2] + f.through[3]);
        const double all = flow_sum(inner, in, out, lane) + through;
        if (lane < n) {
            probe = fmaf((float)all, 0.f, probe);
            if (dg) dg[(long long)(t0 + lane) * H] = (float)all;
            dg_total += all;
        }
    };
    const auto watch = [&](const f32x4 (&acc)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) probe = fmaf(acc[j][i], 0.f, probe);
    };
    if (nc > 0) {
        if (wave == LIGHT) put_decays(lds.d[0]);
        if (kind == DK || (kind == DV && have)) hold();
    }

    for (int ci = 0; ci < nc; ++ci) {
        // (what follows from the lane is worked out anew for each chunk: kept over the loop it fills the registers, masks for every tile among it)
        int lane_ = lane;
        asm volatile("" : "+v"(lane_));
        const int quarter = lane_ >> 4, col = lane_ & 15;
        const int c = nc - 1 - ci, t0 = w.s0 + c * L, n = min(L, w.s1 - t0);
        // ---- operands to the LDS
        const auto put = [&](const Piece<IO>& r, __bf16 (&a)[NS][L][PX], int row) {
            const int o0 = order_of(d0);
            u32x4 t[NS];
            piece_terms<IO>(r, t);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                *reinterpret_cast<uint2*>(&a[s][row][o0]) = uint2{t[s][0], t[s][1]};
                *reinterpret_cast<uint2*>(&a[s][row][o0 + 8]) = uint2{t[s][2], t[s][3]};
            }
        };
#pragma unroll
        for (int i = 0; i < PIECES; ++i) put(ra[i], kind == DQ ? lds.q : kind == DK ? lds.k : lds.v, row0 + 32 * i);
        if (gy_mine) put(rb[0], lds.gy, gy_row);
        if (kind != DQ) {
#pragma unroll
            for (int s = 0; s < 3; ++s)
#pragma unroll
                for (int kx = 0; kx < 2; ++kx) {
                    const u32x4 t = held[s][kx];
                    if (kind == DK) lds.s[s][w4][kx][lane_] = t;
                    else {
                        *reinterpret_cast<uint2*>(&lds.x[s][16 * w4 + col][32 * kx + 8 * quarter]) = uint2{t[0], t[1]};
                        *reinterpret_cast<uint2*>(&lds.x[s][16 * w4 + col][32 * kx + 4 + 8 * quarter]) = uint2{t[2], t[3]};
                    }
                }
        }
        lds_barrier();                                    // (orders the LDS alone: the next chunk's rows and this one's results stay on their way)
        if (ci + 1 < nc) fetch(c - 1);
        else {                                            // (nothing of the last rows is kept)
#pragma unroll
            for (int i = 0; i < PIECES; ++i) ra[i] = Piece<IO>{};
            rb[0] = Piece<IO>{};
        }
        typename S::Decays& dec = lds.d[ci & 1];
        typename S::Flows& flows = lds.f[ci & 1];
        const int r0 = 16 * tw + col;                     // this lane's token
        const auto row_of = [&](const __bf16 (&a)[NS][L][PX], int row, int kx, bf16x8 (&f)[NS]) {
#pragma unroll
            for (int s = 0; s < NS; ++s) f[s] = *reinterpret_cast<const bf16x8*>(&a[s][row][kx * 32 + 8 * quarter]);
        };
        // channels 16 x + col along the lanes, tokens 32 ks + 4 quarter .. and 16 behind those side by side
        const auto across = [&](const __bf16 (&a)[NS][L][PX], int x, int ks, bf16x8 (&f)[NS]) {
#pragma unroll
            for (int s = 0; s < NS; ++s) f[s] = across8(&a[s][32 * ks + 4 * quarter + (col >> 2)][(x >> 1) * 32 + (x & 1) * 4 + 8 * (col & 3)], PX);
        };
        const auto widen4 = [&](const __bf16 (&a)[NS][L][PX], int row, int x, float (&o)[4]) {   // channels 16 x + 4 quarter + i
#pragma unroll
            for (int s = NS - 1; s >= 0; --s) {
                const bf16x4 t = *reinterpret_cast<const bf16x4*>(&a[s][row][order_of(16 * x) + 8 * quarter]);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = s == NS - 1 ? (float)t[i] : o[i] + (float)t[i];
            }
        };
        // acc += what the tokens t >= s of the chunk give: (a_t . mine) D_ts of each, times c_t
        const auto gathered = [&](const __bf16 (&a)[NS][L][PX], const bf16x8 (&mine)[2][NS], const __bf16 (&c_)[NS][L][PX], float gh, float gl, f32x4 (&acc)[NT]) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (2 * ks + 1 < tw) continue;
                if (32 * ks >= n) break;
                float pr[8];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int tt = 2 * ks + hf;
                    f32x4 m = {0.f, 0.f, 0.f, 0.f};
                    if (tt >= tw) {
#pragma unroll
                        for (int kx = 0; kx < 2; ++kx) {
                            bf16x8 f[NS];
                            row_of(a, 16 * tt + col, kx, f);
                            m = mma<2>(m, f, mine[kx]);
                        }
                        const f32x4 th = *reinterpret_cast<const f32x4*>(&dec.gh[16 * tt + 4 * quarter]), tl = *reinterpret_cast<const f32x4*>(&dec.gl[16 * tt + 4 * quarter]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = m[i] * (scale * fast_exp2((th[i] - gh) + (tl[i] - gl)));
                            m[i] = tt > tw || 4 * quarter + i >= col ? x : 0.f;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) pr[4 * hf + i] = m[i];
                }
                bf16x8 fp[3];
                split8<3>(pr, fp);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    bf16x8 f[NS];
                    across(c_, zt0 + j, ks, f);
                    acc[j] = mma<2>(acc[j], f, fp);
                }
            }
        };
        f32x4 acc[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (kind == DQ) {
            if (16 * tw < n) {
                const float gh = dec.gh[r0], gl = dec.gl[r0], dt = dec.dt[r0];
                bf16x8 fo[2][NS];
                row_of(lds.gy, r0, 0, fo[0]);
                row_of(lds.gy, r0, 1, fo[1]);
                f32x4 flow[FLOW ? NT : 1];                // [tile of j]: sums over s < j of the terms of row t
                float in = 0.f;
#pragma unroll
                for (int j = 0; j < (FLOW ? NT : 1); ++j) flow[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (begun(c)) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
#pragma unroll
                        for (int kx = 0; kx < 2; ++kx) {
                            bf16x8 fs[3];
#pragma unroll
                            for (int s = 0; s < 3; ++s) fs[s] = __builtin_bit_cast(bf16x8, lds.s[s][zt0 + j][kx][lane_]);
                            acc[j] = mma<2>(acc[j], fs, fo[kx]);
                        }
                        float q4[4];
                        if constexpr (FLOW) widen4(lds.q, r0, zt0 + j, q4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            acc[j][i] *= dt;
                            if constexpr (FLOW) in = fmaf(q4[i], acc[j][i], in);
                        }
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (2 * ks > tw) break;
                    float pr[8], pf[8];
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int ts = 2 * ks + hf;
                        f32x4 m = {0.f, 0.f, 0.f, 0.f}, mq = {0.f, 0.f, 0.f, 0.f};
                        if (ts <= tw) {
#pragma unroll
                            for (int kx = 0; kx < 2; ++kx) {
                                bf16x8 f[NS];
                                row_of(lds.v, 16 * ts + col, kx, f);
                                m = mma<2>(m, f, fo[kx]);
                                if (FLOW && w4 < NT) {
                                    bf16x8 fq[NS];
                                    row_of(lds.k, 16 * ts + col, kx, f);
                                    row_of(lds.q, r0, kx, fq);
                                    mq = mma<2>(mq, f, fq);
                                }
                            }
                            const f32x4 sh = *reinterpret_cast<const f32x4*>(&dec.gh[16 * ts + 4 * quarter]), sl = *reinterpret_cast<const f32x4*>(&dec.gl[16 * ts + 4 * quarter]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float x = m[i] * (scale * fast_exp2((gh - sh[i]) + (gl - sl[i])));
                                m[i] = ts < tw || 4 * quarter + i <= col ? x : 0.f;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            pr[4 * hf + i] = m[i];
                            pf[4 * hf + i] = m[i] * mq[i];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);    // (what is read ahead of its use fills the registers otherwise)
                    bf16x8 fp[3];
                    split8<3>(pr, fp);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        bf16x8 fk[NS];
                        across(lds.k, zt0 + j, ks, fk);
                        acc[j] = mma<2>(acc[j], fk, fp);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (FLOW && w4 < NT) {                // (the other waves of a 32-token chunk would make the same terms)
                        bf16x8 ff[3];
                        split8<3>(pf, ff);
#pragma unroll
                        for (int j = 2 * ks; j < NT; ++j) {
                            if (j > tw) break;
                            // ones where s < j, row j of the tile in lane col: all of a tile in front of it, none of one behind it
                            u32x4 ones;
#pragma unroll
                            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const unsigned lo = 4 * quarter + 2 * e < col ? 0x3f80u : 0u, hi = 4 * quarter + 2 * e + 1 < col ? 0x3f800000u : 0u;
                                    ones[2 * hf + e] = 2 * ks + hf < j ? 0x3f803f80u : 2 * ks + hf == j ? lo | hi : 0u;
                                }
                            const bf16x8 fu[1] = {__builtin_bit_cast(bf16x8, ones)};
                            flow[j] = mma<2>(flow[j], fu, ff);
                        }
                    }
                }
                if constexpr (FLOW) {
                    in += __shfl_xor(in, 16);
                    in += __shfl_xor(in, 32);
                    if (quarter == 0) flows.in[w4 / NT][r0] = in;
                    float crossing[16];                   // of rows t from j on
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) crossing[4 * j + i] = j < NT && (j < tw || (j == tw && 4 * quarter + i <= col)) ? flow[j < NT ? j : 0][i] : 0.f;
                    int index;
                    const float cf = wkv6_detail::row_sums16(crossing, lane_, index);
                    if ((index >> 2) < NT) flows.inner[w4][16 * (index >> 2) + 4 * quarter + (index & 3)] = cf;
                }
            } else if (FLOW && lane_ < L) flows.inner[w4][lane_] = 0.f;
            watch(acc);
            so.store(acc, t0, r0 < n);
            forget();
        } else if (kind == DK) {
            if constexpr (FLOW) {                         // <S0, X>
                float through = 0.f;
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int s = 0; s < 3; ++s) {
                        const bf16x4 t = *reinterpret_cast<const bf16x4*>(&lds.x[s][16 * w4 + col][order_of(16 * x) + 8 * quarter]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) through = fmaf((float)t[i], st[x][i], through);
                    }
                through = wave_sum(through);
                if (lane_ == 0) flows.through[w4] = through * dec.end;
            }
            fetch_state(max(c - 1, 0));
            if (16 * tw < n) {
                const float gh = dec.gh[r0], gl = dec.gl[r0], dk = dec.dk[r0];
                bf16x8 fv[2][NS];
                row_of(lds.v, r0, 0, fv[0]);
                row_of(lds.v, r0, 1, fv[1]);
                float out = 0.f;
                if (have) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
#pragma unroll
                        for (int kx = 0; kx < 2; ++kx) {
                            bf16x8 fx[3];
#pragma unroll
                            for (int s = 0; s < 3; ++s) fx[s] = *reinterpret_cast<const bf16x8*>(&lds.x[s][16 * (zt0 + j) + col][kx * 32 + 8 * quarter]);
                            acc[j] = mma<2>(acc[j], fx, fv[kx]);
                        }
                        float k4[4];
                        if constexpr (FLOW) widen4(lds.k, r0, zt0 + j, k4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            acc[j][i] *= dk;
                            if constexpr (FLOW) out = fmaf(k4[i], acc[j][i], out);
                        }
                    }
                }
                gathered(lds.gy, fv, lds.q, gh, gl, acc);
                if constexpr (FLOW) {
                    out += __shfl_xor(out, 16);
                    out += __shfl_xor(out, 32);
                    if (quarter == 0) flows.out[w4 / NT][r0] = out;
                }
            }
            have = true;
            watch(acc);
            so.store(acc, t0, r0 < n);
            hold();
            if (wave == LIGHT) {
                if constexpr (FLOW) {
                    if (ci > 0) put_flows(lds.f[(ci + 1) & 1], t0 + L, min(L, w.s1 - t0 - L));
                }
                if (ci + 1 < nc) put_decays(lds.d[(ci + 1) & 1]);
            }
        } else {
            if (16 * tw < n) {
                const float gh = dec.gh[r0], gl = dec.gl[r0], dk = dec.dk[r0];
                bf16x8 fk[2][NS];
                row_of(lds.k, r0, 0, fk[0]);
                row_of(lds.k, r0, 1, fk[1]);
                if (have) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int x = zt0 + j;
#pragma unroll
                        for (int kx = 0; kx < 2; ++kx) {
                            bf16x8 fy[3];
#pragma unroll
                            for (int s = 0; s < 3; ++s) fy[s] = across8(&lds.x[s][32 * kx + 4 * quarter + (col >> 2)][(x >> 1) * 32 + (x & 1) * 4 + 8 * (col & 3)], PX);
                            acc[j] = mma<2>(acc[j], fy, fk[kx]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[j][i] *= dk;
                    }
                }
                gathered(lds.q, fk, lds.gy, gh, gl, acc);
            }
            watch(acc);
            so.store(acc, t0, r0 < n);
            // ---- X in front of the chunk
            const float ed = dec.end;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) st[x][i] *= ed;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (32 * ks >= n) break;
                const f32x4 a0 = *reinterpret_cast<const f32x4*>(&dec.dt[32 * ks + 4 * quarter]), a1 = *reinterpret_cast<const f32x4*>(&dec.dt[32 * ks + 16 + 4 * quarter]);
                bf16x8 fq[NS];
                across(lds.q, w4, ks, fq);
                float x8[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x8[i] = (float)fq[NS - 1][i];
#pragma unroll
                    for (int s = NS - 2; s >= 0; --s) x8[i] += (float)fq[s][i];
                    x8[i] *= i < 4 ? a0[i & 3] : a1[i & 3];
                }
                bf16x8 fd[3];
                split8<3>(x8, fd);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    bf16x8 fo[NS];
                    across(lds.gy, x, ks, fo);
                    st[x] = mma<2>(st[x], fo, fd);
                }
            }
            have = true;
            hold();
        }
        lds_barrier();
    }
    if constexpr (FLOW) {
        if (wave == LIGHT) {
            if (nc > 0) put_flows(lds.f[(nc + 1) & 1], w.s0, min(L, w.s1 - w.s0));
            if (dg_sum) {
#pragma unroll
                for (int d = 32; d; d >>= 1) dg_total += __shfl_xor(dg_total, d);
                if (lane == 0) *dg_sum = dg_total;
            }
        }
    }

    if (p.dstate && w.is_first && kind == DV) {
        const StatePage s(p.dstate + page, 1, p.Dv, p.Dv, p.Dk, v0 + 4 * quarter, zc);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s.store(16 * x + i, st[x][i]);
                probe = fmaf(st[x][i], 0.f, probe);
            }
    }
    if (!(probe == 0.f)) careful.wanted = 1;
    lds_barrier();
    if (nc > 0 && uniform(careful.wanted)) {
        static_assert(sizeof(CarefulBwdLds) <= sizeof(S), "");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // what has been stored arrives in front of what takes its place
        __syncthreads();
        careful_gradients<IO, FLOW, L, BWD_THREADS>(careful, reinterpret_cast<CarefulBwdLds&>(lds), offs);
    }
}

template <typename IO> int launch_decay_bwd(const BwdParams& p, bool vec, hipStream_t st);
extern template int launch_decay_bwd<float>(const BwdParams&, bool, hipStream_t);
extern template int launch_decay_bwd<__hip_bfloat16>(const BwdParams&, bool, hipStream_t);
extern template int launch_decay_bwd<__half>(const BwdParams&, bool, hipStream_t);

template <typename IO>
int launch_decay_bwd(const BwdParams& p, bool vec, hipStream_t st) {
    const dim3 grid = decay_grid(p, p.tk * p.tv), block(BWD_THREADS);
    if (p.dg || p.dg_sums) {
        if (vec) hipLaunchKernelGGL((decay_bwd_kernel<IO, true, true>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((decay_bwd_kernel<IO, true, false>), grid, block, 0, st, p);
    } else {
        if (vec) hipLaunchKernelGGL((decay_bwd_kernel<IO, false, true>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((decay_bwd_kernel<IO, false, false>), grid, block, 0, st, p);
    }
    return check_launch("decay_attention (gradients)");
}

}  // namespace decay
}  // namespace vrwkv
