// Attention whose state decays head by head (gfx950): for one head, with q, k (Dk), v, y (Dv), a log decay g and the state S (Dk, Dv),
//     S_t = exp(g_t) S_{t-1} + k_t v_t^T,      y_t = scale S_t^T q_t.
// A sequence goes in chunks of L tokens.  With G_t = the sum of g over the chunk's tokens up to t and S0 the state in front of the chunk,
//     y_t = scale sum_{s<=t} exp(G_t - G_s) (q_t . k_s) v_s + scale exp(G_t) S0^T q_t,      S = exp(G_end) S0 + sum_s exp(G_end - G_s) k_s v_s^T,
// four matrix products.  The state in front of each chunk, and the same sum back along the tokens (b, c = gy, q in the places of k, v: the gradient of a
// state), which the gradients want (decay_bwd.h), are this kernel's without its outputs.
// Calls of few sequences are cut into segments: a pass makes each segment's own state, a second adds them up, the third starts from them.
// What lies between operands (P, states) has 24 bits, three bf16 terms, in every type: with two, sums that cancel kept 2^-18 of their terms, and 64 x 196 x 12 heads in bf16 took 24.7 us.
// 64 x 196 tokens, 12 heads of 64, bf16: 27 us, 90 MB at 3.3 TB/s.  4 x 16384 in fp16, where rows have two terms: 204 to 214 us, a third of them for the segments' states, 10 to add them
// up, the rest for the outputs, of which the vector units are busy 50 %, the LDS 43, the matrix units 29: bound by a chunk's chain of staging, products, exponentials and products again.
#pragma once
#include "wave_sum.h"
#include "wkv6_chunk_common.h"

namespace vrwkv {
namespace decay {

using wkv6_detail::bf16x4;
using wkv6_detail::bf16x8;
using wkv6_detail::f32x4;
using wkv6_detail::u32x4;

constexpr int TZ = 64;                                    // columns of a state that a workgroup holds
constexpr int THREADS = 256, OUT_THREADS = 512;           // of a workgroup for states; for outputs

// A tensor (batch, token, head, channel), channels side by side; head h of the call reads head h / share.
struct View {
    const void* p;
    long long sb, st, sh;
    int share;
};
struct OutView {
    void* p;
    long long sb, st, sh;
    int f32;                                              // fp32 values of every head, added up and rounded by a kernel behind
};
struct Role {
    View a, b, c;                                         // q, k, v
    OutView o;
    const float* init;                                    // states (N, H, Dk, Dv), or null: zeros
    float* last;                                          // where the states behind the last token go, or null
    float *seg, *seg_decay;                               // [page][head][tile] a segment's state (first its own, then that in front of it), [page][head]; segment_page()
    float* anchors;                                       // [chunk][head][tile]: the state in front of each chunk
    long long sx, sz;                                     // strides of the states' contracted and other index
    int dx, dz, tiles, reverse;                           // (one or two tiles; the roles of a launch have the same)
    float s_upd;                                          // scale of what the states take up
};
struct Call {                                             // sequences, their cut, and the decays
    const void *offsets, *g;
    long long g_sb, g_st, g_sh;
    long long rows;                                       // batch * T
    int off64, g_dtype, N, T, H;                          // T: tokens of a row of the batch (packed: of all sequences)
    int seg_len, nseg, segs;                              // tokens of a segment; segments of a row (0: packed); of the call
    float scale;
    int by_start;                                         // packed: segments' states lie by where the segments start
};
struct Params : Call {
    int n_roles;
    Role role[2];
};
template <typename IO> constexpr int in_terms = std::is_same<IO, float>::value ? 3 : std::is_same<IO, __half>::value ? 2 : 1;   // bf16 numbers that hold an element

// outputs; no outputs: a segment's own state; no outputs: the state in front of each chunk
enum Mode { PLAIN = 0, STATES = 1, CHUNKS = 2 };
// tokens of a chunk: 64 where two workgroups' rows and states fit the LDS of a compute unit (fp32 rows take three times the room of bf16 ones, fp16 rows twice)
template <typename IO, int DX, int MODE>
constexpr int chunk_len = std::is_same<IO, __hip_bfloat16>::value || (std::is_same<IO, __half>::value && (DX == 64 || MODE != PLAIN)) ? 64 : 32;

struct Place {                                            // a workgroup's segment
    int n, first, len;                                    // sequence; its first token and length
    int s0, s1;                                           // the segment's tokens, from the first
    int base;                                             // batch row
    int page;                                             // of the segment's state
    int chunk0;                                           // number of the sequence's first chunk
    int front, back;                                      // packed: where the first sequence begins, and the last one ends
    bool is_last, is_first, valid;
};
__device__ __forceinline__ int offset_at(const Call& p, int n) {
    const long long v = p.off64 ? static_cast<const long long*>(p.offsets)[n] : (long long)static_cast<const int*>(p.offsets)[n];
    return (int)(v < 0 ? 0 : v > p.T ? p.T : v);
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ Place sequence_place(const Call& p, int n, int L) {
    Place w{};
    w.n = n;
    w.valid = true;
    if (p.nseg) {
        w.first = 0;
        w.len = p.T;
        w.base = n;
        w.chunk0 = n * ((p.T + L - 1) / L);
    } else {
        w.first = uniform(offset_at(p, n));
        w.len = uniform(max(0, offset_at(p, n + 1) - w.first));
        w.base = 0;
        w.chunk0 = w.first / L + n;
    }
    return w;
}
// Packed sequences: n's segments have the numbers from first(n) / seg_len + n on, which grow with n and leave each its room whatever its length.
__device__ __forceinline__ int first_segment(const Call& p, int n, int first) { return p.nseg ? n * p.nseg : first / p.seg_len + n; }
// The page of segment j of a sequence that is cut (others have none in use).  Of many packed sequences few can be: in any seg_len tokens at most one first segment of such a
// sequence begins, and one that is not its first, so two pages to each of them do, where a page to each sequence was 2.1 GB for 4096 prompts of 64 tokens and 16 heads of 128 x 64.
__device__ __forceinline__ int segment_page(const Call& p, int n, int first, int j) { return p.by_start ? 2 * (first / p.seg_len + j) + (j == 0 ? 1 : 0) : first_segment(p, n, first) + j; }
__device__ __forceinline__ int segment_count(const Call& p, int len) { return max(1, (len + p.seg_len - 1) / p.seg_len); }

// offs: THREADS_ numbers of shared memory (packed sequences: one read of the offsets where they are fewer than the threads).
template <int THREADS_>
__device__ __forceinline__ Place find_place(const Call& p, int gid, int L, int* offs) {
    Place w{};
    if (p.nseg) {
        w = sequence_place(p, p.nseg == 1 ? gid : gid / p.nseg, L);
    } else if (p.N < THREADS_) {
        const int i = threadIdx.x, o = offset_at(p, min(i, p.N));
        offs[i] = o;
        const int seen = __syncthreads_count(i < p.N && o / p.seg_len + i <= gid), n = __builtin_amdgcn_readfirstlane(seen - 1);
        w.front = __builtin_amdgcn_readfirstlane(offs[0]);
        w.back = __builtin_amdgcn_readfirstlane(offs[p.N]);
        if (n >= 0) {
            w.n = n;
            w.first = __builtin_amdgcn_readfirstlane(offs[n]);
            w.len = max(0, __builtin_amdgcn_readfirstlane(offs[n + 1]) - w.first);
            w.chunk0 = w.first / L + n;
            w.valid = true;
        }
    } else {
        // the last sequence that begins at this segment or in front of it: every step-th one looked at together, then those behind the last that does
        int n = 0, size = p.N, step;
        do {
            step = (size + THREADS_ - 1) / THREADS_;
            const int i = min((int)threadIdx.x * step, size), at = n + min(i, size - 1);
            const int seen = __syncthreads_count(i < size && offset_at(p, at) / p.seg_len + at <= gid);
            if (seen == 0) { n = -1; break; }
            n += (seen - 1) * step;
            size = min(step, size - (seen - 1) * step);
        } while (step > 1);
        n = __builtin_amdgcn_readfirstlane(n);
        if (n >= 0) w = sequence_place(p, n, L);
        w.front = offset_at(p, 0);
        w.back = offset_at(p, p.N);
    }
    if (!w.valid) return w;
    const int j = gid - first_segment(p, w.n, w.first), count = segment_count(p, w.len);
    w.valid = j >= 0 && j < count;
    w.page = segment_page(p, w.n, w.first, j);
    w.s0 = j * p.seg_len;
    w.s1 = min(w.len, w.s0 + p.seg_len);
    w.is_first = j == 0;
    w.is_last = j == count - 1;
    return w;
}
// Workgroups: x: heads, and what varies within one (a power of two); y and z: segments.
constexpr int GRID_Y = 32768;
__device__ __forceinline__ int grid_segment() { return blockIdx.y + GRID_Y * blockIdx.z; }
inline dim3 decay_grid(const Call& p, int within) { return dim3((unsigned)(p.H * within), (unsigned)(p.segs < GRID_Y ? p.segs : GRID_Y), (unsigned)((p.segs + GRID_Y - 1) / GRID_Y)); }

// The eight channels d .. d + 7 of a row: at byte offset `at` of the buffer in one or two loads of 16 bytes where rows come in such pieces (VEC), element by
// element otherwise; `count` of them exist; `ahead` bytes behind, the same for all lanes.  What does not is asked of an offset outside the buffer and arrives as zero, without a branch: loads behind
// branches were waited for one by one, 4.5 of the 5.5 us that a chunk took.
template <typename IO> struct Piece { unsigned w[sizeof(IO) * 2]; };
template <typename IO, bool VEC>
__device__ __forceinline__ Piece<IO> load_piece(__amdgpu_buffer_rsrc_t buf, unsigned at, int count, unsigned ahead) {
    Piece<IO> r;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(IO) / 2; ++i) {
            const auto t = BufRaw<16>::ld(buf, at + 16 * i, ahead);
#pragma unroll
            for (int c = 0; c < 4; ++c) r.w[4 * i + c] = t[c];
        }
    } else if constexpr (sizeof(IO) == 4) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.w[e] = BufRaw<4>::ld(buf, e < count ? at + 4 * e : OOB_OFFSET, ahead);
    } else {
        unsigned short h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = BufRaw<2>::ld(buf, e < count ? at + 2 * e : OOB_OFFSET, ahead);
#pragma unroll
        for (int e = 0; e < 4; ++e) r.w[e] = (unsigned)h[2 * e] | (unsigned)h[2 * e + 1] << 16;
    }
    return r;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) { return make_rsrc(p, 0x7fffffffu); }
// The value stays in scalar registers: read again from the arguments it cost each chunk's fetch 1600 cycles and each result's address as much.
template <typename T>
__device__ __forceinline__ void keep(T& x) { asm volatile("" : "+s"(x)); }

// The arguments' cache lines asked for together: met one after the other, where each is first needed, they cost the start of a workgroup some 2000 cycles.
__device__ __forceinline__ void touch(const Call& c) { asm volatile("" : : "s"(c.offsets), "s"(c.N), "s"(c.segs)); }
__device__ __forceinline__ void touch(const Role& r) { asm volatile("" : : "s"(r.a.p), "s"(r.b.st), "s"(r.c.sh), "s"(r.o.f32), "s"(r.anchors), "s"(r.dx), "s"(r.s_upd)); }

// Four channels of a row, `count` of them there.
template <typename O, bool VEC>
__device__ __forceinline__ void store_quad(__amdgpu_buffer_rsrc_t buf, unsigned at, int count, f32x4 x) {
    O q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = from_f32<O>(x[i]);
    if constexpr (VEC) {
        typename BufRaw<4 * sizeof(O)>::type d;
        __builtin_memcpy(&d, q, sizeof(d));
        BufRaw<4 * sizeof(O)>::st(d, buf, count > 0 ? at : OOB_OFFSET, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            typename BufRaw<sizeof(O)>::type d;
            __builtin_memcpy(&d, &q[i], sizeof(d));
            BufRaw<sizeof(O)>::st(d, buf, i < count ? at + i * (unsigned)sizeof(O) : OOB_OFFSET, 0);
        }
    }
}

// A tensor's rows of one sequence and head, and a thread's pieces of a chunk: rows `row`, `row` + STEP .. in the order that the kernel takes them.  Row i is
// token t0 + i, or back along the tokens t0 + n - 1 - i, which is L - 1 - i from token t0 + n - L on: a thread's offsets stay the same.
template <typename IO, int PIECES, int STEP, bool VEC>
struct Source {
    const char* p;
    int pitch;                                            // bytes from token to token
    unsigned at;
    int row, count;
    __device__ __forceinline__ void open(const View& v, int base, int first, int head, int L, bool rev, int row_, int d, int dim) {
        p = static_cast<const char*>(v.p) + (base * v.sb + (long long)first * v.st + (v.share == 1 ? head : head / v.share) * v.sh) * (int)sizeof(IO);
        pitch = (int)v.st * (int)sizeof(IO);
        keep(p);
        keep(pitch);
        row = row_;
        count = dim - d;
        at = (unsigned)((rev ? L - 1 - row - STEP * (PIECES - 1) : row) * pitch + d * (int)sizeof(IO));
        if (count <= 0) at = OOB_OFFSET;
    }
    // the first of the chunk's tokens in memory (or of the L that end with its last) and its rows
    __device__ __forceinline__ void load(Piece<IO> (&r)[PIECES], int token, int n, bool rev) const {
        const auto buf = buffer_at(p + (long long)token * pitch);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const bool there = row + STEP * i < n;
            r[i] = load_piece<IO, VEC>(buf, there ? at : OOB_OFFSET, there ? count : 0, (unsigned)((rev ? PIECES - 1 - i : i) * STEP * pitch));
        }
    }
};
// Sixteen rows as the products take them from the lanes, straight from memory: a lane's row, and of each 32 channels the four from 4 quarter on and those 16 behind.
template <typename IO, int KX, bool VEC>
struct Fragments {
    const char* p;
    int pitch;
    unsigned at;
    int row, count;
    __device__ __forceinline__ void open(const View& v, int base, int first, int head, int row_, int quarter, int dim) {
        p = static_cast<const char*>(v.p) + (base * v.sb + (long long)first * v.st + (v.share == 1 ? head : head / v.share) * v.sh) * (int)sizeof(IO);
        pitch = (int)v.st * (int)sizeof(IO);
        keep(p);
        keep(pitch);
        row = row_;
        count = dim - 4 * quarter;
        at = (unsigned)(row * pitch + 4 * quarter * (int)sizeof(IO));
    }
    __device__ __forceinline__ void load(Piece<IO> (&r)[KX], int token, int n, bool) const {
        const auto buf = buffer_at(p + (long long)token * pitch);
        const int have = row < n ? count : 0;
#pragma unroll
        for (int i = 0; i < 2 * KX; ++i) {                // fours
            const unsigned ahead = 16 * i * (unsigned)sizeof(IO);
            unsigned* const w = &r[i / 2].w[(i & 1) * (int)sizeof(IO)];
            if constexpr (VEC) {
                const auto t = BufRaw<4 * sizeof(IO)>::ld(buf, 16 * i < have ? at : OOB_OFFSET, ahead);
#pragma unroll
                for (int c = 0; c < (int)sizeof(IO); ++c) w[c] = t[c];
            } else if constexpr (sizeof(IO) == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = BufRaw<4>::ld(buf, 16 * i + e < have ? at + 4 * e : OOB_OFFSET, ahead);
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const unsigned lo = BufRaw<2>::ld(buf, 16 * i + 2 * e < have ? at + 4 * e : OOB_OFFSET, ahead), hi = BufRaw<2>::ld(buf, 16 * i + 2 * e + 1 < have ? at + 4 * e + 2 : OOB_OFFSET, ahead);
                    w[e] = lo | hi << 16;
                }
            }
        }
    }
};
// Where a lane's results go: four channels of a row, and every sixteenth behind them.
template <typename IO, bool VEC>
struct Sink {
    char* p;
    int pitch, f32;
    unsigned at;
    int count;
    __device__ __forceinline__ void open(const OutView& v, int base, int first, int head, int row, int d, int dim) {
        f32 = v.f32;
        const int e = f32 ? 4 : (int)sizeof(IO);
        p = v.p ? static_cast<char*>(v.p) + (base * v.sb + (long long)first * v.st + head * v.sh) * e : nullptr;
        pitch = (int)v.st * e;
        keep(p);
        keep(pitch);
        keep(f32);
        at = (unsigned)(row * pitch + d * e);
        count = dim - d;
    }
    // (called on every way through a chunk, so that what was asked for before is waited for without waiting for this)
    template <int N>
    __device__ __forceinline__ void store(const f32x4 (&x)[N], int token, bool there) const {
        const auto buf = buffer_at(p + (long long)token * pitch);
        const int have = there && p ? count : 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (f32) store_quad<float, VEC>(buf, at + 64 * j, have - 16 * j, x[j]);
            else store_quad<IO, VEC>(buf, at + 16 * j * (unsigned)sizeof(IO), have - 16 * j, x[j]);
        }
    }
};
// A state (N, H, Dk, Dv)'s numbers as a lane of the accumulators has them: x, and the rows behind it, of one column.  Addresses that differ by what is the same for
// all lanes, and no branches: element by element behind its own check, writing the last states took 8 000 of a short sequence's 28 000 cycles.
struct StatePage {
    __amdgpu_buffer_rsrc_t buf;
    unsigned at;
    int step, count;                                      // bytes from row to row; rows from x on
    __device__ __forceinline__ StatePage(const float* p, long long sx, long long sz, int dx, int dz, int x, int z) : buf(buffer_at(p)), step((int)sx * 4), count(z < dz ? dx - x : 0) {
        at = (unsigned)(x * step + z * (int)sz * 4);
    }
    __device__ __forceinline__ float load(int i) const { return __builtin_bit_cast(float, BufRaw<4>::ld(buf, i < count ? at : OOB_OFFSET, (unsigned)(i * step))); }
    __device__ __forceinline__ void store(int i, float v) const { BufRaw<4>::st(__builtin_bit_cast(unsigned, v), buf, i < count ? at : OOB_OFFSET, (unsigned)(i * step)); }
};
// The log decays of a sequence and head.
struct Gates {
    const char* p;
    int pitch, dtype;
    __device__ __forceinline__ void open(const Call& c, int base, int first, int head) {
        const int e = c.g_dtype == VRWKV_F32 ? 4 : 2;
        p = static_cast<const char*>(c.g) + (base * c.g_sb + (long long)first * c.g_st + head * c.g_sh) * e;
        pitch = (int)c.g_st * e;
        dtype = c.g_dtype;
        keep(p);
        keep(pitch);
        keep(dtype);
    }
    // of token `token` + i, as it lies: widened where it is used, so the fetch is ahead, with no branch on its type behind which it would be waited for
    struct Raw {
        unsigned word, half;
    };
    __device__ __forceinline__ Raw fetch(int token, int i, bool there) const {
        const auto buf = buffer_at(p + (long long)token * pitch);
        const unsigned at = (unsigned)(i * pitch);
        return {BufRaw<4>::ld(buf, there && dtype == VRWKV_F32 ? at : OOB_OFFSET, 0), BufRaw<2>::ld(buf, there && dtype != VRWKV_F32 ? at : OOB_OFFSET, 0)};
    }
    __device__ __forceinline__ float widen(Raw r) const {
        const float x = dtype == VRWKV_F32 ? __builtin_bit_cast(float, r.word) : dtype == VRWKV_BF16 ? __builtin_bit_cast(float, r.half << 16) : (float)__builtin_bit_cast(_Float16, (unsigned short)r.half);
        return x < -200.f ? -200.f : x;                   // (exp(-200) is zero in fp32 too; sums of -inf or the lowest value would be -inf, their differences NaN)
    }
};
// x as the sum of n bf16 numbers (two at a time): 16 bits of it with two, all 24 with three
// DOT: heads are subtracted by a dot product each, x + (head0, head1) . (-1, 0), instead of two instructions.  The other product is zero but where the other
// number is no number: for pairs that one sum takes up.
template <int N, bool DOT = false>
__device__ __forceinline__ void split_pair(float x0, float x1, unsigned (&t)[N]) {
    typedef wkv6_detail::bf16x2 pair_t;
    unsigned lo = 0x0000bf80u, hi = 0xbf800000u;          // (kept opaque: as constants they become an inline operand that stands for another pair)
    if (DOT) asm("" : "+s"(lo), "+s"(hi));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        t[i] = wkv6_detail::pack_bf16(x0, x1);
        if (i + 1 < N) {
            if (DOT) {
                const pair_t h = __builtin_bit_cast(pair_t, t[i]);
                x0 = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(pair_t, lo), x0, false);
                x1 = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(pair_t, hi), x1, false);
            } else {
                x0 -= wkv6_detail::bf16_lo(t[i]);
                x1 -= wkv6_detail::bf16_hi(t[i]);
            }
        }
    }
}
template <int N, bool DOT = true>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[N]) {
    u32x4 w[N];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        unsigned o[N];
        split_pair<N, DOT>(x[2 * p], x[2 * p + 1], o);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i][p] = o[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = __builtin_bit_cast(bf16x8, w[i]);
}
template <typename IO>
__device__ __forceinline__ void piece_terms(const Piece<IO>& r, u32x4 (&t)[in_terms<IO>]) {
    constexpr int NS = in_terms<IO>;
    if constexpr (std::is_same<IO, __hip_bfloat16>::value) {
        t[0] = u32x4{r.w[0], r.w[1], r.w[2], r.w[3]};
    } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            unsigned o[NS];
            if constexpr (std::is_same<IO, float>::value)
                split_pair<NS>(__builtin_bit_cast(float, r.w[2 * p]), __builtin_bit_cast(float, r.w[2 * p + 1]), o);
            else
                split_pair<NS>((float)__builtin_bit_cast(_Float16, (unsigned short)r.w[p]), (float)__builtin_bit_cast(_Float16, (unsigned short)(r.w[p] >> 16)), o);
#pragma unroll
            for (int i = 0; i < NS; ++i) t[i][p] = o[i];
        }
    }
}

template <typename IO>
__device__ __forceinline__ void widen_piece(const Piece<IO>& r, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (std::is_same<IO, float>::value) x[e] = __builtin_bit_cast(float, r.w[e]);
        else if constexpr (std::is_same<IO, __half>::value) x[e] = (float)__builtin_bit_cast(_Float16, (unsigned short)(r.w[e / 2] >> (16 * (e & 1))));
        else x[e] = __builtin_bit_cast(float, e & 1 ? r.w[e / 2] & 0xffff0000u : r.w[e / 2] << 16);
    }
}

// acc += a b with both operands sums of bf16 numbers; products beyond the ORDER-th correction are left out.
template <int ORDER, int NA, int NB>
__device__ __forceinline__ f32x4 mma(f32x4 acc, const bf16x8 (&a)[NA], const bf16x8 (&b)[NB]) {
#pragma unroll
    for (int o = (NA + NB - 2 < ORDER ? NA + NB - 2 : ORDER); o >= 0; --o)         // small ones first
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[o - i], acc, 0, 0, 0);
    return acc;
}

// sum over the lanes up to this one: inside 16 lanes, then the rows' totals (DPP moves; lanes without a source add zero)
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CTRL, ROWS, 0xf, false);
    return x + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan_inclusive(double x) {
    x = dpp_add<0x111, 0xf>(x);                           // row_shr:1, 2, 4, 8
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);                           // row_bcast:15 into rows 1 and 3, row_bcast:31 into 2 and 3
    return dpp_add<0x143, 0xc>(x);
}

__device__ __forceinline__ double lane_double(double x, int lane) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
    return __builtin_bit_cast(double, (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)b, lane));
}
// What crosses token `lane`: terms inside the chunk, what it and the tokens behind it receive over the chunk's front, what those in front of it give over its end.
__device__ __forceinline__ double flow_sum(double inner, double in, double out, int lane) {
    double before = wave_scan_inclusive(out);
    before = __shfl_up(before, 1);
    if (lane == 0) before = 0.;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double o = __shfl_down(in, d);
        if (lane + d < 64) in += o;
    }
    return inner + in + before;
}

template <typename IO, int DX, int MODE>
struct Lds {
    static constexpr int L = chunk_len<IO, DX, MODE>, NS = in_terms<IO>;
    static constexpr int PX = DX + 8, PZ = TZ + 8;        // row pitches: 16 rows of a fragment on different banks
    static constexpr bool OUT = MODE == PLAIN;
    // q's rows, each read by one wave or two, come through the LDS (in wide pieces: 64 x 196 x 12 bf16 26.9 us, straight from memory 27.7; 2 x 4150 x 12 fp32 55 and 56) where they
    // leave room for two workgroups, or for one alone either way; fp16 rows, and bf16 ones of more than 64 channels, do not (4 x 16384 x 12 fp16 204 us, with them 232)
    static constexpr bool STAGED = OUT && (NS == 3 || (NS == 1 && DX == 64));
    __bf16 a[STAGED ? NS : 1][STAGED ? L : 1][STAGED ? PX : 8];
    __bf16 b[NS][L][PX];                                  // channels in the order of the state's fragments (as they lie where there are no outputs: read across the rows alone, with fewer bank conflicts)
    // c with its decays to the chunk's end, where it is wanted with them alone and has more terms than one: scaled before it is split, not put together to be scaled
    static constexpr bool SCALED = !OUT && NS > 1;
    __bf16 c[SCALED ? 3 : NS][L][PZ];
    u32x4 s[OUT ? 3 : 1][4][OUT ? DX / 32 : 1][64];   // the state's terms, a lane's fragment side by side
    struct Decays {
        float gh[L], gl[L], dt[L], dk[L];                 // G in powers of two, head and tail; exp(G); exp(G_end - G)
        float end;                                        // exp(G_end)
    } d[2];                                               // this chunk's and the next one's
};

// Where channel d of a row lies in the order that the accumulators' fragments have: inside 32 channels, 4 m .. 4 m + 3 lie at 8 (m & 3) + 4 (m >> 2); of eight from an eighth
// on, the second four 8 behind the first.
__device__ __forceinline__ int order_of(int d) {
    const int m = (d >> 2) & 7;
    return (d & ~31) + 8 * (m & 3) + 4 * (m >> 2);
}

// Packed rows in front of the first sequence and behind the last get zeros, a few from every workgroup of the head and tile.
template <typename IO>
__device__ __forceinline__ void clear_outside(const Params& p, const Role& r, int front, int back, int gid, int z, int h) {
    const int rows = front + max(0, p.T - back);
    const int d = z * TZ + (threadIdx.x & 63);
    for (int i = gid * (OUT_THREADS / 64) + (threadIdx.x >> 6); i < rows; i += p.segs * (OUT_THREADS / 64)) {
        const long long row = i < front ? i : back + (i - front);
        const long long at = row * r.o.st + h * r.o.sh + d;
        if (d < r.dz) static_cast<IO*>(r.o.p)[at] = from_f32<IO>(0.f);
    }
}

// workgroups that a compute unit's LDS holds, up to three: more do not fit the registers
template <size_t BYTES> constexpr int workgroups = 3 * BYTES <= 160 * 1024 ? 3 : 2 * BYTES <= 160 * 1024 ? 2 : 1;
template <size_t BYTES> constexpr int out_workgroups = 2 * BYTES <= 160 * 1024 ? 2 : 1;

// A chunk's decays by one wave, from its log decays (zero behind its last token), those from its front times scale; the sum of the powers of two.
// In 64 bits: a chunk's G may be thousands where a neighbour's difference is a hundredth.
template <int L, typename D>
__device__ __forceinline__ float chunk_decays(D& d, float g, int lane, float scale = 1.f) {
    const double G = wave_scan_inclusive((double)g * 1.4426950408889634);
    const double end = lane_double(G, 63);
    const float gh = (float)G;
    if (lane < L) {
        d.gh[lane] = gh;
        d.gl[lane] = (float)(G - gh);
        d.dt[lane] = fast_exp2(gh) * scale;
        d.dk[lane] = fast_exp2((float)(end - G));
    }
    if (lane == 0) d.end = fast_exp2((float)end);
    return (float)end;
}
// A fragment read across rows: a lane's four of q's row and four of the row 16 behind it.
__device__ __forceinline__ bf16x8 across8(const __bf16* q, int pitch) { return wkv6_detail::cat8(wkv6_detail::lds_read_tr4(q), wkv6_detail::lds_read_tr4(q + 16 * pitch)); }
// c's rows with their decays to the chunk's end, put together from the terms, scaled and split again
template <typename IO, int L, int PZ>
__device__ __forceinline__ void decayed_terms(const __bf16 (&c)[in_terms<IO>][L][PZ], const float* dk, float s_upd, int ks, int column, int quarter, int col, bf16x8 (&f)[3]) {
    float x8[8];
    const f32x4 d0 = *reinterpret_cast<const f32x4*>(&dk[32 * ks + 4 * quarter]), d1 = *reinterpret_cast<const f32x4*>(&dk[32 * ks + 16 + 4 * quarter]);
#pragma unroll
    for (int i = 0; i < 8; ++i) x8[i] = 0.f;
#pragma unroll
    for (int s = in_terms<IO> - 1; s >= 0; --s) {
        const bf16x8 t = across8(&c[s][32 * ks + 4 * quarter + (col >> 2)][column + 4 * (col & 3)], PZ);
#pragma unroll
        for (int i = 0; i < 8; ++i) x8[i] += (float)t[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x8[i] *= d0[i] * s_upd;
        x8[4 + i] *= d1[i] * s_upd;
    }
    split8<3>(x8, f);
}

}  // namespace decay
}  // namespace vrwkv
#include "decay_careful.h"
namespace vrwkv {
namespace decay {

// A segment's own state, or the states in front of a segment's chunks.  Four waves, 16 columns each, several workgroups a compute unit; four more that stage the next
// chunk beside them were slower (4 x 16384 x 12 fp16: 67 us without, 87 with).
template <typename IO, int DX, int MODE, bool VEC>
__global__ __launch_bounds__(THREADS, (workgroups<sizeof(Lds<IO, DX, MODE>)>)) void decay_states_kernel(const Params p) {
    using S = Lds<IO, DX, MODE>;
    constexpr int L = S::L, NS = S::NS, KS = L / 32, NX = DX / 16;
    constexpr int PB = L * DX / 8 / THREADS, PC = L * TZ / 8 / THREADS;
    static_assert(MODE != PLAIN && PB >= 1 && PC >= 1 && L * DX % (8 * THREADS) == 0 && L * TZ % (8 * THREADS) == 0, "");
    __shared__ S lds;
    __shared__ int offs[THREADS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, col = lane & 15;

    // a head's tiles, and the roles of a tile, next to each other: they read the same rows
    int id = blockIdx.x;
    touch(p);
    touch(p.role[0]);
    if (MODE == STATES) touch(p.role[1]);
    const Role& r = p.role[MODE == STATES ? id & (p.n_roles - 1) : 0];
    if (MODE == STATES) id >>= p.n_roles - 1;
    const int z = id & (r.tiles - 1), h = id >> (r.tiles - 1), gid = grid_segment();
    if (gid >= p.segs) return;
    const Place w = find_place<THREADS>(p, gid, L, offs);
    if (!w.valid) return;
    const bool rev = MODE == STATES && r.reverse;
    if (MODE == STATES && (rev ? w.is_first : w.is_last)) return;    // nothing starts behind it
    const int z0 = z * TZ;

    const int nc = (w.s1 - w.s0 + L - 1) / L;
    const int rowx = tid / (DX / 8), dxo = tid % (DX / 8) * 8, rowz = tid / (TZ / 8), dzo = tid % (TZ / 8) * 8;
    constexpr int STEPX = THREADS / (DX / 8), STEPZ = THREADS / (TZ / 8);   // rows between a thread's pieces
    Source<IO, PB, STEPX, VEC> sb;
    Source<IO, PC, STEPZ, VEC> sc;
    Gates gates;
    gates.open(p, w.base, w.first, h);
    sb.open(r.b, w.base, w.first, h, L, rev, rowx, dxo, r.dx);
    sc.open(r.c, w.base, w.first, h, L, rev, rowz, z0 + dzo, r.dz);
    Piece<IO> rb[PB], rc[PC];
    Gates::Raw rg{};
    const auto fetch = [&](int c) {
        const int t0 = w.s0 + c * L, n = min(L, w.s1 - t0), token = rev ? t0 + n - L : t0;
        sb.load(rb, token, n, rev);
        sc.load(rc, token, n, rev);
        if (wave == 0) {
            // back along the tokens a row's decay is that of the token behind it, and none behind the last
            rg = rev ? gates.fetch(t0 + n - 63, 63 - lane, lane < n && t0 + n - lane < w.len) : gates.fetch(t0, lane, lane < n);
        }
    };
    if (nc > 0) fetch(rev ? nc - 1 : 0);

    // ---- the state that the segment starts from: rows 16 x + 4 quarter + i, column 16 wave + col of the tile
    f32x4 st[NX];
    const long long seg_at = (((long long)w.page * p.H + h) * r.tiles + z) * (DX * TZ) + (wave * 64 + lane) * 4;
    bool have = MODE == CHUNKS && (!w.is_first || r.init);
    if (MODE == CHUNKS && !w.is_first) {
#pragma unroll
        for (int x = 0; x < NX; ++x) st[x] = *reinterpret_cast<const f32x4*>(r.seg + seg_at + x * 1024);
    } else if (have) {
        const StatePage s(r.init + ((long long)w.n * p.H + h) * ((long long)r.dx * r.dz), r.sx, r.sz, r.dx, r.dz, 4 * quarter, z0 + 16 * wave + col);
#pragma unroll
        for (int x = 0; x < NX; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[x][i] = s.load(16 * x + i);
    } else {
#pragma unroll
        for (int x = 0; x < NX; ++x) st[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float* const anchors = MODE == CHUNKS ? r.anchors + (((long long)(w.chunk0 + w.s0 / L) * p.H + h) * r.tiles + z) * (DX * TZ) + (wave * 64 + lane) * 4 : nullptr;
    const long long anchor_step = (long long)p.H * r.tiles * (DX * TZ);
    float s_upd = r.s_upd;
    keep(s_upd);

    float seg_log = 0.f;                                  // (STATES: the segment's whole decay, from wave 0,
    unsigned long long forgets = 0;                       //  and whether a token of it keeps nothing)
    const auto put_decays = [&](typename S::Decays& d) {   // wave 0
        const float g = gates.widen(rg), end = chunk_decays<L>(d, g, lane);
        if (MODE == STATES) {
            seg_log += end;
            forgets |= __builtin_amdgcn_ballot_w64(g < LOWEST_DECAY);
        }
    };
    if (nc > 0 && wave == 0) put_decays(lds.d[0]);
    if (S::SCALED) lds_barrier();                         // (c is scaled with them)
    for (int ci = 0; ci < nc; ++ci) {
        // (what follows from the lane is worked out anew for each chunk: kept over the loop it fills the registers)
        int lane_ = lane;
        asm volatile("" : "+v"(lane_));
        const int quarter = lane_ >> 4, col = lane_ & 15;
        const int c = rev ? nc - 1 - ci : ci, t0 = w.s0 + c * L, n = min(L, w.s1 - t0);
        // ---- operands to the LDS
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            u32x4 t[NS];
            piece_terms<IO>(rb[i], t);
#pragma unroll
            for (int s = 0; s < NS; ++s) *reinterpret_cast<u32x4*>(&lds.b[s][rowx + STEPX * i][dxo]) = t[s];
        }
#pragma unroll
        for (int i = 0; i < PC; ++i) {
            const int row = rowz + STEPZ * i;
            if constexpr (S::SCALED) {
                const float f = lds.d[ci & 1].dk[row] * s_upd;
                float x8[8];
                widen_piece<IO>(rc[i], x8);
#pragma unroll
                for (int e = 0; e < 8; ++e) x8[e] *= f;
                bf16x8 t[3];
                split8<3, false>(x8, t);
#pragma unroll
                for (int s = 0; s < 3; ++s) *reinterpret_cast<bf16x8*>(&lds.c[s][row][dzo]) = t[s];
            } else {
                u32x4 t[NS];
                piece_terms<IO>(rc[i], t);
#pragma unroll
                for (int s = 0; s < NS; ++s) *reinterpret_cast<u32x4*>(&lds.c[s][row][dzo]) = t[s];
            }
        }
        lds_barrier();                                    // (orders the LDS alone: the next chunk's rows and what was stored stay on their way)
        if (ci + 1 < nc) fetch(rev ? c - 1 : c + 1);
        typename S::Decays& dec = lds.d[ci & 1];
        if (MODE == CHUNKS && have) {                     // (zeros in front of a first chunk are not kept)
#pragma unroll
            for (int x = 0; x < NX; ++x) *reinterpret_cast<f32x4*>(anchors + c * anchor_step + x * 1024) = st[x];
        }
        if (MODE == CHUNKS && ci + 1 == nc) break;         // (nothing starts behind it)
        // ---- the state behind the chunk
        const float ed = dec.end;
#pragma unroll
        for (int x = 0; x < NX; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[x][i] *= ed;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (32 * ks >= n) break;
            bf16x8 fv[3];
            if constexpr (S::SCALED) {
#pragma unroll
                for (int s = 0; s < 3; ++s) fv[s] = across8(&lds.c[s][32 * ks + 4 * quarter + (col >> 2)][16 * wave + 4 * (col & 3)], S::PZ);
            } else decayed_terms<IO>(lds.c, dec.dk, s_upd, ks, 16 * wave, quarter, col, fv);
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                bf16x8 fk[NS];
#pragma unroll
                for (int s = 0; s < NS; ++s) fk[s] = across8(&lds.b[s][32 * ks + 4 * quarter + (col >> 2)][16 * x + 4 * (col & 3)], S::PX);
                st[x] = mma<2>(st[x], fk, fv);
            }
        }
        have = true;
        if (wave == 0 && ci + 1 < nc) put_decays(lds.d[(ci + 1) & 1]);
        lds_barrier();
    }
    if constexpr (MODE == STATES) {
#pragma unroll
        for (int x = 0; x < NX; ++x) *reinterpret_cast<f32x4*>(r.seg + seg_at + x * 1024) = st[x];
        if (tid == 0 && z == 0) {
            const float d = fast_exp2(seg_log);
            r.seg_decay[(long long)w.page * p.H + h] = d == 0.f && forgets ? -0.f : d;    // (segments_kernel tells a product that is too small from one that is zero)
        }
        __shared__ int careful;
        if (tid == 0) careful = 0;
        float probe = 0.f;
#pragma unroll
        for (int x = 0; x < NX; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) probe = fmaf(st[x][i], 0.f, probe);
        lds_barrier();
        if (!(probe == 0.f)) careful = 1;
        lds_barrier();
        if (uniform(careful)) {
            static_assert(sizeof(CarefulTokens<DX>) <= sizeof(S), "");
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            careful_segment<IO, DX>(reinterpret_cast<CarefulTokens<DX>&>(lds), p, r, w, z, h);
        }
    }
}

// Outputs.  Eight waves of two kinds, which need nothing of each other between two barriers: four take the tokens' outputs (16 tokens each), four the state
// behind the chunk (16 columns each), its terms for the next one and the decays.  (Four waves that did one after the other: one image of 196 tokens 22 % longer; 2 x 4150 x 12
// fp32 8 %; 4 x 16384 x 12 fp16 4 %.)
template <typename IO, int DX, bool VEC>
__global__ __launch_bounds__(OUT_THREADS, (2 * out_workgroups<sizeof(Lds<IO, DX, PLAIN>)>)) void decay_kernel(const Params p) {
    using S = Lds<IO, DX, PLAIN>;
    constexpr int L = S::L, NS = S::NS, NT = L / 16, KX = DX / 32, KS = L / 32, NX = DX / 16;
    constexpr int PB = L * DX / 8 / 256, PC = L * TZ / 8 / 256;   // pieces of a thread of its kind
    static_assert(PB >= 1 && PC >= 1 && L * DX % 2048 == 0 && L * TZ % 2048 == 0, "");
    __shared__ S lds;
    __shared__ int offs[OUT_THREADS];
    const int tid = threadIdx.x & 255, lane = tid & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w4 = wave & 3;

    const Role& r = p.role[0];
    touch(p);
    touch(r);
    const int z = blockIdx.x & (r.tiles - 1), h = blockIdx.x >> (r.tiles - 1), gid = grid_segment();   // a head's tiles next to each other: they read the same rows
    if (gid >= p.segs) return;
    const Place w = find_place<OUT_THREADS>(p, gid, L, offs);
    if (!p.nseg) clear_outside<IO>(p, r, w.front, w.back, gid, z, h);
    if (!w.valid) return;
    const int z0 = z * TZ, nc = (w.s1 - w.s0 + L - 1) / L;
    const bool begun = !w.is_first || r.init;             // there is a state in front
    constexpr int STEPX = 256 / (DX / 8), STEPZ = 256 / (TZ / 8);   // rows between a thread's pieces
    float scale = p.scale;
    keep(scale);
    __shared__ Careful careful;                           // (a result that is not finite is heard of by way of the LDS alone: a barrier that waits for the results on their way took 0.4 us)
    careful_begin(careful);
    float probe = 0.f;                                    // NaN once a result was not finite

    if (wave < 4) {
        const int rowx = tid / (DX / 8), dxo = tid % (DX / 8) * 8, o0 = order_of(dxo);
        const int tw = w4 % NT, zt0 = w4 / NT * NT, t = 16 * tw + col;   // rows 16 tw + col, columns 16 (zt0 + j) + 4 quarter + i
        std::conditional_t<S::STAGED, Source<IO, PB, STEPX, VEC>, Fragments<IO, KX, VEC>> sa;
        Source<IO, PB, STEPX, VEC> sb;
        if constexpr (S::STAGED) sa.open(r.a, w.base, w.first, h, L, false, rowx, dxo, r.dx);
        else sa.open(r.a, w.base, w.first, h, t, quarter, r.dx);
        sb.open(r.b, w.base, w.first, h, L, false, rowx, dxo, r.dx);
        Piece<IO> ra[S::STAGED ? PB : KX], rb[PB];
        const auto fetch = [&](int c) {
            const int t0 = w.s0 + c * L, n = min(L, w.s1 - t0);
            sa.load(ra, t0, n, false);
            sb.load(rb, t0, n, false);
        };
        if (nc > 0) fetch(0);
        Sink<IO, VEC> so;
        so.open(r.o, w.base, w.first, h, t, z0 + 16 * zt0 + 4 * quarter, r.dz);
        for (int c = 0; c < nc; ++c) {
            // (what follows from the lane is worked out anew for each chunk: kept over the loop it fills the registers, masks for every tile among it)
            int lane_ = lane;
            asm volatile("" : "+v"(lane_));
            const int quarter = lane_ >> 4, col = lane_ & 15, t = 16 * tw + col;
            const int t0 = w.s0 + c * L, n = min(L, w.s1 - t0);
            const auto put = [&](const Piece<IO>& piece, __bf16 (&a)[NS][L][S::PX], int row) {
                u32x4 f[NS];
                piece_terms<IO>(piece, f);
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    *reinterpret_cast<uint2*>(&a[s][row][o0]) = uint2{f[s][0], f[s][1]};
                    *reinterpret_cast<uint2*>(&a[s][row][o0 + 8]) = uint2{f[s][2], f[s][3]};
                }
            };
            bf16x8 fa[KX][NS];
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                if constexpr (S::STAGED) put(ra[i], lds.a, rowx + STEPX * i);
                put(rb[i], lds.b, rowx + STEPX * i);
            }
            if constexpr (!S::STAGED) {
#pragma unroll
                for (int kx = 0; kx < KX; ++kx) {
                    u32x4 f[NS];
                    piece_terms<IO>(ra[kx], f);
#pragma unroll
                    for (int s = 0; s < NS; ++s) fa[kx][s] = __builtin_bit_cast(bf16x8, f[s]);
                }
            }
            lds_barrier();                                // (orders the LDS alone: the next chunk's rows and this one's results stay on their way)
            if (c + 1 < nc) fetch(c + 1);
            typename S::Decays& dec = lds.d[c & 1];
            f32x4 acc[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (16 * tw < n) {
                const float gth = dec.gh[t], gtl = dec.gl[t], from_state = dec.dt[t] * scale;
                if constexpr (S::STAGED) {
#pragma unroll
                    for (int kx = 0; kx < KX; ++kx)
#pragma unroll
                        for (int s = 0; s < NS; ++s) fa[kx][s] = *reinterpret_cast<const bf16x8*>(&lds.a[s][t][kx * 32 + 8 * quarter]);
                }
                // what the state in front gives
                if (begun || c > 0) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
#pragma unroll
                        for (int kx = 0; kx < KX; ++kx) {
                            bf16x8 fs[3];
#pragma unroll
                            for (int s = 0; s < 3; ++s) fs[s] = __builtin_bit_cast(bf16x8, lds.s[s][zt0 + j][kx][lane_]);
                            acc[j] = mma<2>(acc[j], fs, fa[kx]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[j][i] *= from_state;
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (2 * ks > tw) break;
                    float pr[8];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int ts = 2 * ks + half;     // tile of 16 tokens s
                        f32x4 m = {0.f, 0.f, 0.f, 0.f};
                        if (ts <= tw) {
#pragma unroll
                            for (int kx = 0; kx < KX; ++kx) {
                                bf16x8 fb[NS];
#pragma unroll
                                for (int s = 0; s < NS; ++s) fb[s] = *reinterpret_cast<const bf16x8*>(&lds.b[s][16 * ts + col][kx * 32 + 8 * quarter]);
                                m = mma<2>(m, fb, fa[kx]);
                            }
                            const f32x4 sh = *reinterpret_cast<const f32x4*>(&dec.gh[16 * ts + 4 * quarter]), sl = *reinterpret_cast<const f32x4*>(&dec.gl[16 * ts + 4 * quarter]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float x = m[i] * (scale * fast_exp2((gth - sh[i]) + (gtl - sl[i])));
                                m[i] = ts < tw || 4 * quarter + i <= col ? x : 0.f;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) pr[4 * half + i] = m[i];
                    }
                    bf16x8 fp[3];
                    split8<3>(pr, fp);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        bf16x8 fc[NS];
#pragma unroll
                        for (int s = 0; s < NS; ++s) fc[s] = across8(&lds.c[s][32 * ks + 4 * quarter + (col >> 2)][16 * (zt0 + j) + 4 * (col & 3)], S::PZ);
                        acc[j] = mma<2>(acc[j], fc, fp);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) probe = fmaf(acc[j][i], 0.f, probe);
            so.store(acc, t0, t < n);
            lds_barrier();
        }
    } else {
        const int rowz = tid / (TZ / 8), dzo = tid % (TZ / 8) * 8;
        constexpr int DECAYS = 7;                         // the wave that has the decays besides
        Source<IO, PC, STEPZ, VEC> sc;
        sc.open(r.c, w.base, w.first, h, L, false, rowz, z0 + dzo, r.dz);
        Gates gates;
        gates.open(p, w.base, w.first, h);
        Piece<IO> rc[PC];
        Gates::Raw rg{};
        const auto fetch = [&](int c) {
            const int t0 = w.s0 + c * L, n = min(L, w.s1 - t0);
            sc.load(rc, t0, n, false);
            if (wave == DECAYS) rg = gates.fetch(t0, lane, lane < n);
        };
        if (nc > 0) fetch(0);
        // the state: rows 16 x + 4 quarter + i, column 16 w4 + col of the tile
        f32x4 st[NX];
        const long long page = ((long long)w.n * p.H + h) * ((long long)r.dx * r.dz);
        const int zc = z0 + 16 * w4 + col;
        if (!w.is_first) {
#pragma unroll
            for (int x = 0; x < NX; ++x) st[x] = *reinterpret_cast<const f32x4*>(r.seg + (((long long)w.page * p.H + h) * r.tiles + z) * (DX * TZ) + ((x * 4 + w4) * 64 + lane) * 4);
        } else if (begun) {
            const StatePage s(r.init + page, r.sx, r.sz, r.dx, r.dz, 4 * quarter, zc);
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) st[x][i] = s.load(16 * x + i);
        } else {
#pragma unroll
            for (int x = 0; x < NX; ++x) st[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        u32x4 held[3][KX];                               // its terms
        const auto hold = [&]() {
#pragma unroll
            for (int kx = 0; kx < KX; ++kx) {
                const float x8[8] = {st[2 * kx][0], st[2 * kx][1], st[2 * kx][2], st[2 * kx][3], st[2 * kx + 1][0], st[2 * kx + 1][1], st[2 * kx + 1][2], st[2 * kx + 1][3]};
                bf16x8 f[3];
                split8<3>(x8, f);
#pragma unroll
                for (int s = 0; s < 3; ++s) held[s][kx] = __builtin_bit_cast(u32x4, f[s]);
            }
        };
        if (nc > 0) {
            if (wave == DECAYS) chunk_decays<L>(lds.d[0], gates.widen(rg), lane);
            hold();
        }
        const bool wanted = r.last && w.is_last;          // the state behind the segment
        for (int c = 0; c < nc; ++c) {
            int lane_ = lane;
            asm volatile("" : "+v"(lane_));
            const int quarter = lane_ >> 4, col = lane_ & 15;
            const int t0 = w.s0 + c * L, n = min(L, w.s1 - t0);
#pragma unroll
            for (int i = 0; i < PC; ++i) {
                u32x4 f[NS];
                piece_terms<IO>(rc[i], f);
#pragma unroll
                for (int s = 0; s < NS; ++s) *reinterpret_cast<u32x4*>(&lds.c[s][rowz + STEPZ * i][dzo]) = f[s];
            }
#pragma unroll
            for (int kx = 0; kx < KX; ++kx)
#pragma unroll
                for (int s = 0; s < 3; ++s) lds.s[s][w4][kx][lane_] = held[s][kx];
            lds_barrier();
            if (c + 1 < nc) fetch(c + 1);
            typename S::Decays& dec = lds.d[c & 1];
            if (c + 1 < nc || wanted) {
                const float ed = dec.end;
#pragma unroll
                for (int x = 0; x < NX; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) st[x][i] *= ed;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (32 * ks >= n) break;
                    bf16x8 fv[3];
                    decayed_terms<IO>(lds.c, dec.dk, 1.f, ks, 16 * w4, quarter, col, fv);
#pragma unroll
                    for (int x = 0; x < NX; ++x) {
                        bf16x8 fk[NS];
#pragma unroll
                        for (int s = 0; s < NS; ++s) fk[s] = across8(&lds.b[s][32 * ks + 4 * quarter + (col >> 2)][(x >> 1) * 32 + (x & 1) * 4 + 8 * (col & 3)], S::PX);
                        st[x] = mma<2>(st[x], fk, fv);
                    }
                }
                if (c + 1 < nc) {
                    hold();
                    if (wave == DECAYS) chunk_decays<L>(lds.d[(c + 1) & 1], gates.widen(rg), lane);
                }
            }
            lds_barrier();
        }
        if (wanted) {
            const StatePage s(r.last + page, r.sx, r.sz, r.dx, r.dz, 4 * quarter, zc);
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s.store(16 * x + i, st[x][i]);
                    probe = fmaf(st[x][i], 0.f, probe);
                }
        }
    }
    if (!(probe == 0.f)) careful.wanted = 1;
    lds_barrier();
    if (nc > 0 && uniform(careful.wanted)) {
        static_assert(sizeof(CarefulLds<DX>) <= sizeof(S), "");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // what has been stored arrives in front of what takes its place
        __syncthreads();
        careful_outputs<IO, DX, L>(careful, reinterpret_cast<CarefulLds<DX>&>(lds), offs);
    }
}

// How the host reaches the instances of each type.
template <typename IO> int launch_decay(const Params& p, int dx, int mode, bool vec, hipStream_t st);
extern template int launch_decay<float>(const Params&, int, int, bool, hipStream_t);
extern template int launch_decay<__hip_bfloat16>(const Params&, int, int, bool, hipStream_t);
extern template int launch_decay<__half>(const Params&, int, int, bool, hipStream_t);

template <typename IO, int DX, bool VEC>
void launch_mode(const Params& p, int mode, dim3 grid, hipStream_t st) {
    if (mode == PLAIN) hipLaunchKernelGGL((decay_kernel<IO, DX, VEC>), grid, dim3(OUT_THREADS), 0, st, p);
    else if (mode == CHUNKS) hipLaunchKernelGGL((decay_states_kernel<IO, DX, CHUNKS, VEC>), grid, dim3(THREADS), 0, st, p);
    else hipLaunchKernelGGL((decay_states_kernel<IO, DX, STATES, VEC>), grid, dim3(THREADS), 0, st, p);
}
// vec: every row of every role in pieces of 16 bytes
template <typename IO>
int launch_decay(const Params& p, int dx, int mode, bool vec, hipStream_t st) {
    const dim3 grid = decay_grid(p, p.role[0].tiles * p.n_roles);
    if (dx <= 64) vec ? launch_mode<IO, 64, true>(p, mode, grid, st) : launch_mode<IO, 64, false>(p, mode, grid, st);
    else vec ? launch_mode<IO, 128, true>(p, mode, grid, st) : launch_mode<IO, 128, false>(p, mode, grid, st);
    return check_launch("decay_attention");
}

}  // namespace decay
}  // namespace vrwkv
