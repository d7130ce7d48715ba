#pragma once
#include "vrwkv_common.h"

namespace vrwkv {

// The sequences of a batch of token rows: row b of the batch whole, or with offsets (N + 1 of 32 or 64 bits, ascending) N of them packed in one row of T tokens,
// n at tokens offsets[n] to offsets[n + 1].  Offsets outside 0 .. T are taken as 0 or T, so that no token outside the rows is named whatever they hold, and a Walk's n is one of the N where begin and end
// are tokens.  Where they do not ascend, begin may lie behind the token that a sequence was found for, or end in front of begin: who counts from one of them into a page of states checks that.
struct Sequences {
    const void* offsets;
    int is64, N, T;
    __device__ __forceinline__ int of_lane(int i) const {
        const long long v = is64 ? static_cast<const long long*>(offsets)[i] : (long long)static_cast<const int*>(offsets)[i];
        return (int)(v < 0 ? 0 : v > T ? T : v);
    }
    // (the same i in all lanes)
    __device__ __forceinline__ int at(int i) const { return __builtin_amdgcn_readfirstlane(of_lane(i)); }
    // The first sequence that ends behind token t, N if there is none, and its tokens [begin, end): 64 offsets at a time, by all lanes of a wave together.
    __device__ __forceinline__ int first_ending_behind(int t, int lane, int& begin, int& end) const {
        int lo = 0, hi = N;                               // the answer is in lo .. hi
        while (hi - lo > WAVE) {
            const int step = (hi - lo + WAVE - 1) / WAVE, i = lo + (lane + 1) * step - 1;   // the last of each piece
            const bool before = i < hi && of_lane(i + 1) <= t;
            const int pieces = __popcll(__ballot(before));
            lo = min(lo + pieces * step, hi);
            hi = min(lo + step - 1, hi);
        }
        lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
        const int i = min(lo + lane, N - 1), from = of_lane(i), to = of_lane(i + 1);   // (the answer's offsets with those that it is found by)
        const int passed = __popcll(__ballot(lo + lane < hi && to <= t)), n = lo + passed;
        begin = n < N ? passed < WAVE ? __builtin_amdgcn_readlane(from, passed) : at(n) : 0x7fffffff;
        end = n < N ? passed < WAVE ? __builtin_amdgcn_readlane(to, passed) : at(n + 1) : 0x7fffffff;
        return n;
    }
    // The tokens [from, to) of [r0, r1) that belong to a sequence.
    __device__ __forceinline__ void inside(int r0, int r1, int& from, int& to) const {
        from = offsets ? max(r0, at(0)) : r0;
        to = offsets ? min(r1, at(N)) : r1;
    }
};

// The sequence that a walk along the tokens of batch row b is in: number n, tokens [begin, end).
struct Walk {
    int n, begin, end;
    __device__ __forceinline__ void read(const Sequences& s) {
        begin = n >= 0 && n < s.N ? s.at(n) : 0x7fffffff;
        end = n >= 0 && n < s.N ? s.at(n + 1) : 0x7fffffff;
    }
    // the one that token t is in (none: one without tokens, perhaps)
    __device__ __forceinline__ void find(const Sequences& s, int b, int t, int lane) {
        if (!s.offsets) {
            n = b, begin = 0, end = s.T;
            return;
        }
        n = s.first_ending_behind(t, lane, begin, end);
    }
    __device__ __forceinline__ void next(const Sequences& s) {
        const int done = end;
        if (!s.offsets) n = s.N;
        else
            for (++n; n < s.N && s.at(n + 1) <= done; ++n) {}
        read(s);
    }
    __device__ __forceinline__ void previous(const Sequences& s) {
        if (!s.offsets) n = -1;
        else
            for (--n; n >= 0 && s.at(n) >= s.at(n + 1); --n) {}
        read(s);
    }
    // whether none begins or ends in [row, row + count)
    __device__ __forceinline__ bool within(int row, int count) const { return (begin < row || begin >= row + count) && (end <= row || end > row + count); }
};

}  // namespace vrwkv
