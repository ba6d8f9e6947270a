// The stream split of decode attention: all (sequence, kv head) token rows laid
// end to end, b-major, and cut into equal segments (attention.hip, cache8.hip).
#pragma once

#include <climits>

#include "ft_common.hpp"

namespace ft {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Device-resident lengths are not read back by the host. A length outside
// [0, span] (span = the cache's row capacity) is clamped into it, so no
// value can make a kernel index past the cache or the block table.
__device__ __forceinline__ int clamp_len(const int* lens, int b, int span) {
    if (!lens) return span;
    return min(max(lens[b], 0), span);
}

constexpr int kStreamScanRows = 2048;        // sequences per launch (LDS prefix)

// Exclusive prefix of the clamped lengths into s_pref[0..batch] (wave 0;
// each lane takes a contiguous run of rows, then a wave scan of the runs),
// and their minimum and maximum into s_mm[0], s_mm[1].
__device__ __forceinline__ void scan_lengths(const int* __restrict__ lens,
                                             int batch, int span, int lane,
                                             long long* s_pref, int* s_mm) {
    const int per = (batch + 63) / 64;
    const int r0 = lane * per;
    long long local = 0;
    int lmin = INT_MAX, lmax = 0;
    for (int i = 0; i < per; ++i)
        if (r0 + i < batch) {
            const int l = clamp_len(lens, r0 + i, span);
            local += l;
            lmin = min(lmin, l);
            lmax = max(lmax, l);
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lmin = min(lmin, __shfl_xor(lmin, o, 64));
        lmax = max(lmax, __shfl_xor(lmax, o, 64));
    }
    if (lane == 0) {
        s_mm[0] = lmin;
        s_mm[1] = lmax;
    }
    long long incl = local;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long y = __shfl_up(incl, o, 64);
        if (lane >= o) incl += y;
    }
    long long run = incl - local;
    for (int i = 0; i < per; ++i)
        if (r0 + i < batch) {
            s_pref[r0 + i] = run;
            run += clamp_len(lens, r0 + i, span);
        }
    if (lane == 63) s_pref[batch] = incl;
}

// A value every lane holds identically, moved to scalar registers (the
// compiler cannot prove that values read from LDS are wave-uniform).
__device__ __forceinline__ long long uniform64(long long x) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)x);
    const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)((unsigned long long)x >> 32));
    return (long long)(((unsigned long long)hi << 32) | lo);
}

// A flat position's place: row (b, kv) and the tokens [t0, t0 + n) of it
// that lie before seg_hi. Everything is wave-uniform.
struct StreamPiece {
    int b, kv, row, t0, n;
    bool whole;       // the row's every token
    long long next;   // the flat position behind the piece
};

__device__ __forceinline__ StreamPiece stream_piece(const long long* s_pref, int batch, int hkv,
                                                    long long pos, long long seg_hi) {
    int lo = 0, hi = batch - 1;  // last sequence starting at or before pos
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (uniform64(s_pref[mid]) * hkv <= pos) lo = mid; else hi = mid - 1;
    }
    StreamPiece p;
    p.b = lo;
    const long long pb = uniform64(s_pref[lo]);
    const long long base = pb * hkv;
    const int len = (int)(uniform64(s_pref[lo + 1]) - pb);
    p.kv = (int)((pos - base) / len);
    p.t0 = (int)(pos - base - (long long)p.kv * len);
    p.next = min(seg_hi, base + (long long)(p.kv + 1) * len);
    p.n = (int)(p.next - pos);
    p.whole = p.t0 == 0 && p.n == len;
    p.row = lo * hkv + p.kv;
    return p;
}

}  // namespace
}  // namespace ft
