// What the decode attention kernels have in common (attention.hip, cache8.hip).
#pragma once

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

// A value every lane holds identically, moved to scalar registers (the
// compiler cannot prove that values read from LDS are wave-uniform).
__device__ __forceinline__ long long uniform64(long long x) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)x);
    const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)((unsigned long long)x >> 32));
    return (long long)(((unsigned long long)hi << 32) | lo);
}

}  // namespace
}  // namespace ft
