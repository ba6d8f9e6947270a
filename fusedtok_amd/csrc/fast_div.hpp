// Division by a size known at launch.
#pragma once

#include <hip/hip_runtime.h>

namespace ft {
namespace {

// Division by a size known at launch, n / d for 0 <= n < 2^31: with l =
// ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1, n / d = (mulhi(m, n) + n)
// >> l (Granlund and Montgomery 1994). Three instructions for the ~25 of a
// 32-bit division.
struct FastDiv {
    unsigned d, m, l;
    FastDiv() = default;
    explicit FastDiv(int by) : d((unsigned)by), m(0), l(0) {
        while ((1ull << l) < d) ++l;
        m = (unsigned)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const {
        return (int)((__umulhi(m, (unsigned)n) + (unsigned)n) >> l);
    }
    __device__ __forceinline__ int up(int n) const {  // ceil(n / d), n <= 2^30
        return div(n + (int)d - 1);
    }
    __device__ __forceinline__ int mod(int n) const { return n - div(n) * (int)d; }
};

}  // namespace
}  // namespace ft
