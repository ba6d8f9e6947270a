// Filtered sampling from given random numbers, for gfx950: for each row of
// logits x[0, n) with temperature T, top-k, top-p, min-p and a number u in
// [0, 1),
//
//   w_i  = rint(2^40 exp((x_i - max) / T))    whole numbers
//   order: x falling, then index; kept: the first k of the order, of them the
//   fewest with p of their sum, of them those with w_i >= min_p 2^40
//   token: the first, in the order of the indices, whose running sum of kept
//   weights passes floor(u * their sum)
//
// T <= 0 (or NaN) takes the largest logit, the first of equals. NaN counts as
// -inf; a row of nothing else gives -1.
//
// Weights come from float64, so that they are the same to a unit in 2^40
// whoever computes them, and every sum of them is exact and the same in any
// order: results depend neither on how a row is cut nor on atomics' order.
//
// The cut. All filters keep a prefix of the order, so what is kept is x > xc,
// and the first q in index order of those with x = xc (and w >= min_p 2^40). A
// histogram of the weights over the distance log2(e) (max - x) / T, in bins of
// 1/16, finds the bin in which a count (k) or a sum (p) is reached; inside it
// histograms over the float's order bits, 1024 wide, narrow it down to the one
// value. Nothing is sorted, and equal logits, thousands in 16 bits, cost
// nothing extra.
//
// n <= 32768: a workgroup a row, its logits in registers, one launch
// (sample_row). Else slices of 8192 tokens, a workgroup each, in four:
//   slice_max   maximum and its index, clears the row's histogram;
//   slice_hist  weights into the row's histogram (or, without a cut, the sum
//               of the slice's kept weights);
//   slice_list  every workgroup finds the bin of the cut from the histogram
//               (the bins, where k and p leave more than one), sums its
//               weights above and lists its logits inside;
//   sample_pick a workgroup a row: the cut, each slice's kept sum, the slice
//               that holds the token, and the token in it.
// What bounds it: one read of the logits from HBM and up to two from the
// caches, and the float64 arithmetic of the weights (12 operations a token).
#include "ft_common.hpp"

#include <algorithm>
#include <climits>

namespace ft {
namespace {

typedef unsigned long long u64;

constexpr int kBins = 656;           // bins of weights that are not 0: log2 distances below 41
constexpr int kSlice = 8192;         // tokens
constexpr int kSliceNT = 256;
constexpr int kRowNT = 1024;
constexpr int kRowMost = 32768;      // tokens of a row that one workgroup holds
constexpr int kMaxVocab = 1 << 22;   // 512 slices; sums of weights below 2^62
constexpr int kLevel = 1024;         // bins of a histogram over order bits

struct SampleArgs {
    const void* x;
    long long ld;
    const float* u;
    const float* temp;  // null: temp_all, and so on
    const int* k;
    const float* p;
    const float* minp;
    float temp_all, p_all, minp_all;
    int k_all;
    long long* out;
    int rows, n, slices;
    // workspace of the sliced form
    float* top;        // [rows][slices]
    int* top_at;       // [rows][slices]
    u64* sum;          // [rows][slices]: kept weights above the cut's bins
    unsigned* listed;  // [rows][slices]
    u64* mass;         // [rows][kBins]
    unsigned* count;   // [rows][kBins]
    unsigned* list;    // [rows][n]: order bits, slice s from kSlice s on
};

// 2^(j / 64), j < 64, in LDS. The caller synchronises.
constexpr int kPowers = 64;
__device__ __forceinline__ void fill_powers(double* s) {
    if (threadIdx.x < kPowers) s[threadIdx.x] = exp2((double)threadIdx.x / kPowers);
}

// rint(2^(40 + t)), t <= 0: with n = rint(64 t), 2^t = 2^(n / 64) 2^f, |f| <=
// 1/128, the series of 2^f to f^4 (the next term is below 4e-14, 0.05 units of
// the largest weight; the exponential by its series alone, to f^11, took twice
// the registers and more time)
__device__ __forceinline__ u64 weight(const double* powers, double t) {
    if (!(t > -41.0)) return 0;
    const double n = rint(t * 64.0), f = fma(n, -1.0 / 64.0, t);
    double s = 9.61812910762847716e-3;   // ln(2)^4 / 24
    s = fma(s, f, 5.55041086648215800e-2);
    s = fma(s, f, 2.40226506959100712e-1);
    s = fma(s, f, 6.93147180559945309e-1);
    s = fma(s, f, 1.0);
    const int k = (int)n;
    // (the last bits of 2^40 2^t + 2^52 are its nearest whole number)
    const double v = ldexp(s * powers[k & 63], (k >> 6) + 40) + 4503599627370496.0;
    return (u64)__double_as_longlong(v) & 0xfffffffffffffull;
}

// A row's parameters, the same in every thread.
struct Row {
    double top, c;  // maximum; log2(e) / T
    double minw;    // least kept weight
    float p;
    int k;          // 0: none
    bool greedy;
    const double* powers;
    __device__ __forceinline__ Row(const SampleArgs& a, int r, float most, const double* s_powers)
        : powers(s_powers) {
        const float t = a.temp ? a.temp[r] : a.temp_all;
        greedy = !(t > 0.0f);
        top = (double)most;
        c = greedy ? 0.0 : 1.4426950408889634074 / (double)t;
        const float m = a.minp ? a.minp[r] : a.minp_all;
        minw = (double)fminf(m, 1.0f) * 1099511627776.0;
        p = a.p ? a.p[r] : a.p_all;
        k = a.k ? a.k[r] : a.k_all;
        if (k < 0 || k >= a.n) k = 0;
    }
    __device__ __forceinline__ bool cut() const { return k > 0 || p < 1.0f; }
    // log2 of the weight over the largest
    __device__ __forceinline__ double far(float x) const {
        return (double)x == top ? 0.0 : ((double)x - top) * c;
    }
    __device__ __forceinline__ u64 weight_at(double t) const { return weight(powers, t); }
    __device__ __forceinline__ u64 weight_of(float x) const { return weight(powers, far(x)); }
    __device__ __forceinline__ bool keeps(u64 w) const { return (double)w >= minw; }
};

__device__ __forceinline__ int bin_of(double t) {
    return t > -41.0 ? (int)(t * -16.0) : kBins;
}

// order bits: larger for larger x, equal for equal ones
__device__ __forceinline__ unsigned order_bits(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);  // -0 -> 0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_bits(unsigned o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

__device__ __forceinline__ u64 shfl64(u64 v, int lane) {
    const unsigned lo = __shfl((unsigned)v, lane, 64), hi = __shfl((unsigned)(v >> 32), lane, 64);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {  // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned lo = __shfl_up((unsigned)v, o, 64);
        const unsigned hi = __shfl_up((unsigned)(v >> 32), o, 64);
        if (lane >= o) v += (u64)hi << 32 | lo;
    }
    return v;
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const unsigned lo = __shfl_xor((unsigned)v, o, 64);
        const unsigned hi = __shfl_xor((unsigned)(v >> 32), o, 64);
        v += (u64)hi << 32 | lo;
    }
    return v;
}
// Exclusive prefix over the workgroup's threads and the total. s: LDS, 16
// words; the caller synchronises before it is used again.
template <int NT>
__device__ __forceinline__ u64 block_scan(u64 v, u64* s, u64& total) {
    const u64 in = wave_scan(v);
    if ((threadIdx.x & 63) == 63) s[threadIdx.x >> 6] = in;
    __syncthreads();
    u64 before = in - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const u64 x = s[w];
        if (w < (int)(threadIdx.x >> 6)) before += x;
        total += x;
    }
    return before;
}

// A thread's tokens: 4 in a row of every 4 NT, from `first` on, x = -inf
// where there is none. NaN becomes -inf.
template <typename T, int NT, int TPT>
__device__ __forceinline__ void load_tokens(const T* row, int first, int end, float (&x)[TPT]) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    const bool vec = ((uintptr_t)(row + first) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int j = 0; j < TPT / 4; ++j) {
        const int i = first + 4 * (j * NT + (int)threadIdx.x);
        v4 v;
        if (vec && i + 4 <= end) {
            v = *reinterpret_cast<const v4*>(row + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * j + e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[4 * j + e] = i + e < end ? (float)row[i + e] : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < TPT; ++j)
        if (!(x[j] >= -INFINITY)) x[j] = -INFINITY;
}

// Between two passes over the tokens: what the first worked out of them in
// float64 is not kept in registers for the second (it would not fit).
template <int TPT>
__device__ __forceinline__ void next_pass(float (&x)[TPT]) {
#pragma unroll
    for (int j = 0; j < TPT; ++j) asm volatile("" : "+v"(x[j]));
}
// In a pass: two tokens' weights at a time, not all at once.
__device__ __forceinline__ void next_pair(int j) {
    if (j & 1) __builtin_amdgcn_sched_barrier(0);
}

// The largest of the workgroup's tokens and its first index. s: 2 words a wave.
template <int NT, int TPT>
__device__ __forceinline__ float block_top(const float (&x)[TPT], int first, float* s, int* s_at,
                                           int& at) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < TPT; ++j) m = fmaxf(m, x[j]);
    m = wave_max(m);
    int i = INT_MAX;
#pragma unroll
    for (int j = TPT - 1; j >= 0; --j)
        if (x[j] == m) i = first + 4 * ((j / 4) * NT + (int)threadIdx.x) + j % 4;
#pragma unroll
    for (int o = 32; o; o >>= 1) i = min(i, __shfl_xor(i, o, 64));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m, s_at[threadIdx.x >> 6] = i;
    __syncthreads();
    float top = s[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) top = fmaxf(top, s[w]);
    at = INT_MAX;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w)
        if (s[w] == top) at = min(at, s_at[w]);
    return top;
}

// A histogram in LDS, bins from the largest values on.
struct Hist {
    u64* mass;
    unsigned* count;
};

// The last bin that is not empty and that a count or a sum of those before it
// has not reached: before < k, or (double)before < want; bin 0 if there is
// none.
struct Crossing {
    int bin;
    u64 mass;        // before it
    unsigned count;  // before it
};
struct CrossState {
    u64 scan[16], scan2[16];
    u64 mass;
    unsigned count;
    int bin;
};
__device__ __forceinline__ Crossing cross(const Hist& h, int bins, u64 mass0, u64 count0,
                                          bool by_count, u64 k, double want, CrossState& s) {
    const int b = threadIdx.x;  // a bin a thread
    const u64 m = b < bins ? h.mass[b] : 0;
    const unsigned c = b < bins ? h.count[b] : 0;
    u64 total;
    if (threadIdx.x == 0) s.bin = 0, s.mass = mass0, s.count = (unsigned)count0;
    const u64 mb = mass0 + block_scan<kRowNT>(m, s.scan, total);
    const u64 cb = count0 + block_scan<kRowNT>(c, s.scan2, total);
    const bool on = c > 0 && (by_count ? cb < k : (double)mb < want);
    if (on) atomicMax(&s.bin, b);
    __syncthreads();
    if (on && s.bin == b) s.mass = mb, s.count = (unsigned)cb;
    __syncthreads();
    const Crossing r{s.bin, s.mass, s.count};
    __syncthreads();
    return r;
}

// The one value at which the count or the sum is reached, among the order
// bits that `each` visits (each(f) calls f(bits, is one) in every thread):
// its bits, the mass and the count before it, and how many have it.
struct Group {
    unsigned bits, of;
    u64 mass, count;
};
template <typename Each>
__device__ __forceinline__ Group resolve(const Row& row, const Hist& h, u64 mass0, u64 count0,
                                         bool by_count, u64 k, double want, CrossState& s,
                                         unsigned* s_range, Each&& each) {
    // the range of the bits
    unsigned lo = ~0u, hi = 0;
    each([&](unsigned o, bool on) {
        if (on) lo = min(lo, o), hi = max(hi, o);
    });
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        lo = min(lo, (unsigned)__shfl_xor(lo, o, 64));
        hi = max(hi, (unsigned)__shfl_xor(hi, o, 64));
    }
    if (threadIdx.x == 0) s_range[0] = ~0u, s_range[1] = 0;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        atomicMin(&s_range[0], lo);
        atomicMax(&s_range[1], hi);
    }
    __syncthreads();
    lo = s_range[0], hi = s_range[1];
    for (;;) {
        const unsigned width = hi - lo;  // the last bit pattern that counts, from hi down
        int shift = 0;
        while ((width >> shift) >= kLevel) ++shift;
        h.mass[threadIdx.x] = 0;
        h.count[threadIdx.x] = 0;
        __syncthreads();
        each([&](unsigned o, bool on) {
            if (!on || o > hi || o < lo) return;
            const unsigned b = (hi - o) >> shift;
            atomicAdd(&h.mass[b], row.weight_of(from_bits(o)));
            atomicAdd(&h.count[b], 1u);
        });
        __syncthreads();
        const Crossing x = cross(h, kLevel, mass0, count0, by_count, k, want, s);
        mass0 = x.mass, count0 = x.count;
        hi -= (unsigned)x.bin << shift;
        if (shift == 0) {
            const Group g{hi, h.count[x.bin], mass0, count0};
            __syncthreads();
            return g;
        }
        const unsigned least = (1u << shift) - 1;
        lo = hi - lo > least ? hi - least : lo;
    }
}

// What is kept: x > xc, and the first q (by index) of those with x = xc (all
// that has weight: xc = -inf, q = 0).
struct Cut {
    float xc;
    u64 q, wc;  // wc: the weight of xc, 0 below min-p
};

// The first q of `of` equal weights w behind `mass` that p keeps: those with a
// sum before them below want.
__device__ __forceinline__ u64 first_below(u64 mass, u64 w, u64 of, double want) {
    const double d = w ? (want - (double)mass) / (double)w : (double)of;
    u64 q = d < 1.0 ? 1 : d >= (double)of ? of : (u64)d;
    while (q > 1 && !((double)(mass + (q - 1) * w) < want)) --q;
    while (q < of && (double)(mass + q * w) < want) ++q;
    return q;
}

// The cut from the histogram of the whole row's weights; each(f, bin) visits
// the order bits of a bin. total: the sum of all.
template <typename Each>
__device__ __forceinline__ Cut find_cut(const Row& row, const Hist& h, u64 total, unsigned tokens,
                                        CrossState& s, const Hist& level, unsigned* s_range,
                                        Each&& each) {
    Cut cut{-INFINITY, 0, 0};
    u64 sum = total;
    // (a k that all weights but zeros come up to cuts nothing)
    const bool by_k = row.k > 0 && (unsigned)row.k < tokens;
    for (int pass = by_k ? 0 : 1; pass < (row.p < 1.0f ? 2 : 1); ++pass) {
        const bool by_count = pass == 0;
        const double want = (double)row.p * (double)sum;
        const Crossing x = cross(h, kBins, 0, 0, by_count, row.k, want, s);
        const Group g = resolve(row, level, x.mass, x.count, by_count, row.k, want, s, s_range,
                                [&](auto&& f) { each(f, x.bin); });
        cut.xc = from_bits(g.bits);
        cut.wc = row.weight_of(cut.xc);
        cut.q = by_count ? (u64)row.k - g.count : first_below(g.mass, cut.wc, g.of, want);
        sum = g.mass + cut.q * cut.wc;
    }
    if (!row.keeps(cut.wc)) cut.wc = 0;
    return cut;
}

__device__ __forceinline__ u64 aim_at(float u, u64 total) {
    const double d = u > 0.0f ? (double)u * (double)total : 0.0;
    const u64 last = total - 1;
    return d >= (double)total ? last : min((u64)d, last);
}

// The first token of the workgroup's whose running sum of kept weights passes
// aim (~0: that of u of their whole sum). `q`: how many of the cut's equals
// may still be kept here.
struct PickState {
    u64 mass[kRowMost / 4096 * 16];
    unsigned ties[kRowMost / 4096 * 16];
    u64 base, q, aim;
    int entry;
    long long token;
};
template <int TPT>
__device__ __forceinline__ void pick(const Row& row, const Cut& cut, const float (&x)[TPT],
                                     int first, u64 q, u64 aim, float u, PickState& s,
                                     long long* out) {
    constexpr int J = TPT / 4, kWaves = kRowNT / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto kept = [&](float v) -> u64 {  // of those above the cut
        if (!(v > cut.xc)) return 0;
        const u64 w = row.weight_of(v);
        return row.keeps(w) ? w : 0;
    };
    auto tie = [&](float v) { return v == cut.xc; };
    // sums of every 256 tokens in a row: (chunk j, wave)
#pragma unroll
    for (int j = 0; j < J; ++j) {
        u64 m = 0;
        unsigned t = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m += kept(x[4 * j + e]);
            t += tie(x[4 * j + e]);
            next_pair(e);
        }
        m = wave_sum64(m);
#pragma unroll
        for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o, 64);
        if (lane == 0) s.mass[j * kWaves + wave] = m, s.ties[j * kWaves + wave] = t;
    }
    __syncthreads();
    if (wave == 0) {
        constexpr int N = J * kWaves, PER = (N + 63) / 64;
        u64 m[PER], t[PER], mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            t[i] = e < N ? s.ties[e] : 0;
            mine += t[i];
        }
        u64 before = wave_scan(mine) - mine;  // equals before the lane's entries
        u64 sum = 0, had[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            had[i] = before;
            const u64 left = q > before ? q - before : 0;
            m[i] = (e < N ? s.mass[e] : 0) + cut.wc * min(left, t[i]);
            before += t[i];
            sum += m[i];
        }
        const u64 in = wave_scan(sum), total = shfl64(in, 63);
        if (aim == ~0ull) aim = aim_at(u, total);
        u64 run = in - sum;
        const u64 hit = __builtin_amdgcn_ballot_w64(in > aim);
        if (hit && lane == __ffsll(hit) - 1) {
            bool done = false;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (!done && run + m[i] > aim) {
                    s.entry = lane * PER + i;
                    s.base = run;
                    s.q = q > had[i] ? q - had[i] : 0;
                    done = true;
                }
                run += m[i];
            }
        }
        if (!hit && lane == 0) s.entry = -1;
        if (lane == 0) s.aim = aim;
    }
    __syncthreads();
    const int entry = s.entry;
    if (entry < 0) {  // nothing has weight: not reached, the largest logit has
        if (threadIdx.x == 0) *out = -1;
        return;
    }
    if (entry % kWaves != wave) return;
    float v[4] = {};
#pragma unroll
    for (int j = 0; j < J; ++j)
        if (j == entry / kWaves)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[4 * j + e];
    unsigned t = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) t += tie(v[e]);
    u64 left = wave_scan(t) - t;
    left = s.q > left ? s.q - left : 0;
    u64 w[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        w[e] = kept(v[e]);
        if (tie(v[e]) && left) w[e] = cut.wc, --left;
        sum += w[e];
    }
    const u64 in = wave_scan(sum) + s.base;
    const u64 hit = __builtin_amdgcn_ballot_w64(in > s.aim);
    if (hit && lane == __ffsll(hit) - 1) {
        u64 run = in - sum;
        int at = 3;
#pragma unroll
        for (int e = 3; e >= 0; --e) {
            u64 upto = run;
#pragma unroll
            for (int f = 0; f < 4; ++f)
                if (f <= e) upto += w[f];
            if (upto > s.aim) at = e;
        }
        *out = (long long)first + 4 * ((entry / kWaves) * kRowNT + (int)threadIdx.x) + at;
    }
}

// ---------------------------------------------------------------------------
// a workgroup a row
// ---------------------------------------------------------------------------
template <typename T, int TPT>
__global__ __launch_bounds__(kRowNT) void sample_row(const SampleArgs a) {
    __shared__ double s_powers[kPowers];
    __shared__ float s_top[16];
    __shared__ int s_at[16];
    __shared__ u64 s_mass[kBins], s_level_mass[kLevel];
    __shared__ unsigned s_count[kBins], s_level_count[kLevel], s_range[2];
    __shared__ CrossState s_cross;
    __shared__ PickState s_pick;
    const int r = blockIdx.x;
    const T* const logits = (const T*)a.x + (long long)r * a.ld;
    float x[TPT];
    load_tokens<T, kRowNT, TPT>(logits, 0, a.n, x);
    fill_powers(s_powers);
    for (int b = threadIdx.x; b < kBins; b += kRowNT) s_mass[b] = 0, s_count[b] = 0;
    int at;
    const float top = block_top<kRowNT, TPT>(x, 0, s_top, s_at, at);
    const Row row(a, r, top, s_powers);
    if (row.greedy || top == -INFINITY) {
        if (threadIdx.x == 0) a.out[r] = top == -INFINITY ? -1 : at;
        return;
    }
    Cut cut{-INFINITY, 0, 0};
    if (row.cut()) {
        u64 mine = 0;
        unsigned some = 0;
#pragma unroll
        for (int j = 0; j < TPT; ++j) {
            const double t = row.far(x[j]);
            const int b = bin_of(t);
            next_pair(j);
            if (b >= kBins) continue;
            const u64 w = row.weight_at(t);
            mine += w;
            ++some;
            atomicAdd(&s_mass[b], w);
            atomicAdd(&s_count[b], 1u);
        }
        u64 total, tokens;
        block_scan<kRowNT>(mine, s_cross.scan, total);
        block_scan<kRowNT>(some, s_cross.scan2, tokens);
        __syncthreads();
        cut = find_cut(row, Hist{s_mass, s_count}, total, (unsigned)tokens, s_cross,
                       Hist{s_level_mass, s_level_count}, s_range, [&](auto&& f, int bin) {
                           next_pass(x);
#pragma unroll
                           for (int j = 0; j < TPT; ++j) {
                               f(order_bits(x[j]), bin_of(row.far(x[j])) == bin);
                               next_pair(j);
                           }
                       });
    }
    next_pass(x);
    pick<TPT>(row, cut, x, 0, cut.q, ~0ull, a.u[r], s_pick, a.out + r);
}

// ---------------------------------------------------------------------------
// slices
// ---------------------------------------------------------------------------
constexpr int kSliceTPT = kSlice / kSliceNT;

template <typename T>
__global__ __launch_bounds__(kSliceNT) void slice_max(const SampleArgs a) {
    __shared__ float s_top[4];
    __shared__ int s_at[4];
    const int r = blockIdx.x / a.slices, s = blockIdx.x - r * a.slices;
    const int lo = s * kSlice, hi = min(lo + kSlice, a.n);
    float x[kSliceTPT];
    load_tokens<T, kSliceNT, kSliceTPT>((const T*)a.x + (long long)r * a.ld, lo, hi, x);
    // the slice's share of the row's histogram
    for (int b = s * kSliceNT + threadIdx.x; b < kBins; b += a.slices * kSliceNT) {
        a.mass[(size_t)r * kBins + b] = 0;
        a.count[(size_t)r * kBins + b] = 0;
    }
    int at;
    const float top = block_top<kSliceNT, kSliceTPT>(x, lo, s_top, s_at, at);
    if (threadIdx.x == 0) {
        a.top[blockIdx.x] = top;
        a.top_at[blockIdx.x] = at;
    }
}

// The row's maximum from its slices', in every lane.
__device__ __forceinline__ float row_top(const SampleArgs& a, int r) {
    float m = -INFINITY;
    for (int s = threadIdx.x & 63; s < a.slices; s += 64)
        m = fmaxf(m, a.top[(size_t)r * a.slices + s]);
    return wave_max(m);
}

template <typename T>
__global__ __launch_bounds__(kSliceNT) void slice_hist(const SampleArgs a) {
    __shared__ double s_powers[kPowers];
    __shared__ u64 s_mass[kBins];
    __shared__ unsigned s_count[kBins];
    __shared__ u64 s_sum[4];
    const int r = blockIdx.x / a.slices, s = blockIdx.x - r * a.slices;
    const int lo = s * kSlice, hi = min(lo + kSlice, a.n);
    float x[kSliceTPT];
    load_tokens<T, kSliceNT, kSliceTPT>((const T*)a.x + (long long)r * a.ld, lo, hi, x);
    fill_powers(s_powers);
    for (int b = threadIdx.x; b < kBins; b += kSliceNT) s_mass[b] = 0, s_count[b] = 0;
    __syncthreads();
    const float top = row_top(a, r);
    const Row row(a, r, top, s_powers);
    if (row.greedy || top == -INFINITY) return;
    if (!row.cut()) {
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < kSliceTPT; ++j) {
            const u64 w = row.weight_of(x[j]);
            if (row.keeps(w)) sum += w;
            next_pair(j);
        }
        sum = wave_sum64(sum);
        if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0) a.sum[blockIdx.x] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        return;
    }
#pragma unroll
    for (int j = 0; j < kSliceTPT; ++j) {
        const double t = row.far(x[j]);
        const int b = bin_of(t);
        next_pair(j);
        if (b >= kBins) continue;
        atomicAdd(&s_mass[b], row.weight_at(t));
        atomicAdd(&s_count[b], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kSliceNT)
        if (s_count[b]) {
            atomicAdd(&a.mass[(size_t)r * kBins + b], s_mass[b]);
            atomicAdd(&a.count[(size_t)r * kBins + b], s_count[b]);
        }
}

// The bins that the cut can be in: [lo, hi], and k's own. Sums are exact but
// for the part of bin `at_k` that k keeps, so p's want lies between two.
struct Span {
    int lo, hi, at_k;  // at_k: -1 none
};
__device__ __forceinline__ Span cut_span(const Row& row, const Hist& h, u64* s_scan, u64* s_scan2,
                                         int* s_bin) {
    constexpr int PER = (kBins + kSliceNT - 1) / kSliceNT;
    u64 m[PER], mine = 0, many = 0, total, tokens;
    unsigned c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = threadIdx.x * PER + i;
        m[i] = b < kBins ? h.mass[b] : 0;
        c[i] = b < kBins ? h.count[b] : 0;
        mine += m[i];
        many += c[i];
    }
    if (threadIdx.x < 3) s_bin[threadIdx.x] = 0;
    u64 mb = block_scan<kSliceNT>(mine, s_scan, total);
    u64 cb = block_scan<kSliceNT>(many, s_scan2, tokens);
    __shared__ u64 s_w[2];
    if (threadIdx.x == 0) s_w[0] = s_w[1] = total;
    const bool by_k = row.k > 0 && (u64)row.k < tokens;
    if (by_k) {
        u64 q = cb;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (c[i] && q < (u64)row.k) atomicMax(&s_bin[2], threadIdx.x * PER + i);
            q += c[i];
        }
    }
    __syncthreads();
    if (by_k) {
        u64 q = mb;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (threadIdx.x * PER + i == s_bin[2]) s_w[0] = q, s_w[1] = q + m[i];
            q += m[i];
        }
    }
    __syncthreads();
    if (row.p < 1.0f) {
        const double w0 = (double)row.p * (double)s_w[0], w1 = (double)row.p * (double)s_w[1];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (c[i] && (double)mb < w0) atomicMax(&s_bin[0], threadIdx.x * PER + i);
            if (c[i] && (double)mb < w1) atomicMax(&s_bin[1], threadIdx.x * PER + i);
            mb += m[i];
        }
    }
    __syncthreads();
    Span x{s_bin[0], s_bin[1], by_k ? s_bin[2] : -1};
    if (!(row.p < 1.0f)) {
        // k alone; where k cuts nothing either, all is kept
        x.lo = by_k ? x.at_k : kBins;
        x.hi = x.lo;
    }
    return x;
}

template <typename T>
__global__ __launch_bounds__(kSliceNT) void slice_list(const SampleArgs a) {
    __shared__ double s_powers[kPowers];
    __shared__ u64 s_scan[4], s_scan2[4], s_sum[4];
    __shared__ int s_bin[3];
    __shared__ unsigned s_n;
    const int r = blockIdx.x / a.slices, s = blockIdx.x - r * a.slices;
    const int lo = s * kSlice, hi = min(lo + kSlice, a.n);
    const float top = row_top(a, r);
    const Row row(a, r, top, s_powers);
    if (row.greedy || top == -INFINITY || !row.cut()) return;
    float x[kSliceTPT];
    load_tokens<T, kSliceNT, kSliceTPT>((const T*)a.x + (long long)r * a.ld, lo, hi, x);
    if (threadIdx.x == 0) s_n = 0;
    fill_powers(s_powers);
    const Span span = cut_span(row, Hist{a.mass + (size_t)r * kBins, a.count + (size_t)r * kBins},
                               s_scan, s_scan2, s_bin);
    u64 sum = 0;
    unsigned* const list = a.list + (size_t)r * a.n + lo;
#pragma unroll
    for (int j = 0; j < kSliceTPT; ++j) {
        const double t = row.far(x[j]);
        const int b = bin_of(t);
        if (b >= kBins) continue;
        if (b < span.lo) {
            const u64 w = row.weight_at(t);
            if (row.keeps(w)) sum += w;
        }
        if ((b >= span.lo && b <= span.hi) || b == span.at_k)
            list[atomicAdd(&s_n, 1u)] = order_bits(x[j]);
    }
    sum = wave_sum64(sum);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        a.sum[blockIdx.x] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        a.listed[blockIdx.x] = s_n;
    }
}

template <typename T>
__global__ __launch_bounds__(kRowNT) void sample_pick(const SampleArgs a) {
    __shared__ double s_powers[kPowers];
    __shared__ u64 s_mass[kBins], s_level_mass[kLevel];
    __shared__ unsigned s_count[kBins], s_level_count[kLevel], s_range[2];
    __shared__ CrossState s_cross;
    __shared__ PickState s_pick;
    __shared__ u64 s_base, s_q;
    __shared__ int s_slice;
    const int r = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float top = row_top(a, r);
    const Row row(a, r, top, s_powers);
    fill_powers(s_powers);
    if (row.greedy || top == -INFINITY) {
        if (wave == 0) {
            int at = INT_MAX;
            for (int s = lane; s < a.slices; s += 64)
                if (a.top[(size_t)r * a.slices + s] == top)
                    at = min(at, a.top_at[(size_t)r * a.slices + s]);
#pragma unroll
            for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
            if (lane == 0) a.out[r] = top == -INFINITY ? -1 : at;
        }
        return;
    }
    const size_t row0 = (size_t)r * a.slices;
    Cut cut{-INFINITY, 0, 0};
    // a slice a thread: kept weights above the cut, and the cut's equals
    u64* const s_sum = s_level_mass;          // (after the cut is found)
    unsigned* const s_ties = s_level_count;
    if (row.cut()) {
        u64 m = 0, c = 0, total, tokens;
        const int b = threadIdx.x;
        if (b < kBins) {
            s_mass[b] = m = a.mass[(size_t)r * kBins + b];
            s_count[b] = c = a.count[(size_t)r * kBins + b];
        }
        block_scan<kRowNT>(m, s_cross.scan, total);
        block_scan<kRowNT>(c, s_cross.scan2, tokens);
        __syncthreads();
        // slice s is wave s % 16's
        cut = find_cut(row, Hist{s_mass, s_count}, total, (unsigned)tokens, s_cross,
                       Hist{s_level_mass, s_level_count}, s_range, [&](auto&& f, int bin) {
                           for (int s = wave; s < a.slices; s += kRowNT / 64) {
                               const unsigned* const list = a.list + (size_t)r * a.n + s * kSlice;
                               const int n = a.listed[row0 + s];
                               for (int i = lane; i < n; i += 64) {
                                   const unsigned o = list[i];
                                   f(o, bin_of(row.far(from_bits(o))) == bin);
                               }
                           }
                       });
        for (int s = wave; s < a.slices; s += kRowNT / 64) {
            u64 sum = 0;
            unsigned ties = 0;
            if (cut.xc > -INFINITY) {
                const unsigned* const list = a.list + (size_t)r * a.n + s * kSlice;
                const int n = a.listed[row0 + s];
                for (int i = lane; i < n; i += 64) {
                    const float v = from_bits(list[i]);
                    if (v > cut.xc) {
                        const u64 w = row.weight_of(v);
                        if (row.keeps(w)) sum += w;
                    }
                    ties += v == cut.xc;
                }
                sum = wave_sum64(sum);
#pragma unroll
                for (int o = 32; o; o >>= 1) ties += __shfl_xor(ties, o, 64);
            }
            if (lane == 0) s_sum[s] = sum + a.sum[row0 + s], s_ties[s] = ties;
        }
    } else {
        for (int s = threadIdx.x; s < a.slices; s += kRowNT)
            s_sum[s] = a.sum[row0 + s], s_ties[s] = 0;
    }
    if (threadIdx.x == 0) s_slice = 0, s_base = 0, s_q = cut.q;
    __syncthreads();
    const int s = threadIdx.x;
    u64 total;
    const u64 ties = s < a.slices ? s_ties[s] : 0;
    const u64 had = block_scan<kRowNT>(ties, s_cross.scan, total);
    const u64 left = cut.q > had ? cut.q - had : 0;
    const u64 mine = s < a.slices ? s_sum[s] + cut.wc * min(left, ties) : 0;
    const u64 before = block_scan<kRowNT>(mine, s_cross.scan2, total);
    const u64 aim = aim_at(a.u[r], total);
    if (before <= aim && aim < before + mine) s_slice = s, s_base = before, s_q = left;
    __syncthreads();
    const int lo = s_slice * kSlice;
    float x[kSlice / kRowNT];
    load_tokens<T, kRowNT, kSlice / kRowNT>((const T*)a.x + (long long)r * a.ld, lo,
                                            min(lo + kSlice, a.n), x);
    pick<kSlice / kRowNT>(row, cut, x, lo, s_q, aim - s_base, 0.f, s_pick, a.out + r);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct SampleShape {
    int slices;  // 0: a workgroup a row
    size_t top, top_at, sum, listed, mass, count, list, bytes;
};

SampleShape sample_shape(int rows, int n) {
    if (rows < 0) inval("sample_filtered_batched: rows must be >= 0");
    if (n < 1) inval("sample of empty logits");
    if (n > kMaxVocab) inval("sample_filtered_batched: at most 2^22 logits a row");
    SampleShape s{};
    if (n <= kRowMost || rows == 0) return s;
    s.slices = (n + kSlice - 1) / kSlice;
    const size_t parts = (size_t)rows * s.slices;
    if (parts > INT_MAX) inval("sample_filtered_batched: too many rows for one call");
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t p = at;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    s.top = take(4 * parts);
    s.top_at = take(4 * parts);
    s.sum = take(8 * parts);
    s.listed = take(4 * parts);
    s.mass = take(8 * (size_t)rows * kBins);
    s.count = take(4 * (size_t)rows * kBins);
    s.list = take(4 * (size_t)rows * n);
    s.bytes = at;
    return s;
}

template <typename T>
void sample_run(const SampleArgs& a, hipStream_t s) {
    if (!a.slices) {
        if (a.n <= 4096) sample_row<T, 4><<<a.rows, kRowNT, 0, s>>>(a);
        else if (a.n <= 8192) sample_row<T, 8><<<a.rows, kRowNT, 0, s>>>(a);
        else if (a.n <= 16384) sample_row<T, 16><<<a.rows, kRowNT, 0, s>>>(a);
        else sample_row<T, 32><<<a.rows, kRowNT, 0, s>>>(a);
        launch_check("sample_filtered_batched kernel launch");
        return;
    }
    const unsigned grid = (unsigned)a.rows * (unsigned)a.slices;
    slice_max<T><<<grid, kSliceNT, 0, s>>>(a);
    slice_hist<T><<<grid, kSliceNT, 0, s>>>(a);
    slice_list<T><<<grid, kSliceNT, 0, s>>>(a);
    sample_pick<T><<<a.rows, kRowNT, 0, s>>>(a);
    launch_check("sample_filtered_batched kernel launch");
}

}  // namespace
}  // namespace ft

using namespace ft;

extern "C" {

int ft_sample_filtered_batched_workspace(int rows, int n, long long* bytes) {
    return guarded([&] {
        if (!bytes) inval("sample_filtered_batched: null operand");
        *bytes = (long long)sample_shape(rows, n).bytes;
    });
}

int ft_sample_filtered_batched_launch(const void* logits, int dtype, long long ld, int rows, int n,
                                      const float* uniforms, const float* temperatures,
                                      float temperature, const int* top_ks, int top_k,
                                      const float* top_ps, float top_p, const float* min_ps,
                                      float min_p, long long* tokens, void* workspace,
                                      long long workspace_bytes, uintptr_t stream) {
    return guarded([&] {
        if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
            inval("sample_filtered_batched: unknown element type");
        const SampleShape sh = sample_shape(rows, n);
        if (!temperatures && !(temperature >= 0.0f)) inval("temperature must be >= 0");
        if (!top_ks && top_k < 0) inval("top_k must be >= 0");
        if (!top_ps && !(top_p > 0.0f && top_p <= 1.0f)) inval("top_p must be in (0, 1]");
        if (!min_ps && !(min_p >= 0.0f && min_p <= 1.0f)) inval("min_p must be in [0, 1]");
        if (rows == 0) return;
        if (rows > 1 && ld < n) inval("sample_filtered_batched: row stride too small");
        if (!logits || !uniforms || !tokens) inval("sample_filtered_batched: null operand");
        if ((uintptr_t)workspace & 15)
            inval("sample_filtered_batched: the workspace must be aligned to 16 bytes");
        if (sh.bytes && (!workspace || workspace_bytes < (long long)sh.bytes))
            inval("sample_filtered_batched: this call needs " + std::to_string(sh.bytes) +
                  " bytes of workspace");
        char* const ws = (char*)workspace;
        SampleArgs a{};
        a.x = logits;
        a.ld = ld;
        a.u = uniforms;
        a.temp = temperatures;
        a.k = top_ks;
        a.p = top_ps;
        a.minp = min_ps;
        a.temp_all = temperature;
        a.k_all = top_k;
        a.p_all = top_p;
        a.minp_all = min_p;
        a.out = tokens;
        a.rows = rows;
        a.n = n;
        a.slices = sh.slices;
        a.top = (float*)(ws + sh.top);
        a.top_at = (int*)(ws + sh.top_at);
        a.sum = (u64*)(ws + sh.sum);
        a.listed = (unsigned*)(ws + sh.listed);
        a.mass = (u64*)(ws + sh.mass);
        a.count = (unsigned*)(ws + sh.count);
        a.list = (unsigned*)(ws + sh.list);
        const hipStream_t s = as_stream(stream);
        if (dtype == FT_DT_F32) sample_run<float>(a, s);
        else if (dtype == FT_DT_BF16) sample_run<bf16>(a, s);
        else sample_run<f16>(a, s);
    });
}

}  // extern "C"
