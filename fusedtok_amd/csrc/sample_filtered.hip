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
// order: results depend neither on how a row is cut nor on atomics' order. The
// products p * sum and u * sum are float64, as are the sums that p * sum is
// compared with.
//
// The cut. All filters keep a prefix of the order, so what is kept is x > xc,
// and the first q in index order of those with x = xc (and w >= min_p 2^40). A
// histogram of the weights over the distance log2(e) (max - x) / T, in bins of
// 1/16, finds the bin in which a count (k) or a sum (p) is reached; inside it
// histograms over the float's order bits, 512 wide, narrow it down to the one
// value. Nothing is sorted, and equal logits, thousands in 16 bits, cost
// nothing extra.
//
// The floor. With k, the k-th largest of the largest logits of 256 parts of the
// row is a bound that the first k are not below, whatever lies in the parts.
// Below it neither histogram nor list need a logit, and the weights of few are
// worked out (2 rows of 32000, k = 40: 4.4 us for the histogram, 11.7 without).
//
// n <= 32768: a workgroup a row, its logits in LDS, one launch (sample_row).
// Above that they do not fit beside the rest; slices of 8192 tokens, a workgroup
// each, in four launches:
//   slice_max   maximum and its index, the parts' maxima, clears the row's
//               histogram;
//   slice_hist  weights into the slice's histogram and the row's (or, without
//               a cut, the sum of the slice's kept weights);
//   slice_list  every workgroup finds the bin of the cut from the row's
//               histogram (the bins, where k and p leave more than one, and
//               those of min-p), sums its own bins above and lists its logits
//               inside;
//   sample_pick a workgroup a row: the cut, each slice's kept sum, the slice
//               that holds the token, and the token in it.
//
// What bounds it. One read of the logits from HBM and two from the caches: 64
// rows of 128256 float32 (32.8 MB, a quarter of them without k) 5.5 + 13.7 +
// 11.8 + 20 us, 52-54 a call, the reads at 5.1 TB/s 6.4; 301 of 50257 bf16, p
// alone, 8 + 24 + 16.5 + 26, 70 a call. slice_hist without a floor waits for the LDS
// (a table's word and an atomic a token) and float64 (10 operations a token),
// slice_list for the row's bins, sample_pick and sample_row (2 x 32000: 21.9 us)
// for their 30 steps, one behind the other, with a barrier between each: 1024
// threads instead of 512 took 25 and 46 us for sample_pick's 21 and 27. Without k
// sample_row has every token's two atomics in one histogram besides (64 x 32000,
// p alone: 43 us a call, 24.5 with k = 50).
#include "ft_common.hpp"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace ft {
namespace {

typedef unsigned long long u64;

constexpr int kBins = 657;           // bins of weights that are not 0: log2 distances below 41
constexpr int kSlice = 8192;         // tokens
constexpr int kSliceNT = 256;
constexpr int kRowNT = 512;
constexpr int kRowMost = 32768;      // tokens of a row that one workgroup holds in LDS
constexpr int kMaxVocab = 1 << 22;   // 512 slices; sums of weights below 2^62
constexpr int kMinBins = 3;
constexpr int kGroups = 16;          // parts of a slice
constexpr int kFloorOf = 256;        // parts of a row whose largest logits give its floor
constexpr int kLevel = kRowNT;         // bins of a histogram over order bits

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
    float* groups;     // [rows][slices][kGroups]: the largest of each part of a slice
    float* floors;     // [rows]: below it none of the first k
    u64* sum;          // [rows][slices]: kept weights above the listed bins
    u64* part;         // [rows][slices][kBins]: the slices' histograms
    unsigned* listed;  // [rows][slices]
    u64* mass;         // [rows][kBins]
    unsigned* count;   // [rows][kBins]
    unsigned* list;    // [rows][n]: order bits, slice s from kSlice s on
};

// 2^(j / 64), and 2^40 times it in LDS (the caller synchronises).
constexpr int kPowers = 64;
__device__ const double kPowerTable[kPowers] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};
__device__ __forceinline__ void fill_powers(double* s) {
    if (threadIdx.x < kPowers) s[threadIdx.x] = 1099511627776.0 * kPowerTable[threadIdx.x];
}

// Distances t are in 1/64 of log2, 0 or less; from kFar on a weight is 0.
constexpr double kFar = -41.0 * kPowers;
// (the high words of numbers below 2624 in magnitude are below its own)
__device__ __forceinline__ bool near(double t) {
    return ((unsigned)(__double_as_longlong(t) >> 32) & 0x7fffffffu) < 0x40a48000u;
}
static_assert(kFar == -2624.0, "near's constant");
// t to the nearest whole number, as an int and as a double: its last bits
// after the addition (a conversion and a rounding take four times as long)
constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
__device__ __forceinline__ int nearest(double t) { return (int)__double_as_longlong(t + kRound); }

// rint(2^(40 + t / 64)): with n the nearest to t, 2^(t / 64) = 2^(n / 64) 2^(f / 64),
// |f| <= 1/2, the series of 2^(f / 64) to f^4 (the next term is below 4e-14, 0.05
// units of the largest weight; the exponential by its series alone, to the
// 11th power, took twice the registers and more time)
// (weight_near: of a t that is not much below kFar, where it is 0)
__device__ __forceinline__ u64 weight_near(const double* powers, double t) {
    const int k = nearest(t);
    const double f = t - ((t + kRound) - kRound);
    double s = 5.732851688640402e-10;  // (ln(2) / 64)^4 / 24
    s = fma(s, f, 2.1173137155464774e-07);
    s = fma(s, f, 5.864904955056169e-05);
    s = fma(s, f, 1.0830424696249145e-02);
    s = fma(s, f, 1.0);
    // 2^(40 + n / 64): the power's exponent moved, in its high word; then the
    // last bits of its product + 2^52 are the nearest whole number
    const double power = powers[k & 63];
    const double p = __hiloint2double(__double2hiint(power) + ((k << 14) & (int)0xfff00000),
                                      __double2loint(power));
    const double v = fma(s, p, 4503599627370496.0);
    return (u64)__double_as_longlong(v) & 0xfffffffffffffull;
}
__device__ __forceinline__ u64 weight(const double* powers, double t) {
    const u64 w = weight_near(powers, t);
    return near(t) ? w : 0;
}

// A row's parameters, the same in every thread.
struct Row {
    double top, c;  // maximum; 64 log2(e) / T
    u64 minw;       // least kept weight
    float p, minp;
    int k;          // 0: none
    bool greedy, infinite;
    const double* powers;
    __device__ __forceinline__ Row(const SampleArgs& a, int r, float most, const double* s_powers)
        : powers(s_powers) {
        const float t = a.temp ? a.temp[r] : a.temp_all;
        greedy = !(t > 0.0f);
        // (the same in every lane: a branch on it costs a token nothing)
        const int bits = __builtin_amdgcn_readfirstlane(__float_as_int(most));
        top = (double)__int_as_float(bits);
        infinite = bits == 0x7f800000;
        c = greedy ? 0.0 : 92.332482616893658 / (double)t;
        minp = a.minp ? a.minp[r] : a.minp_all;
        minp = minp < 1.0f ? fmaxf(minp, 0.0f) : 1.0f;  // (NaN: 1)
        minw = (u64)ceil((double)minp * 1099511627776.0);
        p = a.p ? a.p[r] : a.p_all;
        k = a.k ? a.k[r] : a.k_all;
        // (the first token alone: a limit of 0 would never be open)
        if (p <= 0.0f) k = 1, p = 1.0f;
        if (k < 0 || k >= a.n) k = 0;
    }
    __device__ __forceinline__ bool cut() const { return k > 0 || p < 1.0f; }
    // 64 log2 of the weight over the largest (infinite ones share the mass)
    __device__ __forceinline__ double far(float x) const {
        if (infinite) return x == INFINITY ? 0.0 : 2.0 * kFar;
        return finite_far(x);
    }
    __device__ __forceinline__ double finite_far(float x) const { return ((double)x - top) * c; }
    // the first of the kMinBins bins that may hold weights on both sides of
    // min-p: those before it are kept, those behind them not
    __device__ __forceinline__ int least_bin() const {
        return minp > 0.0f ? max((int)(-16.0f * log2f(minp)) - 1, 0) : kBins;
    }
    // floats that no logit of bin b lies outside of (a NaN: no bound)
    __device__ __forceinline__ float2 around(int b) const {
        const double lo = top - (4.0 * b + 3.75) / c, hi = top - (4.0 * b - 0.75) / c;
        const double room = 1e-12 * (fabs(top) + fabs(lo));
        const float f = (float)(lo - room), g = (float)(hi + room);
        return make_float2(f - (fabsf(f) * 0x1p-22f + 0x1p-126f),
                           g + (fabsf(g) * 0x1p-22f + 0x1p-126f));
    }
    // no logit of bin b or one before it lies below it, nor below floor
    __device__ __forceinline__ float least_of(int b, float floor) const {
        return fmaxf(around(b).x, floor);  // (of a NaN: the other)
    }
    __device__ __forceinline__ u64 weight_of(float x) const { return weight(powers, far(x)); }
    __device__ __forceinline__ bool keeps(u64 w) const { return w >= minw; }
};

// the bin, 1/16 of log2 wide; kBins and more: none (with weights of 0 the last
// bin ends a little behind kFar)
constexpr double kFarthest = -65536.0;
__device__ __forceinline__ int bin_near(double t) { return -nearest(t) >> 2; }  // t > kFarthest
__device__ __forceinline__ int bin_of(double t) { return t > kFarthest ? bin_near(t) : kBins; }

// order bits: larger for larger x, equal for equal ones
__device__ __forceinline__ unsigned order_bits(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);  // -0 -> 0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_bits(unsigned o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// v of the lane that a DPP control names, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 lane64(u64 v, int lane) {  // the same in every lane
    const unsigned lo = __builtin_amdgcn_readlane((int)v, lane);
    const unsigned hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (u64)hi << 32 | lo;
}
// Inclusive prefix over a wave: shifts by 1, 2, 4 and 8 in rows of 16, then
// the last lane of a row to the next, of a half to the other.
__device__ __forceinline__ u64 wave_scan(u64 v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ u64 wave_sum64(u64 v) { return lane64(wave_scan(v), 63); }
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

// A bound that the k-th largest logit is not below: of kFloorOf parts' largest
// ones, 4 a lane (`parts` of them: the rest is -inf), the k-th, to 16 bits of
// its order bits. Where there are fewer than k, the least finite value. What
// lies below is none of the first k, or has no weight: neither the histogram
// nor the list needs it.
__device__ __forceinline__ float floor_of(float4 g, int k, int parts) {
    if (k <= 0 || k > parts) return -FLT_MAX;
    const unsigned o[4] = {order_bits(g.x), order_bits(g.y), order_bits(g.z), order_bits(g.w)};
    unsigned at = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const unsigned next = at | 1u << bit;
        int many = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) many += __popcll(__builtin_amdgcn_ballot_w64(o[i] >= next));
        if (many >= k) at = next;
    }
    return at > order_bits(-FLT_MAX) ? from_bits(at) : -FLT_MAX;
}

// Two at once. s: 32 words.
template <int NT>
__device__ __forceinline__ void block_scan2(u64& v, u64& w, u64* s, u64& all_v, u64& all_w) {
    const u64 in_v = wave_scan(v), in_w = wave_scan(w);
    if ((threadIdx.x & 63) == 63) {
        s[threadIdx.x >> 6] = in_v;
        s[16 + (threadIdx.x >> 6)] = in_w;
    }
    __syncthreads();
    v = in_v - v, w = in_w - w;
    all_v = all_w = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        const u64 x = s[i], y = s[16 + i];
        if (i < (int)(threadIdx.x >> 6)) v += x, w += y;
        all_v += x, all_w += y;
    }
}

// A thread's tokens: 4 in a row of every 4 NT, from `first` on, x = -inf
// where there is none; NaN stays, every comparison with it is false. All loads
// are unconditional and converted behind the last one: a conversion in a branch
// waits there for its load (301 rows of 50257 bf16: slice_max 11 us so).
template <typename T, int NT, int TPT>
__device__ __forceinline__ void load_tokens(const T* row, int first, int end, float (&x)[TPT]) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    const T* const p = row + first;
    const int len = end - first, mine = 4 * (int)threadIdx.x;
    v4 v[TPT / 4];
    if (len >= 4 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0) {
        const int whole = len & ~3;
#pragma unroll
        for (int j = 0; j < TPT / 4; ++j)
            v[j] = *reinterpret_cast<const v4*>(p + min(4 * j * NT + mine, whole - 4));
#pragma unroll
        for (int j = 0; j < TPT / 4; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[4 * j + e] = 4 * j * NT + mine < whole ? (float)v[j][e] : -INFINITY;
        }
        if (whole < len) {  // the last one to three
            float rest[3];
#pragma unroll
            for (int e = 0; e < 3; ++e) rest[e] = whole + e < len ? (float)p[whole + e] : -INFINITY;
#pragma unroll
            for (int j = 0; j < TPT / 4; ++j)
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (4 * j * NT + mine == whole) x[4 * j + e] = rest[e];
        }
    } else {
#pragma unroll
        for (int j = 0; j < TPT / 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = p[min(4 * j * NT + mine + e, len - 1)];
#pragma unroll
        for (int j = 0; j < TPT / 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[4 * j + e] = 4 * j * NT + mine + e < len ? (float)v[j][e] : -INFINITY;
    }
}

// The largest of the workgroup's tokens and its first index, and of each 16
// threads. s: 2 words a wave.
template <int NT, int TPT>
__device__ __forceinline__ float block_top(const float (&x)[TPT], int first, float* s, int* s_at,
                                           float* groups, int& at) {
    static_assert(NT == 16 * kGroups, "parts of 16 threads");
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < TPT; ++j) m = fmaxf(m, x[j]);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 15) == 0) groups[threadIdx.x >> 4] = m;
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
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

// ---------------------------------------------------------------------------
// What a row's workgroup holds in LDS.
// ---------------------------------------------------------------------------
constexpr int kFew = kRowNT / 8;  // logits that are ranked by comparing all with all
constexpr int kFirst = 512;       // logits above a floor that are listed
constexpr int kWaves = kRowNT / 64;
constexpr int kChunk = 4 * kRowNT;  // tokens of a pass of the workgroup

struct Group {  // the logits of one value: bits, how many, mass and count before
    unsigned bits, of;
    u64 mass, count;
};
struct RowState {
    double powers[kPowers];
    // the histogram, bins from the largest values on; then (scan_bins) the sums
    // before each bin
    u64 mass[kBins + 1];
    unsigned count[kBins + 1];
    u64 level_mass[kLevel];
    unsigned level_count[kLevel];
    unsigned first[kFirst], firsts;  // sample_row's logits above a floor
    u64 few_w[kFew];
    unsigned few_key[kFew];
    u64 scan[32];
    u64 chunk_mass[kRowMost / kChunk * kWaves];
    unsigned chunk_ties[kRowMost / kChunk * kWaves];
    Group group;
    u64 base, q, aim, before_mass;
    unsigned few, best, before_count;
    int bin, level_bin, entry, slice;
    float top[kWaves];
    int top_at[kWaves];
    __attribute__((aligned(16))) float parts[kFloorOf];
};

// The tokens [first, end) of a row into s_x, up to a whole chunk (-inf behind
// the end), at most MOST of them. Returns their largest and,
// in `at`, its first index; PARTS: and leaves the parts' largest.
template <typename T, int MOST, bool PARTS>
__device__ __forceinline__ float stage_tokens(const T* row, int first, int end, float* s_x,
                                              RowState& s, int& at) {
    float x[MOST / kRowNT];
    load_tokens<T, kRowNT, MOST / kRowNT>(row, first, end, x);
    float m = -INFINITY;
    at = INT_MAX;
#pragma unroll
    for (int j = 0; j < MOST / kChunk; ++j) {
        const int i = 4 * (j * kRowNT + (int)threadIdx.x);
        if (first + j * kChunk < end)
            *reinterpret_cast<float4*>(s_x + i) =
                make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (x[4 * j + e] > m) m = x[4 * j + e], at = first + i + e;
    }
    const float mine = m;
    if (PARTS) {
        constexpr int LANES = kRowNT / kFloorOf;
        float part = m;
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) part = fmaxf(part, __shfl_xor(part, o, 64));
        if (threadIdx.x % LANES == 0) s.parts[threadIdx.x / LANES] = part;
    }
    m = wave_max(m);
    if (mine != m) at = INT_MAX;
#pragma unroll
    for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    if ((threadIdx.x & 63) == 0) s.top[threadIdx.x >> 6] = m, s.top_at[threadIdx.x >> 6] = at;
    __syncthreads();
    float top = s.top[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s.top[w]);
    at = INT_MAX;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        if (s.top[w] == top) at = min(at, s.top_at[w]);
    return top;
}

// The histogram becomes the sums before each bin; returns the whole sum, the
// tokens of it are count[kBins].
__device__ __forceinline__ u64 scan_bins(RowState& s) {
    constexpr int PER = (kBins + kRowNT - 1) / kRowNT;
    u64 m[PER], c[PER], mass = 0, count = 0, total, tokens;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = threadIdx.x * PER + i;
        m[i] = b < kBins ? s.mass[b] : 0;
        c[i] = b < kBins ? s.count[b] : 0;
        mass += m[i];
        count += c[i];
    }
    block_scan2<kRowNT>(mass, count, s.scan, total, tokens);
    u64 mb = mass, cb = count;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = threadIdx.x * PER + i;
        if (b < kBins) s.mass[b] = mb, s.count[b] = (unsigned)cb;
        mb += m[i];
        cb += c[i];
    }
    if (threadIdx.x == 0) s.mass[kBins] = total, s.count[kBins] = (unsigned)tokens;
    __syncthreads();
    return total;
}

// A threshold in the order: a count or a sum (of weights before) to be reached.
struct Limit {
    bool by_count;
    u64 k;
    double want;
    __device__ __forceinline__ bool open(u64 mass, u64 count) const {
        return by_count ? count < k : (double)mass < want;
    }
    // open before a bin and not behind it: one bin, as both sums rise
    __device__ __forceinline__ bool closes(u64 mass, u64 count, u64 mass1, u64 count1) const {
        return open(mass, count) && !open(mass1, count1);
    }
};

// The bin in which the limit is reached. Every limit is open at 0 (k >= 1; p > 0, so
// want > 0) and not behind all weights (k is at most their count; p < 1), so it
// is one bin, here and in the narrower histograms of that bin.
__device__ __forceinline__ int limit_bin(const Limit& l, RowState& s) {
    if (threadIdx.x == 0) s.bin = 0;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kRowNT)
        if (l.closes(s.mass[b], s.count[b], s.mass[b + 1], s.count[b + 1])) s.bin = b;
    __syncthreads();
    return s.bin;
}

// The one value at which the limit is reached, among the n order bits that
// `each` visits (each(f) calls f(bits, one) in every thread, one() telling
// whether they are of them), with mass0 and count0 before them, all in [lo, hi]. Few are compared all with all, 8
// threads each; more are narrowed down by histograms, 512 wide, first.
template <typename Each>
__device__ __forceinline__ Group resolve(const Row& row, const Limit& l, unsigned n, u64 mass0,
                                         u64 count0, unsigned lo, unsigned hi, RowState& s,
                                         Each&& each) {
    while (n > kFew) {
        int shift = 0;
        while (((hi - lo) >> shift) >= kLevel) ++shift;
        s.level_mass[threadIdx.x] = 0;
        s.level_count[threadIdx.x] = 0;
        // (a word of its own: s.bin may still be read by the waves behind)
        if (threadIdx.x == 0) s.level_bin = 0;
        __syncthreads();
        each([&](unsigned o, auto&& one) {
            if (o > hi || o < lo || !one()) return;
            const unsigned b = (hi - o) >> shift;
            atomicAdd(&s.level_mass[b], row.weight_of(from_bits(o)));
            atomicAdd(&s.level_count[b], 1u);
        });
        __syncthreads();
        const unsigned c = s.level_count[threadIdx.x];
        const u64 m = s.level_mass[threadIdx.x];
        u64 mb = m, cb = c, total, tokens;
        block_scan2<kRowNT>(mb, cb, s.scan, total, tokens);
        mb += mass0, cb += count0;
        if (l.closes(mb, cb, mb + m, cb + c)) s.level_bin = threadIdx.x;
        __syncthreads();
        const int bin = s.level_bin;
        if (threadIdx.x == bin) s.before_mass = mb, s.before_count = (unsigned)cb, s.few = c;
        __syncthreads();
        mass0 = s.before_mass, count0 = s.before_count, n = s.few;
        hi -= (unsigned)bin << shift;
        const unsigned span = (1u << shift) - 1;
        lo = hi - lo > span ? hi - span : lo;
        __syncthreads();
        if (shift == 0) return Group{hi, n, mass0, count0};  // one value
    }
    if (threadIdx.x == 0) s.few = 0, s.best = 0;
    __syncthreads();
    each([&](unsigned o, auto&& one) {
        if (o > hi || o < lo || !one()) return;
        s.few_key[atomicAdd(&s.few, 1u)] = o;
    });
    __syncthreads();
    // (weights after: a wave goes through a loop's body for each lane's find)
    if (threadIdx.x < n) s.few_w[threadIdx.x] = row.weight_of(from_bits(s.few_key[threadIdx.x]));
    __syncthreads();
    const unsigned mine = threadIdx.x >> 3;
    const unsigned key = mine < n ? s.few_key[mine] : 0;
    u64 m = 0;
    unsigned c = 0, of = 0;
    if (mine < n)
        for (unsigned i = threadIdx.x & 7; i < n; i += 8) {
            const unsigned o = s.few_key[i];
            if (o > key) m += s.few_w[i], ++c;
            of += o == key;
        }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const unsigned a = __shfl_xor((unsigned)m, o, 64), b = __shfl_xor((unsigned)(m >> 32), o, 64);
        m += (u64)b << 32 | a;
        c += __shfl_xor(c, o, 64);
        of += __shfl_xor(of, o, 64);
    }
    const bool first = (threadIdx.x & 7) == 0 && mine < n;
    if (first && l.open(mass0 + m, count0 + c)) atomicMax(&s.best, c + 1);
    __syncthreads();
    const unsigned best = s.best ? s.best - 1 : 0;
    if (first && c == best) s.group = Group{key, of, mass0 + m, count0 + c};
    __syncthreads();
    const Group g = s.group;
    __syncthreads();
    return g;
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

// The cut from the scanned histogram of the whole row's weights, `total` their
// sum; each(f, bin) visits the order bits of a bin.
template <typename Each>
__device__ __forceinline__ Cut find_cut(const Row& row, u64 total, RowState& s, Each&& each) {
    Cut cut{-INFINITY, 0, 0};
    u64 sum = total;
    // (a k beyond all weights that are not 0 cuts nothing)
    const bool by_k = row.k > 0 && (unsigned)row.k <= s.count[kBins];
    for (int pass = by_k ? 0 : 1; pass < (row.p < 1.0f ? 2 : 1); ++pass) {
        const Limit l{pass == 0, (u64)row.k, (double)row.p * (double)sum};
        const int bin = limit_bin(l, s);
        const float2 about = row.around(bin);
        const Group g = resolve(row, l, s.count[bin + 1] - s.count[bin], s.mass[bin], s.count[bin],
                                about.x >= -INFINITY ? order_bits(about.x) : 0,
                                about.y <= INFINITY ? order_bits(about.y) : ~0u, s,
                                [&](auto&& f) { each(f, bin); });
        cut.xc = from_bits(g.bits);
        cut.wc = row.weight_of(cut.xc);
        cut.q = l.by_count ? (u64)row.k - g.count : first_below(g.mass, cut.wc, g.of, l.want);
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

// The first of the staged tokens (n of them, `first` the first one's index)
// whose running sum of kept weights passes aim (~0: that of u of their whole
// sum). q: how many of the cut's equals may still be kept here.
__device__ __forceinline__ void pick(const Row& row, const Cut& cut, const float* s_x, int n,
                                     int first, u64 q, u64 aim, float u, RowState& s,
                                     long long* out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunks = (n + kChunk - 1) / kChunk;
    auto kept = [&](float v) -> u64 {  // of those above the cut (no branch: four at once)
        const u64 w = row.weight_of(v);
        return v > cut.xc && row.keeps(w) ? w : 0;
    };
    auto tie = [&](float v) { return v == cut.xc; };
    // sums of every 256 tokens in a row: (chunk j, wave)
    for (int j = 0; j < chunks; ++j) {
        const float4 x = *reinterpret_cast<const float4*>(s_x + 4 * (j * kRowNT + threadIdx.x));
        const float most = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
        if (!__builtin_amdgcn_ballot_w64(most >= cut.xc)) {  // nothing is kept here
            if (lane == 0) s.chunk_mass[j * kWaves + wave] = 0, s.chunk_ties[j * kWaves + wave] = 0;
            continue;
        }
        u64 m = kept(x.x) + kept(x.y) + kept(x.z) + kept(x.w);
        unsigned t = tie(x.x) + tie(x.y) + tie(x.z) + tie(x.w);
        if (__builtin_amdgcn_ballot_w64(m | t)) {
            // (in one word: 256 weights are at most 2^48)
            const u64 both = wave_sum64(m | (u64)t << 52);
            m = both & ((1ull << 52) - 1);
            t = (unsigned)(both >> 52);
        }
        if (lane == 0) s.chunk_mass[j * kWaves + wave] = m, s.chunk_ties[j * kWaves + wave] = t;
    }
    __syncthreads();
    if (wave == 0) {
        constexpr int PER = kRowMost / kChunk * kWaves / 64;
        const int entries = chunks * kWaves;
        u64 m[PER], t[PER], had[PER], mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            t[i] = e < entries ? s.chunk_ties[e] : 0;
            mine += t[i];
        }
        u64 before = wave_scan(mine) - mine, sum = 0;  // equals before the lane's entries
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            had[i] = before;
            const u64 left = q > before ? q - before : 0;
            m[i] = (e < entries ? s.chunk_mass[e] : 0) + cut.wc * min(left, t[i]);
            before += t[i];
            sum += m[i];
        }
        const u64 in = wave_scan(sum), total = lane64(in, 63);
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
    const int at = 4 * ((entry / kWaves) * kRowNT + (int)threadIdx.x);
    const float4 x = *reinterpret_cast<const float4*>(s_x + at);
    const float v[4] = {x.x, x.y, x.z, x.w};
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
        int e = 0;
#pragma unroll
        for (int f = 0; f < 3; ++f) {
            run += w[f];
            if (run <= s.aim) e = f + 1;
        }
        *out = (long long)first + at + e;
    }
}

// ---------------------------------------------------------------------------
// a workgroup a row, its logits in LDS
// ---------------------------------------------------------------------------
template <typename T, int MOST>
__global__ __launch_bounds__(kRowNT) void sample_row(const SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    RowState& s = *reinterpret_cast<RowState*>(smem);
    float* const s_x = reinterpret_cast<float*>(smem + ((sizeof(RowState) + 15) & ~(size_t)15));
    const int r = blockIdx.x;
    for (int b = threadIdx.x; b < kBins; b += kRowNT) s.mass[b] = 0, s.count[b] = 0;
    fill_powers(s.powers);
    if (threadIdx.x == 0) s.firsts = 0;
    int at;
    const float top = stage_tokens<T, MOST, true>((const T*)a.x + (long long)r * a.ld, 0, a.n, s_x, s, at);
    const Row row(a, r, top, s.powers);
    if (row.greedy || top == -INFINITY) {
        if (threadIdx.x == 0) a.out[r] = top == -INFINITY ? -1 : at;
        return;
    }
    const int chunks = (a.n + kChunk - 1) / kChunk;
    Cut cut{-INFINITY, 0, 0};
    if (row.cut()) {
        const float floor =
            floor_of(*reinterpret_cast<const float4*>(s.parts + 4 * (threadIdx.x & 63)), row.k,
                     kFloorOf);
        const float near_floor = row.least_of(kBins - 1, floor);
        const bool few = floor > -FLT_MAX;
        for (int j = 0; j < chunks; ++j) {
            const float4 x = *reinterpret_cast<const float4*>(s_x + 4 * (j * kRowNT + threadIdx.x));
            const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!(v[e] >= near_floor)) continue;
                const double t = row.far(v[e]);
                const int b = min(bin_of(t), kBins);  // (kBins: nobody's)
                atomicAdd(&s.mass[b], weight(s.powers, t));
                atomicAdd(&s.count[b], 1u);
                if (few) {
                    const unsigned i = atomicAdd(&s.firsts, 1u);
                    if (i < kFirst) s.first[i] = order_bits(v[e]);
                }
            }
        }
        __syncthreads();
        // (a floor's finds are looked through again, not the row)
        const unsigned firsts = few ? s.firsts : kFirst + 1;
        const u64 total = scan_bins(s);
        cut = find_cut(row, total, s, [&](auto&& f, int bin) {
            if (firsts <= kFirst) {
                for (unsigned i = threadIdx.x; i < firsts; i += kRowNT) {
                    const unsigned o = s.first[i];
                    f(o, [&] { return bin_of(row.far(from_bits(o))) == bin; });
                }
                return;
            }
            const float2 about = row.around(bin);
            const float least = row.least_of(bin, floor);
            const float* const x0 = s_x + 4 * threadIdx.x;
            u64 some = 0;  // the thread's tokens about the bin
#pragma unroll 4
            for (int j = 0; j < chunks; ++j) {
                const float4 x = *reinterpret_cast<const float4*>(x0 + j * kChunk);
                const float v[4] = {x.x, x.y, x.z, x.w};
                unsigned in = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    in |= v[e] >= least && !(v[e] > about.y) ? 1u << e : 0;
                some |= (u64)in << (4 * j);
            }
            for (; some; some &= some - 1) {
                const int j = __ffsll(some) - 1;
                const float v = x0[(j >> 2) * kChunk + (j & 3)];
                f(order_bits(v), [&] { return bin_of(row.far(v)) == bin; });
            }
        });
    }
    pick(row, cut, s_x, a.n, 0, cut.q, ~0ull, a.u[r], s, a.out + r);
}

// ---------------------------------------------------------------------------
// slices
// ---------------------------------------------------------------------------
constexpr int kSliceTPT = kSlice / kSliceNT;

// f(token, its place j) for a thread's tokens of a slice (-inf behind its end),
// AHEAD loads under way: all loads first left every workgroup of a CU loading
// and then computing at the same time. A load is unconditional and its values
// are touched only when their turn comes, so nothing waits for it before: whole
// slices of aligned rows 4 tokens at once, others one by one, the last one again
// behind the end.
template <typename T, int AHEAD>
struct Tokens {
    typedef T v4 __attribute__((ext_vector_type(4)));
    static constexpr int kSteps = kSliceTPT / 4;
    const T* row;
    int lo, hi;
    bool whole;
    v4 x[AHEAD];
    template <bool WHOLE>
    __device__ __forceinline__ v4 load(int j) const {
        const int i = lo + 4 * (j * kSliceNT + (int)threadIdx.x);
        if (WHOLE) return *reinterpret_cast<const v4*>(row + i);
        v4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = row[min(i + e, hi - 1)];
        return v;
    }
    __device__ __forceinline__ Tokens(const SampleArgs& a, int r, int first, int end)
        : row((const T*)a.x + (long long)r * a.ld), lo(first), hi(end),
          whole(first + kSlice <= end && ((uintptr_t)(row + first) & (4 * sizeof(T) - 1)) == 0) {
        if (whole) start<true>();
        else start<false>();
    }
    template <bool WHOLE>
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) x[j] = load<WHOLE>(j);
    }
    template <bool WHOLE, typename F>
    __device__ __forceinline__ void run(F&& f) {
#pragma unroll 1
        for (int j0 = 0; j0 < kSteps; j0 += AHEAD)
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int j = 4 * (j0 + q), i = lo + j * kSliceNT + 4 * (int)threadIdx.x;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    f(WHOLE || i + e < hi ? (float)x[q][e] : -INFINITY, j + e);
                if (j0 + AHEAD < kSteps) x[q] = load<WHOLE>(j0 + AHEAD + q);
            }
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) {
        if (whole) run<true>(f);
        else run<false>(f);
    }
};

// (8 waves a SIMD: 301 x 50257 bf16 in 8.1 us, with the registers of 5 in 9.7)
template <typename T>
__global__ __launch_bounds__(kSliceNT, 8) void slice_max(const SampleArgs a) {
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
    const float top = block_top<kSliceNT, kSliceTPT>(
        x, lo, s_top, s_at, a.groups + (size_t)blockIdx.x * kGroups, at);
    if (threadIdx.x == 0) {
        a.top[blockIdx.x] = top;
        a.top_at[blockIdx.x] = at;
    }
}

// The row's maximum from its slices', in every lane: a lane's first one, then
// the rest.
__device__ __forceinline__ float slice_top(const SampleArgs& a, int r) {
    const int s = threadIdx.x & 63;
    return s < a.slices ? a.top[(size_t)r * a.slices + s] : -INFINITY;
}
__device__ __forceinline__ float row_top(const SampleArgs& a, int r, float m) {
    for (int s = (threadIdx.x & 63) + 64; s < a.slices; s += 64)
        m = fmaxf(m, a.top[(size_t)r * a.slices + s]);
    return wave_max(m);
}

template <typename T>
__global__ __launch_bounds__(kSliceNT) void slice_hist(const SampleArgs a) {
    __shared__ double s_powers[kPowers];
    // A histogram a wave, mass and count in one word: 2048 tokens, so at most
    // 2^51 and 2^11. (One of both for the workgroup: two atomics a token, and
    // LDS is what the loop waits for.) The last bin: weights that are 0.
    constexpr int kCountAt = 52;
    static_assert(kSliceTPT * 64 <= 1 << 11, "a wave's tokens");
    __shared__ u64 s_hist[kSliceNT / 64][kBins + 1];
    __shared__ u64 s_sum[4];
    const int r = blockIdx.x / a.slices, s = blockIdx.x - r * a.slices;
    const int lo = s * kSlice, hi = min(lo + kSlice, a.n);
    const float some = slice_top(a, r);
    const int parts = min(a.slices * kGroups, kFloorOf);
    float4 of_parts = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (4 * (int)(threadIdx.x & 63) < parts)
        of_parts = *reinterpret_cast<const float4*>(a.groups + (size_t)r * a.slices * kGroups +
                                                    4 * (threadIdx.x & 63));
    Tokens<T, 2> tokens(a, r, lo, hi);
    fill_powers(s_powers);
    for (int b = threadIdx.x; b < kSliceNT / 64 * (kBins + 1); b += kSliceNT) s_hist[0][b] = 0;
    __syncthreads();
    const float top = row_top(a, r, some);
    const Row row(a, r, top, s_powers);
    if (row.greedy || top == -INFINITY) return;
    if (!row.cut()) {
        u64 sum = 0;
        tokens.each([&](float x, int) {
            const u64 w = row.weight_of(x);
            if (row.keeps(w)) sum += w;
        });
        sum = wave_sum64(sum);
        if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0) a.sum[blockIdx.x] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        return;
    }
    const float floor = floor_of(of_parts, row.k, parts);
    if (s == 0 && threadIdx.x == 0) a.floors[r] = floor;
    const float least = row.least_of(kBins - 1, floor);
    u64* const hist = s_hist[threadIdx.x >> 6];
    auto add = [&](int b, u64 w) { atomicAdd(&hist[b], w | 1ull << kCountAt); };
    // (where T is so small that the bound's own rounding is far: all checks)
    if (row.infinite || !(row.far(least) > kFarthest))
        tokens.each([&](float x, int) {
            const double t = row.far(x);
            const int b = bin_of(t);
            if (x >= floor && b < kBins) add(b, weight(s_powers, t));
        });
    else
        tokens.each([&](float x, int) {
            if (!(x >= least)) return;
            const double t = row.finite_far(x);
            add(min(bin_near(t), kBins), weight_near(s_powers, t));
        });
    __syncthreads();
    u64* const part = a.part + (size_t)blockIdx.x * kBins;
    for (int b = threadIdx.x; b < kBins; b += kSliceNT) {
        u64 mass = 0;
        unsigned count = 0;
#pragma unroll
        for (int w = 0; w < kSliceNT / 64; ++w) {
            const u64 v = s_hist[w][b];
            mass += v & ((1ull << kCountAt) - 1);
            count += (unsigned)(v >> kCountAt);
        }
        part[b] = mass;
        if (count) {
            atomicAdd(&a.mass[(size_t)r * kBins + b], mass);
            atomicAdd(&a.count[(size_t)r * kBins + b], count);
        }
    }
}

// A thread's bins of the row's histogram.
struct BinRun {
    static constexpr int PER = (kBins + kSliceNT - 1) / kSliceNT;
    u64 m[PER];
    unsigned c[PER];
    __device__ __forceinline__ void load(const SampleArgs& a, int r) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int b = threadIdx.x * PER + i;
            m[i] = b < kBins ? a.mass[(size_t)r * kBins + b] : 0;
            c[i] = b < kBins ? a.count[(size_t)r * kBins + b] : 0;
        }
    }
};

// The bins that the cut can be in: [lo, hi], and k's own. Sums are exact but
// for the part of bin `at_k` that k keeps, so p's want lies between two.
struct Span {
    int lo, hi, at_k;  // at_k: -1 none
};
__device__ __forceinline__ Span cut_span(const Row& row, const BinRun& h, u64* s_scan,
                                         int* s_bin) {
    constexpr int PER = BinRun::PER;
    const u64(&m)[PER] = h.m;
    const unsigned(&c)[PER] = h.c;
    u64 mine = 0, many = 0, total, tokens;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += m[i], many += c[i];
    if (threadIdx.x < 3) s_bin[threadIdx.x] = 0;
    block_scan2<kSliceNT>(mine, many, s_scan, total, tokens);
    u64 mb = mine;
    const u64 cb = many;
    __shared__ u64 s_w[2];
    if (threadIdx.x == 0) s_w[0] = s_w[1] = total;
    const bool by_k = row.k > 0 && (u64)row.k <= tokens;
    if (by_k) {
        u64 q = cb;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (q < (u64)row.k && q + c[i] >= (u64)row.k) s_bin[2] = threadIdx.x * PER + i;
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
            const u64 next = mb + m[i];
            if ((double)mb < w0 && !((double)next < w0)) s_bin[0] = threadIdx.x * PER + i;
            if ((double)mb < w1 && !((double)next < w1)) s_bin[1] = threadIdx.x * PER + i;
            mb = next;
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
    __shared__ u64 s_scan[32], s_sum[4];
    __shared__ int s_bin[3];
    __shared__ unsigned s_n;
    const int r = blockIdx.x / a.slices, s = blockIdx.x - r * a.slices;
    const int lo = s * kSlice, hi = min(lo + kSlice, a.n);
    __shared__ T s_near[kSlice];
    const float some = slice_top(a, r), floor = a.floors[r];
    BinRun bins;
    bins.load(a, r);
    u64 own[BinRun::PER];  // the slice's
#pragma unroll
    for (int i = 0; i < BinRun::PER; ++i) {
        const int b = threadIdx.x + i * kSliceNT;
        own[i] = b < kBins ? a.part[(size_t)blockIdx.x * kBins + b] : 0;
    }
    // (on their way while the bins are searched)
    Tokens<T, 4> tokens(a, r, lo, hi);
    const float top = row_top(a, r, some);
    const Row row(a, r, top, nullptr);
    if (row.greedy || top == -INFINITY || !row.cut()) return;
    if (threadIdx.x == 0) s_n = 0;
    const Span span = cut_span(row, bins, s_scan, s_bin);
    // Above the bins that are listed all is kept: with min-p's own bin among
    // them, and its own bins' sums at hand, a slice works out no weight here.
    const int at_p = row.least_bin();
    const int all = min(span.lo, at_p);
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < BinRun::PER; ++i)
        if ((int)threadIdx.x + i * kSliceNT < all) sum += own[i];
    unsigned* const list = a.list + (size_t)r * a.n + lo;
    // logits outside the listed bins are seen without their float64 distance
    const float least = row.least_of(min(max(span.hi, span.at_k), kBins - 1), floor);
    const float most = row.around(min(all, kBins - 1)).y;
    unsigned some_of = 0;  // the thread's tokens that may be listed
    tokens.each([&](float x, int j) {
        if (x >= least && !(x > most)) {
            some_of |= 1u << j;
            s_near[j * kSliceNT + threadIdx.x] = (T)x;
        }
    });
    while (some_of) {
        const int j = __ffs(some_of) - 1;
        some_of &= some_of - 1;
        const float x = (float)s_near[j * kSliceNT + threadIdx.x];
        const int b = bin_of(row.far(x));
        if (b < kBins && ((b >= span.lo && b <= span.hi) || b == span.at_k ||
                          (b >= at_p && b < at_p + kMinBins && b < span.lo)))
            list[atomicAdd(&s_n, 1u)] = order_bits(x);
    }
    sum = wave_sum64(sum);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        a.sum[blockIdx.x] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        a.listed[blockIdx.x] = s_n;
    }
}

constexpr int kListMost = 12288;  // listed logits of a row that are held in LDS

template <typename T>
__global__ __launch_bounds__(kRowNT) void sample_pick(const SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    RowState& s = *reinterpret_cast<RowState*>(smem);
    // the list; then a slice's tokens
    unsigned* const s_list =
        reinterpret_cast<unsigned*>(smem + ((sizeof(RowState) + 15) & ~(size_t)15));
    __shared__ unsigned s_off[kMaxVocab / kSlice + 1];
    const int r = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int b = threadIdx.x;
    const size_t row0 = (size_t)r * a.slices;
    // (slice s in thread s)
    const unsigned listed = b < a.slices ? a.listed[row0 + b] : 0;
    for (int i = b; i < kBins; i += kRowNT) {
        s.mass[i] = a.mass[(size_t)r * kBins + i];
        s.count[i] = a.count[(size_t)r * kBins + i];
    }
    const float u = a.u[r];
    const float top = row_top(a, r, slice_top(a, r));
    const Row row(a, r, top, s.powers);
    fill_powers(s.powers);
    if (row.greedy || top == -INFINITY) {
        if (wave == 0) {
            int at = INT_MAX;
            for (int t = lane; t < a.slices; t += 64)
                if (a.top[row0 + t] == top) at = min(at, a.top_at[row0 + t]);
#pragma unroll
            for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
            if (lane == 0) a.out[r] = top == -INFINITY ? -1 : at;
        }
        return;
    }
    Cut cut{-INFINITY, 0, 0};
    // a slice's kept weights, and the cut's equals in it
    u64* const s_sum = s.level_mass;  // (after the cut is found)
    unsigned* const s_ties = s.level_count;
    if (row.cut()) {
        u64 all;
        const u64 off = block_scan<kRowNT>(listed, s.scan, all);
        if (b < a.slices) s_off[b] = (unsigned)off;
        if (b == 0) s_off[a.slices] = (unsigned)all;
        __syncthreads();
        const bool held = all <= kListMost;
        // slice t is wave t % kWaves'
        auto slices = [&](auto&& f) {
            for (int t = wave; t < a.slices; t += kWaves) {
                const unsigned n = s_off[t + 1] - s_off[t];
                const unsigned* const list = a.list + (size_t)r * a.n + t * kSlice;
                for (unsigned i = lane; i < n; i += 64) f(list[i]);
            }
        };
        if (held)
            for (int t = wave; t < a.slices; t += kWaves)
                for (unsigned i = lane; i < s_off[t + 1] - s_off[t]; i += 64)
                    s_list[s_off[t] + i] = a.list[(size_t)r * a.n + t * kSlice + i];
        const u64 total = scan_bins(s);  // (synchronises)
        cut = find_cut(row, total, s, [&](auto&& f, int bin) {
            if (held)
                for (unsigned i = b; i < (unsigned)all; i += kRowNT) {
                    const unsigned o = s_list[i];
                    f(o, [&] { return bin_of(row.far(from_bits(o))) == bin; });
                }
            else
                slices([&](unsigned o) {
                    f(o, [&] { return bin_of(row.far(from_bits(o))) == bin; });
                });
        });
        // (also where nothing is cut off: min-p's bins are listed, not summed)
        for (int t = wave; t < a.slices; t += kWaves) {
            u64 sum = 0;
            unsigned ties = 0;
            const unsigned n = s_off[t + 1] - s_off[t];
            const unsigned* const list =
                held ? s_list + s_off[t] : a.list + (size_t)r * a.n + t * kSlice;
            for (unsigned i = lane; i < n; i += 64) {
                const float v = from_bits(list[i]);
                if (v > cut.xc) {
                    const u64 w = row.weight_of(v);
                    if (row.keeps(w)) sum += w;
                }
                ties += v == cut.xc;
            }
            sum = wave_sum64(sum);
            ties = (unsigned)wave_sum64(ties);
            if (lane == 0) s_sum[t] = sum + a.sum[row0 + t], s_ties[t] = ties;
        }
    } else if (b < a.slices) {
        s_sum[b] = a.sum[row0 + b], s_ties[b] = 0;
    }
    if (b == 0) s.slice = 0, s.base = 0, s.q = cut.q;
    __syncthreads();
    u64 total;
    const u64 ties = b < a.slices ? s_ties[b] : 0;
    const u64 had = block_scan<kRowNT>(ties, s.scan, total);
    const u64 left = cut.q > had ? cut.q - had : 0;
    const u64 mine = b < a.slices ? s_sum[b] + cut.wc * min(left, ties) : 0;
    const u64 before = block_scan<kRowNT>(mine, s.scan + 16, total);
    const u64 aim = aim_at(u, total);
    if (before <= aim && aim < before + mine) s.slice = b, s.base = before, s.q = left;
    __syncthreads();
    const int lo = s.slice * kSlice, hi = min(lo + kSlice, a.n);
    const u64 base = s.base, q = s.q;
    float* const s_x = reinterpret_cast<float*>(s_list);
    int at;
    stage_tokens<T, kSlice, false>((const T*)a.x + (long long)r * a.ld, lo, hi, s_x, s, at);
    pick(row, cut, s_x, hi - lo, lo, q, aim - base, 0.f, s, a.out + r);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct SampleShape {
    int slices;  // 0: a workgroup a row
    size_t top, top_at, groups, floors, sum, part, listed, mass, count, list, bytes;
};

SampleShape sample_shape(int rows, int n) {
    if (rows < 0) inval("sample_filtered_batched: rows must be >= 0");
    if (n < 1) inval("sample of empty logits");
    if (n > kMaxVocab) inval("sample_filtered_batched: at most 2^22 logits a row");
    SampleShape s{};
    // (a launch has fewer than 2^32 threads)
    if ((long long)rows * kRowNT >= 1LL << 32)
        inval("sample_filtered_batched: too many rows for one call");
    if (n <= kRowMost || rows == 0) return s;
    s.slices = (n + kSlice - 1) / kSlice;
    const size_t parts = (size_t)rows * s.slices;
    if (parts * kSliceNT >= 1ULL << 32)
        inval("sample_filtered_batched: too many rows for one call");
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t p = at;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    s.top = take(4 * parts);
    s.top_at = take(4 * parts);
    s.groups = take(4 * parts * kGroups);
    s.floors = take(4 * (size_t)rows);
    s.sum = take(8 * parts);
    s.part = take(8 * parts * kBins);
    s.listed = take(4 * parts);
    s.mass = take(8 * (size_t)rows * kBins);
    s.count = take(4 * (size_t)rows * kBins);
    s.list = take(4 * (size_t)rows * n);
    s.bytes = at;
    return s;
}

constexpr size_t kStateBytes = (sizeof(RowState) + 15) & ~(size_t)15;

template <typename T, int MOST>
void row_run(const SampleArgs& a, hipStream_t s) {
    const size_t lds = kStateBytes + (size_t)(a.n + kChunk - 1) / kChunk * kChunk * 4;
    allow_lds((const void*)sample_row<T, MOST>, lds);
    sample_row<T, MOST><<<a.rows, kRowNT, lds, s>>>(a);
}

template <typename T>
void sample_run(const SampleArgs& a, hipStream_t s) {
    if (!a.slices) {
        if (a.n <= 4096) row_run<T, 4096>(a, s);
        else if (a.n <= 16384) row_run<T, 16384>(a, s);
        else row_run<T, 32768>(a, s);
        launch_check("sample_filtered_batched kernel launch");
        return;
    }
    const unsigned grid = (unsigned)a.rows * (unsigned)a.slices;
    slice_max<T><<<grid, kSliceNT, 0, s>>>(a);
    slice_hist<T><<<grid, kSliceNT, 0, s>>>(a);
    slice_list<T><<<grid, kSliceNT, 0, s>>>(a);
    const size_t lds = kStateBytes + 4 * (size_t)kListMost;
    allow_lds((const void*)sample_pick<T>, lds);
    sample_pick<T><<<a.rows, kRowNT, lds, s>>>(a);
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
        a.groups = (float*)(ws + sh.groups);
        a.floors = (float*)(ws + sh.floors);
        a.sum = (u64*)(ws + sh.sum);
        a.part = (u64*)(ws + sh.part);
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
