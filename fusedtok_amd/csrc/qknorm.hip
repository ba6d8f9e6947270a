// Norms of query and key heads with the rotation, for gfx950: a projection's
// rows [T, (Hq + 2 Hkv) * D] (q heads, k heads, v heads) become rotated q and
// k heads and v heads, dense or with k and v in a paged cache's slots.
//
//   n  = x * (1 / sqrt(mean(x^2) + eps)) * w     (a head's D values; no
//                                                 weights: n = x)
//   (a, b) = pair j of the first R values, (j, j + R/2) or (2j, 2j + 1)
//   a' = a cos - b sin, b' = b cos + a sin,  angle = pos[axis(j)] theta^(-2j/R)
//
// The values past R keep their norm; v is copied. Everything is float32 but
// the angle (float64), rounded once at the end.
//
// What bounds it: HBM, each value read and written once (16384 tokens of 32 + 2 *
// 8 heads, D = 128, bf16: 403 MB in 70-74 us, 5.4-5.8 TB/s, with the same inputs
// again and again, 88 with others from call to call; stores that bypass the
// caches: 87-91 us without, or with loads that do too, same inputs), and for few
// tokens latency (64 tokens 5.6 us). Where the pieces are not whole 16 bytes
// (VEC false: rows or halves of the rotated part) loads and stores are single
// elements: the same tokens 241 us in unaligned rows, 231 with D = 80, R = 40 (D = 80
// whole: 81).
//
// Work split. A head is a group of lanes, 16 bytes of each half of its pairs
// a lane (D = 128, 2-byte types: 8 lanes, 8 heads a wave); a workgroup takes
// a few tokens and goes through their heads. Each pair's cosine and sine are
// computed once a token and workgroup and shared through LDS: a lane's own
// pairs are the same for every head, its weights stay in registers. The norm
// is a butterfly over the group.
//
// The angle. theta^(-2j/R) = 2^(-(2j/R) log2 theta) with the exponent in two
// float64 parts, so it is right to a float64 step, as far positions need it
// (a position of 2^31 scales its error to 5e-7); pos * freq is reduced to
// +-pi/4 in float64, the sine and cosine of what is left are their Taylor
// series in float32 (next terms 2e-9 and 1e-10).
#include "ft_common.hpp"

#include <algorithm>
#include <cmath>

namespace ft {
namespace {

constexpr int kMaxHead = 512;
constexpr int kMaxAxes = 4;
constexpr int kMaxTok = 8;  // tokens of a workgroup, at most

template <typename T>
struct QkArgs {
    const T* qkv;
    long long ld;
    const float* qw;
    const float* kw;
    const int* pos;
    const int* slots;  // null: dense k and v
    T* q;
    T* k;
    T* v;
    long long slot_end;  // blocks * page
    int tokens, hq, hkv, dim, rot, page;
    int axes, end[kMaxAxes];  // axis a holds pairs [end[a - 1], end[a])
    double log_hi, log_lo;    // log2(theta)
    double inv_rot;           // 1 / rot
    float eps;
    int lanes_log2;           // lanes a head
    int tt, heads;            // tokens and heads of a workgroup
};

// cosine and sine of a (float64 radians, below 2^41: what is left of it after
// quarter turns is within pi / 4 and right to 6e-17; from 2^48 on it is not)
__device__ __forceinline__ float2 cos_sin(double a) {
    const double n = rint(a * 0.63661977236758134308);  // 2 / pi
    double r = fma(n, -1.57079632679489655800, a);      // pi / 2 in two parts
    r = fma(n, -6.12323399573676603587e-17, r);
    const float x = (float)r, x2 = x * x;
    const float s = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.0f / 362880, -1.0f / 5040),
                                               1.0f / 120), -1.0f / 6), x);
    const float c = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.0f / 3628800, 1.0f / 40320),
                                                    -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int k = (int)(long long)n & 3;
    const float co = k & 1 ? s : c, si = k & 1 ? c : s;
    return make_float2(k == 1 || k == 2 ? -co : co, k >= 2 ? -si : si);
}

// VEC: every lane's chunks are whole 16-byte pieces (qk_run)
template <typename T, bool NEOX, bool VEC>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const QkArgs<T> a) {
    constexpr int NP = 16 / sizeof(T);  // pairs a lane
    typedef T vec __attribute__((ext_vector_type(NP)));
    extern __shared__ __attribute__((aligned(16))) char smem[];
    long long* const s_row = reinterpret_cast<long long*>(smem);        // kMaxTok
    float2* const s_trig = reinterpret_cast<float2*>(smem + 8 * kMaxTok);  // [tt][rot / 2]

    const int tid = threadIdx.x;
    const int half = a.dim >> 1, rp = a.rot >> 1;
    const int t0 = blockIdx.x * a.tt, nt = min(a.tt, a.tokens - t0);
    const int all = a.hq + 2 * a.hkv;
    const int h0 = blockIdx.y * a.heads, nh = min(a.heads, all - h0);

    const int lph = 1 << a.lanes_log2;
    const int p0 = (tid & (lph - 1)) * NP;  // the lane's first pair
    const int step = 256 >> a.lanes_log2;   // heads a pass
    // element of pair p: first, second
    auto at0 = [&](int p) { return NEOX ? (p < rp ? p : p + rp) : 2 * p; };
    auto at1 = [&](int p) { return NEOX ? (p < rp ? p + rp : p + half) : 2 * p + 1; };
    const bool lane_on = p0 < half;
    // the lane's 16-byte pieces: both halves of its pairs, or its pairs in a row
    const int c0 = NEOX ? at0(p0) : 2 * p0, c1 = NEOX ? at1(p0) : 2 * p0 + NP;

    // A head's values as they come, and as pairs. Loads are unconditional (a lane
    // past the head reads its start) and nothing touches their values before
    // their turn: a conversion or a branch around them waits for them at once.
    const int l0 = lane_on ? c0 : 0, l1 = lane_on ? c1 : 0;
    vec raw0, raw1;
    auto load = [&](const T* row) {
        if constexpr (VEC) {
            raw0 = *reinterpret_cast<const vec*>(row + l0);
            raw1 = *reinterpret_cast<const vec*>(row + l1);
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const bool on = p0 + i < half;
                raw0[i] = row[on ? at0(p0 + i) : 0];
                raw1[i] = row[on ? at1(p0 + i) : 0];
            }
        }
    };
    auto unpack = [&](float (&x)[NP], float (&y)[NP]) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            T u = raw0[i], w = raw1[i];
            if constexpr (VEC && !NEOX) {
                u = 2 * i < NP ? raw0[(2 * i) % NP] : raw1[(2 * i) % NP];
                w = 2 * i < NP ? raw0[(2 * i + 1) % NP] : raw1[(2 * i + 1) % NP];
            }
            const bool on = VEC ? lane_on : p0 + i < half;
            x[i] = on ? (float)u : 0.0f;
            y[i] = on ? (float)w : 0.0f;
        }
    };
    auto store = [&](T* row, const float (&x)[NP], const float (&y)[NP]) {
        if constexpr (VEC) {
            if (!lane_on) return;
            vec u, w;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                if constexpr (NEOX) {
                    u[i] = (T)x[i];
                    w[i] = (T)y[i];
                } else if (2 * i < NP) {
                    u[(2 * i) % NP] = (T)x[i];
                    u[(2 * i + 1) % NP] = (T)y[i];
                } else {
                    w[(2 * i) % NP] = (T)x[i];
                    w[(2 * i + 1) % NP] = (T)y[i];
                }
            }
            __builtin_nontemporal_store(u, reinterpret_cast<vec*>(row + c0));
            __builtin_nontemporal_store(w, reinterpret_cast<vec*>(row + c1));
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i)
                if (p0 + i < half) {
                    row[at0(p0 + i)] = (T)x[i];
                    row[at1(p0 + i)] = (T)y[i];
                }
        }
    };

    // the first head's values are on their way while the angles are computed
    int tok = 0, head = tid >> a.lanes_log2;
    while (head >= nh && tok < nt) head -= nh, ++tok;
    const T* const rows = a.qkv + (long long)t0 * a.ld + (long long)h0 * a.dim;
    if (tok < nt) load(rows + tok * a.ld + (long long)head * a.dim);

    // weights of the lane's pairs
    float wq0[NP], wq1[NP], wk0[NP], wk1[NP];
    const bool norm = a.qw != nullptr;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p = min(p0 + i, half - 1);
        wq0[i] = norm ? a.qw[at0(p)] : 1.0f;
        wq1[i] = norm ? a.qw[at1(p)] : 1.0f;
        wk0[i] = norm ? a.kw[at0(p)] : 1.0f;
        wk1[i] = norm ? a.kw[at1(p)] : 1.0f;
    }

    for (int e = tid; e < nt * rp; e += 256) {
        const int t = e / rp, j = e - t * rp;
        int axis = 0;
        while (axis + 1 < a.axes && j >= a.end[axis]) ++axis;
        const int pos = a.pos[(long long)axis * a.tokens + t0 + t];
        // 2j log2(theta) / R in two parts
        const double m = 2.0 * j, r = a.rot;
        const double hi = m * a.log_hi, lo = fma(m, a.log_hi, -hi) + m * a.log_lo;
        const double e0 = hi * a.inv_rot, e1 = (fma(-e0, r, hi) + lo) * a.inv_rot;
        const double f = exp2(-e0);
        s_trig[e] = cos_sin((double)pos * fma(-0.69314718055994530942 * e1, f, f));
    }
    if (tid < nt) {
        if (!a.slots) {
            s_row[tid] = (long long)(t0 + tid) * a.hkv * a.dim;
        } else {
            const long long s = a.slots[t0 + tid];
            const long long b = s / a.page;
            s_row[tid] = s < 0 || s >= a.slot_end
                             ? -1 : (b * a.hkv * a.page + (s - b * a.page)) * a.dim;
        }
    }
    __syncthreads();

    const long long kv_head = (a.slots ? (long long)a.page : 1) * a.dim;
    const float inv_dim = 1.0f / (float)a.dim;
    while (tok < nt) {
        const int h = h0 + head, t = tok;
        float u[NP], w[NP];
        unpack(u, w);
        head += step;
        while (head >= nh && tok < nt) head -= nh, ++tok;
        if (tok < nt) load(rows + tok * a.ld + (long long)head * a.dim);

        if (h < a.hq + a.hkv) {
            const bool is_q = h < a.hq;
            if (norm) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < NP; ++i) s = fmaf(u[i], u[i], fmaf(w[i], w[i], s));
                for (int o = lph >> 1; o; o >>= 1) s += __shfl_xor(s, o, 64);
                const float inv = 1.0f / sqrtf(s * inv_dim + a.eps);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    u[i] *= inv * (is_q ? wq0[i] : wk0[i]);
                    w[i] *= inv * (is_q ? wq1[i] : wk1[i]);
                }
            }
            const float2* const trig = s_trig + t * rp;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                if (p0 + i >= rp) continue;
                const float2 cs = trig[p0 + i];
                const float b = fmaf(w[i], cs.x, u[i] * cs.y);
                u[i] = fmaf(u[i], cs.x, -(w[i] * cs.y));
                w[i] = b;
            }
        }
        if (h < a.hq) {
            store(a.q + ((long long)(t0 + t) * a.hq + h) * a.dim, u, w);
        } else if (s_row[t] >= 0) {
            const bool is_k = h < a.hq + a.hkv;
            const int kv = h - a.hq - (is_k ? 0 : a.hkv);
            store((is_k ? a.k : a.v) + s_row[t] + kv * kv_head, u, w);
        }
    }
}

inline bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T>
void qk_run(QkArgs<T> a, bool neox, hipStream_t s) {
    constexpr int NP = 16 / sizeof(T);
    const int half = a.dim / 2, rp = a.rot / 2;
    // Whole 16-byte pieces: aligned rows, and no piece across the end of the
    // rotated part's halves (neighbouring pairs lie in one row anyway).
    const bool vec = half % NP == 0 && (!neox || rp % NP == 0) &&
                     a.ld * sizeof(T) % 16 == 0 && on16(a.qkv) && on16(a.q) && on16(a.k) &&
                     on16(a.v);
    a.lanes_log2 = 0;
    while ((NP << a.lanes_log2) < half) ++a.lanes_log2;
    const int all = a.hq + 2 * a.hkv, step = 256 >> a.lanes_log2;
    // As many tokens a workgroup, up to kMaxTok, as leave two workgroups a CU
    // (angles and weights are shared further: 16384 tokens of 48 heads 137, 102,
    // 84, 78 us at 1, 2, 4, 8; 6001 of 20 50, 30, 22, 18.5, and 24 at 16); few tokens
    // have their heads spread over workgroups of one pass.
    const int cus = dev_info().cu_count;
    a.tt = 1;
    while (a.tt < kMaxTok && a.tokens / (2 * a.tt) >= 2 * cus) a.tt *= 2;
    a.heads = all;
    if (a.tokens < 4 * cus) a.heads = std::min(all, step);
    const dim3 grid((a.tokens + a.tt - 1) / a.tt, (all + a.heads - 1) / a.heads);
    if (grid.y > 65535) inval("qk_norm_rope: too many heads");
    // (a launch has fewer than 2^32 threads)
    if ((long long)grid.x * 256 >= 1LL << 32) inval("qk_norm_rope: too many tokens for one call");
    const size_t lds = 8 * kMaxTok + (size_t)a.tt * rp * sizeof(float2);
    if (neox && vec) qk_norm_rope_kernel<T, true, true><<<grid, 256, lds, s>>>(a);
    else if (neox) qk_norm_rope_kernel<T, true, false><<<grid, 256, lds, s>>>(a);
    else if (vec) qk_norm_rope_kernel<T, false, true><<<grid, 256, lds, s>>>(a);
    else qk_norm_rope_kernel<T, false, false><<<grid, 256, lds, s>>>(a);
    launch_check("qk_norm_rope kernel launch");
}

int qk_norm_rope(const void* qkv, int dtype, long long ld, const float* q_weight,
                 const float* k_weight, const int* positions, int axes, const int* sections,
                 int rotary_dim, double theta, float eps, int neox, void* q_out, void* k_out,
                 void* v_out, bool paged, const int* slots, int tokens, int q_heads, int kv_heads,
                 int dim, int blocks, int page, uintptr_t stream) {
    return guarded([&] {
        if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
            inval("qk_norm_rope: unknown element type");
        if (tokens < 0 || q_heads < 1 || kv_heads < 1)
            inval("qk_norm_rope: tokens >= 0 and heads >= 1 are required");
        if (dim < 2 || dim % 2 || dim > kMaxHead)
            inval("dim must be even and at most 512");
        if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > dim)
            inval("rotary_dim must be even, at least 2 and at most dim");
        // (an angle is below 2^31 / theta: cos_sin's range)
        if (!(theta >= 0x1p-10) || !std::isfinite(theta))
            inval("theta must be at least 2^-10 and finite");
        if (!(eps >= 0.0f)) inval("eps must be >= 0");
        if (axes < 1 || axes > kMaxAxes) inval("positions must have 1 to 4 axes");
        if ((long long)q_heads + 2LL * kv_heads > (1 << 20)) inval("qk_norm_rope: too many heads");
        if (ld < (long long)(q_heads + 2 * kv_heads) * dim)
            inval("qk_norm_rope: qkv row stride too small");
        int end[kMaxAxes] = {};
        if (axes > 1) {
            if (!sections) inval("several axes of positions need sections");
            long long sum = 0;
            for (int i = 0; i < axes; ++i) {
                if (sections[i] < 0) inval("sections must be >= 0");
                sum += sections[i];
                if (sum > rotary_dim / 2) break;
                end[i] = (int)sum;
            }
            if (sum != rotary_dim / 2) inval("sections must sum to rotary_dim / 2");
        }
        if (!q_weight != !k_weight) inval("q_weight and k_weight are given together or not at all");
        if (paged && (blocks < 0 || page < 1))
            inval("qk_norm_rope: blocks >= 0 and page >= 1 are required");
        if (tokens == 0) return;
        if (!qkv || !positions || !q_out || (paged && !slots) ||
            ((!paged || blocks > 0) && (!k_out || !v_out)))
            inval("qk_norm_rope: null operand");
        const double l = std::log2(theta);
        const double l_lo = (double)(std::log2((long double)theta) - (long double)l);
        auto go = [&](auto zero) {
            using T = decltype(zero);
            QkArgs<T> a{};
            a.qkv = (const T*)qkv;
            a.ld = ld;
            a.qw = q_weight;
            a.kw = k_weight;
            a.pos = positions;
            a.slots = paged ? slots : nullptr;
            a.q = (T*)q_out;
            a.k = (T*)k_out;
            a.v = (T*)v_out;
            a.slot_end = paged ? (long long)blocks * page : 0;
            a.tokens = tokens;
            a.hq = q_heads;
            a.hkv = kv_heads;
            a.dim = dim;
            a.rot = rotary_dim;
            a.page = page;
            a.axes = axes;
            for (int i = 0; i < kMaxAxes; ++i) a.end[i] = end[i];
            a.log_hi = l;
            a.log_lo = l_lo;
            a.inv_rot = 1.0 / rotary_dim;
            a.eps = eps;
            qk_run(a, neox != 0, as_stream(stream));
        };
        if (dtype == FT_DT_F32) go(0.0f);
        else if (dtype == FT_DT_BF16) go((bf16)0.0f);
        else go((f16)0.0f);
    });
}

}  // namespace
}  // namespace ft

extern "C" {

int ft_qk_norm_rope_launch(const void* qkv, int dtype, long long ld, const float* q_weight,
                           const float* k_weight, const int* positions, int axes,
                           const int* sections, int rotary_dim, double theta, float eps, int neox,
                           void* q_out, void* k_out, void* v_out, int tokens, int q_heads,
                           int kv_heads, int dim, uintptr_t stream) {
    return ft::qk_norm_rope(qkv, dtype, ld, q_weight, k_weight, positions, axes, sections,
                            rotary_dim, theta, eps, neox, q_out, k_out, v_out, false, nullptr,
                            tokens, q_heads, kv_heads, dim, 0, 1, stream);
}

int ft_qk_norm_rope_kv_append_paged_launch(
    const void* qkv, int dtype, long long ld, const float* q_weight, const float* k_weight,
    const int* positions, int axes, const int* sections, int rotary_dim, double theta, float eps,
    int neox, void* q_out, void* k_pool, void* v_pool, const int* slots, int tokens, int q_heads,
    int kv_heads, int dim, int blocks, int page, uintptr_t stream) {
    return ft::qk_norm_rope(qkv, dtype, ld, q_weight, k_weight, positions, axes, sections,
                            rotary_dim, theta, eps, neox, q_out, k_pool, v_pool, true, slots,
                            tokens, q_heads, kv_heads, dim, blocks, page, stream);
}

}  // extern "C"
