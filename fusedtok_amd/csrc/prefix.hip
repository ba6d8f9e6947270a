// Decode attention of a batch whose sequences share long prefixes, for gfx950:
//
//   out[b, h] = softmax(q[b, h] . K / sqrt(D)) . V  over the tokens of the
//   prefix of b's group, then b's own, both in one paged cache.
//
// q, out [B, Hq, D]; k_pool, v_pool [blocks, Hkv, P, D]; group g is the
// sequences [off_g, off_g+1), its prefix lies in row g of prefix_table, a
// sequence's own tokens in its row of table.
//
// Work split. An entry is a group's prefix or a sequence's own tokens: rows
// (the q heads of its sequences that read one kv head) against n tokens. Its
// units are (kv head, tile of rows), n tokens each; all units are laid end to
// end and every workgroup takes one equal contiguous segment of that range,
// whatever the mix of lengths. A segment is one or more pieces, one a unit it
// touches; a piece leaves a float32 partial (m, l, acc[D]) a row, which
// prefix_combine folds by the log-sum-exp rule: of each (b, h) the pieces of
// the group's prefix and of its own tokens. A piece's partials start at row
// 16 (8 segment + granules of the units before it), a granule being 16 rows of
// a tile, 8 of them at most: pieces are ordered in both, so the places are
// disjoint and both kernels work them out from the plan (the entries' sums),
// which every workgroup scans by itself and the first leaves for the combine.
// Nothing else passes between workgroups and the workspace is the caller's.
//
// A unit's cost is its tokens times a cost a token, by the rows of its tile,
// and its start: equal shares of tokens alone left 131071 tokens of 64 rows at
// 200 us, the workgroups with many short units behind; with costs 117 (both with
// two parts of a weight, below; 122 with three).
//
// What bounds it: HBM, each K / V row read once a tile of rows of a kv head (up
// to 128 rows on the matrix cores, so once for a group of 128 rows and fewer). A
// prefix of 8192 tokens and 64 sequences of 16-2000, 32 / 8 heads, D = 128, bf16:
// 296 MB in 70 + 6.1 us (attention and combine; 4.2 TB/s); 5 prefixes of
// 1000-16000 and 48 of 0-3001, 64 / 8 heads, fp16: 469 MB in 90 + 6.9 (5.2); 131071 tokens
// of 16 sequences: 553 MB in 110 + 8.1 (5.0). Own tokens alone (64 x 4000) reach
// 6.1 TB/s. What the prefixes lose is the matrix cores' chain from scores to
// products (128 rows of bf16 behind 131071 tokens: 174 us, the matrix cores busy
// for 43% of them, the products with V three times; 152 and 64 us for the first
// case with two parts of a weight, whose error showed in the output's last bits)
// and the ~6 us of a segment's start, as long as two steps of 64 tokens
// for each piece. Loads two steps ahead gained nothing.
#include "attn_common.hpp"
#include "fast_div.hpp"
#include "ft_common.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace ft {
namespace {

constexpr int kMaxDimP = 512;
constexpr int kMaxEntries = 4096;  // groups and sequences of a call (their sums are in LDS)
constexpr int kGranule = 16;       // rows
constexpr int kTileGranules = 8;   // of a tile, at most

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// What the combine needs of one of a sequence's two entries.
struct Part {
    long long start;  // of the first unit's tokens in the range of all
    long long whole;  // from unit to unit
    int gran;         // granules before it
    int n;            // tokens (0: none)
    int rows;         // rows a kv head
    int first;        // its first sequence
};
struct Parts {
    Part prefix, own;
};

struct PrefixArgs {
    const void* q;
    const void* k;
    const void* v;
    const int* ptable;
    const int* plens;
    const int* offsets;
    const int* table;
    const int* lens;
    void* out;
    float* ml;       // [rows][2]
    float* acc;      // [rows][dim]
    Parts* parts;    // [batch]
    long long* seg;  // the segments' length
    int batch, hq, hkv, gq, groups, blocks, pwidth, twidth, dim;
    FastDiv page, gdiv;
    float scale_log2;
    int segs, min_seg, start_cost, cost[3];
};

// Which kernel takes a call.
enum Kind { kGeneral, kFloat, kHalf };

// Rows of a tile. On the matrix cores up to 16 rows leave the keys of a step to
// the four waves, more are shared out to them, 16 each or (kHalf) 32.
template <Kind KIND>
__device__ __forceinline__ int tile_rows(int rows) {
    if (KIND == kGeneral || rows <= 16) return 16;
    return KIND == kFloat || rows <= 64 ? 64 : 128;
}
__device__ __forceinline__ int up(int a, int b) { return (a + b - 1) / b; }

// The cost of a unit of n tokens: its start and its tokens, in the order of
// the range that is cut into segments.
template <Kind KIND>
__device__ __forceinline__ int token_cost(const PrefixArgs& a, int rows) {
    return a.cost[KIND == kGeneral || rows <= 16 ? 0 : KIND == kFloat || rows <= 64 ? 1 : 2];
}
template <Kind KIND>
__device__ __forceinline__ long long unit_cost(const PrefixArgs& a, int rows, int n) {
    return n ? a.start_cost + (long long)n * token_cost<KIND>(a, rows) : 0;
}

// The plan, in LDS: sum of the tokens of all units before an entry, granules
// before it, and the groups' first sequences.
struct Plan {
    long long* start;  // [E + 1]
    int* gran;         // [E]
    int* first;        // [G + 1]
    int entries;
    static size_t bytes(int entries, int groups) {
        return 8 * (size_t)(entries + 1) + 4 * (size_t)entries + 4 * (size_t)(groups + 1);
    }
};

// offsets in [0, batch] and not falling, whatever their values: the running
// maximum of the clamped ones. So no sequence is in two groups.
__device__ __forceinline__ int clamped_offset(const PrefixArgs& a, int g) {
    if (!a.offsets) return g ? a.batch : 0;
    return min(max(a.offsets[g], 0), a.batch);
}

__device__ __forceinline__ int entry_tokens(const PrefixArgs& a, int e) {
    return e < a.groups ? clamp_len(a.plens, e, a.pwidth * (int)a.page.d)
                        : clamp_len(a.lens, e - a.groups, a.twidth * (int)a.page.d);
}
__device__ __forceinline__ int entry_rows(const PrefixArgs& a, const Plan& p, int e) {
    return e < a.groups ? (p.first[e + 1] - p.first[e]) * a.gq : a.gq;
}

template <Kind KIND>
__device__ void make_plan(const PrefixArgs& a, const Plan& p, long long* s_sum, int* s_cnt) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the groups' first sequences: thread t takes offsets [t per, ...)
    {
        const int n = a.groups + 1, per = up(n, 256);
        const int lo = min(tid * per, n), hi = min(lo + per, n);
        int most = 0;
        for (int g = lo; g < hi; ++g) p.first[g] = most = max(most, clamped_offset(a, g));
        int run = most;
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(run, o, 64);
            if (lane >= o) run = max(run, x);
        }
        if (lane == 63) s_cnt[wave] = run;
        int before = __shfl_up(run, 1, 64);
        if (lane == 0) before = 0;
        __syncthreads();
        for (int w = 0; w < wave; ++w) before = max(before, s_cnt[w]);
        for (int g = lo; g < hi; ++g) p.first[g] = max(p.first[g], before);
        __syncthreads();
    }
    const int E = p.entries, per = up(E, 256);
    const int lo = min(tid * per, E), hi = min(lo + per, E);
    long long sum = 0;
    int gran = 0;
    for (int e = lo; e < hi; ++e) {
        const int rows = entry_rows(a, p, e);
        p.start[e] = sum;
        p.gran[e] = gran;
        sum += unit_cost<KIND>(a, rows, entry_tokens(a, e)) * a.hkv *
               up(rows, tile_rows<KIND>(rows));
        gran += a.hkv * up(rows, kGranule);
    }
    long long s = sum;
    int c = gran;
    for (int o = 1; o < 64; o <<= 1) {
        const long long x = __shfl_up(s, o, 64);
        const int y = __shfl_up(c, o, 64);
        if (lane >= o) s += x, c += y;
    }
    if (lane == 63) s_sum[wave] = s, s_cnt[wave] = c;
    __syncthreads();
    s -= sum, c -= gran;
    for (int w = 0; w < wave; ++w) s += s_sum[w], c += s_cnt[w];
    for (int e = lo; e < hi; ++e) p.start[e] += s, p.gran[e] += c;
    if (tid == 255) p.start[E] = s + sum;
    __syncthreads();
}

// The cost of a segment: an equal share.
__device__ __forceinline__ long long segment(const PrefixArgs& a, long long total) {
    const long long s = (total + a.segs - 1) / a.segs;
    return s < a.min_seg ? a.min_seg : s;
}

// The combine's copy of the plan, sequence by sequence.
template <Kind KIND>
__device__ void leave_plan(const PrefixArgs& a, const Plan& p, long long seg) {
    if (threadIdx.x == 0) *a.seg = seg;
    auto part = [&](int e, int first) {
        const int n = entry_tokens(a, e), rows = entry_rows(a, p, e);
        return Part{p.start[e] + a.start_cost, unit_cost<KIND>(a, rows, n), p.gran[e], n, rows,
                    first};
    };
    for (int b = threadIdx.x; b < a.batch; b += 256) {
        int lo = 0, hi = a.groups;  // the last g with first[g] <= b
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            (p.first[mid] <= b ? lo : hi) = mid;
        }
        Parts x{};
        if (a.groups > 0 && p.first[lo] <= b && b < p.first[lo + 1]) x.prefix = part(lo, p.first[lo]);
        x.own = part(a.groups + b, b);
        a.parts[b] = x;
    }
}

// A segment's piece that starts at pos: the unit's tokens whose costs begin in
// the segment; none where that is the unit's start alone.
struct Piece {
    int entry, first, rows, kv, row0;  // row0: the tile's first row
    int t0, n;
    const int* table;
    size_t slot;     // its partials' first row
    long long next;  // the position behind it
};
template <Kind KIND>
__device__ __forceinline__ Piece piece_at(const PrefixArgs& a, const Plan& p, long long pos,
                                          long long end) {
    int lo = 0, hi = p.entries;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (p.start[mid] <= pos ? lo : hi) = mid;
    }
    Piece x;
    x.entry = __builtin_amdgcn_readfirstlane(lo);
    const int n = entry_tokens(a, x.entry);
    x.rows = entry_rows(a, p, x.entry);
    const bool own = x.entry >= a.groups;
    x.first = own ? x.entry - a.groups : p.first[x.entry];
    const int tr = tile_rows<KIND>(x.rows), tiles = up(x.rows, tr);
    const int w = token_cost<KIND>(a, x.rows);
    const long long whole = unit_cost<KIND>(a, x.rows, n), off = pos - p.start[x.entry];
    const int unit = (int)(off / whole);
    const long long in = off - unit * whole, base = pos - in;
    const long long stop = min(whole, end - base);
    auto token = [&](long long c) {
        // (below 2^34: the float64 quotient's floor is exact)
        return c <= a.start_cost ? 0 : (int)((double)(c - a.start_cost + w - 1) / (double)w);
    };
    x.t0 = token(in);
    x.n = token(stop) - x.t0;
    x.next = base + stop;
    x.kv = unit / tiles;
    const int tile = unit - x.kv * tiles;
    x.row0 = tile * tr;
    x.table = own ? a.table + (size_t)x.first * a.twidth : a.ptable + (size_t)x.entry * a.pwidth;
    const size_t gran = (size_t)kTileGranules * blockIdx.x + p.gran[x.entry] +
                        (size_t)x.kv * up(x.rows, kGranule) + tile * (tr / kGranule);
    x.slot = gran * kGranule;
    // (the same in every lane)
    x.first = __builtin_amdgcn_readfirstlane(x.first);
    x.rows = __builtin_amdgcn_readfirstlane(x.rows);
    x.kv = __builtin_amdgcn_readfirstlane(x.kv);
    x.row0 = __builtin_amdgcn_readfirstlane(x.row0);
    x.t0 = __builtin_amdgcn_readfirstlane(x.t0);
    x.n = __builtin_amdgcn_readfirstlane(x.n);
    x.slot = (size_t)uniform64((long long)x.slot);
    x.next = uniform64(x.next);
    return x;
}

// Row r of an entry: sequence first + r / gq, q head kv * gq + r % gq.
__device__ __forceinline__ size_t q_row(const PrefixArgs& a, const Piece& p, int r) {
    const int s = a.gdiv.div(r);
    return (size_t)(p.first + s) * a.hq + (size_t)p.kv * a.gq + (r - s * a.gq);
}

// ---------------------------------------------------------------------------
// bf16 / fp16 on the matrix cores, dim a multiple of 8 up to D (64 or 128; a
// smaller dim's missing 16-byte chunks are zero), 16-byte aligned.
//
// A step is 64 tokens: K and V rows go through two LDS stages, the next one's
// loads in flight while this one is computed. Everything is transposed, so an
// accumulator's lane holds one row (r = lane % 16, g = lane / 16; operands of
// v_mfma_f32_16x16x32: A[r][8g+j], B[8g+j][r], C[4g+i][r]):
//
//   scores  S^T[key][row] = K . Q^T, Q in registers for the whole piece;
//   softmax online, a row's keys in 4 lanes; the maximum moves only when a
//           step's exceeds it by 8 (log2), so weights are at most 2^8;
//   PV      O^T[dim][row] += V^T . P^T, P straight from the scores: lane (r, g)
//           holds keys 4g+i of each block of 16, so two blocks fill its 8
//           slots, and V^T comes in the same order by ds_read_b64_tr_b16.
//   weights in parts of the storage type, what one leaves in the next: three
//           for bf16, 8 bits each, all 24 of a float32; two for fp16, 22 bits
//           (2^-22 of a weight, as the exponential's own error; there times 2^7,
//           so that parts down to 2^-32 of the maximum are held). Sums are
//           float32.
//
// Tiles of up to 16 rows (KEYS): wave w takes keys 16w .. of each step with a
// softmax of its own, merged at the piece's end. One block of 16 keys leaves
// half of the slots empty: they hold the second parts, against the same V.
// Larger ones: 16 QB rows a wave, all 64 keys, a product for each part.
// ---------------------------------------------------------------------------
template <typename T> struct PMma;
template <> struct PMma<bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static constexpr float kUp = 1.0f;
    static constexpr int kParts = 3;
    __device__ __forceinline__ static f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // two weights' parts, packed, each the upper half of what is left
    __device__ __forceinline__ static void split(float a, float b, int (&part)[kParts]) {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const unsigned u = __float_as_uint(a), w = __float_as_uint(b);
            part[i] = (int)((u >> 16) | (w & 0xffff0000u));
            a -= __uint_as_float(u & 0xffff0000u);
            b -= __uint_as_float(w & 0xffff0000u);
        }
    }
};
template <> struct PMma<f16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static constexpr float kUp = 128.0f;
    static constexpr int kParts = 2;
    __device__ __forceinline__ static f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    // (the first truncated, the second rounded)
    __device__ __forceinline__ static void split(float a, float b, int (&part)[kParts]) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef f16 t2 __attribute__((ext_vector_type(2)));
        const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
        const f2 rest = {a - (float)h[0], b - (float)h[1]};
        part[0] = __builtin_bit_cast(int, h);
        part[1] = __builtin_bit_cast(int, __builtin_convertvector(rest, t2));
    }
};

template <int D>
struct PCfg {
    static constexpr int kPitch = 2 * D + 16;        // bytes of a staged row
    static constexpr int kStage = 2 * 64 * kPitch;   // K rows, then V rows
    static constexpr int kChunks = 64 * D / 8 / 256; // 16-byte chunks a thread, each of K and V
    static constexpr int kS = D / 32;                // k-steps of the scores
    static constexpr int kDB = D / 16;               // blocks of dims
};

// A lane's share of its row's partials: D / 16 times 4 dims, piece(x, d) giving
// the x-th and its first dim. KEYS: the waves' softmaxes over their keys are
// merged through LDS first.
template <int D, bool FULL, bool KEYS, typename F>
__device__ __forceinline__ void leave_partials(const PrefixArgs& a, const Piece& pc, int r, float m,
                                               float l, float scale, char* smem,
                                               float (*s_ml)[2][16], F&& piece) {
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int dim = FULL ? D : a.dim;
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if constexpr (!KEYS) {
        if (r >= pc.rows) return;
        const size_t row = pc.slot + (r - pc.row0);
        if (g == 0) {
            a.ml[2 * row] = m;
            a.ml[2 * row + 1] = l;
        }
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            int d;
            const f32x4 v = piece(x, d);
            if (FULL || d < dim) *reinterpret_cast<f32x4*>(a.acc + row * dim + d) = v * scale;
        }
    } else {
        constexpr int kRow = D + 4;
        float* const s_acc = reinterpret_cast<float*>(smem);
        if (g == 0) {
            s_ml[wave][0][r16] = m;
            s_ml[wave][1][r16] = l;
        }
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            int d;
            const f32x4 v = piece(x, d);
            *reinterpret_cast<f32x4*>(s_acc + (16 * wave + r16) * kRow + d) = v;
        }
        __syncthreads();
        const int rr = tid >> 4;
        if (pc.row0 + rr < pc.rows) {
            float top = -INFINITY, sum = 0.f, f[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ml[w][0][rr]);
            const float top_use = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                f[w] = __builtin_amdgcn_exp2f(s_ml[w][0][rr] - top_use);
                sum += f[w] * s_ml[w][1][rr];
            }
            const size_t row = pc.slot + rr;
            if ((tid & 15) == 0) {
                a.ml[2 * row] = top;
                a.ml[2 * row + 1] = sum;
            }
#pragma unroll
            for (int x = 0; x < D / 64; ++x) {
                const int d = 64 * x + 4 * (tid & 15);
                f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    y += f[w] * *reinterpret_cast<const f32x4*>(s_acc + (16 * w + rr) * kRow + d);
                if (FULL || d < dim)
                    *reinterpret_cast<f32x4*>(a.acc + row * dim + d) = y * scale;
            }
        }
        __syncthreads();
    }
}

template <typename T, int D, bool FULL, int QB, bool KEYS>
__device__ __forceinline__ void prefix_piece(const PrefixArgs& a, const Piece& pc, char* smem,
                                             float (*s_ml)[2][16]) {
    using M = PMma<T>;
    using V8 = typename M::v8;
    using C = PCfg<D>;
    constexpr int KB = KEYS ? 1 : 4;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int dim = FULL ? D : a.dim;
    const T* const kp = (const T*)a.k;
    const T* const vp = (const T*)a.v;

    // the wave's Q as B operands; rows past the entry's are zero
    const int wrow = pc.row0 + (KEYS ? 0 : 16 * QB * wave);  // its first row
    const bool active = wrow < pc.rows;
    V8 qf[QB][C::kS];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int r = wrow + 16 * qb + r16;
        const bool on = r < pc.rows;
        const T* const row = (const T*)a.q + q_row(a, pc, on ? r : pc.row0) * dim;
#pragma unroll
        for (int s = 0; s < C::kS; ++s) {
            V8 x = {};
            if (on && (FULL || 32 * s + 8 * g < dim))
                x = *reinterpret_cast<const V8*>(row + 32 * s + 8 * g);
            qf[qb][s] = x;
        }
    }

    const int steps = (pc.n + 63) >> 6;
    // Nothing of a step's loads is waited for or branched on before its turn:
    // lane l's table entry of step st (past the piece: its last token's) ..
    auto entry_of = [&](int st) {
        return pc.table[a.page.div(pc.t0 + min(64 * st + lane, pc.n - 1))];
    };
    // .. which of them count: in the piece, and a block of the pools
    auto held_of = [&](int st, int ent) {
        return __builtin_amdgcn_ballot_w64(64 * st + lane < pc.n &&
                                           (unsigned)ent < (unsigned)a.blocks);
    };
    // .. and the rows, 16 bytes a thread; block 0's where there is none
    const int ch = tid % (D / 8);
    const bool ch_on = FULL || 8 * ch < dim;
    const size_t col = ch_on ? 8 * ch : 0;
    struct Rows {
        i32x4 k[C::kChunks], v[C::kChunks];
    };
    auto load = [&](int st, int ent, Rows& x) {
        ent = (unsigned)ent < (unsigned)a.blocks ? ent : 0;
#pragma unroll
        for (int j = 0; j < C::kChunks; ++j) {
            const int row = (tid + 256 * j) / (D / 8);
            const int e = __shfl(ent, row, 64);
            const int t = pc.t0 + min(64 * st + row, pc.n - 1);
            const size_t off =
                (((size_t)e * a.hkv + pc.kv) * a.page.d + a.page.mod(t)) * dim + col;
            if constexpr (KEYS) {  // read once
                x.k[j] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(kp + off));
                x.v[j] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(vp + off));
            } else {
                x.k[j] = *reinterpret_cast<const i32x4*>(kp + off);
                x.v[j] = *reinterpret_cast<const i32x4*>(vp + off);
            }
        }
    };
    // rows that do not count are zero, so that nothing in them is infinite
    auto stage = [&](int st, unsigned long long held, Rows& x) {
        char* const ks = smem + (st & 1) * C::kStage;
        char* const vs = ks + 64 * C::kPitch;
        if (held != ~0ull || !FULL) {
#pragma unroll
            for (int j = 0; j < C::kChunks; ++j)
                if (!ch_on || !(held >> ((tid + 256 * j) / (D / 8)) & 1))
                    x.k[j] = x.v[j] = i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < C::kChunks; ++j) {
            const int at = (tid + 256 * j) / (D / 8) * C::kPitch + 16 * ch;
            *reinterpret_cast<i32x4*>(ks + at) = x.k[j];
            *reinterpret_cast<i32x4*>(vs + at) = x.v[j];
        }
    };

    f32x4 o[C::kDB][QB];
#pragma unroll
    for (int db = 0; db < C::kDB; ++db)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run[QB], l_run[QB];  // the maximum in log2 units, as it was subtracted
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) m_run[qb] = -INFINITY, l_run[qb] = 0.f;
    const float c2 = a.scale_log2;

    auto compute = [&](int st, unsigned long long held) {
        if (active) {
            const char* const ks = smem + (st & 1) * C::kStage;
            const char* const vs = ks + 64 * C::kPitch;
            const int k0 = KEYS ? 16 * wave : 0;  // the wave's first key
            // the softmax and the staging go ahead of the SIMD's other wave's
            // matrix instructions, which fill the gaps
            __builtin_amdgcn_s_setprio(0);
            f32x4 sc[KB][QB];
#pragma unroll
            for (int s = 0; s < C::kS; ++s)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const V8 kf = *reinterpret_cast<const V8*>(
                        ks + (k0 + 16 * kb + r16) * C::kPitch + (32 * s + 8 * g) * 2);
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb)
                        sc[kb][qb] = M::mma(kf, qf[qb][s],
                                            s ? sc[kb][qb] : f32x4{0.f, 0.f, 0.f, 0.f});
                }
            __builtin_amdgcn_s_setprio(1);
            if (held != ~0ull) {  // past the piece, or no block
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const unsigned bits = (unsigned)(held >> (k0 + 16 * kb + 4 * g));
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(bits >> i & 1)) {
#pragma unroll
                            for (int qb = 0; qb < QB; ++qb) sc[kb][qb][i] = -INFINITY;
                        }
                }
            }
            constexpr int KS = KEYS ? 1 : 2;  // k-steps of the PV product
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                float top = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[kb][qb][i]);
                top = max4_rows(top) * c2;
                const bool moved = top > m_run[qb] + 8.0f;
                const float m_new = moved ? top : m_run[qb];
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = __builtin_amdgcn_exp2f(m_run[qb] - m_use);
                m_run[qb] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sc[kb][qb][i] = __builtin_amdgcn_exp2f(fmaf(sc[kb][qb][i], c2, -m_use));
                        sum += sc[kb][qb][i];
                    }
                l_run[qb] = l_run[qb] * alpha + sum;
                if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
                    for (int db = 0; db < C::kDB; ++db) o[db][qb] *= alpha;
                }
            }
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                // the weights' operands: a part each, or (KEYS) two of them in one
                constexpr int OPS = KEYS ? (M::kParts + 1) / 2 : M::kParts;
                i32x4 pw[QB][OPS];
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int w = 0; w < (KEYS ? 2 : 4); ++w) {
                        const f32x4 p = sc[KEYS ? 0 : 2 * x + (w >> 1)][qb];
                        int part[M::kParts];
                        M::split(p[2 * (w & 1)] * M::kUp, p[2 * (w & 1) + 1] * M::kUp, part);
#pragma unroll
                        for (int i = 0; i < (KEYS ? 2 * OPS : OPS); ++i)
                            pw[qb][KEYS ? i / 2 : i][KEYS ? w + 2 * (i & 1) : w] =
                                i < M::kParts ? part[i] : 0;
                    }
                __builtin_amdgcn_s_setprio(0);
                // V^T: dims 16 db + r, keys k0 + 32 x + 4g + (0..3) and 16 more
#pragma unroll
                for (int db = 0; db < C::kDB; ++db) {
                    typedef short v4s __attribute__((ext_vector_type(4)));
                    typedef short v8s __attribute__((ext_vector_type(8)));
                    const char* const p = vs + (k0 + 32 * x + 4 * g + (r16 >> 2)) * C::kPitch +
                                          (16 * db + 4 * (r16 & 3)) * 2;
                    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) v4s*)(p));
                    v4s hi = lo;
                    if constexpr (!KEYS)
                        hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) v4s*)(p + 16 * C::kPitch));
                    const v8s vt = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    const V8 vf = __builtin_bit_cast(V8, vt);
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                        for (int i = 0; i < OPS; ++i)
                            o[db][qb] = M::mma(vf, __builtin_bit_cast(V8, pw[qb][i]), o[db][qb]);
                }
            }
        }
        __builtin_amdgcn_s_setprio(1);
    };
    // (Loads of two steps ahead, where 16 rows a wave leave the registers, were
    // no faster: 64 sequences of 4000 tokens 174 for 169 us.)
    int ent = entry_of(0), next = entry_of(1);
    unsigned long long held = held_of(0, ent), held_next = 0;
    Rows x;
    load(0, ent, x);
    stage(0, held, x);
    __syncthreads();
    for (int st = 0; st < steps; ++st) {
        if (st + 1 < steps) {
            ent = next;
            next = entry_of(st + 2);
            load(st + 1, ent, x);
            held_next = held_of(st + 1, ent);
        }
        __builtin_amdgcn_sched_barrier(0);  // the loads stay ahead
        compute(st, held);
        if (st + 1 < steps) stage(st + 1, held_next, x);
        held = held_next;
        __syncthreads();
    }

    // lane (r, g) holds dims 16 db + 4g + i of row r
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
        leave_partials<D, FULL, KEYS>(a, pc, wrow + 16 * qb + r16, m_run[qb], l_run[qb],
                                      1.0f / M::kUp, smem, s_ml, [&](int x, int& d) {
                                          d = 16 * x + 4 * g;
                                          return o[x][qb];
                                      });
}

template <typename T, int D, bool FULL>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefix_attn(const PrefixArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float s_ml[4][2][16];
    __shared__ long long s_sum[4];
    __shared__ int s_cnt[4];
    Plan p;
    p.entries = a.groups + a.batch;
    p.start = reinterpret_cast<long long*>(smem + 2 * PCfg<D>::kStage);
    p.gran = reinterpret_cast<int*>(p.start + p.entries + 1);
    p.first = p.gran + p.entries;
    make_plan<kHalf>(a, p, s_sum, s_cnt);
    const long long total = uniform64(p.start[p.entries]);
    const long long seg = segment(a, total);
    if (blockIdx.x == 0) leave_plan<kHalf>(a, p, seg);
    long long pos = (long long)blockIdx.x * seg;
    const long long end = min(pos + seg, total);
    while (pos < end) {
        const Piece pc = piece_at<kHalf>(a, p, pos, end);
        pos = pc.next;
        if (pc.n == 0) continue;
        if (pc.rows <= 16) prefix_piece<T, D, FULL, 1, true>(a, pc, smem, s_ml);
        else if (pc.rows <= 64) prefix_piece<T, D, FULL, 1, false>(a, pc, smem, s_ml);
        else prefix_piece<T, D, FULL, 2, false>(a, pc, smem, s_ml);
    }
}

// ---------------------------------------------------------------------------
// float32 on the float32 matrix instructions, dim a multiple of 4 up to D (64 or
// 128), 16-byte aligned: the same steps of 64 tokens, tiles of 16 rows (KEYS) and
// of 64, one LDS stage. With v_mfma_f32_16x16x4 (A[r][g], B[g][r], C[4g+i][r]) a
// lane reads 4 dims at a time, 16 j + 4g .., and its four products take one of
// them each: any order of dims serves the scores. V is read the same way, dims
// 64 h + 4r .. of key 4g + i, so product c has dims 64 h + 4 m + c for m = 0..15 and a lane
// ends with dims 64 h + 16g + 4i + c. Weights are float32, all 24 bits. What
// bounds it: the matrix cores from 64 rows on (154 TFLOP/s at most), else memory.
// ---------------------------------------------------------------------------
template <int D, bool FULL, bool KEYS>
__device__ __forceinline__ void prefix_piece_f32(const PrefixArgs& a, const Piece& pc, char* smem,
                                                 float (*s_ml)[2][16]) {
    constexpr int kPitch = 4 * D + 16, kChunks = D / 16, KB = KEYS ? 1 : 4;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int dim = FULL ? D : a.dim;
    const float* const kp = (const float*)a.k;
    const float* const vp = (const float*)a.v;
    const int wrow = pc.row0 + (KEYS ? 0 : 16 * wave);
    const bool active = wrow < pc.rows;

    f32x4 qf[kChunks];
    {
        const bool on = wrow + r16 < pc.rows;
        const float* const row = (const float*)a.q + q_row(a, pc, on ? wrow + r16 : pc.row0) * dim;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            qf[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (on && (FULL || 16 * j + 4 * g < dim))
                qf[j] = *reinterpret_cast<const f32x4*>(row + 16 * j + 4 * g);
        }
    }
    const int steps = (pc.n + 63) >> 6;
    // (as prefix_piece)
    auto entry_of = [&](int st) {
        return pc.table[a.page.div(pc.t0 + min(64 * st + lane, pc.n - 1))];
    };
    auto held_of = [&](int st, int ent) {
        return __builtin_amdgcn_ballot_w64(64 * st + lane < pc.n &&
                                           (unsigned)ent < (unsigned)a.blocks);
    };
    const int ch = tid % (D / 4);
    const bool ch_on = FULL || 4 * ch < dim;
    const size_t col = ch_on ? 4 * ch : 0;
    f32x4 kx[kChunks], vx[kChunks];
    auto load = [&](int st, int ent) {
        ent = (unsigned)ent < (unsigned)a.blocks ? ent : 0;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int row = (tid + 256 * j) / (D / 4);
            const int e = __shfl(ent, row, 64);
            const int t = pc.t0 + min(64 * st + row, pc.n - 1);
            const size_t off =
                (((size_t)e * a.hkv + pc.kv) * a.page.d + a.page.mod(t)) * dim + col;
            kx[j] = *reinterpret_cast<const f32x4*>(kp + off);
            vx[j] = *reinterpret_cast<const f32x4*>(vp + off);
        }
    };
    char* const ks = smem;
    char* const vs = smem + 64 * kPitch;
    auto stage = [&](unsigned long long held) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int row = (tid + 256 * j) / (D / 4);
            if (!ch_on || !(held >> row & 1)) kx[j] = vx[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            *reinterpret_cast<f32x4*>(ks + row * kPitch + 16 * ch) = kx[j];
            *reinterpret_cast<f32x4*>(vs + row * kPitch + 16 * ch) = vx[j];
        }
    };
    f32x4 o[D / 64][4];
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[h][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;
    const float c2 = a.scale_log2;
    const int k0 = KEYS ? 16 * wave : 0;

    int ent = entry_of(0), next = entry_of(1);
    load(0, ent);
    unsigned long long held = held_of(0, ent), held_next = 0;
    stage(held);
    __syncthreads();
    for (int st = 0; st < steps; ++st) {
        if (st + 1 < steps) {
            ent = next;
            next = entry_of(st + 2);
            load(st + 1, ent);
            held_next = held_of(st + 1, ent);
        }
        __builtin_amdgcn_sched_barrier(0);  // the loads stay ahead
        if (active) {
            f32x4 sc[KB];
            float top = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                f32x4 part[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) part[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < kChunks; ++j) {
                    const f32x4 kf = *reinterpret_cast<const f32x4*>(
                        ks + (k0 + 16 * kb + r16) * kPitch + (16 * j + 4 * g) * 4);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        part[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c], qf[j][c], part[c], 0,
                                                                       0, 0);
                }
                sc[kb] = (part[0] + part[1]) + (part[2] + part[3]);
                const unsigned bits = (unsigned)(held >> (k0 + 16 * kb + 4 * g));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!(bits >> i & 1)) sc[kb][i] = -INFINITY;
                    top = fmaxf(top, sc[kb][i]);
                }
            }
            const float m_new = fmaxf(m_run, max4_rows(top) * c2);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
            m_run = m_new;
            float sum = 0.f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[kb][i] = __builtin_amdgcn_exp2f(fmaf(sc[kb][i], c2, -m_use));
                    sum += sc[kb][i];
                }
            l_run = l_run * alpha + sum;
            if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
                for (int h = 0; h < D / 64; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[h][c] *= alpha;
            }
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 vf = *reinterpret_cast<const f32x4*>(
                            vs + (k0 + 16 * kb + 4 * g + i) * kPitch + (64 * h + 4 * r16) * 4);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            o[h][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[c], sc[kb][i],
                                                                           o[h][c], 0, 0, 0);
                    }
        }
        __syncthreads();
        if (st + 1 < steps) stage(held_next);
        held = held_next;
        __syncthreads();
    }
    leave_partials<D, FULL, KEYS>(a, pc, wrow + r16, m_run, l_run, 1.0f, smem, s_ml,
                                  [&](int x, int& d) {
                                      d = 64 * (x / 4) + 16 * g + 4 * (x % 4);
                                      return f32x4{o[x / 4][0][x % 4], o[x / 4][1][x % 4],
                                                   o[x / 4][2][x % 4], o[x / 4][3][x % 4]};
                                  });
}

template <int D, bool FULL>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefix_attn_f32(const PrefixArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float s_ml[4][2][16];
    __shared__ long long s_sum[4];
    __shared__ int s_cnt[4];
    Plan p;
    p.entries = a.groups + a.batch;
    p.start = reinterpret_cast<long long*>(smem + 2 * 64 * (4 * D + 16));
    p.gran = reinterpret_cast<int*>(p.start + p.entries + 1);
    p.first = p.gran + p.entries;
    make_plan<kFloat>(a, p, s_sum, s_cnt);
    const long long total = uniform64(p.start[p.entries]);
    const long long seg = segment(a, total);
    if (blockIdx.x == 0) leave_plan<kFloat>(a, p, seg);
    long long pos = (long long)blockIdx.x * seg;
    const long long end = min(pos + seg, total);
    while (pos < end) {
        const Piece pc = piece_at<kFloat>(a, p, pos, end);
        pos = pc.next;
        if (pc.n == 0) continue;
        if (pc.rows <= 16) prefix_piece_f32<D, FULL, true>(a, pc, smem, s_ml);
        else prefix_piece_f32<D, FULL, false>(a, pc, smem, s_ml);
    }
}

// ---------------------------------------------------------------------------
// Every other head dim and alignment: 16 rows of a piece against 64
// tokens a step on the vector ALU, which bounds it (64 sequences of 16-2000 tokens
// behind 8192, 32 / 8 heads, D = 256, bf16: 4.7 ms, 592 MB). Thread (row, x) scores tokens x, x + 16, ..
// of the step; then threads own 4 dims of a few rows.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void prefix_general(const PrefixArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ long long s_sum[4];
    __shared__ int s_cnt[4];
    __shared__ long long s_off[64];  // the step's rows in the pools, -1: none
    __shared__ float s_p[16][64], s_alpha[16];
    const int tid = threadIdx.x, dim = a.dim, dc = dim / 4;
    float* const s_q = reinterpret_cast<float*>(smem);  // [16][dim]
    Plan p;
    p.entries = a.groups + a.batch;
    p.start = reinterpret_cast<long long*>(smem + 64 * (size_t)dim);
    p.gran = reinterpret_cast<int*>(p.start + p.entries + 1);
    p.first = p.gran + p.entries;
    make_plan<kGeneral>(a, p, s_sum, s_cnt);
    const long long total = uniform64(p.start[p.entries]);
    const long long seg = segment(a, total);
    if (blockIdx.x == 0) leave_plan<kGeneral>(a, p, seg);
    const T* const kp = (const T*)a.k;
    const T* const vp = (const T*)a.v;

    const int row = tid >> 4, x16 = tid & 15;
    // dims 4 d4 .. of rows y0, y0 + ys, ..
    const int ys = 256 / dc < 16 ? 256 / dc : 16;
    const int d4 = tid % dc, y0 = tid / dc;

    long long pos = (long long)blockIdx.x * seg;
    const long long end = min(pos + seg, total);
    while (pos < end) {
        const Piece pc = piece_at<kGeneral>(a, p, pos, end);
        pos = pc.next;
        if (pc.n == 0) continue;
        const int rows = min(16, pc.rows - pc.row0);
        for (int i = tid; i < 16 * dim; i += 256) {
            const int r = i / dim;
            s_q[i] = r < rows ? St<T>::ld((const T*)a.q + q_row(a, pc, pc.row0 + r) * dim +
                                          (i - r * dim)) : 0.f;
        }
        float4 acc[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) acc[y] = make_float4(0.f, 0.f, 0.f, 0.f);
        float m_run = -INFINITY, l_run = 0.f;
        for (int st = 0; st < pc.n; st += 64) {
            const int n = min(64, pc.n - st);
            if (tid < 64) {
                long long off = -1;
                if (tid < n) {
                    const int t = pc.t0 + st + tid, e = pc.table[a.page.div(t)];
                    if ((unsigned)e < (unsigned)a.blocks)
                        off = (((long long)e * a.hkv + pc.kv) * a.page.d + a.page.mod(t)) * dim;
                }
                s_off[tid] = off;
            }
            __syncthreads();
            float s[4], top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long long off = s_off[x16 + 16 * j];
                s[j] = -INFINITY;
                if (off < 0) continue;
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                for (int c = 0; c < dc; ++c) {
                    const float4 kv = St<T>::ld4(kp + off + 4 * c);
                    const float4 qv = *reinterpret_cast<const float4*>(s_q + row * dim + 4 * c);
                    part[0] = fmaf(kv.x, qv.x, part[0]);
                    part[1] = fmaf(kv.y, qv.y, part[1]);
                    part[2] = fmaf(kv.z, qv.z, part[2]);
                    part[3] = fmaf(kv.w, qv.w, part[3]);
                }
                s[j] = ((part[0] + part[1]) + (part[2] + part[3])) * a.scale_log2;
                top = fmaxf(top, s[j]);
            }
            for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
            const float m_new = fmaxf(m_run, top);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = exp2f(m_run - m_use);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = exp2f(s[j] - m_use);
                s_p[row][x16 + 16 * j] = w;
                sum += w;
            }
            for (int o = 8; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
            l_run = l_run * alpha + sum;
            m_run = m_new;
            if (x16 == 0) s_alpha[row] = alpha;
            __syncthreads();
            if (y0 < ys) {
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    if (y0 + y * ys >= rows) break;
                    const float al = s_alpha[y0 + y * ys];
                    acc[y].x *= al; acc[y].y *= al; acc[y].z *= al; acc[y].w *= al;
                }
                for (int t = 0; t < n; ++t) {
                    const long long off = s_off[t];
                    if (off < 0) continue;
                    const float4 vv = St<T>::ld4(vp + off + 4 * d4);
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        if (y0 + y * ys >= rows) break;
                        const float w = s_p[y0 + y * ys][t];
                        acc[y].x = fmaf(w, vv.x, acc[y].x);
                        acc[y].y = fmaf(w, vv.y, acc[y].y);
                        acc[y].z = fmaf(w, vv.z, acc[y].z);
                        acc[y].w = fmaf(w, vv.w, acc[y].w);
                    }
                }
            }
            __syncthreads();
        }
        if (y0 < ys) {
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                if (y0 + y * ys >= rows) break;
                *reinterpret_cast<float4*>(a.acc + (pc.slot + y0 + y * ys) * dim + 4 * d4) = acc[y];
            }
        }
        if (row < rows && x16 == 0) {
            a.ml[2 * (pc.slot + row)] = m_run;
            a.ml[2 * (pc.slot + row) + 1] = l_run;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// The fold. A workgroup takes HEADS heads of a sequence: one, its pieces shared
// out to the four waves; or, where there are heads enough for every CU, four:
// a wave each, or all waves for one after another where one has many pieces.
// A wave's lanes are
// groups of dim / 4 that take pieces in turn; the first of them are on their
// way before their maxima are known. What bounds it: the chain plan -> maxima
// -> weights (4.5 us), the partials' bytes for long prefixes of many rows.
// ---------------------------------------------------------------------------
constexpr int kAlone = 32;  // pieces of a head that one wave folds
constexpr int kAhead = 4;

// A head's pieces: n0 of the prefix, then n1 of its own tokens.
struct Pieces {
    int n0, n1;
    size_t row0, row1;  // first partials; the next is one segment's granules on
    __device__ __forceinline__ size_t row(int i) const {
        const bool own = i >= n0;
        return (own ? row1 : row0) + (size_t)(kTileGranules * kGranule) * (own ? i - n0 : i);
    }
};

// floor(x / d), below 2^20 (a segment's number): an estimate, one off at most
__device__ __forceinline__ long long quotient(long long x, long long d, double inv) {
    long long q = (long long)((double)x * inv);
    if (q * d > x) --q;
    return (q + 1) * d <= x ? q + 1 : q;
}

template <Kind KIND>
__device__ __forceinline__ void find_pieces(const PrefixArgs& a, const Part& x, long long seg,
                                            double inv, int kv, int b, int j, int& n,
                                            size_t& row) {
    n = 0;
    row = 0;
    if (x.n == 0) return;
    const int r = (b - x.first) * a.gq + j;
    const int tr = tile_rows<KIND>(x.rows);
    const int log = tr == 16 ? 4 : tr == 64 ? 6 : 7, tile = r >> log;
    const int tiles = (x.rows + tr - 1) >> log;
    const long long lo = x.start + ((long long)kv * tiles + tile) * x.whole;
    const long long s0 = quotient(lo, seg, inv);
    const long long hi = lo + (long long)token_cost<KIND>(a, x.rows) * (x.n - 1);
    n = (int)(quotient(hi, seg, inv) - s0) + 1;
    const size_t gran = (size_t)kTileGranules * s0 + x.gran +
                        (size_t)kv * ((x.rows + kGranule - 1) / kGranule) +
                        tile * (tr / kGranule);
    row = gran * kGranule + (r - (tile << log));
}

template <typename T, Kind KIND, int HEADS>
__global__ __launch_bounds__(256) void prefix_combine(const PrefixArgs a) {
    __shared__ Pieces s_pieces[4];
    __shared__ float s_m[4], s_l[4];
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* const s_acc = reinterpret_cast<float*>(smem);  // [4][dim]
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.y, h = HEADS * blockIdx.x + wave % HEADS, dim = a.dim;
    const long long seg = *a.seg;
    const Parts parts = a.parts[b];
    Pieces mine{0, 0, 0, 0};
    if (h < a.hq) {
        const int kv = a.gdiv.div(h), j = h - kv * a.gq;
        const double inv = 1.0 / (double)seg;
        find_pieces<KIND>(a, parts.prefix, seg, inv, kv, b, j, mine.n0, mine.row0);
        find_pieces<KIND>(a, parts.own, seg, inv, kv, b, j, mine.n1, mine.row1);
    }
    if (lane == 0) s_pieces[wave] = mine;
    __syncthreads();
    int most = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) most = max(most, s_pieces[w].n0 + s_pieces[w].n1);

    int size = 1;  // lanes a piece
    while (size < 64 && 4 * size < dim) size *= 2;
    const int groups = 64 / size, group = lane / size, d0 = 4 * (lane & (size - 1));
    // pieces first, first + step, .. of `pc`: their maximum and sum, and 4 dims
    // from d on in the lanes of group 0
    auto fold = [&](const Pieces& pc, int first, int step, int d, float& m, float& l) {
        const int n = pc.n0 + pc.n1;
        float4 x[kAhead];
        float xm[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = first + step * (group + groups * k);
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            xm[k] = -INFINITY;
            if (i < n && d < dim) {
                const size_t r = pc.row(i);
                xm[k] = a.ml[2 * r];
                x[k] = *reinterpret_cast<const float4*>(a.acc + r * dim + d);
            }
        }
        m = -INFINITY;
        l = 0.f;
        float l_first = 0.f, m_first = -INFINITY;
        {
            const int i = first + step * lane;
            if (i < n) {
                const size_t r = pc.row(i);
                m_first = a.ml[2 * r];
                l_first = a.ml[2 * r + 1];
            }
            m = m_first;
        }
        for (int i = first + step * (lane + 64); i < n; i += 64 * step)
            m = fmaxf(m, a.ml[2 * pc.row(i)]);
        m = wave_max(m);
        const float m_use = m == -INFINITY ? 0.f : m;
        l = exp2f(m_first - m_use) * l_first;
        for (int i = first + step * (lane + 64); i < n; i += 64 * step) {
            const size_t r = pc.row(i);
            l += exp2f(a.ml[2 * r] - m_use) * a.ml[2 * r + 1];
        }
        l = wave_sum(l);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float f, const float4& v) {
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
        };
#pragma unroll
        for (int k = 0; k < kAhead; ++k) add(exp2f(xm[k] - m_use), x[k]);
        if (d < dim) {
#pragma unroll 4
            for (int i = first + step * (group + groups * kAhead); i < n; i += step * groups) {
                const size_t r = pc.row(i);
                add(exp2f(a.ml[2 * r] - m_use), *reinterpret_cast<const float4*>(a.acc + r * dim + d));
            }
        }
        for (int o = size; o < 64; o *= 2) {
            acc.x += __shfl_xor(acc.x, o, 64);
            acc.y += __shfl_xor(acc.y, o, 64);
            acc.z += __shfl_xor(acc.z, o, 64);
            acc.w += __shfl_xor(acc.w, o, 64);
        }
        return acc;
    };
    // a sum of 0 (no token) gives zeros, one that is not a number itself
    auto scale = [](float l) { return l > 0.f ? 1.0f / l : l; };

    if (HEADS > 1 && most <= kAlone) {
        if (h >= a.hq) return;
        for (int d = d0; d < ((dim + 255) & ~255); d += 256) {
            float m, l;
            const float4 x = fold(mine, 0, 1, d, m, l);
            const float f = scale(l);
            if (group == 0 && d < dim)
                St<T>::st4((T*)a.out + ((size_t)b * a.hq + h) * dim + d,
                           make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
            if (size < 64) break;
        }
        return;
    }
    for (int k = 0; k < HEADS && HEADS * (int)blockIdx.x + k < a.hq; ++k) {
        const Pieces pc = s_pieces[k];
        for (int d = d0; d < ((dim + 255) & ~255); d += 256) {
            float m, l;
            const float4 x = fold(pc, wave, 4, d, m, l);
            if (group == 0 && d < dim) *reinterpret_cast<float4*>(s_acc + wave * dim + d) = x;
            if (lane == 0) s_m[wave] = m, s_l[wave] = l;
            if (size < 64) break;
        }
        __syncthreads();
        float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
        top = top == -INFINITY ? 0.f : top;
        float f[4], total = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            f[w] = exp2f(s_m[w] - top);
            total += f[w] * s_l[w];
        }
        const float inv = scale(total);
        for (int d = tid; d < dim; d += 256) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) x = fmaf(f[w], s_acc[w * dim + d], x);
            St<T>::st((T*)a.out + ((size_t)b * a.hq + HEADS * blockIdx.x + k) * dim + d, x * inv);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// The cost of a unit's start (its table, Q and first rows arriving, its partials)
// and of a token with up to 16, 64 and 128 rows (float32: up to 16 and 64, where the
// matrix cores bound it). They balance the workgroups:
// with starts free, 16 sequences of 1-500 tokens behind 131071 shared ones took
// 215 us, a few workgroups being full of starts, for 120; 128 rows are bound by
// the matrix cores (64 sequences behind 8192, by graph replays: 78 us at 6, 88 at 4, 80 at 8).
constexpr int kStartCost = 768;
constexpr int kTokenCost[3] = {4, 4, 6}, kTokenCostFloat[3] = {4, 10, 10};
// The least cost of a segment (4 sequences behind 500 tokens, D = 64: 12.5 us, 14.3
// at 1024, 17 at 2048).
constexpr int kMinSegment = 256;

struct PrefixShape {
    int dtype, batch, hq, hkv, groups, page, pwidth, twidth, dim, segs;
    Kind kind;
    size_t ml, acc, parts, seg, bytes;  // offsets in the workspace
};

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

void check_shape(int dtype, int batch, int hq, int hkv, int groups, int page, int pwidth,
                 int twidth, int dim) {
    if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
        inval("attention: unknown element type");
    if (batch < 0 || groups < 0 || hq < 1 || hkv < 1 || pwidth < 0 || twidth < 0)
        inval("attention shapes must satisfy batch, groups, widths >= 0, heads >= 1");
    if (hq % hkv != 0) inval("q heads must be a multiple of kv heads (contiguous GQA groups)");
    if (dim < 4 || dim % 4 != 0 || dim > kMaxDimP)
        inval("dim must be a multiple of 4 and at most 512");
    if (page < 1) inval("page must be >= 1");
    if ((long long)page * pwidth > INT_MAX / 2 || (long long)page * twidth > INT_MAX / 2)
        inval("attention: a table's capacity must be below 2^30 tokens");
    if ((long long)batch + groups > kMaxEntries)
        inval("attention: at most 4096 sequences and groups together");
    if ((long long)batch * hq >= 1 << 24) inval("attention problem too large for one launch");
}

PrefixShape prefix_shape(int dtype, int batch, int hq, int hkv, int groups, int page, int pwidth,
                         int twidth, int dim) {
    PrefixShape s{dtype, batch, hq, hkv, groups, page, pwidth, twidth, dim};
    s.kind = dim > 128 ? kGeneral : dtype == FT_DT_F32 ? kFloat : dim % 8 == 0 ? kHalf : kGeneral;
    s.segs = 2 * dev_info().cu_count;
    const size_t gq = hq / hkv;
    // granules of every unit (the rows of a group that is not empty are rounded
    // up once), and 8 a segment more
    const size_t granules = (size_t)kTileGranules * s.segs +
                            hkv * (batch * gq / kGranule + std::min(groups, batch)) +
                            (size_t)batch * hkv * ((gq + kGranule - 1) / kGranule);
    const size_t rows = granules * kGranule;
    s.ml = 0;
    s.acc = align256(rows * 8);
    s.parts = s.acc + align256(rows * dim * 4);
    s.seg = s.parts + align256(sizeof(Parts) * (size_t)batch);
    s.bytes = s.seg + 256;
    if (batch == 0) s.bytes = 0;
    return s;
}

template <typename T, int D>
void wide_run(const PrefixArgs& a, int segs, hipStream_t s) {
    const size_t lds = 2 * PCfg<D>::kStage + Plan::bytes(a.groups + a.batch, a.groups);
    if (a.dim == D) {
        allow_lds((const void*)prefix_attn<T, D, true>, lds);
        prefix_attn<T, D, true><<<segs, 256, lds, s>>>(a);
    } else {
        allow_lds((const void*)prefix_attn<T, D, false>, lds);
        prefix_attn<T, D, false><<<segs, 256, lds, s>>>(a);
    }
}

template <int D>
void float_run(const PrefixArgs& a, int segs, hipStream_t s) {
    const size_t lds = 2 * 64 * (4 * D + 16) + Plan::bytes(a.groups + a.batch, a.groups);
    if (a.dim == D) {
        allow_lds((const void*)prefix_attn_f32<D, true>, lds);
        prefix_attn_f32<D, true><<<segs, 256, lds, s>>>(a);
    } else {
        allow_lds((const void*)prefix_attn_f32<D, false>, lds);
        prefix_attn_f32<D, false><<<segs, 256, lds, s>>>(a);
    }
}

template <typename T, Kind KIND>
void combine_run(const PrefixArgs& a, hipStream_t s) {
    const size_t lds = 16 * (size_t)a.dim;
    if ((long long)a.batch * a.hq > 4 * dev_info().cu_count)
        prefix_combine<T, KIND, 4><<<dim3((a.hq + 3) / 4, a.batch), 256, lds, s>>>(a);
    else
        prefix_combine<T, KIND, 1><<<dim3(a.hq, a.batch), 256, lds, s>>>(a);
    launch_check("shared-prefix combine kernel launch");
}

template <typename T>
void prefix_run(const PrefixShape& sh, const PrefixArgs& a, hipStream_t s) {
    constexpr Kind kFast = std::is_same<T, float>::value ? kFloat : kHalf;
    if (sh.kind == kGeneral) {
        const size_t lds = 64 * (size_t)sh.dim + Plan::bytes(sh.groups + sh.batch, sh.groups);
        allow_lds((const void*)prefix_general<T>, lds);
        prefix_general<T><<<a.segs, 256, lds, s>>>(a);
        launch_check("shared-prefix attention kernel launch");
        combine_run<T, kGeneral>(a, s);
        return;
    }
    if constexpr (kFast == kFloat) {
        if (sh.dim <= 64) float_run<64>(a, a.segs, s);
        else float_run<128>(a, a.segs, s);
    } else {
        if (sh.dim <= 64) wide_run<T, 64>(a, a.segs, s);
        else wide_run<T, 128>(a, a.segs, s);
    }
    launch_check("shared-prefix attention kernel launch");
    combine_run<T, kFast>(a, s);
}

}  // namespace
}  // namespace ft

using namespace ft;

extern "C" {

int ft_attention_decode_paged_prefix_workspace(int dtype, int batch, int q_heads, int kv_heads,
                                               int groups, int page, int prefix_width,
                                               int tbl_width, int dim, long long* bytes) {
    return guarded([&] {
        if (!bytes) inval("attention: null operand");
        check_shape(dtype, batch, q_heads, kv_heads, groups, page, prefix_width, tbl_width, dim);
        *bytes = (long long)prefix_shape(dtype, batch, q_heads, kv_heads, groups, page,
                                         prefix_width, tbl_width, dim).bytes;
    });
}

int ft_attention_decode_paged_prefix_launch(
    const void* q, int dtype, const void* k_pool, const void* v_pool, const int* prefix_table,
    const int* prefix_lens, const int* group_offsets, const int* table, const int* lens, void* out,
    void* workspace, long long workspace_bytes, int batch, int q_heads, int kv_heads, int groups,
    int blocks, int page, int prefix_width, int tbl_width, int dim, uintptr_t stream) {
    return guarded([&] {
        check_shape(dtype, batch, q_heads, kv_heads, groups, page, prefix_width, tbl_width, dim);
        if (blocks < 0) inval("attention: blocks must be >= 0");
        if (groups > 1 && !group_offsets) inval("attention: several groups need group_offsets");
        if (batch == 0) return;
        if (!q || !out || (groups > 0 && prefix_width > 0 && !prefix_table) ||
            (tbl_width > 0 && !table) || (blocks > 0 && (!k_pool || !v_pool)))
            inval("attention: null operand");
        const size_t by = dtype == FT_DT_F32 ? 16 : 8;   // 4 elements
        auto off = [&](const void* p, size_t n) { return ((uintptr_t)p % n) != 0; };
        if (off(q, by) || off(k_pool, by) || off(v_pool, by) || off(out, by))
            inval("attention: operands must be aligned to 4 elements");
        if (off(workspace, 16)) inval("attention: the workspace must be aligned to 16 bytes");
        PrefixShape sh = prefix_shape(dtype, batch, q_heads, kv_heads, groups, page, prefix_width,
                                      tbl_width, dim);
        if (!workspace || workspace_bytes < (long long)sh.bytes)
            inval("attention: this call needs " + std::to_string(sh.bytes) +
                  " bytes of workspace");
        // whole 16-byte chunks, and a block to read, on the matrix-core path
        if (blocks == 0 || off(q, 16) || off(k_pool, 16) || off(v_pool, 16)) sh.kind = kGeneral;
        char* const ws = (char*)workspace;
        PrefixArgs a{};
        a.q = q;
        a.k = k_pool;
        a.v = v_pool;
        a.ptable = prefix_table;
        a.plens = prefix_lens;
        a.offsets = group_offsets;
        a.table = table;
        a.lens = lens;
        a.out = out;
        a.ml = (float*)(ws + sh.ml);
        a.acc = (float*)(ws + sh.acc);
        a.parts = (Parts*)(ws + sh.parts);
        a.seg = (long long*)(ws + sh.seg);
        a.batch = batch;
        a.hq = q_heads;
        a.hkv = kv_heads;
        a.gq = q_heads / kv_heads;
        a.groups = groups;
        a.blocks = blocks;
        a.pwidth = prefix_width;
        a.twidth = tbl_width;
        a.dim = dim;
        a.page = FastDiv(page);
        a.gdiv = FastDiv(a.gq);
        a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)dim));
        a.segs = sh.segs;
        a.min_seg = kMinSegment;
        a.start_cost = kStartCost;
        for (int i = 0; i < 3; ++i)
            a.cost[i] = sh.kind == kFloat ? kTokenCostFloat[i] : kTokenCost[i];
        // no more workgroups than the tables' capacity can fill
        const long long gq = a.gq, c = a.cost[2];
        const long long most =
            kv_heads * ((batch * gq / kGranule + std::min(groups, batch)) *
                            (kStartCost + c * page * prefix_width) +
                        batch * ((gq + kGranule - 1) / kGranule) *
                            (kStartCost + c * page * tbl_width));
        a.segs = (int)std::min<long long>(sh.segs, most / a.min_seg + 1);
        const hipStream_t s = as_stream(stream);
        if (dtype == FT_DT_F32) prefix_run<float>(sh, a, s);
        else if (dtype == FT_DT_BF16) prefix_run<bf16>(sh, a, s);
        else prefix_run<f16>(sh, a, s);
    });
}

}  // extern "C"
