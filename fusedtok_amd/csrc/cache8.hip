// A paged KV cache held in 8 bits, for gfx950: block tables and slot maps
// from lengths, the append of fresh keys and values, and decode attention.
//
// The cache. k_pool / v_pool are int8 [blocks, kv heads, page, dim], k_scales /
// v_scales float32 [blocks, kv heads]; the value at row r of block n, head h is
// code * scale[n, h]. A slot is block * page + row.
#include "attn_common.hpp"
#include "fast_div.hpp"
#include "ft_common.hpp"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace ft {
namespace {

constexpr int kMaxDim8 = 512;
constexpr int kMaxPage8 = 1024;      // rows of a block (the append's row map in LDS)
constexpr int kExtendSeqs = 4096;    // sequences of one table call (their prefixes in LDS)

void check_pools(int blocks, int hkv, int page, int dim) {
    if (blocks < 0 || hkv < 1 || dim < 1) inval("int8 cache: blocks >= 0, kv heads >= 1, dim >= 1");
    if (dim % 4 != 0 || dim > kMaxDim8)
        inval("int8 cache: dim must be a multiple of 4 and at most 512");
    if (page < 1 || page > kMaxPage8) inval("int8 cache: page must be in [1, 1024]");
    if ((long long)blocks * page > INT_MAX) inval("int8 cache: slots must fit 31 bits");
    if ((long long)blocks * page * hkv > UINT_MAX)
        inval("int8 cache: blocks * page * kv heads must fit 32 bits");
}

// Rows are read 4 elements at a time at least: every row starts at a multiple
// of 4 elements (dim % 4 == 0) where the tensor does.
void check_aligned(const void* p, size_t bytes, const char* what) {
    if ((uintptr_t)p % bytes)
        inval(std::string("int8 cache: ") + what + " must be aligned to " +
              std::to_string(bytes) + " bytes");
}
inline size_t size_of(int dtype) { return dtype == FT_DT_F32 ? 4 : 2; }

// ---------------------------------------------------------------------------
// Block tables and slot maps.
//
// Sequence b holds lens[b] tokens in ceil(lens[b] / P) blocks and gets
// counts[b] more: with end_b = min(lens[b] + counts[b], S P) it needs
// n_b = ceil(end_b / P) - ceil(lens[b] / P) fresh blocks. With N_b the sum of
// n over the sequences before it, its j-th is free[n_free - 1 - (N_b + j)],
// -1 where the list has no such entry. Fresh token i of sequence b sits at
// position lens[b] + i, at row (sum of counts before b) + i of the outputs.
//
// Every workgroup scans the lengths by itself (a few thousand at most, from
// L2) and takes its share of the tokens and of the fresh blocks, finding a
// token's sequence in the prefix by bisection: one launch without a hand-over
// between workgroups. A token's slot is worked out from the free list, not
// from the table entry that another workgroup may be writing. What bounds it:
// launch and the dependent chain length -> scan -> bisection -> table: 3.9 us
// for 64 sequences, 7.3 for 2000, 5.4 for 125k tokens of 32 prompts.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void block_table_extend_kernel(
    int* __restrict__ table, const int* __restrict__ lens, const int* __restrict__ counts,
    const int* __restrict__ free_blocks, int free_len, const int* __restrict__ n_free,
    int* __restrict__ slots, int* __restrict__ positions, int* __restrict__ offsets,
    int* __restrict__ lens_out, int* __restrict__ n_free_out, int batch, FastDiv page, int width,
    int tokens) {
    constexpr int PER = kExtendSeqs / 256;
    __shared__ int s_off[kExtendSeqs + 1];   // fresh tokens before sequence b (saturated)
    __shared__ int s_need[kExtendSeqs + 1];  // fresh blocks before sequence b
    __shared__ int s_len[kExtendSeqs];
    __shared__ long long s_toks[4];
    __shared__ int s_blocks[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int span = width * (int)page.d;  // <= 2^30
    const int have = *n_free;

    // each thread's run of sequences, all loaded before any is used
    const int per = (batch + 255) / 256, b0 = tid * per;
    int len[PER], add[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool in = i < per && b0 + i < batch;
        len[i] = in ? lens[b0 + i] : 0;
        add[i] = in ? counts[b0 + i] : 0;
    }
    long long toks = 0;
    int need = 0;  // all sequences': at most the table's entries, which fit
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        len[i] = min(max(len[i], 0), span);
        add[i] = max(add[i], 0);
        toks += add[i];
        need += page.up(len[i] + min(add[i], span - len[i])) - page.up(len[i]);
    }
    long long it = toks;  // inclusive over the wave, then the workgroup
    int in = need;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long yt = __shfl_up(it, o, 64);
        const int yn = __shfl_up(in, o, 64);
        if (lane >= o) {
            it += yt;
            in += yn;
        }
    }
    if (lane == 63) {
        s_toks[wave] = it;
        s_blocks[wave] = in;
    }
    __syncthreads();
    long long rt = it - toks, all = 0;
    int rn = in - need, fresh = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) {
            rt += s_toks[w];
            rn += s_blocks[w];
        }
        all += s_toks[w];
        fresh += s_blocks[w];
    }
    const int total = (int)min(all, (long long)INT_MAX);
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (i < per && b0 + i < batch) {
            const int b = b0 + i, off = (int)min(rt, (long long)INT_MAX);
            const int end = len[i] + min(add[i], span - len[i]);
            s_off[b] = off;
            s_need[b] = rn;
            s_len[b] = len[i];
            if (blockIdx.x == 0) {
                offsets[b] = off;
                lens_out[b] = end;
            }
            rt += add[i];
            rn += page.up(end) - page.up(len[i]);
        }
    if (tid == 0) {
        s_off[batch] = total;
        s_need[batch] = fresh;
        if (blockIdx.x == 0) {
            offsets[batch] = total;
            *n_free_out = (int)max((long long)have - fresh, (long long)INT_MIN);
        }
    }
    __syncthreads();

    // last b of s[0..batch) with s[b] <= x (x < s[batch])
    auto find = [&](const int* s, int x) {
        int lo = 0, hi = batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s[mid] <= x) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    auto taken = [&](int k) {  // the k-th fresh block
        const long long at = (long long)have - 1 - k;
        return at >= 0 && at < free_len ? free_blocks[at] : -1;
    };

    // the tokens, then the fresh blocks
    const long long items = (long long)tokens + fresh, stride = gridDim.x * 256;
    for (long long t = blockIdx.x * 256 + tid; t < items; t += stride) {
        if (t >= tokens) {
            const int k = (int)(t - tokens), b = find(s_need, k);
            table[(size_t)b * width + page.up(s_len[b]) + (k - s_need[b])] = taken(k);
            continue;
        }
        int slot = -1, pos = 0;
        if (t < total) {
            const int b = find(s_off, (int)t), n = s_len[b];
            const long long p = (long long)n + (t - s_off[b]);
            pos = (int)min(p, (long long)INT_MAX);
            if (p < span) {
                const int col = page.div(pos), first = page.up(n);
                const int block = col < first ? table[(size_t)b * width + col]
                                              : taken(s_need[b] + col - first);
                const long long s = (long long)block * (int)page.d + (pos - col * (int)page.d);
                if (block >= 0 && s <= INT_MAX) slot = (int)s;
            }
        }
        slots[t] = slot;
        positions[t] = pos;
    }
}

// ---------------------------------------------------------------------------
// Append. Fresh row i (k_new[i], v_new[i]: [kv heads, dim]) goes to slot
// slots[i]; a slot outside the pools is skipped. The rows next to each other
// in `slots` that share a block are a run. With a = max |x| over a run's
// finite values of one head,
//   scale' = max(held, f32(a / 127), 2^-120),
//   code   = clamp(rint(f32(x * f32(1 / scale'))), -127, 127), NaN -> 0,
// held being the block's scale, or 0 where row 0 is in the run (the block
// starts over). Where scale' > held and row 0 is not in the run, the block's
// other rows become rint(f32(code * f32(held / scale'))): zeros where held was
// 0. All float32, IEEE divisions: codes are the same on every path.
// ---------------------------------------------------------------------------
constexpr float kLeastScale = 0x1p-120f;

__device__ __forceinline__ signed char code8(float x, float inv) {
    const float v = rintf(x * inv);
    return v == v ? (signed char)fmaxf(-127.0f, fminf(127.0f, v)) : (signed char)0;
}

// V values of a row as they are stored, in 32-bit words.
template <typename T, int V>
struct Raw {
    static constexpr int kWords = V * (int)sizeof(T) / 4;
    // the bits of the type's infinity: magnitudes from there are not finite
    static constexpr unsigned kInf = sizeof(T) == 4 ? 0x7f800000u
                                     : std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;
    typedef unsigned vec __attribute__((ext_vector_type(kWords)));
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    vec w;
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T* p) {
        w = *reinterpret_cast<const vec*>(p);
    }
    // max of m and the magnitudes' bits (both halves of m for a 16-bit type):
    // magnitudes order as their bits do
    __device__ __forceinline__ unsigned most(unsigned m) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4)
                m = max(m, w[i] & 0x7fffffffu);
            else
                m = __builtin_bit_cast(
                    unsigned,
                    __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                              __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu)));
        }
        return m;
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return value_of(w[i / 2] >> (i % 2 * 16));
    }
    static __device__ __forceinline__ float value_of(unsigned bits) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
        else return (float)__builtin_bit_cast(T, (unsigned short)bits);
    }
};

// Low bytes of rint(x inv) of four values, |x inv| < 127.5: added to 1.5 * 2^23
// the product rounds to a whole number, half to even, whose low byte is the
// sum's. The product is rounded by itself first.
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d, float inv) {
#pragma clang fp contract(off)
    constexpr float kWhole = 12582912.0f;
    const unsigned x = __float_as_uint(a * inv + kWhole), y = __float_as_uint(b * inv + kWhole);
    const unsigned z = __float_as_uint(c * inv + kWhole), w = __float_as_uint(d * inv + kWhole);
    return __builtin_amdgcn_perm(y, x, 0x0c0c0400u) | __builtin_amdgcn_perm(w, z, 0x04000c0cu);
}

template <int V>
struct Codes {
    unsigned w[V / 4];
} __attribute__((aligned(V)));

// UT threads (a wave or a workgroup) have a run, kv head and pool at a time.
// How runs are found is chosen by the number of fresh rows, since how many
// there are a run the host does not know:
//   few rows        (a decode step) a unit a row; those that start no run end;
//   up to 1024      every workgroup lists the starts of all runs in LDS, and
//                   the units share them out;
//   more            a unit a window of as many rows as a block has (64 at most):
//                   the runs that start in it, one after another (about one, in
//                   prompts).
// (8 heads, D = 128, blocks of 16, graph replays, us, the three in turn: a step
// of 64 sequences 5.1, 6.2, 23.8, of 512 8.4, 8.7, 23.2, of 1024 12.6, 13.2, 23.4;
// a prompt of 512 tokens 9.7, 6.3, 5.8, of 2048 28.7, 10.3, 6.2.)
// A lane has V values of a row; the first kKeep passes of a run
// stay in registers between the maximum and the codes, so a run is read once.
// Rows in order, as a sequence's are, need no map; others (gaps, a slot twice)
// go by a map in LDS from the block's row to the last fresh row for it. Values
// stay as they are stored: the maximum is one of their bits (two instructions
// for two 16-bit values), and only a run with an infinity or NaN in it, which
// the maximum shows, goes through the code that looks at each value.
//
// What bounds it: memory latency in a decode step (4 us for 64 rows); a step
// whose scales grow reads and writes its blocks' other rows too (graph replays,
// 64 rows 4.4 us for 4.3, of blocks of 64 6.8 for 5.2, 512 rows 12.0 for 8.1). For
// prompts, HBM: 30k rows, 8 heads, D = 128, bf16, 38.7 us, 4.7 TB/s read and
// written, where a large copy has 4.8. (Values widened and compared one by one:
// 61 us, bound by the vector ALU.)
constexpr long long kRowEach = 16;  // units a CU, at most, where each row has its own
constexpr int kListTokens = 1024;   // rows whose runs are listed, at most
constexpr int kListWgs = 4;         // workgroups a CU of a listed call, at most

template <typename T, int V, int UT, bool LISTED>
__global__ __launch_bounds__(256) void kv_append8_kernel(
    const T* __restrict__ k_new, const T* __restrict__ v_new, const int* __restrict__ slots,
    signed char* __restrict__ k_pool, signed char* __restrict__ v_pool,
    float* __restrict__ k_scales, float* __restrict__ v_scales, int tokens, FastDiv heads, int dim,
    int nslots, FastDiv page, FastDiv lanes, int window, long long first_wg, long long units) {
    constexpr int kKeep = 4, kUnits = 256 / UT;
    __shared__ int s_map[kUnits][kMaxPage8];
    __shared__ int s_runs[LISTED ? kListTokens : 1];
    __shared__ unsigned s_red[4];
    const int lane = threadIdx.x & 63;
    const int ut = UT == 64 ? lane : (int)threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long unit = (first_wg + blockIdx.x) * kUnits + (UT == 64 ? wave : 0);
    if (!LISTED && unit >= units) return;
    int* const map = s_map[UT == 64 ? wave : 0];
    const int hkv = (int)heads.d;
    const size_t row_stride = (size_t)hkv * dim;
    auto sync = [&] {
        if (UT == 64) wave_lds_order();
        else __syncthreads();
    };
    auto unit_max = [&](unsigned v) {  // over the unit's threads
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
        if (UT == 64) return v;
        if (lane == 0) s_red[wave] = v;
        __syncthreads();
        v = max(max(s_red[0], s_red[1]), max(s_red[2], s_red[3]));
        __syncthreads();
        return v;
    };
    auto slot_of = [&](int t) { return t >= 0 && t < tokens ? slots[t] : -1; };
    auto block_of = [&](int s) { return s >= 0 && s < nslots ? page.div(s) : -1; };

    // the run of K or V (is_v), head h, whose first fresh row is i, in `block`
    auto run = [&](int i, int block, bool is_v, int h) {
        const T* const x = (is_v ? v_new : k_new) + (size_t)h * dim;
        signed char* const pool = is_v ? v_pool : k_pool;
        float* const scales = is_v ? v_scales : k_scales;
        const int slot0 = slots[i], row0 = page.mod(slot0);
        // its length, and whether its rows are in order
        int n = 0;
        bool ordered = true;
        for (;; n += 64) {
            const int s = slot_of(i + n + lane);
            const unsigned long long out = __ballot(block_of(s) != block);
            const int got = out ? __builtin_ctzll(out) : 64;
            ordered = ordered && !__any(lane < got && s != slot0 + n + lane);
            if (got < 64) {
                n += got;
                break;
            }
        }
        n = __builtin_amdgcn_readfirstlane(n);
        bool over = row0 == 0;
        if (!ordered) {
            sync();
            for (int r = ut; r < (int)page.d; r += UT) map[r] = -1;
            sync();
            for (int k = ut; k < n; k += UT) atomicMax(&map[page.mod(slots[i + k])], i + k);
            sync();
            over = map[0] >= 0;
        }
        const int base = ordered ? row0 : 0;                 // the rows gone over
        const int nvec = (ordered ? n : (int)page.d) * (int)lanes.d;
        // the fresh row for the j-th vector of them, -1 where there is none
        auto source = [&](int r) { return ordered ? i + r : map[r]; };
        using R = Raw<T, V>;
        R keep[kKeep];
        auto load = [&](int j, R& v) {
            const int r = lanes.div(j), src = source(r);
            if (src >= 0) v.load(x + src * row_stride + V * (j - r * (int)lanes.d));
            else v.zero();
        };
        unsigned bits = 0;
#pragma unroll
        for (int p = 0; p < kKeep; ++p) {
            const int j = p * UT + ut;
            if (j < nvec) load(j, keep[p]);
        }
#pragma unroll
        for (int p = 0; p < kKeep; ++p)
            if (p * UT + ut < nvec) bits = keep[p].most(bits);
        for (int j = kKeep * UT + ut; j < nvec; j += UT) {
            R v;
            load(j, v);
            bits = v.most(bits);
        }
        const size_t bh = (size_t)block * hkv + h;
        const float held = over ? 0.0f : scales[bh];
        if constexpr (sizeof(T) == 2) bits = max(bits & 0xffffu, bits >> 16);
        bits = unit_max(bits);
        float most = R::value_of(bits);
        const bool finite = bits < R::kInf;
        if (!finite) {  // of the finite values alone
            float m = 0.0f;
            for (int j = ut; j < nvec; j += UT) {
                R v;
                load(j, v);
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    const float a = fabsf(v.value(c));
                    m = fmaxf(m, a < INFINITY ? a : 0.0f);
                }
            }
            most = __uint_as_float(unit_max(__float_as_uint(m)));
        }
        const float now = fmaxf(fmaxf(held, most / 127.0f), kLeastScale);
        const float inv = 1.0f / now;
        signed char* const codes = pool + bh * page.d * dim;
        auto store = [&](int j, const R& v) {
            const int r = lanes.div(j);
            if (source(r) < 0) return;
            Codes<V> o;
#pragma unroll
            for (int c = 0; c < V; c += 4)
                o.w[c / 4] = codes4(v.value(c), v.value(c + 1), v.value(c + 2),
                                    v.value(c + 3), inv);
            if (!finite) {
#pragma unroll
                for (int c = 0; c < V; c += 4) {
                    o.w[c / 4] = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o.w[c / 4] |= (unsigned)(unsigned char)code8(v.value(c + i), inv)
                                      << (8 * i);
                }
            }
            *reinterpret_cast<Codes<V>*>(codes + (size_t)(base + r) * dim +
                                         V * (j - r * (int)lanes.d)) = o;
        };
#pragma unroll
        for (int p = 0; p < kKeep; ++p) {
            const int j = p * UT + ut;
            if (j < nvec) store(j, keep[p]);
        }
        for (int j = kKeep * UT + ut; j < nvec; j += UT) {
            R v;
            load(j, v);
            store(j, v);
        }
        if (!over && now > held) {  // the block's other rows
            const float ratio = held / now;
            for (int j = ut; j < (int)(page.d * lanes.d); j += UT) {
                const int r = lanes.div(j);
                if (ordered ? (unsigned)(r - row0) < (unsigned)n : map[r] >= 0) continue;
                Codes<V>* p = reinterpret_cast<Codes<V>*>(codes + (size_t)V * j);
                Codes<V> o = *p;
#pragma unroll
                for (int c = 0; c < V / 4; ++c) {
                    const unsigned u = o.w[c];
                    o.w[c] = codes4((float)(signed char)u, (float)(signed char)(u >> 8),
                                    (float)(signed char)(u >> 16), (float)((int)u >> 24),
                                    ratio);
                }
                *p = o;
            }
        }
        if (ut == 0) scales[bh] = now;
    };

    if constexpr (LISTED) {
        // the starts of all runs: a thread looks at consecutive fresh rows
        constexpr int PER = kListTokens / 256;
        const int per = (tokens + 255) / 256, t0 = (int)threadIdx.x * per;
        int s[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) s[k] = k < per ? slot_of(t0 + k) : -1;
        int before = block_of(slot_of(t0 - 1));
        unsigned starts = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int block = block_of(s[k]);
            if (block >= 0 && block != before) starts |= 1u << k;
            before = block;
        }
        const int mine = __popc(starts);
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(incl, o, 64);
            if (lane >= o) incl += y;
        }
        if (lane == 63) s_red[wave] = incl;
        __syncthreads();
        int at = incl - mine, runs = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < wave) at += s_red[w];
            runs += s_red[w];
        }
        for (; starts; starts &= starts - 1) s_runs[at++] = t0 + __builtin_ctz(starts);
        __syncthreads();  // (s_red is free again too)
        const int all = runs * 2 * hkv;  // <= 2 tokens * heads
        const int step = (int)gridDim.x * kUnits;
        for (int u = (int)unit; u < all; u += step) {
            const int rk = heads.div(u);  // (run, K or V)
            const int i = __builtin_amdgcn_readfirstlane(s_runs[rk >> 1]);
            run(i, block_of(slots[i]), rk & 1, u - rk * hkv);
        }
    } else {
        // (units / 2 <= tokens * heads < 2^31: checked by the host)
        const bool is_v = unit >= units / 2;
        const int wh = (int)(is_v ? unit - units / 2 : unit);
        const int h = heads.mod(wh), first = heads.div(wh) * window;
        const int mine = lane < window ? block_of(slot_of(first + lane)) : -1;
        unsigned long long starts =
            __ballot(mine >= 0 && block_of(slot_of(first + lane - 1)) != mine);
        for (; starts; starts &= starts - 1) {
            const int at = __builtin_ctzll(starts);
            run(first + at, __shfl(mine, at, 64), is_v, h);
        }
    }
}

template <typename T, int V, int UT>
void append8_run(const T* k_new, const T* v_new, const int* slots, signed char* k_pool,
                 signed char* v_pool, float* k_scales, float* v_scales, int tokens, int hkv,
                 int dim, int blocks, int page, hipStream_t s) {
    const int cus = dev_info().cu_count;
    const long long pairs = 2LL * tokens * hkv;  // one a row, head and pool
    const bool row_each = pairs <= kRowEach * cus;
    const bool listed = !row_each && tokens <= kListTokens;
    const int window = row_each ? 1 : std::min(page, 64);  // (a lane a row)
    const long long units = 2LL * ((tokens + window - 1) / window) * hkv;
    const long long wgs = listed ? std::min((pairs * UT + 255) / 256, (long long)kListWgs * cus)
                                 : (units * UT + 255) / 256;
    const auto kernel = listed ? kv_append8_kernel<T, V, UT, true> : kv_append8_kernel<T, V, UT, false>;
    // (a grid's threads fit 32 bits; units share nothing, so a call may take several)
    constexpr long long kGrid = (1LL << 24) - 1;
    for (long long at = 0; at < wgs; at += kGrid) {
        kernel<<<(unsigned)std::min(kGrid, wgs - at), 256, 0, s>>>(
            k_new, v_new, slots, k_pool, v_pool, k_scales, v_scales, tokens, FastDiv(hkv), dim,
            blocks * page, FastDiv(page), FastDiv(dim / V), window, at, units);
        launch_check("int8 kv append kernel launch");
    }
}

template <typename T>
void append8(const T* k_new, const T* v_new, const int* slots, signed char* k_pool,
             signed char* v_pool, float* k_scales, float* v_scales, int tokens, int hkv, int dim,
             int blocks, int page, hipStream_t s) {
    auto go = [&](auto v, auto ut) {
        append8_run<T, decltype(v)::value, decltype(ut)::value>(
            k_new, v_new, slots, k_pool, v_pool, k_scales, v_scales, tokens, hkv, dim, blocks,
            page, s);
    };
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    using Wave = std::integral_constant<int, 64>;
    using Group = std::integral_constant<int, 256>;
    auto aligned = [](const void* p, size_t by) { return (uintptr_t)p % by == 0; };
    const bool eight = dim % 8 == 0 && aligned(k_new, 16) && aligned(v_new, 16) &&
                       aligned(k_pool, 8) && aligned(v_pool, 8);
    // a wave has a run where a block stays in its registers, else a workgroup
    // (16384 prompt tokens, 8 heads, D = 128: blocks of 16 22.3 us by waves, 43.0
    // by workgroups; blocks of 64 28.2 and 22.8)
    const bool wave = page * (dim / (eight ? 8 : 4)) <= 4 * 64;
    if (eight && wave) go(I8{}, Wave{});
    else if (eight) go(I8{}, Group{});
    else if (wave) go(I4{}, Wave{});
    else go(I4{}, Group{});
}

// ---------------------------------------------------------------------------
// Decode attention.
//
//   s_t = (q . kcode_t) kscale(t) / sqrt(D),  out = sum_t softmax(s)_t vscale(t) vcode_t
//
// The partial of a stretch of tokens is (m = max s, l = sum exp2(s - m),
// acc = sum exp2(s - m) v), in log2 units and float32; partials of one row
// fold by the log-sum-exp rule (attn8_combine). A stretch without a token that
// counts has m = -inf, l = 0. A table entry outside [0, blocks) is a hole:
// its tokens weigh nothing, and nothing is read for them.
// ---------------------------------------------------------------------------

// floor(a / b) for 0 <= a, b > 0 and a quotient below 2^20, by way of a float32
// one, which is then off by at most one (a 64-bit division, or a float64 one,
// costs a kernel's start 0.2-0.3 us).
__device__ __forceinline__ int small_div(long long a, long long b) {
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
    const long long r = a - q * b;
    return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

// Where the pieces of row (b, head) lie in the workspace: piece i at slot
// at(i), `tile` q heads a slot. count 0: no token; -1: the row is stored
// already.
struct Chunked8 {  // attn8_general: a slot per (row, chunk)
    int cmax, chunk;
    struct Row {
        size_t first;
        int count;
        __device__ __forceinline__ size_t at(int i) const { return first + i; }
    };
    __device__ __forceinline__ Row row(const int* lens, int span, int b, int vrow,
                                       int vrows) const {
        const int len = clamp_len(lens, b, span);
        return Row{((size_t)b * vrows + vrow) * cmax, (len + chunk - 1) / chunk};
    }
};

struct Streamed8 {  // attn8_stream: two slots a segment (kernel comment)
    const long long* pref;  // prefix of the lengths [batch + 1], then the segment length
    int batch;
    struct Row {
        int s_lo;
        long long end, seg;
        int count;
        __device__ __forceinline__ size_t at(int i) const {
            const int s = s_lo + i;
            return (size_t)(2 * s + (end >= (s + 1) * seg ? 1 : 0));
        }
    };
    __device__ __forceinline__ Row row(const int*, int, int b, int vrow, int vrows) const {
        const long long seg = pref[batch + 1], p0 = pref[b], len = pref[b + 1] - p0;
        const long long start = p0 * vrows + vrow * len;
        if (len == 0) return Row{0, 0, seg, 0};
        const int lo = small_div(start, seg), hi = small_div(start + len - 1, seg);
        return Row{lo, start + len, seg, lo == hi ? -1 : hi - lo + 1};
    }
};

constexpr int kMaxPieces8 = 4096;  // of a row (their weights are kept in LDS)
constexpr int kWavePieces8 = 32;   // folded by one wave, at most

// `per` (1 or 4) q heads a workgroup, a wave each; a head of many pieces is
// folded by the whole workgroup, afterwards. Where heads are few, gridDim.y
// workgroups share the dims of one of many pieces. Bound by latency: the row's
// place, its pieces' (m, l) and sums, the launch; 4-7 us of kernel.
template <typename T, typename Pieces>
__global__ __launch_bounds__(256) void attn8_combine(
    const float* __restrict__ ws_ml, const float* __restrict__ ws_acc,
    const int* __restrict__ lens, T* __restrict__ out, Pieces pieces, int heads, int hq, int hkv,
    int dim, int span, int tile, int tiles, int per) {
    __shared__ float s_w[kMaxPieces8];
    __shared__ float4 s_acc[256];
    __shared__ float s_max[4], s_sum[4];
    __shared__ int s_many[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = hq / hkv, dc = dim / 4;
    auto row_of = [&](int head) {
        const int b = head / hq, hh = head - b * hq, kv = hh / group, gi = hh - kv * group;
        return pieces.row(lens, span, b, kv * tiles + gi / tile, hkv * tiles);
    };
    auto in_tile = [&](int head) { return head % hq % group % tile; };
    const float2* const ml = reinterpret_cast<const float2*>(ws_ml);
    // (a piece of no weight has l = 0)
    auto weight = [&](float2 p, float mx) { return p.y == 0.0f ? 0.0f : exp2f(p.x - mx); };
    auto store = [&](int head, int d4, float4 a, float l) {
        if (l == 0.0f) a = make_float4(0.f, 0.f, 0.f, 0.f);
        else a = make_float4(a.x / l, a.y / l, a.z / l, a.w / l);
        St<T>::st4(out + (size_t)head * dim + 4 * d4, a);
    };

    // dims [4 v0, 4 v0 + 4 nv) of one head by the whole workgroup
    auto fold = [&](int head, const typename Pieces::Row& row, int v0, int nv) {
        constexpr int kAhead = 8;
        const int np = row.count, ng = 256 / nv, tg = tid / nv, d4 = v0 + tid - tg * nv;
        const int gi = in_tile(head);
        auto at = [&](int i) { return row.at(i) * tile + gi; };
        auto piece = [&](int i) {
            return tg < ng && i < np
                       ? *reinterpret_cast<const float4*>(ws_acc + at(i) * dim + 4 * d4)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        const float2 p0 = tid < np ? ml[at(tid)] : make_float2(-INFINITY, 0.0f);
        float4 x[kAhead];  // under way before the weights are known
#pragma unroll
        for (int k = 0; k < kAhead; ++k) x[k] = piece(tg + k * ng);
        float mx = p0.x;
        for (int i = tid + 256; i < np; i += 256) mx = fmaxf(mx, ml[at(i)].x);
        mx = wave_max(mx);
        if (lane == 0) s_max[wave] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        float l = 0.0f;
        for (int i = tid; i < np; i += 256) {
            const float2 p = i == tid ? p0 : ml[at(i)];
            const float w = weight(p, mx);
            s_w[i] = w;
            l += w * p.y;
        }
        l = wave_sum(l);
        if (lane == 0) s_sum[wave] = l;
        __syncthreads();
        l = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](int i, float4 v) {
            const float w = tg < ng && i < np ? s_w[i] : 0.0f;
            a.x += w * v.x; a.y += w * v.y; a.z += w * v.z; a.w += w * v.w;
        };
#pragma unroll
        for (int k = 0; k < kAhead; ++k) add(tg + k * ng, x[k]);
        for (int i = tg + kAhead * ng; i < np; i += kAhead * ng) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) x[k] = piece(i + k * ng);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) add(i + k * ng, x[k]);
        }
        s_acc[tid] = a;
        __syncthreads();
        // the groups' sums, halved until one is left
        for (int n = ng; n > 1;) {
            const int half = (n + 1) >> 1;
            if (tg + half < n) {
                const float4 v = s_acc[tid + half * nv];
                a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
                s_acc[tid] = a;
            }
            n = half;
            __syncthreads();
        }
        if (tg == 0) store(head, d4, a, l);
        __syncthreads();  // LDS is the next head's
    };

    if (per == 1) {
        const auto row = row_of(blockIdx.x);
        const int nv = dc / gridDim.y;
        if (row.count > kWavePieces8) return fold(blockIdx.x, row, blockIdx.y * nv, nv);
        if (blockIdx.y) return;
    }
    {
        const int head = blockIdx.x * per + wave;
        bool many = false;
        if (wave < per && head < heads) {
            const auto row = row_of(head);
            const int np = row.count, gi = in_tile(head);
            many = np > kWavePieces8 || (np >= 0 && 64 % dc != 0);
            if (!many && np >= 0) {
                const size_t slot = row.at(min(lane, np)) * tile + gi;
                const float2 p = lane < np ? ml[slot] : make_float2(-INFINITY, 0.0f);
                const int grp = lane / dc, d4 = lane - grp * dc, ng = 64 / dc;
                float4 x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // (under way before the weights are known)
                    const int i = grp + k * ng;
                    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (i < np)
                        x[k] = *reinterpret_cast<const float4*>(
                            ws_acc + (row.at(i) * tile + gi) * dim + 4 * d4);
                }
                const float mx = wave_max(p.x), w = weight(p, mx), l = wave_sum(w * p.y);
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                auto add = [&](int i, float4 v) {
                    const float wi = __shfl(w, i & 63, 64);
                    if (i < np) {
                        a.x += wi * v.x; a.y += wi * v.y; a.z += wi * v.z; a.w += wi * v.w;
                    }
                };
#pragma unroll
                for (int k = 0; k < 4; ++k) add(grp + k * ng, x[k]);
                for (int i0 = 4 * ng; i0 < np; i0 += ng) {
                    const int i = i0 + grp;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (i < np)
                        v = *reinterpret_cast<const float4*>(
                            ws_acc + (row.at(i) * tile + gi) * dim + 4 * d4);
                    add(i, v);
                }
                for (int o = dc; o < 64; o <<= 1) {
                    a.x += __shfl_xor(a.x, o, 64);
                    a.y += __shfl_xor(a.y, o, 64);
                    a.z += __shfl_xor(a.z, o, 64);
                    a.w += __shfl_xor(a.w, o, 64);
                }
                if (grp == 0) store(head, d4, a, l);
            }
        }
        if (lane == 0) s_many[wave] = many;
    }
    __syncthreads();
    for (int k = 0; k < per; ++k)
        if (s_many[k]) fold(blockIdx.x * per + k, row_of(blockIdx.x * per + k), 0, dc);
}

template <typename T, typename Pieces>
void combine8(const float* ml, const float* acc, const int* lens, T* out, const Pieces& pieces,
              int batch, int hq, int hkv, int dim, int span, int tile, int tiles, hipStream_t s) {
    const int heads = batch * hq;
    // few heads have many pieces each: a workgroup a head, or one for 32 of its
    // dims (one row of 131072 tokens, 8 heads, attention and combine, graph
    // replays: 32.7 us without, 22.8 with); many have few: four a workgroup (4096
    // heads, 128 rows of 500 tokens, both: 49.3 and 37.5)
    const int per = heads >= 4 * dev_info().cu_count && 256 % dim == 0 ? 4 : 1;
    const int parts = per == 1 && heads < dev_info().cu_count && dim % 32 == 0 ? dim / 32 : 1;
    attn8_combine<T, Pieces><<<dim3((heads + per - 1) / per, parts), 256, 0, s>>>(
        ml, acc, lens, out, pieces, heads, hq, hkv, dim, span, tile, tiles, per);
    launch_check("int8 decode attention combine launch");
}

// ---------------------------------------------------------------------------
// The other head dims (attn8_general): one workgroup per (sequence, kv head, chunk of
// tokens), 8 q heads at a time, dot products on the vector ALU, 256 tokens at
// a time with a running maximum.
// ---------------------------------------------------------------------------
constexpr int kGen8Heads = 8, kGen8Step = 256;

template <typename T>
__global__ __launch_bounds__(256) void attn8_general(
    const T* __restrict__ q, const signed char* __restrict__ k_pool,
    const signed char* __restrict__ v_pool, const float* __restrict__ k_scales,
    const float* __restrict__ v_scales, const int* __restrict__ table,
    const int* __restrict__ lens, float* __restrict__ ws_ml, float* __restrict__ ws_acc, int hq,
    int hkv, int dim, int blocks, int page, int width, int span, int chunk, float scale_log2) {
    __shared__ float s_sc[kGen8Heads][kGen8Step];
    __shared__ float s_vs[kGen8Step];
    __shared__ long long s_row[kGen8Step];  // element offset of the token's row, -1 a hole
    __shared__ float s_m[kGen8Heads], s_l[kGen8Heads], s_alpha[kGen8Heads];
    __shared__ float4 s_red[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int c = blockIdx.x, kv = blockIdx.y, b = blockIdx.z, cmax = gridDim.x;
    const int group = hq / hkv, len = clamp_len(lens, b, span), lo = c * chunk;
    if (lo >= len) return;
    const int hi = min(lo + chunk, len), dc = dim / 4;
    const int ng = 256 / dc, tg = tid / dc, d4 = tid - tg * dc;
    for (int g0 = 0; g0 < group; g0 += kGen8Heads) {
        const int gc = min(kGen8Heads, group - g0);
        const T* qg = q + ((size_t)b * hq + (size_t)kv * group + g0) * dim;
        float4 acc[kGen8Heads];
#pragma unroll
        for (int g = 0; g < kGen8Heads; ++g) acc[g] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tid < kGen8Heads) {
            s_m[tid] = -INFINITY;
            s_l[tid] = 0.0f;
        }
        for (int t0 = lo; t0 < hi; t0 += kGen8Step) {
            const int n = min(kGen8Step, hi - t0);
            if (tid < n) {  // scores: a thread a token
                const int t = t0 + tid, ent = table[(size_t)b * width + t / page];
                const bool ok = (unsigned)ent < (unsigned)blocks;
                const size_t bh = (size_t)(ok ? ent : 0) * hkv + kv;
                const long long row = ok ? (long long)((bh * page + t % page) * dim) : -1;
                const float ks = ok ? k_scales[bh] * scale_log2 : 0.0f;
                float part[kGen8Heads] = {};
                if (ok) {
                    const char4* kr = reinterpret_cast<const char4*>(k_pool + row);
                    for (int j = 0; j < dc; ++j) {
                        const char4 kk = kr[j];
#pragma unroll
                        for (int g = 0; g < kGen8Heads; ++g)
                            if (g < gc) {
                                const float4 qq = St<T>::ld4(qg + (size_t)g * dim + 4 * j);
                                part[g] += qq.x * kk.x + qq.y * kk.y + qq.z * kk.z + qq.w * kk.w;
                            }
                    }
                }
                s_row[tid] = row;
                s_vs[tid] = ok ? v_scales[bh] : 0.0f;
#pragma unroll
                for (int g = 0; g < kGen8Heads; ++g) s_sc[g][tid] = ok ? part[g] * ks : -INFINITY;
            }
            __syncthreads();
            for (int g = wave; g < gc; g += 4) {
                float m = -INFINITY;
                for (int t = lane; t < n; t += 64) m = fmaxf(m, s_sc[g][t]);
                const float was = s_m[g];
                m = fmaxf(was, wave_max(m));
                const float top = m == -INFINITY ? 0.0f : m;
                float l = 0.0f;
                for (int t = lane; t < n; t += 64) {
                    const float p = exp2f(s_sc[g][t] - top);
                    l += p;
                    s_sc[g][t] = s_row[t] >= 0 ? p * s_vs[t] : 0.0f;
                }
                l = wave_sum(l);
                if (lane == 0) {
                    const float alpha = exp2f(was - top);
                    s_alpha[g] = alpha;
                    s_l[g] = s_l[g] * alpha + l;
                    s_m[g] = m;
                }
            }
            __syncthreads();
            if (tg < ng) {
#pragma unroll
                for (int g = 0; g < kGen8Heads; ++g)
                    if (g < gc) {
                        const float al = s_alpha[g];
                        acc[g].x *= al; acc[g].y *= al; acc[g].z *= al; acc[g].w *= al;
                    }
                for (int t = tg; t < n; t += ng) {
                    if (s_row[t] < 0) continue;
                    const char4 vv = *reinterpret_cast<const char4*>(v_pool + s_row[t] + 4 * d4);
#pragma unroll
                    for (int g = 0; g < kGen8Heads; ++g)
                        if (g < gc) {
                            const float w = s_sc[g][t];
                            acc[g].x += w * vv.x; acc[g].y += w * vv.y;
                            acc[g].z += w * vv.z; acc[g].w += w * vv.w;
                        }
                }
            }
            __syncthreads();
        }
        const size_t slot0 = (((size_t)b * hkv + kv) * cmax + c) * group + g0;
#pragma unroll
        for (int g = 0; g < kGen8Heads; ++g) {
            if (g >= gc) break;
            s_red[tid] = acc[g];
            __syncthreads();
            if (tg == 0) {
                float4 a = s_red[d4];
                for (int j = 1; j < ng; ++j) {
                    const float4 o = s_red[j * dc + d4];
                    a.x += o.x; a.y += o.y; a.z += o.z; a.w += o.w;
                }
                *reinterpret_cast<float4*>(ws_acc + (slot0 + g) * dim + 4 * d4) = a;
            }
            __syncthreads();
        }
        if (tid < gc) {
            ws_ml[(slot0 + tid) * 2] = s_m[tid];
            ws_ml[(slot0 + tid) * 2 + 1] = s_l[tid];
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Tokens of a segment, at least (a power of two, whole steps). Calls of few
// tokens take segments of one row each: of 64 tokens while those are at most
// four a CU (eight at D = 64), else of 128 while those do not outnumber the
// waves. Attention and combine together, graph replays: 4 rows of 500-1000
// tokens, 8 kv heads, D = 128, 13.6 us at 64, 14.7 at 128, 15.8 as equal
// segments; 8 rows of 1000-2000 16.8 at 128 (18.7 at 64, measured with a weight of
// two parts), 21.4 equal; 32 rows of 500-1000 20.5 at 128, 22.9 equal.
constexpr int kMinSeg8 = 64;
constexpr int kScanRows8 = 1024;  // sequences of a launch (their prefixes are in LDS)

// ---------------------------------------------------------------------------
// dim a multiple of 16 up to 256 (attn8_stream): matrix cores, each K / V byte
// read once. The kernel is built for D = 64, 128 and 256; another dim runs in
// the next larger (FULL false), its rows' missing chunks never read and zero.
//
// Work split. The rows are (sequence b, kv head, tile of up to 16 q heads),
// b-major, len_b tokens each, laid end to end; every WAVE takes one equal
// contiguous segment of that range, whatever the length mix; for few tokens
// (kMinSeg8) each row is rounded up to whole segments, so that none has two
// rows. A segment is one or more pieces, one per row it touches. A piece that
// is a whole row is normalised and stored; another leaves its partial in the
// segment's slot 1 if its row reaches the segment's end, else in slot 0: a
// segment has at most one of each. Waves share nothing but the length prefix,
// so after it there is no barrier and no merge in the kernel. (More segments
// than waves, or smaller ones behind the large, cost more at their starts than
// the even end saves: 32 ragged rows, with the combine, 224 against 214 us with
// twice as many.)
//
// A step is TOK tokens (32; 64 for D = 64), K and V of the next one - of the
// next piece at a piece's end - in flight in registers while this one is
// computed from the wave's own LDS staging. With r = lane % 16, g = lane / 16
// (v_mfma_f32_16x16x32_bf16: A[r][8g+i], B[8g+i][r], C[4g+i][r]):
//
//  loads    whole 128-byte lines per instruction, non-temporal, of rows whose
//           places the lanes have worked out from the table (a lane a token)
//           and hand out by shuffles;
//  scores   S^T[tok][head] = K . Q^T. Codes become bf16 (exact: 8 bits); q
//           goes in as 1, 2 or 3 bf16 parts (bf16, fp16, float32: all its
//           bits), so every product is exact and sums are float32. Any order
//           of dims serves if q has the same: the lane reads 16-byte chunks.
//           (Integer products with q in base-256 digits take 56 vector
//           instructions a step less, but the loop waited on memory either way,
//           with a weight of two parts: 32 ragged rows 197 us both, 4 short ones
//           8.7 against 8.1);
//  softmax  lane (r, g) holds head r's scores of tokens 4g+i (+ 16 a tile);
//           scaled by the block's K scale, running maximum over the 4 lanes
//           of a head; the weight takes the block's V scale, then goes into 3
//           bf16 parts: all its bits, small ones too, so that products are
//           exact here as well. (Two parts leave out up to 2^-15, always
//           downwards, and a result in a hundred is another fp16 number.)
//           (Groups of up to 4 heads could fill the 16 columns with copies that
//           share the tokens out: a quarter of the exponentials, and 1-2% of
//           the time.);
//  PV       O^T[dim][head] = V^T . W^T, codes widened to bf16 (exact). The
//           weights are where B wants them; for A, lane (r, g) reads dims
//           (D/16) r .. of its 8 tokens from the staging and pairs the tokens
//           up while it widens them, so the transpose costs nothing. Lane
//           (r, g) ends with D/4 consecutive dims of head r.
//
// Masked tokens (behind the piece, holes) weigh 0 exactly: score -inf, V scale
// 0, the row read in its place a real one (its own last, or block 0's).
//
// What bounds it: HBM, and the vector ALU behind it. After the first 6 us
// (lengths, piece, table, first rows) 32 rows of 512-32768 tokens, 32 / 8 heads,
// D = 128, bf16, read at 6.4 TB/s (202 us in all; bare reads of such pages reach
// 6.7-6.8); 64 rows of 4097, 64 / 8 heads, fp16, take 94.5 us, 2 rows of 131071,
// D = 64, 51.4. The vector ALU is busy 63-70% of the cycles, the matrix cores
// 20-23%. (A weight of two parts, which is not exact: 197, 94.1 and 48.8 us.) Two
// waves a SIMD: at three the registers spill (226 against 210 us for the first of
// these, all else equal, in an earlier form). For short rows, latency: 5.6 us for
// 4 rows of 128-1024 tokens, D = 64, and 4.2 for the combine.
// ---------------------------------------------------------------------------
typedef float f32x4_8 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int stream_occ(int dim) { return dim > 128 ? 1 : 2; }

template <typename T, int D>
struct Stream8 {
    static constexpr int kTok = D == 64 ? 64 : 32;   // tokens a step
    static constexpr int kLoads = kTok * D / 1024;   // 16-byte loads a lane and pool
    static constexpr int kRowsPer = 1024 / D;        // rows a load instruction covers
    static constexpr int kChunks = D / 16;           // 16-byte chunks of a row
    static constexpr int kW = 3;                     // weight parts: all 24 bits
    static constexpr int kOcc = stream_occ(D);       // waves a SIMD
    static constexpr int kLds = 2 * kTok * D + 8 * kTok;  // bytes a wave
    static constexpr int kQ = std::is_same<T, float>::value ? 3 : std::is_same<T, f16>::value ? 2 : 1;  // q parts
};

// upper halves of two float32 (as two bf16, truncated)
__device__ __forceinline__ unsigned pack_hi(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float byte_f(unsigned x, int i) {
    return (float)(signed char)(x >> (8 * i));
}
// 8 codes to bf16
__device__ __forceinline__ b16x8 widen8(unsigned a, unsigned b) {
    u32x4 o;
    o[0] = pack_hi(byte_f(a, 0), byte_f(a, 1));
    o[1] = pack_hi(byte_f(a, 2), byte_f(a, 3));
    o[2] = pack_hi(byte_f(b, 0), byte_f(b, 1));
    o[3] = pack_hi(byte_f(b, 2), byte_f(b, 3));
    return __builtin_bit_cast(b16x8, o);
}
// Exclusive prefix of the clamped lengths, each rounded up to a multiple of
// `to` (a power of two), by one wave.
__device__ __forceinline__ void scan8(const int* __restrict__ lens, int batch, int span, int lane,
                                      int to, long long* pref) {
    const int per = (batch + 63) >> 6, b0 = lane * per;
    auto len = [&](int i) {
        return b0 + i < batch ? (clamp_len(lens, b0 + i, span) + to - 1) & -to : 0;
    };
    long long sum = 0;
    for (int i = 0; i < per; ++i) sum += len(i);
    long long incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long y = __shfl_up(incl, o, 64);
        if (lane >= o) incl += y;
    }
    long long at = incl - sum;
    for (int i = 0; i < per; ++i) {
        const int n = len(i);
        if (b0 + i < batch) pref[b0 + i] = at;
        at += n;
    }
    if (lane == 63) pref[batch] = incl;
}

// A stretch of one row: tokens [t0, t0 + n) of sequence b for q heads [h0, h0 +
// heads), up to flat position next. (No padding: the compiler keeps a copied
// struct's padding in LDS, and to place it reads the workgroup's size from the
// dispatch packet in host memory, 3-7 us at the kernel's start.)
struct Piece8 {
    long long next;
    int b, kv, t0, n;
    int h0, heads;
    int whole;  // the row's every token
    int ends;   // the row reaches the segment's end
};

// The row that holds flat position pos (in units of 1 / vrows of the prefix),
// cut at seg_end: the sequences' ends are counted 64 at a time, by the lanes.
__device__ __forceinline__ Piece8 piece8(const long long* s_pref, int batch, int vrows,
                                         long long pos, long long seg_end, int lane, int group,
                                         int tile, const FastDiv& tiles,
                                         const long long* s_tokens) {
    int b = 0;
    for (int step = (batch + 63) >> 6;; step = 1) {
        const int at = b + (lane + 1) * step;
        b += step * __popcll(__ballot(at <= batch && s_pref[min(at, batch)] * vrows <= pos));
        if (step == 1) break;
        // (the coarse count's last stretch may hold fewer than 64 sequences)
    }
    Piece8 p;
    p.b = b;
    const long long pb = uniform64(s_pref[b]), base = pb * vrows;
    const int len = (int)(uniform64(s_pref[b + 1]) - pb);
    // (s_pref may be of padded lengths, s_tokens is of the true ones)
    const int end = (int)(uniform64(s_tokens[b + 1]) - uniform64(s_tokens[b]));
    const int v = __builtin_amdgcn_readfirstlane(small_div(pos - base, len));
    const long long row_end = base + (long long)(v + 1) * len;
    p.t0 = (int)(pos - base - (long long)v * len);
    p.next = min(seg_end, row_end);
    p.n = min((int)(p.next - pos), end - p.t0);
    p.whole = p.t0 == 0 && p.n == end;
    p.ends = row_end >= seg_end;
    p.kv = tiles.div(v);
    const int first = (v - p.kv * (int)tiles.d) * tile;
    p.h0 = p.kv * group + first;
    p.heads = min(tile, group - first);
    return p;
}

template <typename T, int D, bool FULL>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(Stream8<T, D>::kOcc, Stream8<T, D>::kOcc)))
void attn8_stream(const T* __restrict__ q, const signed char* __restrict__ k_pool,
                  const signed char* __restrict__ v_pool, const float* __restrict__ k_scales,
                  const float* __restrict__ v_scales, const int* __restrict__ table,
                  const int* __restrict__ lens, float* __restrict__ ws_ml,
                  float* __restrict__ ws_acc, long long* __restrict__ pref_out,
                  T* __restrict__ out, int batch, int hq, int hkv, int tile, FastDiv tiles,
                  int blocks, FastDiv page, int width, int span, int nseg, int short_segs,
                  float scale_log2, float inv_nseg, int dim_) {
    using C = Stream8<T, D>;
    constexpr int TOK = C::kTok, NL = C::kLoads, SUB = TOK / 32, KE = D / 64;
    __shared__ __align__(16) char s_stage[4][C::kLds];
    __shared__ long long s_prefix[3][kScanRows8 + 1];  // of lens, rounded up to 1, 64, 128

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int dim = FULL ? D : dim_;
    if (wave < 3) scan8(lens, batch, span, lane, wave ? kMinSeg8 * wave : 1, s_prefix[wave]);
    __syncthreads();
    const int vrows = hkv * (int)tiles.d, group = hq / hkv;
    // few tokens: a segment a stretch of S tokens of one row
    const long long pad1 = uniform64(s_prefix[1][batch]) * vrows;
    const long long pad2 = uniform64(s_prefix[2][batch]) * vrows;
    const int few = pad1 <= (long long)short_segs * kMinSeg8   ? 1
                    : pad2 <= (long long)nseg * (2 * kMinSeg8) ? 2
                                                               : 0;
    const long long* const s_pref = s_prefix[few];
    const long long total = uniform64(s_pref[batch]) * vrows;
    long long S = kMinSeg8 * few;
    if (!few) {
        // at least total / nseg, whole steps (float32, off by 2^-22: rounded up)
        S = max((long long)((float)total * inv_nseg) + 1, (long long)kMinSeg8);
        S = (S + TOK - 1) & ~(long long)(TOK - 1);
    }
    if (blockIdx.x == 0) {  // the combine's copy of the prefix, and S
        for (int i = tid; i <= batch; i += 256) pref_out[i] = s_pref[i];
        if (tid == 0) pref_out[batch + 1] = S;
    }
    const int seg = blockIdx.x * 4 + wave;
    const long long seg_lo = (long long)seg * S;
    if (seg >= nseg || seg_lo >= total) return;
    const long long seg_hi = min(seg_lo + S, total);

    char* const sk = &s_stage[wave][0];
    char* const sv = sk + TOK * D;
    float2* const ss = reinterpret_cast<float2*>(sv + TOK * D);
    // Row w's 16-byte chunk c in the K staging: the 16 lanes of a fragment
    // read (16 rows, one chunk) hit 16 different 16-byte bank groups.
    auto k_at = [&](int w, int c) {
        const int x = D == 64 ? (w >> 2) & 3 : D == 128 ? (w >> 1) & 7 : w & 15;
        return w * D + 16 * (c ^ x);
    };
    // Row w of the V staging: the rows 4g + i of one i, read together, next to
    // each other.
    auto v_at = [&](int w) { return ((w & ~15) | ((w & 3) << 2) | ((w >> 2) & 3)) * D; };
    const int my = lane & (TOK - 1);                 // the lane's token of a step
    const int lc = lane % C::kChunks, lr = lane / C::kChunks;  // its place in a load
    // the lane's i-th score of 32 tokens is that of token at(i)
    auto at = [&](int i) { return 16 * (i >> 2) + 4 * g + (i & 3); };

    // ---- a step's loads ------------------------------------------------------
    auto steps = [&](const Piece8& p) { return (p.n + TOK - 1) / TOK; };
    auto token = [&](const Piece8& p, int st) { return p.t0 + min(st * TOK + my, p.n - 1); };
    auto entry = [&](const Piece8& p, int st) {
        return table[(size_t)p.b * width + page.div(token(p, min(st, steps(p) - 1)))];
    };
    u32x4 kt[NL], vt[NL];
    const bool has = FULL || 16 * lc < dim;  // the row has the lane's chunk
    if (!FULL) {
#pragma unroll
        for (int i = 0; i < NL; ++i) kt[i] = vt[i] = u32x4{0, 0, 0, 0};
    }
    float ksn, vsn;
    unsigned long long seen;  // lanes whose token of the loaded step counts
    auto issue = [&](const Piece8& p, int st, int ent) {
        const int t = token(p, st);
        const bool held = (unsigned)ent < (unsigned)blocks;
        const unsigned bh = (unsigned)(held ? ent : 0) * hkv + p.kv;
        const unsigned row = bh * page.d + page.mod(t);
        const bool ok = held && st * TOK + my < p.n;
        seen = __ballot(ok);
        ksn = k_scales[bh];  // (not touched before the step is staged: a use here
        vsn = v_scales[bh];  // would wait for loads behind them, at a join)
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const unsigned rw = __shfl(row, C::kRowsPer * i + lr, 64);
            const size_t off = (size_t)rw * dim + 16 * lc;
            if (has) {
                kt[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k_pool + off));
                vt[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(v_pool + off));
            }
        }
    };
    // ---- a row's q: column r's dims 64 e + 16 g .. + 15 ----------------------
    typedef T tx8 __attribute__((ext_vector_type(8)));
    tx8 qx[KE][2];
    auto load_q = [&](const Piece8& p) {
        const T* row = q + ((size_t)p.b * hq + p.h0 + (r < p.heads ? r : 0)) * dim;
#pragma unroll
        for (int e = 0; e < KE; ++e)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                if (!FULL) qx[e][f] = tx8{};
                if (FULL || 64 * e + 16 * g < dim)
                    qx[e][f] = *reinterpret_cast<const tx8*>(row + 64 * e + 16 * g + 8 * f);
            }
    };

    Piece8 pc = piece8(s_pref, batch, vrows, seg_lo, seg_lo + S, lane, group, tile, tiles, s_prefix[0]);
    int ent = entry(pc, 0);
    load_q(pc);
    issue(pc, 0, ent);
    ent = entry(pc, 1);

    for (;;) {
        const int nsteps = steps(pc);
        const bool more = pc.next < seg_hi;
        Piece8 nx = pc;
        // B operand of the score products: q in parts, each truncated
        b16x8 qf[KE][2][C::kQ];
#pragma unroll
        for (int e = 0; e < KE; ++e)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                if constexpr (C::kQ == 1) {
                    qf[e][f][0] = qx[e][f];
                } else {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = (float)qx[e][f][i];
#pragma unroll
                    for (int p = 0; p < C::kQ; ++p) {
                        u32x4 o;
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[i] = pack_hi(x[2 * i], x[2 * i + 1]);
                        qf[e][f][p] = __builtin_bit_cast(b16x8, o);
                        if (p + 1 < C::kQ) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                x[i] -= __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u);
                        }
                    }
                }
            }
        f32x4_8 acc[C::kChunks];
#pragma unroll
        for (int i = 0; i < C::kChunks; ++i) acc[i] = f32x4_8{0.f, 0.f, 0.f, 0.f};
        float m_run = -INFINITY, l_run = 0.0f;

        for (int st = 0; st < nsteps; ++st) {
            // ---- this step into the staging, the next one on its way -------
            wave_lds_order();  // (the step before has read it)
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int w = C::kRowsPer * i + lr;
                *reinterpret_cast<u32x4*>(sk + k_at(w, lc)) = kt[i];
                *reinterpret_cast<u32x4*>(sv + v_at(w) + 16 * lc) = vt[i];
            }
            const unsigned long long now = seen;
            if (TOK == 64 || lane < 32) {
                const bool ok = now >> lane & 1;
                ss[my] = make_float2(ok ? ksn * scale_log2 : 0.0f, ok ? vsn : 0.0f);
            }
            wave_lds_order();
            if (st + 1 < nsteps) {
                const int e = ent;
                ent = entry(pc, st + 2);
                issue(pc, st + 1, e);
            } else if (more) {
                nx = piece8(s_pref, batch, vrows, pc.next, seg_lo + S, lane, group, tile, tiles, s_prefix[0]);
                const int e = entry(nx, 0);
                ent = entry(nx, 1);
                issue(nx, 0, e);
            }
            __builtin_amdgcn_sched_barrier(0);

            // ---- scores ------------------------------------------------------
            float x[8 * SUB], vsc[8 * SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f32x4_8 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < KE; ++e) {
                        const u32x4 kc = *reinterpret_cast<const u32x4*>(
                            sk + k_at(32 * u + 16 * h + r, 4 * e + g));
#pragma unroll
                        for (int f = 0; f < 2; ++f) {
                            const b16x8 a = widen8(kc[2 * f], kc[2 * f + 1]);
#pragma unroll
                            for (int p = C::kQ - 1; p >= 0; --p)
                                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[e][f][p], c, 0,
                                                                            0, 0);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 sc = ss[32 * u + at(4 * h + i)];
                        x[8 * u + 4 * h + i] = c[i] * sc.x;
                        vsc[8 * u + 4 * h + i] = sc.y;
                    }
                }
            }
            if (now != ~0ull) {
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!(now >> (32 * u + at(i)) & 1)) x[8 * u + i] = -INFINITY;
            }
            // ---- running softmax ---------------------------------------------
            float top = x[0];
#pragma unroll
            for (int i = 1; i < 8 * SUB; ++i) top = fmaxf(top, x[i]);
            top = fmaxf(m_run, max4_rows(top));
            const float base = top == -INFINITY ? 0.0f : top;
            if (__any(top != m_run)) {
                const float alpha = __builtin_amdgcn_exp2f(m_run - base);
                l_run *= alpha;
#pragma unroll
                for (int i = 0; i < C::kChunks; ++i) acc[i] *= alpha;
                m_run = top;
            }
            // ---- weights and PV, 32 tokens at a time -------------------------
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = __builtin_amdgcn_exp2f(x[8 * u + i] - base);
                    l_run += p;
                    w[i] = p * vsc[8 * u + i];
                }
                // bf16 parts, each truncated, the first the largest: all bits of
                // a weight from 2^-110 up (the products keep subnormal parts,
                // whose last bit is 2^-133; 2^-13 of the least scale) (an
                // infinity, which only a scale that is not finite makes, leaves
                // NaN behind it)
                b16x8 wp[C::kW];
#pragma unroll
                for (int p = 0; p < C::kW; ++p) {
                    u32x4 o;
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = pack_hi(w[2 * i], w[2 * i + 1]);
                    wp[p] = __builtin_bit_cast(b16x8, o);
                    if (p + 1 < C::kW) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            w[i] -= __uint_as_float(__float_as_uint(w[i]) & 0xffff0000u);
                    }
                }
                const char* vr[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    vr[i] = sv + v_at(32 * u + (i < 4 ? 0 : 16) + 4 * g + (i & 3)) + (D / 16) * r;
#pragma unroll
                for (int j = 0; j < C::kChunks / 4; ++j) {  // 4 dims of the lane's D / 16
                    unsigned c[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        c[i] = *reinterpret_cast<const unsigned*>(vr[i] + 4 * j);
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        u32x4 o;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            o[i] = pack_hi(byte_f(c[2 * i], d), byte_f(c[2 * i + 1], d));
                        const b16x8 a = __builtin_bit_cast(b16x8, o);
#pragma unroll
                        for (int p = C::kW - 1; p >= 0; --p)
                            acc[4 * j + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                a, wp[p], acc[4 * j + d], 0, 0, 0);
                    }
                }
            }
        }
        // ---- the row, or its partial -----------------------------------------
        l_run += __shfl_xor(l_run, 16, 64);
        l_run += __shfl_xor(l_run, 32, 64);
        if (r < pc.heads) {
            // dims (D/4) g + (D/16) i + d of head r: acc[d][i]
            if (pc.whole) {
                T* o = out + ((size_t)pc.b * hq + pc.h0 + r) * dim + (D / 4) * g;
                const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < C::kChunks; d += 4) {
                        if (!FULL && (D / 4) * g + (D / 16) * i + d >= dim) continue;
                        float y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (std::is_same<T, float>::value)
                                y[e] = l_run == 0.0f ? 0.0f : acc[d + e][i] / l_run;
                            else
                                y[e] = l_run == 0.0f ? 0.0f : acc[d + e][i] * inv;
                        }
                        St<T>::st4(o + (D / 16) * i + d, make_float4(y[0], y[1], y[2], y[3]));
                    }
            } else {
                const size_t slot = (2 * (size_t)seg + (size_t)pc.ends) * tile + r;
                float* o = ws_acc + slot * dim + (D / 4) * g;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < C::kChunks; d += 4) {
                        if (!FULL && (D / 4) * g + (D / 16) * i + d >= dim) continue;
                        *reinterpret_cast<float4*>(o + (D / 16) * i + d) = make_float4(
                            acc[d][i], acc[d + 1][i], acc[d + 2][i], acc[d + 3][i]);
                    }
                if (g == 0) {
                    ws_ml[slot * 2] = m_run;
                    ws_ml[slot * 2 + 1] = l_run;
                }
            }
        }
        if (!more) break;
        load_q(nx);
        pc = nx;
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct Attn8Shape {
    int batch, hq, hkv, page, width, dim, span;
    bool stream;
    int tile, tiles, nseg, short_segs;  // stream
    int cmax, chunk;                    // general
    size_t slots, bytes;                // slots: (partial, q head) pairs
};

Attn8Shape attn8_shape(int dtype, int batch, int hq, int hkv, int page, int width, int dim) {
    check_pools(0, hkv, page, dim);
    if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
        inval("attention: unknown element type");
    if (batch < 0 || hq < 1 || width < 0) inval("attention: batch >= 0, q heads >= 1, width >= 0");
    if (hq % hkv != 0) inval("q heads must be a multiple of kv heads (contiguous GQA groups)");
    const long long span = (long long)width * page;
    if (span > (1LL << 30)) inval("table capacity too large");
    if ((long long)std::min(batch, kScanRows8) * hq >= 1 << 24)
        inval("attention problem too large for one launch");
    if (hq >= 1 << 20) inval("attention: too many q heads");
    Attn8Shape s{};
    s.batch = batch; s.hq = hq; s.hkv = hkv; s.page = page; s.width = width; s.dim = dim;
    s.span = (int)span;
    if (batch == 0) return s;
    const int cus = dev_info().cu_count, group = hq / hkv;
    s.stream = span > 0 && dim % 16 == 0 && dim <= 256;
    if (s.stream) {
        s.tiles = (group + 15) / 16;
        s.tile = (group + s.tiles - 1) / s.tiles;
        s.tiles = (group + s.tile - 1) / s.tile;
        const int occ = stream_occ(dim);
        const long long rows = (long long)std::min(batch, kScanRows8) * hkv * s.tiles;
        const long long most = rows * ((span + kMinSeg8 - 1) / kMinSeg8);
        s.nseg = (int)std::min(std::min((long long)4 * cus * occ, most), (long long)kMaxPieces8);
        s.short_segs = std::min(s.nseg, (dim <= 64 ? 8 : 4) * cus);
        s.slots = (size_t)2 * s.nseg * s.tile;
    } else {
        if (hkv > 65535 || batch > 65535) inval("attention: batch and kv heads must be <= 65535");
        // about 16 workgroups a CU, at least 256 tokens each
        const long long units =
            std::min((long long)kMaxPieces8, std::max(1LL, 16LL * cus / ((long long)batch * hkv)));
        s.chunk = (int)std::max(1LL, (span + units - 1) / units);
        s.chunk = (s.chunk + kGen8Step - 1) / kGen8Step * kGen8Step;
        s.cmax = (int)((span + s.chunk - 1) / s.chunk);
        s.tile = group;
        s.tiles = 1;
        if ((long long)batch * hq >= 1 << 24 || (long long)batch * hkv * s.cmax >= 1 << 24)
            inval("attention problem too large for one launch");
        s.slots = (size_t)batch * hq * s.cmax;
    }
    s.bytes = (((s.slots * 2 + 63) & ~(size_t)63) + s.slots * dim) * sizeof(float) +
              (s.stream ? (std::min(batch, kScanRows8) + 2) * sizeof(long long) : 0);
    return s;
}

struct Attn8Args {
    const void* q;
    const signed char *kp, *vp;
    const float *ks, *vs;
    const int *table, *lens;
    void *out, *ws;
    int blocks;
};

template <typename T, int D>
void attn8_stream_run(const Attn8Shape& sh, const Attn8Args& a, float* ml, float* acc,
                      hipStream_t s) {
    const int dim = sh.dim;
    long long* pref = (long long*)(acc + sh.slots * dim);
    const float scale = (1.0f / sqrtf((float)dim)) * kLog2e;
    const float inv_nseg = (1.0f + 0x1p-21f) / (float)sh.nseg;
    const auto kernel = dim == D ? attn8_stream<T, D, true> : attn8_stream<T, D, false>;
    for (int b0 = 0; b0 < sh.batch; b0 += kScanRows8) {
        const int nb = std::min(kScanRows8, sh.batch - b0);
        const T* q = (const T*)a.q + (size_t)b0 * sh.hq * dim;
        T* out = (T*)a.out + (size_t)b0 * sh.hq * dim;
        const int* lens = a.lens ? a.lens + b0 : nullptr;
        kernel<<<(sh.nseg + 3) / 4, 256, 0, s>>>(
            q, a.kp, a.vp, a.ks, a.vs, a.table + (size_t)b0 * sh.width, lens, ml, acc, pref, out,
            nb, sh.hq, sh.hkv, sh.tile, FastDiv(sh.tiles), a.blocks, FastDiv(sh.page), sh.width,
            sh.span, sh.nseg, sh.short_segs, scale, inv_nseg, dim);
        launch_check("int8 decode attention kernel launch");
        combine8(ml, acc, lens, out, Streamed8{pref, nb}, nb, sh.hq, sh.hkv, dim, sh.span, sh.tile,
                 sh.tiles, s);
    }
}

template <typename T>
void attn8_run(const Attn8Shape& sh, const Attn8Args& a, hipStream_t s) {
    float* ml = (float*)a.ws;
    float* acc = ml + ((sh.slots * 2 + 63) & ~(size_t)63);
    if (sh.stream && a.blocks > 0) {
        if (sh.dim <= 64) attn8_stream_run<T, 64>(sh, a, ml, acc, s);
        else if (sh.dim <= 128) attn8_stream_run<T, 128>(sh, a, ml, acc, s);
        else attn8_stream_run<T, 256>(sh, a, ml, acc, s);
        return;
    }
    // (a cache without a block or a row: the combine alone, which writes zeros)
    const bool any = sh.span > 0 && a.blocks > 0;
    if (any) {
        attn8_general<T><<<dim3(sh.cmax, sh.hkv, sh.batch), 256, 0, s>>>(
            (const T*)a.q, a.kp, a.vp, a.ks, a.vs, a.table, a.lens, ml, acc, sh.hq, sh.hkv, sh.dim,
            a.blocks, sh.page, sh.width, sh.span, sh.chunk,
            (1.0f / sqrtf((float)sh.dim)) * kLog2e);
        launch_check("int8 decode attention kernel launch");
    }
    combine8(ml, acc, any ? a.lens : nullptr, (T*)a.out, Chunked8{sh.cmax, std::max(sh.chunk, 1)},
             sh.batch, sh.hq, sh.hkv, sh.dim, any ? sh.span : 0, sh.tile, sh.tiles, s);
}

}  // namespace
}  // namespace ft

using namespace ft;

extern "C" {

int ft_block_table_extend_launch(int* table, const int* lens, const int* counts,
                                 const int* free_blocks, int free_len, const int* n_free,
                                 int* slots, int* positions, int* offsets, int* lens_out,
                                 int* n_free_out, int batch, int page, int tbl_width, int tokens,
                                 uintptr_t stream) {
    return guarded([&] {
        if (batch < 0 || batch > kExtendSeqs)
            inval("block_table_extend: batch must be in [0, 4096]");
        if (page < 1 || page > kMaxPage8 || tbl_width < 0 || tokens < 0 || free_len < 0)
            inval("block_table_extend: page in [1, 1024], width >= 0, tokens >= 0");
        if ((long long)tbl_width * page > (1LL << 30)) inval("table capacity too large");
        if ((long long)tbl_width * batch > INT_MAX) inval("block_table_extend: table too large");
        if (!n_free || !n_free_out || !offsets || (tokens && (!slots || !positions)) ||
            (batch && (!lens || !counts || !lens_out || (tbl_width && !table))) ||
            (free_len && !free_blocks))
            inval("block_table_extend: null operand");
        // a thread a token or fresh block, of which there is about one a sequence
        // and one a page of tokens
        const unsigned grid = grid_1d((long long)tokens + tokens / page + batch, 256,
                                      4 * dev_info().cu_count);
        block_table_extend_kernel<<<grid, 256, 0, as_stream(stream)>>>(
            table, lens, counts, free_blocks, free_len, n_free, slots, positions, offsets,
            lens_out, n_free_out, batch, FastDiv(page), tbl_width, tokens);
        launch_check("block table kernel launch");
    });
}

int ft_kv_append_paged_int8_launch(const void* k_new, const void* v_new, int dtype,
                                   const int* slots, signed char* k_pool, signed char* v_pool,
                                   float* k_scales, float* v_scales, int tokens, int kv_heads,
                                   int dim, int blocks, int page, uintptr_t stream) {
    return guarded([&] {
        check_pools(blocks, kv_heads, page, dim);
        if (tokens < 0) inval("kv_append_paged_int8: tokens must be >= 0");
        if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
            inval("kv_append_paged_int8: unknown element type");
        if (tokens == 0 || blocks == 0) return;
        if (!k_new || !v_new || !slots || !k_pool || !v_pool || !k_scales || !v_scales)
            inval("kv_append_paged_int8: null operand");
        check_aligned(k_new, 4 * size_of(dtype), "k_new");
        check_aligned(v_new, 4 * size_of(dtype), "v_new");
        check_aligned(k_pool, 4, "k_pool");
        check_aligned(v_pool, 4, "v_pool");
        // (twice as many, a grid's step on top, are counted in 31 bits)
        if ((long long)tokens * kv_heads > (1LL << 29))
            inval("kv_append_paged_int8: too many rows for one call");
        const hipStream_t s = as_stream(stream);
        auto go = [&](auto zero) {
            using T = decltype(zero);
            append8((const T*)k_new, (const T*)v_new, slots, k_pool, v_pool, k_scales, v_scales,
                    tokens, kv_heads, dim, blocks, page, s);
        };
        if (dtype == FT_DT_F32) go(0.0f);
        else if (dtype == FT_DT_BF16) go((bf16)0.0f);
        else go((f16)0.0f);
    });
}

int ft_attention_decode_paged_int8_workspace(int dtype, int batch, int q_heads, int kv_heads,
                                             int page, int tbl_width, int dim, long long* bytes) {
    return guarded([&] {
        if (!bytes) inval("attention: null operand");
        *bytes = (long long)attn8_shape(dtype, batch, q_heads, kv_heads, page, tbl_width, dim).bytes;
    });
}

int ft_attention_decode_paged_int8_launch(const void* q, int dtype, const signed char* k_pool,
                                          const signed char* v_pool, const float* k_scales,
                                          const float* v_scales, const int* table,
                                          const int* lens, void* out, void* workspace,
                                          long long workspace_bytes, int batch, int q_heads,
                                          int kv_heads, int blocks, int page, int tbl_width,
                                          int dim, uintptr_t stream) {
    return guarded([&] {
        check_pools(blocks, kv_heads, page, dim);
        // (without a block, one launch writes every head's zeros)
        if (blocks == 0 && (long long)batch * q_heads >= 1 << 24)
            inval("attention problem too large for one launch");
        // whole 16-byte chunks of a row on the matrix-core path
        const size_t by = dim % 16 == 0 ? 16 : 4;
        check_aligned(k_pool, by, "k_pool");
        check_aligned(v_pool, by, "v_pool");
        check_aligned(q, std::max(by, 4 * size_of(dtype)), "q");
        check_aligned(out, std::max(by, 4 * size_of(dtype)), "out");
        check_aligned(workspace, 16, "the workspace");
        const Attn8Shape sh =
            attn8_shape(dtype, batch, q_heads, kv_heads, page, tbl_width, dim);
        if (batch == 0) return;
        if (!q || !out || (sh.span > 0 && !table) ||
            (sh.span > 0 && blocks > 0 && (!k_pool || !v_pool || !k_scales || !v_scales)))
            inval("attention: null operand");
        if (sh.bytes && (!workspace || workspace_bytes < (long long)sh.bytes))
            inval("attention: this call needs " + std::to_string(sh.bytes) +
                  " bytes of workspace");
        const Attn8Args a{q,   k_pool,    v_pool, k_scales, v_scales, table,
                          lens, out, workspace, blocks};
        const hipStream_t s = as_stream(stream);
        if (dtype == FT_DT_F32) attn8_run<float>(sh, a, s);
        else if (dtype == FT_DT_BF16) attn8_run<bf16>(sh, a, s);
        else attn8_run<f16>(sh, a, s);
    });
}

}  // extern "C"
