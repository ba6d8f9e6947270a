// A paged KV cache held in 8 bits, for gfx950: block tables and slot maps
// from lengths, the append of fresh keys and values, and decode attention.
//
// The cache. k_pool / v_pool are int8 [blocks, kv heads, page, dim], k_scales /
// v_scales float32 [blocks, kv heads]; the value at row r of block n, head h is
// code * scale[n, h]. A slot is block * page + row.
#include "attn_stream.hpp"
#include "ft_common.hpp"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace ft {
namespace {

constexpr int kMaxDim8 = 512;
constexpr int kMaxPage8 = 1024;      // rows of a block (the append's row map in LDS)
constexpr int kExtendSeqs = 4096;    // sequences of one table call (two prefixes in LDS)

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
// launch and the dependent chain length -> scan -> bisection -> table.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void block_table_extend_kernel(
    int* __restrict__ table, const int* __restrict__ lens, const int* __restrict__ counts,
    const int* __restrict__ free_blocks, int free_len, const int* __restrict__ n_free,
    int* __restrict__ slots, int* __restrict__ positions, int* __restrict__ offsets,
    int* __restrict__ lens_out, int* __restrict__ n_free_out, int batch, int page, int width,
    int tokens) {
    __shared__ int s_off[kExtendSeqs + 1];   // fresh tokens before sequence b (saturated)
    __shared__ int s_need[kExtendSeqs + 1];  // fresh blocks before sequence b
    __shared__ long long s_wave[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long span = (long long)width * page;

    const int per = (batch + 255) / 256;
    const int b0 = min(batch, tid * per), b1 = min(batch, b0 + per);
    auto len_of = [&](int b) { return min((long long)max(lens[b], 0), span); };
    auto need_of = [&](long long len, long long add) {
        const long long end = min(len + add, span);
        return (end + page - 1) / page - (len + page - 1) / page;
    };
    long long toks = 0, need = 0;
    for (int b = b0; b < b1; ++b) {
        const long long add = max(counts[b], 0);
        toks += add;
        need += need_of(len_of(b), add);
    }
    long long it = toks, in = need;  // inclusive over the wave, then the workgroup
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long yt = __shfl_up(it, o, 64), yn = __shfl_up(in, o, 64);
        if (lane >= o) {
            it += yt;
            in += yn;
        }
    }
    if (lane == 63) {
        s_wave[0][wave] = it;
        s_wave[1][wave] = in;
    }
    __syncthreads();
    long long rt = it - toks, rn = in - need;
    long long all_t = 0, all_n = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) {
            rt += s_wave[0][w];
            rn += s_wave[1][w];
        }
        all_t += s_wave[0][w];
        all_n += s_wave[1][w];
    }
    const int total = (int)min(all_t, (long long)INT_MAX);
    const int fresh = (int)all_n;  // <= batch * width, which fits (the table's entries)
    for (int b = b0; b < b1; ++b) {
        s_off[b] = (int)min(rt, (long long)INT_MAX);
        s_need[b] = (int)rn;
        const long long add = max(counts[b], 0), len = len_of(b);
        if (blockIdx.x == 0) {
            offsets[b] = (int)min(rt, (long long)INT_MAX);
            lens_out[b] = (int)min(len + add, span);
        }
        rt += add;
        rn += need_of(len, add);
    }
    const int have = *n_free;
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

    const int stride = gridDim.x * 256;
    for (long long t = blockIdx.x * 256 + tid; t < tokens; t += stride) {
        int slot = -1, pos = 0;
        if (t < total) {
            const int b = find(s_off, (int)t);
            const int len = (int)len_of(b);
            const long long p = (long long)len + (t - s_off[b]);
            pos = (int)min(p, (long long)INT_MAX);
            if (p < span) {
                const int col = (int)(p / page), first = (int)(((long long)len + page - 1) / page);
                const int block = col < first ? table[(size_t)b * width + col]
                                              : taken(s_need[b] + col - first);
                const long long s = (long long)block * page + p % page;
                if (block >= 0 && s <= INT_MAX) slot = (int)s;
            }
        }
        slots[t] = slot;
        positions[t] = pos;
    }
    for (long long k = blockIdx.x * 256 + tid; k < fresh; k += stride) {
        const int b = find(s_need, (int)k);
        const int first = (int)((len_of(b) + page - 1) / page);
        table[(size_t)b * width + first + (k - s_need[b])] = taken((int)k);
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
// starts over). Where scale' > held > 0 the block's other rows become
// rint(f32(code * f32(held / scale'))). All float32, IEEE divisions: codes
// are the same on every path.
// ---------------------------------------------------------------------------
constexpr float kLeastScale = 0x1p-120f;

__device__ __forceinline__ signed char code8(float x, float inv) {
    const float v = rintf(x * inv);
    return v == v ? (signed char)fmaxf(-127.0f, fminf(127.0f, v)) : (signed char)0;
}

// One wave per (token, kv head, K or V): the wave whose token starts a run
// does the whole run.
template <typename T>
__global__ __launch_bounds__(64) void kv_append8_kernel(
    const T* __restrict__ k_new, const T* __restrict__ v_new, const int* __restrict__ slots,
    signed char* __restrict__ k_pool, signed char* __restrict__ v_pool,
    float* __restrict__ k_scales, float* __restrict__ v_scales, int tokens, int hkv, int dim,
    int nslots, int page) {
    __shared__ int s_src[kMaxPage8];  // row of the block -> its fresh row, or -1
    const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y;
    auto block_of = [&](int t) {
        const int s = slots[t];
        return s >= 0 && s < nslots ? s / page : -1;
    };
    const int block = block_of(i);
    if (block < 0 || (i > 0 && block_of(i - 1) == block)) return;
    const T* x = blockIdx.z ? v_new : k_new;
    signed char* codes = (blockIdx.z ? v_pool : k_pool) + ((size_t)block * hkv + h) * page * dim;
    float* scale = (blockIdx.z ? v_scales : k_scales) + (size_t)block * hkv + h;

    for (int r = lane; r < page; r += 64) s_src[r] = -1;
    __syncthreads();
    for (long long t = i;; t += 64) {
        const bool in = t + lane < tokens && block_of((int)t + lane) == block;
        const unsigned long long out = __ballot(!in);
        const int n = out ? __builtin_ctzll(out) : 64;
        if (lane < n) atomicMax(&s_src[slots[t + lane] % page], (int)t + lane);
        if (n < 64) break;
    }
    __syncthreads();
    const int dc = dim / 4;
    float most = 0.0f;
    for (int j = lane; j < page * dc; j += 64) {
        const int r = j / dc, src = s_src[r];
        if (src < 0) continue;
        const float4 v = St<T>::ld4(x + ((size_t)src * hkv + h) * dim + 4 * (j - r * dc));
        const float e[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
        for (int c = 0; c < 4; ++c)
            if (e[c] < INFINITY) most = fmaxf(most, e[c]);
    }
    most = wave_max(most);
    const bool over = s_src[0] >= 0;
    const float held = over ? 0.0f : *scale;
    const float now = fmaxf(fmaxf(held, most / 127.0f), kLeastScale);
    const float inv = 1.0f / now, ratio = held / now;
    const bool grown = !over && now > held;
    for (int j = lane; j < page * dc; j += 64) {
        const int r = j / dc, src = s_src[r];
        char4* p = reinterpret_cast<char4*>(codes + (size_t)r * dim + 4 * (j - r * dc));
        if (src >= 0) {
            const float4 v = St<T>::ld4(x + ((size_t)src * hkv + h) * dim + 4 * (j - r * dc));
            *p = make_char4(code8(v.x, inv), code8(v.y, inv), code8(v.z, inv), code8(v.w, inv));
        } else if (grown) {
            const char4 c = *p;
            *p = make_char4(code8(c.x, ratio), code8(c.y, ratio), code8(c.z, ratio),
                            code8(c.w, ratio));
        }
    }
    __syncthreads();
    if (lane == 0) *scale = now;
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

// Where the pieces of row (b, head) lie in the workspace: piece i at slot
// at(i), `rows` q heads a slot. count 0: no token; -1: the row is stored
// already.
struct Chunked8 {  // attn8_general: a slot per (row, chunk)
    int cmax, chunk;
    struct Row {
        size_t first;
        int count;
        __device__ __forceinline__ size_t at(int i) const { return first + i; }
    };
    __device__ __forceinline__ Row row(int b, int vrow, int vrows, int len) const {
        return Row{((size_t)b * vrows + vrow) * cmax, (len + chunk - 1) / chunk};
    }
};

struct Streamed8 {  // attn8_stream: two slots a segment (kernel comment)
    const long long* pref;  // prefix of the lengths [batch + 1], then the segment length
    int batch;
    struct Row {
        long long s_lo, end, seg;
        int count;
        __device__ __forceinline__ size_t at(int i) const {
            const long long s = s_lo + i;
            return (size_t)(2 * s + (end >= (s + 1) * seg ? 1 : 0));
        }
    };
    __device__ __forceinline__ Row row(int b, int vrow, int vrows, int len) const {
        const long long seg = pref[batch + 1], start = pref[b] * vrows + (long long)vrow * len;
        if (len == 0) return Row{0, 0, seg, 0};
        const long long lo = start / seg, hi = (start + len - 1) / seg;
        return Row{lo, start + len, seg, lo == hi ? -1 : (int)(hi - lo + 1)};
    }
};

// One workgroup per (sequence, q head).
template <typename T, typename Pieces>
__global__ __launch_bounds__(256) void attn8_combine(
    const float* __restrict__ ws_ml, const float* __restrict__ ws_acc,
    const int* __restrict__ lens, T* __restrict__ out, Pieces pieces, int hq, int hkv, int dim,
    int span, int tile, int tiles) {
    __shared__ float s_red[4];
    __shared__ float4 s_acc[256];
    const int tid = threadIdx.x, b = blockIdx.x / hq, hh = blockIdx.x - b * hq;
    const int group = hq / hkv, kv = hh / group, gi = hh - kv * group, dc = dim / 4;
    T* o = out + (size_t)blockIdx.x * dim;
    const auto row = pieces.row(b, kv * tiles + gi / tile, hkv * tiles, clamp_len(lens, b, span));
    const int np = row.count;
    if (np < 0) return;
    auto slot = [&](int i) { return row.at(i) * tile + gi % tile; };
    float mx = -INFINITY;
    for (int i = tid; i < np; i += 256) mx = fmaxf(mx, ws_ml[slot(i) * 2]);
    mx = block_max<256>(mx, s_red);
    auto weight = [&](int i) {
        return ws_ml[slot(i) * 2 + 1] == 0.0f ? 0.0f : exp2f(ws_ml[slot(i) * 2] - mx);
    };
    float l = 0.0f;
    for (int i = tid; i < np; i += 256) l += weight(i) * ws_ml[slot(i) * 2 + 1];
    l = block_sum<256>(l, s_red);
    const int ng = 256 / dc, tg = tid / dc, d4 = tid - tg * dc;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (tg < ng) {
#pragma unroll 4
        for (int i = tg; i < np; i += ng) {
            const float w = weight(i);
            const float4 x = *reinterpret_cast<const float4*>(ws_acc + slot(i) * dim + 4 * d4);
            a.x += w * x.x; a.y += w * x.y; a.z += w * x.z; a.w += w * x.w;
        }
    }
    s_acc[tid] = a;
    __syncthreads();
    if (tg != 0) return;
    for (int j = 1; j < ng; ++j) {
        const float4 x = s_acc[j * dc + d4];
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    }
    if (l == 0.0f) a = make_float4(0.f, 0.f, 0.f, 0.f);
    else a = make_float4(a.x / l, a.y / l, a.z / l, a.w / l);
    St<T>::st4(o + 4 * d4, a);
}

// ---------------------------------------------------------------------------
// Any head dim (attn8_general): one workgroup per (sequence, kv head, chunk of
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
// D = 64, 128, 256 (attn8_stream): matrix cores, each K / V byte read once.
//
// Work split. The rows are (sequence b, kv head, tile of up to 16 q heads),
// b-major, len_b tokens each, laid end to end; every WAVE takes one equal
// contiguous segment of that range, whatever the length mix. A segment is one
// or more pieces, one per row it touches. A piece that is a whole row is
// normalised and stored; another leaves its partial in the segment's slot 1
// if its row reaches the segment's end, else in slot 0: a segment has at most
// one of each. Waves share nothing but the length prefix, so after it there
// is no barrier and no merge in the kernel.
//
// A step is TOK tokens (32; 64 for D = 64), K and V of the next one in flight
// in registers while this one is computed from the wave's own LDS staging.
// With r = lane % 16, g = lane / 16 (v_mfma_f32_16x16x32_bf16: A[r][8g+i],
// B[8g+i][r], C[4g+i][r]):
//
//  loads    whole 128-byte lines per instruction, non-temporal, of rows whose
//           places the lanes have worked out from the table (a lane a token)
//           and hand out by shuffles;
//  scores   S^T[tok][head] = K . Q^T. Codes become bf16 (exact: 8 bits); q
//           goes in as 1, 2 or 3 bf16 parts (bf16, fp16, float32: all its
//           bits), so every product is exact and sums are float32. Any order
//           of dims serves if q has the same: the lane reads 16-byte chunks;
//  softmax  lane (r, g) holds head r's scores of tokens 4g+i (+ 16 a tile);
//           scaled by the block's K scale, running maximum over the 4 lanes
//           of a head; the weight takes the block's V scale, then goes into 2
//           bf16 parts (3 for float32 outputs), which hold any float's
//           magnitude: small weights count as they weigh;
//  PV       O^T[dim][head] = V^T . W^T. The weights are where B wants them; for
//           A, lane (r, g) reads dims (D/16) r .. of its 8 tokens from the
//           staging and pairs the tokens up while it widens them, so the
//           transpose costs nothing. Lane (r, g) ends with D/4 consecutive
//           dims of head r.
//
// Masked tokens (behind the piece, holes) weigh 0 exactly: score -inf, V scale
// 0, the row read in its place a real one (its own last, or block 0's).
// ---------------------------------------------------------------------------
typedef float f32x4_8 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <typename T, int D>
struct Stream8 {
    static constexpr int kTok = D == 64 ? 64 : 32;   // tokens a step
    static constexpr int kLoads = kTok * D / 1024;   // 16-byte loads a lane and pool
    static constexpr int kRowsPer = 1024 / D;        // rows a load instruction covers
    static constexpr int kChunks = D / 16;           // 16-byte chunks of a row
    static constexpr int kQ = std::is_same<T, float>::value ? 3 : std::is_same<T, f16>::value ? 2 : 1;
    static constexpr int kW = std::is_same<T, float>::value ? 3 : 2;  // weight parts
    static constexpr int kOcc = D == 256 ? 1 : std::is_same<T, float>::value ? 2 : 3;  // waves a SIMD
    static constexpr int kLds = 2 * kTok * D + 8 * kTok;  // bytes a wave
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
// x[8] as N bf16 parts, each truncated, the first the largest (an infinity
// leaves NaN behind it: only a scale that is not finite makes one).
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], b16x8 (&part)[N]) {
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int p = 0; p < N; ++p) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = pack_hi(rest[2 * i], rest[2 * i + 1]);
        part[p] = __builtin_bit_cast(b16x8, o);
        if (p + 1 < N) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float hi = __uint_as_float(__float_as_uint(rest[i]) & 0xffff0000u);
                rest[i] -= hi;
            }
        }
    }
}
__device__ __forceinline__ f32x4_8 mma8(b16x8 a, b16x8 b, f32x4_8 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <typename T, int D>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(Stream8<T, D>::kOcc, Stream8<T, D>::kOcc)))
void attn8_stream(const T* __restrict__ q, const signed char* __restrict__ k_pool,
                  const signed char* __restrict__ v_pool, const float* __restrict__ k_scales,
                  const float* __restrict__ v_scales, const int* __restrict__ table,
                  const int* __restrict__ lens, float* __restrict__ ws_ml,
                  float* __restrict__ ws_acc, long long* __restrict__ pref_out,
                  T* __restrict__ out, int batch, int hq, int hkv, int tile, int tiles,
                  int blocks, int page, int page_shift, int width, int span, int nseg, int min_seg,
                  float scale_log2) {
    using C = Stream8<T, D>;
    constexpr int TOK = C::kTok, NL = C::kLoads, SUB = TOK / 32, KE = D / 64;
    __shared__ __align__(16) char s_stage[4][C::kLds];
    __shared__ long long s_pref[kStreamScanRows + 1];
    __shared__ int s_mm[2];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    if (wave == 0) scan_lengths(lens, batch, span, lane, s_pref, s_mm);
    __syncthreads();
    const int vrows = hkv * tiles;
    const long long total = uniform64(s_pref[batch]) * vrows;
    long long S = max((total + nseg - 1) / nseg, (long long)min_seg);
    S = (S + TOK - 1) / TOK * TOK;
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

    long long pos = seg_lo;
    while (pos < seg_hi) {
        const StreamPiece pc = stream_piece(s_pref, batch, vrows, pos, seg_hi);
        const int b = pc.b, kv = pc.kv / tiles, t0 = pc.t0, n = pc.n;
        const int h0 = kv * (hq / hkv) + (pc.kv - kv * tiles) * tile;     // first q head
        const int heads = min(tile, (kv + 1) * (hq / hkv) - h0);
        const int* trow = table + (size_t)b * width;
        const int nsteps = (n + TOK - 1) / TOK;

        auto token = [&](int st) { return t0 + min(st * TOK + my, n - 1); };
        auto entry = [&](int st) {
            const int t = token(st);
            return trow[page_shift >= 0 ? t >> page_shift : t / page];
        };
        u32x4 kt[NL], vt[NL];
        float ksn, vsn;
        unsigned long long seen;  // lanes whose token of the loaded step counts
        auto issue = [&](int st, int ent) {
            const int t = token(st);
            const bool held = (unsigned)ent < (unsigned)blocks;
            const unsigned bh = (unsigned)(held ? ent : 0) * hkv + kv;
            const unsigned row = bh * page + (page_shift >= 0 ? t & (page - 1) : t % page);
            const bool ok = held && st * TOK + my < n;
            seen = __ballot(ok);
            const float ks = k_scales[bh], vs = v_scales[bh];
            ksn = ok ? ks * scale_log2 : 0.0f;
            vsn = ok ? vs : 0.0f;
#pragma unroll
            for (int p = 0; p < NL; ++p) {
                const unsigned rw = __shfl(row, C::kRowsPer * p + lr, 64);
                const size_t off = (size_t)rw * D + 16 * lc;
                kt[p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k_pool + off));
                vt[p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(v_pool + off));
            }
        };

        int ent = entry(0);
        // B operand of the score products: Q[head r], parts
        b16x8 qf[KE][2][C::kQ];
        {
            const T* qrow = q + ((size_t)b * hq + h0 + (r < heads ? r : 0)) * D;
#pragma unroll
            for (int e = 0; e < KE; ++e)
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float4 y = St<T>::ld4(qrow + 64 * e + 16 * g + 8 * f + 4 * i);
                        x[4 * i] = y.x; x[4 * i + 1] = y.y; x[4 * i + 2] = y.z; x[4 * i + 3] = y.w;
                    }
                    split8<C::kQ>(x, qf[e][f]);
                }
        }
        issue(0, ent);
        ent = entry(min(1, nsteps - 1));

        f32x4_8 acc[C::kChunks];
#pragma unroll
        for (int i = 0; i < C::kChunks; ++i) acc[i] = f32x4_8{0.f, 0.f, 0.f, 0.f};
        float m_run = -INFINITY, l_run = 0.0f;

        for (int st = 0; st < nsteps; ++st) {
            // ---- this step into the staging, the next one on its way -------
            wave_lds_order();  // (the step before has read it)
#pragma unroll
            for (int p = 0; p < NL; ++p) {
                const int w = C::kRowsPer * p + lr;
                *reinterpret_cast<u32x4*>(sk + k_at(w, lc)) = kt[p];
                *reinterpret_cast<u32x4*>(sv + v_at(w) + 16 * lc) = vt[p];
            }
            if (TOK == 64 || lane < 32) ss[my] = make_float2(ksn, vsn);
            const unsigned long long now = seen;
            wave_lds_order();
            if (st + 1 < nsteps) {
                const int e = ent;
                ent = entry(min(st + 2, nsteps - 1));
                issue(st + 1, e);
            }
            __builtin_amdgcn_sched_barrier(0);

            // ---- scores ------------------------------------------------------
            float x[8 * SUB], vsc[8 * SUB];
#pragma unroll
            for (int h = 0; h < 2 * SUB; ++h) {
                f32x4_8 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < KE; ++e) {
                    const u32x4 kc = *reinterpret_cast<const u32x4*>(sk + k_at(16 * h + r, 4 * e + g));
#pragma unroll
                    for (int f = 0; f < 2; ++f) {
                        const b16x8 a = widen8(kc[2 * f], kc[2 * f + 1]);
#pragma unroll
                        for (int p = C::kQ - 1; p >= 0; --p) s = mma8(a, qf[e][f][p], s);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 sc = ss[16 * h + 4 * g + i];
                    x[4 * h + i] = s[i] * sc.x;
                    vsc[4 * h + i] = sc.y;
                }
            }
            if (now != ~0ull) {
#pragma unroll
                for (int h = 0; h < 2 * SUB; ++h) {
                    const unsigned bits = (unsigned)(now >> (16 * h + 4 * g));
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(bits >> i & 1)) x[4 * h + i] = -INFINITY;
                }
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
                b16x8 wp[C::kW];
                split8<C::kW>(w, wp);
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
                            acc[4 * j + d] = mma8(a, wp[p], acc[4 * j + d]);
                    }
                }
            }
        }

        // ---- the row, or its partial -----------------------------------------
        l_run += __shfl_xor(l_run, 16, 64);
        l_run += __shfl_xor(l_run, 32, 64);
        if (r < heads) {
            // dims (D/4) g + (D/16) i + d of head r: acc[d][i]
            if (pc.whole) {
                T* o = out + ((size_t)b * hq + h0 + r) * D + (D / 4) * g;
                const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < C::kChunks; d += 4) {
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
                const long long end = uniform64(s_pref[b]) * vrows +
                                      (long long)(pc.kv + 1) * (uniform64(s_pref[b + 1]) -
                                                                uniform64(s_pref[b]));
                const size_t slot =
                    (2 * (size_t)seg + (end >= seg_lo + S ? 1 : 0)) * tile + r;
                float* o = ws_acc + slot * D + (D / 4) * g;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < C::kChunks; d += 4)
                        *reinterpret_cast<float4*>(o + (D / 16) * i + d) = make_float4(
                            acc[d][i], acc[d + 1][i], acc[d + 2][i], acc[d + 3][i]);
                if (g == 0) {
                    ws_ml[slot * 2] = m_run;
                    ws_ml[slot * 2 + 1] = l_run;
                }
            }
        }
        pos = pc.next;
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct Attn8Shape {
    int batch, hq, hkv, page, width, dim, span;
    bool stream;
    int tile, tiles, nseg, min_seg;  // stream
    int cmax, chunk;                 // general
    size_t slots, bytes;             // slots: (partial, q head) pairs
};

constexpr int kMinSeg8 = 64;  // tokens of a segment, at least

template <int D>
int stream_occ(int dtype) {
    return dtype == FT_DT_F32 ? Stream8<float, D>::kOcc
                              : dtype == FT_DT_F16 ? Stream8<f16, D>::kOcc : Stream8<bf16, D>::kOcc;
}

Attn8Shape attn8_shape(int dtype, int batch, int hq, int hkv, int page, int width, int dim) {
    check_pools(0, hkv, page, dim);
    if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
        inval("attention: unknown element type");
    if (batch < 0 || hq < 1 || width < 0) inval("attention: batch >= 0, q heads >= 1, width >= 0");
    if (hq % hkv != 0) inval("q heads must be a multiple of kv heads (contiguous GQA groups)");
    const long long span = (long long)width * page;
    if (span > (1LL << 30)) inval("table capacity too large");
    if ((long long)batch * hq > INT_MAX) inval("attention: too many rows");
    Attn8Shape s{};
    s.batch = batch; s.hq = hq; s.hkv = hkv; s.page = page; s.width = width; s.dim = dim;
    s.span = (int)span;
    if (batch == 0) return s;
    const int cus = dev_info().cu_count, group = hq / hkv;
    s.stream = span > 0 && (dim == 64 || dim == 128 || dim == 256);
    if (s.stream) {
        s.tiles = (group + 15) / 16;
        s.tile = (group + s.tiles - 1) / s.tiles;
        s.tiles = (group + s.tile - 1) / s.tile;
        const int occ = dim == 64 ? stream_occ<64>(dtype)
                                  : dim == 128 ? stream_occ<128>(dtype) : stream_occ<256>(dtype);
        s.min_seg = kMinSeg8;
        const long long rows = (long long)std::min(batch, kStreamScanRows) * hkv * s.tiles;
        const long long most = rows * ((span + s.min_seg - 1) / s.min_seg);
        s.nseg = (int)std::min((long long)4 * cus * occ, most);
        s.slots = (size_t)2 * s.nseg * s.tile;
    } else {
        if (hkv > 65535 || batch > 65535) inval("attention: batch and kv heads must be <= 65535");
        // about 16 workgroups a CU, at least 256 tokens each
        const long long units = std::max(1LL, 16LL * cus / ((long long)batch * hkv));
        s.chunk = (int)std::max(1LL, (span + units - 1) / units);
        s.chunk = (s.chunk + kGen8Step - 1) / kGen8Step * kGen8Step;
        s.cmax = (int)((span + s.chunk - 1) / s.chunk);
        s.tile = group;
        s.tiles = 1;
        s.slots = (size_t)batch * hq * s.cmax;
    }
    s.bytes = (((s.slots * 2 + 63) & ~(size_t)63) + s.slots * dim) * sizeof(float) +
              (s.stream ? (std::min(batch, kStreamScanRows) + 2) * sizeof(long long) : 0);
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
    long long* pref = (long long*)(acc + sh.slots * D);
    int shift = -1;
    if ((sh.page & (sh.page - 1)) == 0)
        for (shift = 0; (1 << shift) < sh.page;) ++shift;
    const float scale = (1.0f / sqrtf((float)D)) * kLog2e;
    for (int b0 = 0; b0 < sh.batch; b0 += kStreamScanRows) {
        const int nb = std::min(kStreamScanRows, sh.batch - b0);
        const T* q = (const T*)a.q + (size_t)b0 * sh.hq * D;
        T* out = (T*)a.out + (size_t)b0 * sh.hq * D;
        const int* lens = a.lens ? a.lens + b0 : nullptr;
        attn8_stream<T, D><<<(sh.nseg + 3) / 4, 256, 0, s>>>(
            q, a.kp, a.vp, a.ks, a.vs, a.table + (size_t)b0 * sh.width, lens, ml, acc, pref, out,
            nb, sh.hq, sh.hkv, sh.tile, sh.tiles, a.blocks, sh.page, shift, sh.width, sh.span,
            sh.nseg, sh.min_seg, scale);
        launch_check("int8 decode attention kernel launch");
        attn8_combine<T, Streamed8><<<(unsigned)(nb * sh.hq), 256, 0, s>>>(
            ml, acc, lens, out, Streamed8{pref, nb}, sh.hq, sh.hkv, D, sh.span, sh.tile, sh.tiles);
        launch_check("int8 decode attention combine launch");
    }
}

template <typename T>
void attn8_run(const Attn8Shape& sh, const Attn8Args& a, hipStream_t s) {
    float* ml = (float*)a.ws;
    float* acc = ml + ((sh.slots * 2 + 63) & ~(size_t)63);
    if (sh.stream && a.blocks > 0) {
        if (sh.dim == 64) attn8_stream_run<T, 64>(sh, a, ml, acc, s);
        else if (sh.dim == 128) attn8_stream_run<T, 128>(sh, a, ml, acc, s);
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
    attn8_combine<T, Chunked8><<<(unsigned)(sh.batch * sh.hq), 256, 0, s>>>(
        ml, acc, any ? a.lens : nullptr, (T*)a.out, Chunked8{sh.cmax, std::max(sh.chunk, 1)}, sh.hq,
        sh.hkv, sh.dim, any ? sh.span : 0, sh.tile, sh.tiles);
    launch_check("int8 decode attention combine launch");
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
        if (page < 1 || tbl_width < 0 || tokens < 0 || free_len < 0)
            inval("block_table_extend: page >= 1, width >= 0, tokens >= 0");
        if ((long long)tbl_width * page > (1LL << 30)) inval("table capacity too large");
        if ((long long)tbl_width * batch > INT_MAX) inval("block_table_extend: table too large");
        if (!n_free || !n_free_out || !offsets || (tokens && (!slots || !positions)) ||
            (batch && (!lens || !counts || !lens_out || (tbl_width && !table))) ||
            (free_len && !free_blocks))
            inval("block_table_extend: null operand");
        const unsigned grid = std::min(256u, grid_1d(tokens, 2048));
        block_table_extend_kernel<<<grid, 256, 0, as_stream(stream)>>>(
            table, lens, counts, free_blocks, free_len, n_free, slots, positions, offsets,
            lens_out, n_free_out, batch, page, tbl_width, tokens);
        launch_check("block table kernel launch");
    });
}

int ft_kv_append_paged_int8_launch(const void* k_new, const void* v_new, int dtype,
                                   const int* slots, signed char* k_pool, signed char* v_pool,
                                   float* k_scales, float* v_scales, int tokens, int kv_heads,
                                   int dim, int blocks, int page, uintptr_t stream) {
    return guarded([&] {
        check_pools(blocks, kv_heads, page, dim);
        if (tokens < 0 || kv_heads > 65535) inval("kv_append_paged_int8: tokens >= 0, heads <= 65535");
        if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
            inval("kv_append_paged_int8: unknown element type");
        if (tokens == 0 || blocks == 0) return;
        if (!k_new || !v_new || !slots || !k_pool || !v_pool || !k_scales || !v_scales)
            inval("kv_append_paged_int8: null operand");
        check_aligned(k_new, 4 * size_of(dtype), "k_new");
        check_aligned(v_new, 4 * size_of(dtype), "v_new");
        check_aligned(k_pool, 4, "k_pool");
        check_aligned(v_pool, 4, "v_pool");
        const hipStream_t s = as_stream(stream);
        auto go = [&](auto zero) {
            using T = decltype(zero);
            kv_append8_kernel<T><<<dim3(tokens, kv_heads, 2), 64, 0, s>>>(
                (const T*)k_new, (const T*)v_new, slots, k_pool, v_pool, k_scales, v_scales,
                tokens, kv_heads, dim, blocks * page, page);
        };
        if (dtype == FT_DT_F32) go(0.0f);
        else if (dtype == FT_DT_BF16) go((bf16)0.0f);
        else go((f16)0.0f);
        launch_check("int8 kv append kernel launch");
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
        // whole 16-byte chunks of a row on the matrix-core path
        const size_t by = dim % 16 == 0 ? 16 : 4;
        check_aligned(k_pool, by, "k_pool");
        check_aligned(v_pool, by, "v_pool");
        check_aligned(q, 4 * size_of(dtype), "q");
        check_aligned(out, 4 * size_of(dtype), "out");
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
