// A paged KV cache held in 8 bits, for gfx950: block tables and slot maps
// from lengths, the append of fresh keys and values, and decode attention.
//
// The cache. k_pool / v_pool are int8 [blocks, kv heads, page, dim], k_scales /
// v_scales float32 [blocks, kv heads]; the value at row r of block n, head h is
// code * scale[n, h]. A slot is block * page + row.
#include <climits>

#include "ft_common.hpp"

#include <algorithm>

namespace ft {
namespace {

constexpr int kMaxDim8 = 512;
constexpr int kMaxPage8 = 1024;      // rows of a block (the append's row map in LDS)
constexpr int kExtendSeqs = 4096;    // sequences of one table call (two prefixes in LDS)
constexpr float kLog2e = 1.4426950408889634f;

void check_pools(int blocks, int hkv, int page, int dim) {
    if (blocks < 0 || hkv < 1 || dim < 1) inval("int8 cache: blocks >= 0, kv heads >= 1, dim >= 1");
    if (dim % 4 != 0 || dim > kMaxDim8)
        inval("int8 cache: dim must be a multiple of 4 and at most 512");
    if (page < 1 || page > kMaxPage8) inval("int8 cache: page must be in [1, 1024]");
    if ((long long)blocks * page > INT_MAX) inval("int8 cache: slots must fit 31 bits");
    if ((long long)blocks * page * hkv > UINT_MAX)
        inval("int8 cache: blocks * page * kv heads must fit 32 bits");
}

// Rows are read 4 elements at a time: every row starts at a multiple of 4
// elements (dim % 4 == 0) where the tensor does.
void check_aligned(const void* p, size_t bytes, const char* what) {
    if ((uintptr_t)p % bytes)
        inval(std::string("int8 cache: ") + what + " must be aligned to 4 elements");
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
// Decode attention, any shape (attn8_general): one workgroup per (sequence, kv
// head, chunk of tokens), 8 q heads at a time, dot products on the vector ALU.
// Each leaves the float32 partial (m, l, acc[D]) of every q head, in log2
// units; attn8_combine folds a row's partials by the log-sum-exp rule. A table
// entry outside [0, blocks) is a hole: its tokens weigh nothing.
// ---------------------------------------------------------------------------
constexpr int kGen8Heads = 8, kGen8Chunk = 256;

__device__ __forceinline__ int clamp_len8(const int* lens, int b, int span) {
    return lens ? min(max(lens[b], 0), span) : span;
}

template <typename T>
__global__ __launch_bounds__(256) void attn8_general(
    const T* __restrict__ q, const signed char* __restrict__ k_pool,
    const signed char* __restrict__ v_pool, const float* __restrict__ k_scales,
    const float* __restrict__ v_scales, const int* __restrict__ table,
    const int* __restrict__ lens, float* __restrict__ ws_ml, float* __restrict__ ws_acc, int hq,
    int hkv, int dim, int blocks, int page, int width, int span, float scale_log2) {
    __shared__ float s_sc[kGen8Heads][kGen8Chunk];
    __shared__ float s_vs[kGen8Chunk];
    __shared__ long long s_row[kGen8Chunk];  // element offset of the token's row, -1 a hole
    __shared__ float s_m[kGen8Heads], s_l[kGen8Heads];
    __shared__ float4 s_red[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int c = blockIdx.x, kv = blockIdx.y, b = blockIdx.z, cmax = gridDim.x;
    const int group = hq / hkv, len = clamp_len8(lens, b, span), t0 = c * kGen8Chunk;
    if (t0 >= len) return;
    const int n = min(kGen8Chunk, len - t0), dc = dim / 4;
    float my_ks = 0.0f;
    if (tid < n) {
        const int t = t0 + tid, ent = table[(size_t)b * width + t / page];
        const bool ok = (unsigned)ent < (unsigned)blocks;
        const size_t bh = (size_t)(ok ? ent : 0) * hkv + kv;
        s_row[tid] = ok ? (long long)((bh * page + t % page) * dim) : -1;
        s_vs[tid] = ok ? v_scales[bh] : 0.0f;
        my_ks = ok ? k_scales[bh] * scale_log2 : 0.0f;
    }
    __syncthreads();
    for (int g0 = 0; g0 < group; g0 += kGen8Heads) {
        const int gc = min(kGen8Heads, group - g0);
        const T* qg = q + ((size_t)b * hq + (size_t)kv * group + g0) * dim;
        if (tid < n) {  // scores: a thread a token
            float part[kGen8Heads] = {};
            if (s_row[tid] >= 0) {
                const char4* kr = reinterpret_cast<const char4*>(k_pool + s_row[tid]);
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
#pragma unroll
            for (int g = 0; g < kGen8Heads; ++g)
                s_sc[g][tid] = s_row[tid] >= 0 ? part[g] * my_ks : -INFINITY;
        }
        __syncthreads();
        for (int g = wave; g < gc; g += 4) {
            float m = -INFINITY;
            for (int t = lane; t < n; t += 64) m = fmaxf(m, s_sc[g][t]);
            m = wave_max(m);
            const float top = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            for (int t = lane; t < n; t += 64) {
                const float p = exp2f(s_sc[g][t] - top);
                l += p;
                s_sc[g][t] = s_row[t] >= 0 ? p * s_vs[t] : 0.0f;
            }
            l = wave_sum(l);
            if (lane == 0) {
                s_m[g] = m;
                s_l[g] = l;
            }
        }
        __syncthreads();
        const int ng = 256 / dc, tg = tid / dc, d4 = tid - tg * dc;
        const size_t slot0 = (((size_t)b * hkv + kv) * cmax + c) * group + g0;
        for (int g = 0; g < gc; ++g) {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            if (tg < ng)
                for (int t = tg; t < n; t += ng) {
                    if (s_row[t] < 0) continue;
                    const char4 vv = *reinterpret_cast<const char4*>(v_pool + s_row[t] + 4 * d4);
                    const float w = s_sc[g][t];
                    a.x += w * vv.x; a.y += w * vv.y; a.z += w * vv.z; a.w += w * vv.w;
                }
            s_red[tid] = a;
            __syncthreads();
            if (tg == 0) {
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

// One workgroup per (sequence, q head).
template <typename T>
__global__ __launch_bounds__(256) void attn8_combine(const float* __restrict__ ws_ml,
                                                     const float* __restrict__ ws_acc,
                                                     const int* __restrict__ lens,
                                                     T* __restrict__ out, int hq, int hkv, int dim,
                                                     int span, int cmax) {
    __shared__ float s_red[4];
    __shared__ float4 s_acc[256];
    const int tid = threadIdx.x, b = blockIdx.x / hq, hh = blockIdx.x - b * hq;
    const int group = hq / hkv, kv = hh / group, gi = hh - kv * group, dc = dim / 4;
    T* o = out + (size_t)blockIdx.x * dim;
    const int np = (clamp_len8(lens, b, span) + kGen8Chunk - 1) / kGen8Chunk;
    auto slot = [&](int i) { return (((size_t)b * hkv + kv) * cmax + i) * group + gi; };
    float mx = -INFINITY;
    for (int i = tid; i < np; i += 256) mx = fmaxf(mx, ws_ml[slot(i) * 2]);
    mx = block_max<256>(mx, s_red);
    // (a piece of no weight, l = 0, has m = -inf)
    auto weight = [&](int i) {
        return ws_ml[slot(i) * 2 + 1] == 0.0f ? 0.0f : exp2f(ws_ml[slot(i) * 2] - mx);
    };
    float l = 0.0f;
    for (int i = tid; i < np; i += 256) l += weight(i) * ws_ml[slot(i) * 2 + 1];
    l = block_sum<256>(l, s_red);
    const int ng = 256 / dc, tg = tid / dc, d4 = tid - tg * dc;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (tg < ng)
        for (int i = tg; i < np; i += ng) {
            const float w = weight(i);
            const float4 x = *reinterpret_cast<const float4*>(ws_acc + slot(i) * dim + 4 * d4);
            a.x += w * x.x; a.y += w * x.y; a.z += w * x.z; a.w += w * x.w;
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

struct Attn8Shape {
    int batch, hq, hkv, page, width, dim, span, cmax;
    size_t slots, bytes;
};

Attn8Shape attn8_shape(int batch, int hq, int hkv, int page, int width, int dim) {
    check_pools(0, hkv, page, dim);
    if (batch < 0 || hq < 1 || width < 0) inval("attention: batch >= 0, q heads >= 1, width >= 0");
    if (hq % hkv != 0) inval("q heads must be a multiple of kv heads (contiguous GQA groups)");
    const long long span = (long long)width * page;
    if (span > (1LL << 30)) inval("table capacity too large");
    Attn8Shape s{batch, hq, hkv, page, width, dim, (int)span, 0, 0, 0};
    s.cmax = (int)((span + kGen8Chunk - 1) / kGen8Chunk);
    s.slots = (size_t)batch * hq * s.cmax;
    s.bytes = (((s.slots * 2 + 63) & ~(size_t)63) + s.slots * dim) * sizeof(float);
    return s;
}

template <typename T>
void attn8_run(const Attn8Shape& sh, const void* q, const signed char* kp, const signed char* vp,
               const float* ks, const float* vs, const int* table, const int* lens, void* out,
               int blocks, void* ws, hipStream_t s) {
    float* ml = (float*)ws;
    float* acc = ml + ((sh.slots * 2 + 63) & ~(size_t)63);
    if (sh.hkv > 65535 || sh.batch > 65535) inval("attention: batch and kv heads must be <= 65535");
    const float scale = (1.0f / sqrtf((float)sh.dim)) * kLog2e;
    if (sh.cmax) {
        attn8_general<T><<<dim3(sh.cmax, sh.hkv, sh.batch), 256, 0, s>>>(
            (const T*)q, kp, vp, ks, vs, table, lens, ml, acc, sh.hq, sh.hkv, sh.dim, blocks,
            sh.page, sh.width, sh.span, scale);
        launch_check("int8 decode attention kernel launch");
    }
    attn8_combine<T><<<(unsigned)(sh.batch * sh.hq), 256, 0, s>>>(
        ml, acc, lens, (T*)out, sh.hq, sh.hkv, sh.dim, sh.span, sh.cmax);
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

int ft_attention_decode_paged_int8_workspace(int batch, int q_heads, int kv_heads, int page,
                                             int tbl_width, int dim, long long* bytes) {
    return guarded([&] {
        if (!bytes) inval("attention: null operand");
        *bytes = (long long)attn8_shape(batch, q_heads, kv_heads, page, tbl_width, dim).bytes;
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
        const Attn8Shape sh = attn8_shape(batch, q_heads, kv_heads, page, tbl_width, dim);
        check_pools(blocks, kv_heads, page, dim);
        if (dtype != FT_DT_F32 && dtype != FT_DT_BF16 && dtype != FT_DT_F16)
            inval("attention: unknown element type");
        if (batch == 0) return;
        if (!q || !out || (sh.span > 0 && !table) ||
            (sh.span > 0 && blocks > 0 && (!k_pool || !v_pool || !k_scales || !v_scales)))
            inval("attention: null operand");
        if (sh.bytes && (!workspace || workspace_bytes < (long long)sh.bytes))
            inval("attention: this call needs " + std::to_string(sh.bytes) +
                  " bytes of workspace");
        check_aligned(q, 4 * size_of(dtype), "q");
        check_aligned(out, 4 * size_of(dtype), "out");
        check_aligned(k_pool, 4, "k_pool");
        check_aligned(v_pool, 4, "v_pool");
        check_aligned(workspace, 16, "the workspace");
        const hipStream_t s = as_stream(stream);
        if (dtype == FT_DT_F32)
            attn8_run<float>(sh, q, k_pool, v_pool, k_scales, v_scales, table, lens, out, blocks,
                             workspace, s);
        else if (dtype == FT_DT_BF16)
            attn8_run<bf16>(sh, q, k_pool, v_pool, k_scales, v_scales, table, lens, out, blocks,
                            workspace, s);
        else
            attn8_run<f16>(sh, q, k_pool, v_pool, k_scales, v_scales, table, lens, out, blocks,
                           workspace, s);
    });
}

}  // extern "C"
