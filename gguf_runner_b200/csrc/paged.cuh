// Pages of a KV cache, the launch plan of a batch, and the kernels that write rows into pages and read them back.
//
// A page holds page_size consecutive positions of one sequence in one layer, [KV head][position][head_dim], so that the rows
// of a KV head that attention walks are contiguous. Formats: bf16, or int8 codes with one f32 scale per (position, KV head):
// the head is the unit that attention reads and that heads are sharded by, and its scale then multiplies a whole score or a
// whole softmax weight, which leaves the codes exact operands of the tensor cores. Code and scale follow the rule of the
// 8-bit row caches (src/engine/runtime/inference.rs:1906-1916): m = max |x|, s = m / 127, code = round(x * (127 / m)), half
// away from zero, each step in f32; m = 0 gives s = 1. A head with a value that is not finite gets scale NaN, so that it
// reads back as NaN instead of as a finite row.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "rope_math.cuh"

namespace ggr {

constexpr int kKvQ8Head = 5;     // GGR_KV_Q8_HEAD
constexpr int kPageRowsMin = 16; // rows of the smallest page: one key tile of the warp-level kernels

struct PageView {
    unsigned char* k;
    unsigned char* v;
    float* ks;  // [layer][page][KV head][position], 8-bit pages only
    float* vs;
    int fmt, D, Hkv, page_log2, n_pages;
    __host__ __device__ int64_t row(int layer, int page, int h, int r) const {
        return ((((int64_t)layer * n_pages + page) * Hkv + h) << page_log2) + r;
    }
};

// One piece of attention work: packed rows [row0, row0 + rows) of a sequence against keys [key0, key1). Row r of a sequence
// and KV head stands for its new token r / G and query head r % G of the group, so that a key tile serves all heads that
// share it, whatever the number of tokens.
struct PagedItem {
    int tok0;   // row of the sequence's first new token in q and out
    int pos0;   // its position
    int n_tok;  // new tokens of the sequence
    int row0, rows;
    int key0, key1;  // key0 is a multiple of the kernel's key tile; the last piece ends with the visible keys
    int src;    // paged: index of the sequence's first page in the table; packed: row of its first key
    int part;   // key splits: first partial state of the row tile (in tiles), else -1
    int split, n_split;
    int ticket;
    int kvh;    // tcgen05 kernel only: its items are dealt over all KV heads; row0 is then a token, not a packed row
    int lin;    // and the dense row of the sequence's first key where tiles come from dense rows
    int unused[2];
};

// What a launch reads from the plan on the device.
struct PlanView {
    const int* counts;       // [0] items, [1] table entries, [2] tokens of the list that the launch walks
    const PagedItem* items;
    const int* table;        // page ids, sequence after sequence
};

struct AppendArgs {
    PageView pages;
    RopeParams rope;
    const int* counts;       // [2] tokens
    const int* tok_pos;      // position of every new token
    const int* tok_slot;     // page * page_size + row in the page
    int layer, rotate, write_q, in_bf16, q_bf16;
    int Hq, tokens_per_cta, heads;  // heads: of q (when it is rotated), k and v together
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    int64_t q_stride, k_stride, v_stride, qo_stride;  // elements between rows
};

template <bool BF16>
__device__ __forceinline__ void load8_any(const void* p, int64_t at, float x[8]) {
    if constexpr (BF16)
        load8_in<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(p) + at, x);
    else
        load8_in<float>(static_cast<const float*>(p) + at, x);
}

// RoPE and append of a few tokens per CTA. D / 16 lanes share a head, each with elements [8 j, 8 j + 8) of its lower and of
// its upper half, so that both kinds of RoPE pairs of a fully rotated head lie in one lane and its largest element takes
// log2(D / 16) shuffles. Bound by the bytes of the rows; one token per CTA while tokens are few (a token step is latency:
// the angles of a token, one load, one store), several when there are more CTAs than SMs to hold them.
template <bool BF16>
__global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs a) {
    extern __shared__ float sm[];  // cos [tokens_per_cta][half], sin
    const int D = a.pages.D, lanes = D / 16, half = a.rope.rope_half;
    const int total = a.counts[2], t0 = blockIdx.x * a.tokens_per_cta;
    if (t0 >= total) return;
    const int n = min(a.tokens_per_cta, total - t0);
    float* cs = sm;
    float* sn = sm + a.tokens_per_cta * half;
    if (a.rotate) {
        for (int i = threadIdx.x; i < n * half; i += 256) {
            const int t = i / half, f = i - t * half;
            const float angle = __fmul_rn(__fmul_rn((float)a.tok_pos[t0 + t], a.rope.freqs[f]), a.rope.fscale);
            sincosf(angle, &sn[i], &cs[i]);
        }
        __syncthreads();
    }
    const int Hkv = a.pages.Hkv, nq = a.write_q ? a.Hq : 0;
    const int tasks = n * a.heads * lanes;
    // whole warps take part in the shuffles of the last round
    for (int task = threadIdx.x; task < ((tasks + 31) & ~31); task += 256) {
        const bool live = task < tasks;
        const int unit = live ? task / lanes : 0, j = task & (lanes - 1);
        const int t = unit / a.heads, h = unit - t * a.heads, tok = t0 + t;
        const int kind = h < nq ? 0 : (h < nq + Hkv ? 1 : 2), hh = kind == 0 ? h : (kind == 1 ? h - nq : h - nq - Hkv);
        const void* src = kind == 0 ? a.q : (kind == 1 ? a.k : a.v);
        const int64_t at = tok * (kind == 0 ? a.q_stride : (kind == 1 ? a.k_stride : a.v_stride)) + (int64_t)hh * D;
        const int e0 = j * 8, e1 = D / 2 + j * 8;
        float x[8], y[8];
        if (live) {
            load8_any<BF16>(src, at + e0, x);
            load8_any<BF16>(src, at + e1, y);
        } else {
#pragma unroll
            for (int p = 0; p < 8; ++p) x[p] = y[p] = 0.0f;
        }
        if (a.rotate && kind < 2 && live) {
            const float* c = cs + t * half;
            const float* s = sn + t * half;
            if (a.rope.rope_dim != D) {  // part of a head: partners may lie in other lanes
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    x[p] = rope_elem(src, at, e0 + p, D, a.rope, c, s, BF16);
                    y[p] = rope_elem(src, at, e1 + p, D, a.rope, c, s, BF16);
                }
            } else if (a.rope.style == 0) {
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    const float lo = x[p], hi = y[p], cc = c[e0 + p], ss = s[e0 + p];
                    x[p] = __fsub_rn(__fmul_rn(lo, cc), __fmul_rn(hi, ss));
                    y[p] = __fadd_rn(__fmul_rn(lo, ss), __fmul_rn(hi, cc));
                }
            } else {
#pragma unroll
                for (int p = 0; p < 8; p += 2) {
                    const float x0 = x[p], x1 = x[p + 1], y0 = y[p], y1 = y[p + 1];
                    const int i0 = (e0 + p) >> 1, i1 = (e1 + p) >> 1;
                    x[p] = __fsub_rn(__fmul_rn(x0, c[i0]), __fmul_rn(x1, s[i0]));
                    x[p + 1] = __fadd_rn(__fmul_rn(x0, s[i0]), __fmul_rn(x1, c[i0]));
                    y[p] = __fsub_rn(__fmul_rn(y0, c[i1]), __fmul_rn(y1, s[i1]));
                    y[p + 1] = __fadd_rn(__fmul_rn(y0, s[i1]), __fmul_rn(y1, c[i1]));
                }
            }
        }
        float top = 0.0f, step = 1.0f;
        if (a.pages.fmt == kKvQ8Head) {
            bool odd = false;  // a value that is not finite: max would lose a NaN
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                top = fmaxf(top, fmaxf(fabsf(x[p]), fabsf(y[p])));
                odd |= !isfinite(x[p]) | !isfinite(y[p]);
            }
            if (odd) top = INFINITY;
            if (top < 1e-36f) top = 0.0f;  // 127 / m would overflow: such a row counts as zeros
            for (int o = lanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (!live) continue;
        if (kind == 0) {
            if (a.rope.do_prescale && a.rotate) {
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    x[p] = __fmul_rn(x[p], a.rope.q_prescale);
                    y[p] = __fmul_rn(y[p], a.rope.q_prescale);
                }
            }
            const int64_t to = tok * a.qo_stride + (int64_t)hh * D;
            if (a.q_bf16) {
                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.q_out) + to;
                *reinterpret_cast<uint4*>(o + e0) = pack8(x);
                *reinterpret_cast<uint4*>(o + e1) = pack8(y);
            } else {
                float* o = static_cast<float*>(a.q_out) + to;
                store8_f32(o + e0, x);
                store8_f32(o + e1, y);
            }
            continue;
        }
        const int slot = a.tok_slot[tok];
        const int64_t row = a.pages.row(a.layer, slot >> a.pages.page_log2, hh, slot & ((1 << a.pages.page_log2) - 1));
        unsigned char* pool = kind == 1 ? a.pages.k : a.pages.v;
        if (a.pages.fmt == KV_BF16) {
            __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(pool) + row * D;
            *reinterpret_cast<uint4*>(o + e0) = pack8(x);
            *reinterpret_cast<uint4*>(o + e1) = pack8(y);
            continue;
        }
        const bool finite = top < INFINITY;
        const float inv = top > 0.0f && finite ? __fdiv_rn(127.0f, top) : 0.0f;
        if (top > 0.0f) step = finite ? __fdiv_rn(top, 127.0f) : NAN;
        uint32_t w[4] = {0, 0, 0, 0};
        if (finite) {
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                w[p >> 2] |= (uint32_t)(uint8_t)q8_code(x[p], inv) << (8 * (p & 3));
                w[2 + (p >> 2)] |= (uint32_t)(uint8_t)q8_code(y[p], inv) << (8 * (p & 3));
            }
        }
        *reinterpret_cast<uint2*>(pool + row * D + e0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(pool + row * D + e1) = make_uint2(w[2], w[3]);
        if (j == 0) (kind == 1 ? a.pages.ks : a.pages.vs)[row] = step;
    }
}

struct ReadArgs {
    PageView pages;
    const int* counts;       // [1] table entries
    const int* table;
    const int2* entries;     // of every table entry: row of its first position in the dense output, rows in use
    int layer;
    void* k_out;
    void* v_out;
    int64_t k_stride, v_stride;  // elements between dense rows
    // kReadHalf: the new tokens' q goes into f16 rows as well
    const __nv_bfloat16* q;
    __half* q_out;
    int64_t q_stride;
    int q_dim;
};

// kReadHalf: f16 operands of the tcgen05 kernel. V is taken times 64, so that values of 6e-8 to 1000 keep the precision of a
// bf16 row or better; what f16 cannot hold (or was not finite) becomes NaN, and rows that meet it are computed again from the
// pages in f32.
enum ReadOut { kReadF32 = 0, kReadBf16 = 1, kReadHalf = 2 };
constexpr float kReadVScale = 64.0f;

__device__ __forceinline__ uint32_t half2_or_nan(float x, float y) {
    const __half2 h = __floats2half2_rn(fabsf(x) <= 65504.0f ? x : NAN, fabsf(y) <= 65504.0f ? y : NAN);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Rows of all sequences out of their pages: a warp-wide task is 16 elements of one row, a CTA takes blocks of 16 rows of one
// KV head of K and of V. The page ids of four blocks are fetched before the rows of any, and the rows of four before the
// first is stored: a block alone is two dependent loads.
template <int FMT, int D, int OUT>
__global__ void __launch_bounds__(256) paged_read_kernel(ReadArgs a) {
    constexpr int per_row = D / 16, rows_per_pass = 128 / per_row;  // 128 threads for K, 128 for V
    constexpr int passes = (16 + rows_per_pass - 1) / rows_per_pass;
    constexpr int UN = 4 / passes > 0 ? 4 / passes : 1;
    const int sub_log2 = a.pages.page_log2 - 4, Hkv = a.pages.Hkv;
    const bool is_v = threadIdx.x >= 128;
    const int tid = threadIdx.x & 127, r0 = tid / per_row, e = (tid % per_row) * 16;
    const int64_t blocks = ((int64_t)a.counts[1] << sub_log2) * Hkv;
    const unsigned char* pool = is_v ? a.pages.v : a.pages.k;
    const float* scales = is_v ? a.pages.vs : a.pages.ks;
    void* out = is_v ? a.v_out : a.k_out;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    for (int64_t b0 = (int64_t)blockIdx.x * UN; b0 < blocks; b0 += (int64_t)gridDim.x * UN) {
        int slot[UN], dense[UN], used[UN], head[UN];  // of a block's first row: where it lies in the pool and in the output
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int64_t b = b0 + u, s = b / Hkv;
            const int entry = (int)(s >> sub_log2), sub = (int)(s & ((1 << sub_log2) - 1)) * 16;
            head[u] = (int)(b - s * Hkv);
            slot[u] = dense[u] = used[u] = 0;
            if (b < blocks) {
                const int2 at = a.entries[entry];
                slot[u] = (a.table[entry] << a.pages.page_log2) + sub;
                dense[u] = at.x + sub;
                used[u] = max(0, min(16, at.y - sub));
            }
        }
        uint4 raw[UN * passes][FMT == KV_BF16 ? 2 : 1];
        float scale[UN * passes];
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int p = 0; p < passes; ++p) {
                const int r = p * rows_per_pass + r0, i = u * passes + p;
                if (r >= used[u]) continue;
                const int64_t row = a.pages.row(a.layer, slot[u] >> a.pages.page_log2, head[u], (slot[u] & ((1 << a.pages.page_log2) - 1)) + r);
                if constexpr (FMT == KV_BF16) {
                    const uint4* src = reinterpret_cast<const uint4*>(pool + (row * D + e) * 2);
                    raw[i][0] = __ldg(src);
                    raw[i][1] = __ldg(src + 1);
                } else {
                    raw[i][0] = __ldg(reinterpret_cast<const uint4*>(pool + row * D + e));
                    scale[i] = __ldg(scales + row);
                }
            }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int p = 0; p < passes; ++p) {
                const int r = p * rows_per_pass + r0, i = u * passes + p;
                if (r >= used[u]) continue;
                float x[16];
                if constexpr (FMT == KV_BF16) {
                    unpack8(raw[i][0], x);
                    unpack8(raw[i][1], x + 8);
                } else {
                    const uint32_t w[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
                    if (OUT == kReadHalf && is_v) scale[i] *= kReadVScale;
#pragma unroll
                    for (int q = 0; q < 16; ++q) x[q] = (float)(int8_t)(w[q >> 2] >> (8 * (q & 3))) * scale[i];
                }
                const int64_t to = (int64_t)(dense[u] + r) * stride + (int64_t)head[u] * D + e;
                if constexpr (OUT == kReadHalf) {
                    uint4* o = reinterpret_cast<uint4*>(static_cast<__half*>(out) + to);
                    o[0] = make_uint4(half2_or_nan(x[0], x[1]), half2_or_nan(x[2], x[3]), half2_or_nan(x[4], x[5]), half2_or_nan(x[6], x[7]));
                    o[1] = make_uint4(half2_or_nan(x[8], x[9]), half2_or_nan(x[10], x[11]), half2_or_nan(x[12], x[13]), half2_or_nan(x[14], x[15]));
                } else if constexpr (OUT == kReadBf16) {
                    uint4* o = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + to);
                    if constexpr (FMT == KV_BF16) {
                        o[0] = raw[i][0];
                        o[1] = raw[i][1];
                    } else {
                        o[0] = pack8(x);
                        o[1] = pack8(x + 8);
                    }
                } else {
                    float* o = static_cast<float*>(out) + to;
                    store8_f32(o, x);
                    store8_f32(o + 8, x + 8);
                }
            }
    }
    if constexpr (OUT == kReadHalf) {
        const int vecs = a.q_dim / 8;
        const int64_t n = (int64_t)a.counts[2] * vecs;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
            const int64_t row = i / vecs, d = (i - row * vecs) * 8;
            float x[8];
            load8_in<__nv_bfloat16>(a.q + row * a.q_stride + d, x);
            *reinterpret_cast<uint4*>(a.q_out + row * a.q_dim + d) =
                make_uint4(half2_or_nan(x[0], x[1]), half2_or_nan(x[2], x[3]), half2_or_nan(x[4], x[5]), half2_or_nan(x[6], x[7]));
        }
    }
}

}  // namespace ggr
