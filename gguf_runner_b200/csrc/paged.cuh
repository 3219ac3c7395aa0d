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
struct alignas(16) PagedItem {
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
    const double* freqs;     // of the layer's kind, in 64 bits
    const int* counts;       // [2] tokens
    const int* tok_pos;      // position of every new token
    const int* tok_slot;     // page * page_size + row in the page
    int layer, rotate, write_q, in_bf16, q_bf16;
    int Hq, tokens_per_cta, heads;  // heads: of q (when it is rotated), k and v together
    unsigned heads_inv;             // 2^32 / heads, rounded up: task numbers are divided by a multiplication
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    int64_t q_stride, k_stride, v_stride, qo_stride;  // elements between rows
};

// 16 bytes of a row, as they lie and as E f32 elements (E = 4 of f32, 8 of bf16 rows).
template <bool BF16>
__device__ __forceinline__ uint4 load_raw(const void* p, int64_t at) {
    return *reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(p) + at * (BF16 ? 2 : 4));
}
template <bool BF16, int E>
__device__ __forceinline__ void unpack_raw(const uint4& v, float (&x)[E]) {
    if constexpr (BF16) {
        unpack8(v, x);
    } else {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    }
}
// Codes of four elements, rounded half away from zero. (|x * inv| is at most 127 but for its own rounding, so nothing saturates.)
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
    int c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (int)roundf(__fmul_rn(x[i], inv));
    uint32_t hi, w;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(hi) : "r"(c[3]), "r"(c[2]), "r"(0));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(c[1]), "r"(c[0]), "r"(hi));
    return w;
}
template <int E>
__device__ __forceinline__ void store_bf16(__nv_bfloat16* p, const float (&x)[E]) {
    if constexpr (E == 8) {
        *reinterpret_cast<uint4*>(p) = pack8(x);
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

// RoPE (by cache position, in 64-bit angles) and append of a few tokens per CTA. A lane has E elements of the lower half of a head and E of the upper, 16 bytes each,
// so that both kinds of RoPE pairs of a fully rotated head lie in one lane, a warp's loads are whole lines, and the head's
// largest element takes log2(D / 2E) shuffles. Bound by the bytes of the rows; one token per CTA while tokens are few (a token
// step is latency: the angles of a token, one load, one store), several when there are more CTAs than SMs to hold them. A
// thread requests the rows of two tasks before it works on either.
template <bool BF16>
__global__ void __launch_bounds__(256, 4) paged_append_kernel(AppendArgs a) {
    constexpr int E = BF16 ? 8 : 4, UN = 2;
    extern __shared__ float sm[];  // cos [tokens_per_cta][half], sin
    const int D = a.pages.D, lanes_log2 = 31 - __clz(D / (2 * E)), lanes = 1 << lanes_log2, half = a.rope.rope_half;
    const int total = a.counts[2], t0 = blockIdx.x * a.tokens_per_cta;
    if (t0 >= total) return;
    const int n = min(a.tokens_per_cta, total - t0);
    const int Hkv = a.pages.Hkv, nq = a.write_q ? a.Hq : 0, tasks = n * a.heads * lanes;
    struct Task {
        const void* src;
        int64_t at;
        int t, kind, head, j;
        bool live;
    };
    auto task_of = [&](int i) {
        Task k;
        k.live = i < tasks;
        const int unit = k.live ? i >> lanes_log2 : 0;
        k.j = i & (lanes - 1);
        k.t = (int)__umulhi((unsigned)unit, a.heads_inv);
        const int h = unit - k.t * a.heads;
        k.kind = h < nq ? 0 : (h < nq + Hkv ? 1 : 2);
        k.head = k.kind == 0 ? h : (k.kind == 1 ? h - nq : h - nq - Hkv);
        k.src = k.kind == 0 ? a.q : (k.kind == 1 ? a.k : a.v);
        k.at = (t0 + k.t) * (k.kind == 0 ? a.q_stride : (k.kind == 1 ? a.k_stride : a.v_stride)) + (int64_t)k.head * D;
        return k;
    };
    uint4 x[UN], y[UN];
    auto fetch = [&](int i, uint4& lo, uint4& hi) {
        const Task k = task_of(i);
        lo = hi = make_uint4(0, 0, 0, 0);
        if (!k.live) return;
        lo = load_raw<BF16>(k.src, k.at + k.j * E);
        hi = load_raw<BF16>(k.src, k.at + D / 2 + k.j * E);
    };
    float* cs = sm;
    float* sn = sm + a.tokens_per_cta * half;
    if (a.rotate) {
        for (int i = threadIdx.x; i < n * half; i += 256) {
            const int t = i / half, f = i - t * half;
            // The angle of a far position in 32 bits is off by its position times 2^-24 (2e-4 at 3000, against 6e-8 of the
            // rotation itself): it is taken in 64 bits and brought into one turn before it becomes an f32.
            const double angle = (double)a.tok_pos[t0 + t] * a.freqs[f] * (double)a.rope.fscale;
            const double turns = rint(angle * 0.15915494309189535);
            sincosf((float)fma(turns, -6.283185307179586, angle), &sn[i], &cs[i]);
        }
    }
    // (so far only the plan was read; the rows may be the work of the launch in front)
    grid_wait();
    grid_allow_dependents();
#pragma unroll
    for (int u = 0; u < UN; ++u) fetch(threadIdx.x + u * 256, x[u], y[u]);
    __syncthreads();
    auto finish = [&](const Task& k, const uint4& raw_x, const uint4& raw_y) {
        float x[E], y[E];
        unpack_raw<BF16, E>(raw_x, x);
        unpack_raw<BF16, E>(raw_y, y);
        const int e0 = k.j * E, e1 = D / 2 + k.j * E, tok = t0 + k.t;
        if (a.rotate && k.kind < 2 && k.live) {
            const float* c = cs + k.t * half;
            const float* s = sn + k.t * half;
            if (a.rope.rope_dim != D) {  // part of a head: partners may lie in other lanes
#pragma unroll
                for (int p = 0; p < E; ++p) {
                    x[p] = rope_elem(k.src, k.at, e0 + p, D, a.rope, c, s, BF16);
                    y[p] = rope_elem(k.src, k.at, e1 + p, D, a.rope, c, s, BF16);
                }
            } else if (a.rope.style == 0) {
#pragma unroll
                for (int p = 0; p < E; ++p) {
                    const float lo = x[p], hi = y[p], cc = c[e0 + p], ss = s[e0 + p];
                    x[p] = __fsub_rn(__fmul_rn(lo, cc), __fmul_rn(hi, ss));
                    y[p] = __fadd_rn(__fmul_rn(lo, ss), __fmul_rn(hi, cc));
                }
            } else {
#pragma unroll
                for (int p = 0; p < E; p += 2) {
                    const float x0 = x[p], x1 = x[p + 1], y0 = y[p], y1 = y[p + 1];
                    const int i0 = (e0 + p) >> 1, i1 = (e1 + p) >> 1;
                    x[p] = __fsub_rn(__fmul_rn(x0, c[i0]), __fmul_rn(x1, s[i0]));
                    x[p + 1] = __fadd_rn(__fmul_rn(x0, s[i0]), __fmul_rn(x1, c[i0]));
                    y[p] = __fsub_rn(__fmul_rn(y0, c[i1]), __fmul_rn(y1, s[i1]));
                    y[p + 1] = __fadd_rn(__fmul_rn(y0, s[i1]), __fmul_rn(y1, c[i1]));
                }
            }
        }
        float top = 0.0f;
        if (a.pages.fmt == kKvQ8Head) {  // (whole warps take part)
            bool odd = false;  // a value that is not finite: max would lose a NaN
#pragma unroll
            for (int p = 0; p < E; ++p) {
                top = fmaxf(top, fmaxf(fabsf(x[p]), fabsf(y[p])));
                odd |= !isfinite(x[p]) | !isfinite(y[p]);
            }
            if (odd) top = INFINITY;
            if (top < 1e-36f) top = 0.0f;  // 127 / m would overflow: such a row counts as zeros
            for (int o = lanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (!k.live) return;
        if (k.kind == 0) {
            if (a.rope.do_prescale && a.rotate) {
#pragma unroll
                for (int p = 0; p < E; ++p) {
                    x[p] = __fmul_rn(x[p], a.rope.q_prescale);
                    y[p] = __fmul_rn(y[p], a.rope.q_prescale);
                }
            }
            const int64_t to = tok * a.qo_stride + (int64_t)k.head * D;
            if (a.q_bf16) {
                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.q_out) + to;
                store_bf16<E>(o + e0, x);
                store_bf16<E>(o + e1, y);
            } else {
                float* o = static_cast<float*>(a.q_out) + to;
#pragma unroll
                for (int p = 0; p < E; p += 4) {
                    *reinterpret_cast<float4*>(o + e0 + p) = make_float4(x[p], x[p + 1], x[p + 2], x[p + 3]);
                    *reinterpret_cast<float4*>(o + e1 + p) = make_float4(y[p], y[p + 1], y[p + 2], y[p + 3]);
                }
            }
            return;
        }
        const int slot = a.tok_slot[tok];
        const int64_t row = a.pages.row(a.layer, slot >> a.pages.page_log2, k.head, slot & ((1 << a.pages.page_log2) - 1));
        unsigned char* pool = k.kind == 1 ? a.pages.k : a.pages.v;
        if (a.pages.fmt == KV_BF16) {
            __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(pool) + row * D;
            store_bf16<E>(o + e0, x);
            store_bf16<E>(o + e1, y);
            return;
        }
        const bool finite = top < INFINITY;
        const float inv = top > 0.0f && finite ? __fdiv_rn(127.0f, top) : 0.0f;
        uint32_t w[E / 2] = {};
        if (finite) {
#pragma unroll
            for (int p = 0; p < E; p += 4) {
                w[p >> 2] = codes4(x + p, inv);
                w[(E + p) >> 2] = codes4(y + p, inv);
            }
        }
        if constexpr (E == 8) {
            *reinterpret_cast<uint2*>(pool + row * D + e0) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2*>(pool + row * D + e1) = make_uint2(w[2], w[3]);
        } else {
            *reinterpret_cast<uint32_t*>(pool + row * D + e0) = w[0];
            *reinterpret_cast<uint32_t*>(pool + row * D + e1) = w[1];
        }
        if (k.j == 0) (k.kind == 1 ? a.pages.ks : a.pages.vs)[row] = top > 0.0f ? (finite ? __fdiv_rn(top, 127.0f) : NAN) : 1.0f;
    };
    const int whole = (tasks + 31) & ~31;
    for (int i0 = threadIdx.x; i0 < whole; i0 += 256 * UN) {
        if (i0 != (int)threadIdx.x) {
#pragma unroll
            for (int u = 0; u < UN; ++u) fetch(i0 + u * 256, x[u], y[u]);
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (i0 + u * 256 < whole) finish(task_of(i0 + u * 256), x[u], y[u]);
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

// kReadHalf: f16 operands of the tcgen05 kernel. V is taken times 64, so that values of 1.2e-7 to 1023 keep the precision of a
// bf16 row or better (smaller ones are off by at most 2^-31); what f16 cannot hold (or was not finite) becomes NaN, and rows that
// meet it are computed again from the pages in f32.
enum ReadOut { kReadF32 = 0, kReadBf16 = 1, kReadHalf = 2 };
constexpr float kReadVScale = 64.0f;

__device__ __forceinline__ uint32_t half2_or_nan(float x, float y) {
    const __half2 h = __floats2half2_rn(fabsf(x) <= 65504.0f ? x : NAN, fabsf(y) <= 65504.0f ? y : NAN);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Byte `i` of codes offset to 0 .. 255, as the f32 code: the byte becomes the low bits of 2^23 + code + 128. (Conversion instructions
// run at a quarter of the rate: with them that pipe was 59 % busy, and 170 MB of int8 pages into bf16 rows took 29.5 us instead of
// 29.2.)
__device__ __forceinline__ float code_value(uint32_t w, int i) { return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)) - 8388736.0f; }

// Rows of all sequences out of their pages. A thread has 16 bytes of output at a time (E elements), so that a warp's stores, and
// its loads, are whole lines; a CTA takes blocks of 16 rows of one KV head of K and of V, UN of them at once: the page ids of
// all are fetched before the rows of any, and all rows before the first is stored (a block alone is two dependent loads). Rows come
// by plain loads: the launch in front may still write them while this one's CTAs are there already, waiting for it.
template <int FMT, int D, int OUT>
__global__ void __launch_bounds__(256) paged_read_kernel(ReadArgs a) {
    constexpr int E = OUT == kReadF32 ? 4 : 8;
    constexpr int per_row = D / E, rows_per_pass = 256 / per_row > 16 ? 16 : 256 / per_row, passes = 16 / rows_per_pass;
    constexpr int used_threads = rows_per_pass * per_row;  // (head_dim 64 in 16 bits: half of them)
    constexpr int UN = passes >= 4 ? 1 : (passes == 2 ? 2 : 4);
    const int sub_log2 = a.pages.page_log2 - 4, Hkv = a.pages.Hkv;
    const int tid = threadIdx.x % used_threads, r0 = tid / per_row, e = (tid % per_row) * E;
    const bool idle = threadIdx.x >= used_threads;
    grid_wait();
    grid_allow_dependents();
    const int64_t blocks = ((int64_t)a.counts[1] << sub_log2) * Hkv;
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
                used[u] = idle ? 0 : max(0, min(16, at.y - sub));
            }
        }
        uint32_t raw[2][UN * passes][FMT == KV_BF16 ? E / 2 : E / 4];
        float scale[2][UN * passes];
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int p = 0; p < passes; ++p)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int r = p * rows_per_pass + r0, i = u * passes + p;
                    if (r >= used[u]) continue;
                    const int64_t row = a.pages.row(a.layer, slot[u] >> a.pages.page_log2, head[u], (slot[u] & ((1 << a.pages.page_log2) - 1)) + r);
                    const unsigned char* src = (v ? a.pages.v : a.pages.k) + (row * D + e) * (FMT == KV_BF16 ? 2 : 1);
                    if constexpr (FMT == KV_BF16 && E == 8) {
                        const uint4 x = *reinterpret_cast<const uint4*>(src);
                        raw[v][i][0] = x.x, raw[v][i][1] = x.y, raw[v][i][2] = x.z, raw[v][i][3] = x.w;
                    } else if constexpr (FMT == KV_BF16 || E == 8) {
                        const uint2 x = *reinterpret_cast<const uint2*>(src);
                        raw[v][i][0] = x.x, raw[v][i][1] = x.y;
                    } else {
                        raw[v][i][0] = *reinterpret_cast<const uint32_t*>(src);
                    }
                    if constexpr (FMT != KV_BF16) scale[v][i] = (v ? a.pages.vs : a.pages.ks)[row];
                }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int p = 0; p < passes; ++p)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int r = p * rows_per_pass + r0, i = u * passes + p;
                    if (r >= used[u]) continue;
                    float x[E];
                    if constexpr (FMT == KV_BF16) {
#pragma unroll
                        for (int q = 0; q < E; q += 2) {
                            x[q] = __uint_as_float(raw[v][i][q / 2] << 16);
                            x[q + 1] = __uint_as_float(raw[v][i][q / 2] & 0xffff0000u);
                        }
                    } else {
                        const float f = OUT == kReadHalf && v ? scale[v][i] * kReadVScale : scale[v][i];
#pragma unroll
                        for (int q = 0; q < E; ++q) x[q] = code_value(raw[v][i][q >> 2] ^ 0x80808080u, q & 3) * f;
                    }
                    void* out = v ? a.v_out : a.k_out;
                    const int64_t to = (int64_t)(dense[u] + r) * (v ? a.v_stride : a.k_stride) + (int64_t)head[u] * D + e;
                    if constexpr (OUT == kReadF32) {
                        *reinterpret_cast<float4*>(static_cast<float*>(out) + to) = make_float4(x[0], x[1], x[2], x[3]);
                    } else if constexpr (OUT == kReadHalf) {
                        *reinterpret_cast<uint4*>(static_cast<__half*>(out) + to) =
                            make_uint4(half2_or_nan(x[0], x[1]), half2_or_nan(x[2], x[3]), half2_or_nan(x[4], x[5]), half2_or_nan(x[6], x[7]));
                    } else if constexpr (FMT == KV_BF16) {
                        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + to) = make_uint4(raw[v][i][0], raw[v][i][1], raw[v][i][2], raw[v][i][3]);
                    } else {
                        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + to) = pack8(x);
                    }
                }
    }
    if constexpr (OUT == kReadHalf) {
        const int vecs = a.q_dim / 8;
        const int64_t n = (int64_t)a.counts[2] * vecs;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
            const int64_t row = i / vecs, d = (i - row * vecs) * 8;
            float x[8];
            unpack8(*reinterpret_cast<const uint4*>(a.q + row * a.q_stride + d), x);
            *reinterpret_cast<uint4*>(a.q_out + row * a.q_dim + d) =
                make_uint4(half2_or_nan(x[0], x[1]), half2_or_nan(x[2], x[3]), half2_or_nan(x[4], x[5]), half2_or_nan(x[6], x[7]));
        }
    }
}

}  // namespace ggr
