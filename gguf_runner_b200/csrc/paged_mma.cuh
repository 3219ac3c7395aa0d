// Attention over pages (or over packed rows) on the warp-level tensor-core instructions: single tokens, short chunks, and
// everything in 32-bit precision or at head_dim 256. attention_token of the reference (src/engine/runtime/inference.rs:
// 1970-2530) for each new token of a batch, as one online softmax over the visible keys
//     o = sum_j p_j v_j / sum_j p_j,   p_j = 2^((s_j - m) c),   s_j = q . k_j,   c = scale * log2 e.
//
// Two forms of one tile step (16 rows x 16 keys, PagedMma::step):
//  - paged_splitk_kernel: the six to twelve warps of a CTA share 16 rows and split the keys between them, each
//    with a ring of its own that TMA fills; states are merged in shared memory, and over CTAs by the last one to finish a row
//    tile. Bound by the bytes of the cache: for a few tokens times G heads every cache byte is read once.
//  - paged_rows_kernel: eight warps with 16 rows each walk the same keys through one ring, which a ninth warp fills.
//
// Precision. bf16 rows: q is an exact operand, softmax weights are rounded once to bf16. f32 rows: q and the weights go in as
// three bf16 parts (24 bits), f32 keys and values as three bf16 planes, of which the products up to the weight of 2^-16 are
// taken (six of nine; the others are below an f32 rounding). Two parts (16 bits) were measured first: 3.9e-6 from 64 bits
// (2-norm) instead of 2e-7.
// 8-bit pages: f16 operands, in which a code is exact and costs two instructions per pair instead of four in bf16. A row of q is
// brought to [1, 2) by a power of two; a weight (at most 4, the reference maximum being at most two powers of two behind) times
// the scale of V is taken relative to the largest such scale so far and times 2^13, so that f16 reaches 2^-38 of the largest
// term. bf16 rows: one f16 part (11 bits); f32 rows: two (22 bits).
// In split-K form f32 tiles have eight rows, and the other eight of the tensor core's sixteen hold the second part: one or two
// instructions per product instead of two or three, and both halves of a row lie in one lane.
//
// Keys that only some rows of a tile see get weight 0, and 0 times an infinity or NaN in a value would spoil the other rows:
// a row whose result is not finite is computed again, by a warp of its own, by paged_row_again (unless it must be NaN: see there).
// Rows of a tile that nobody sees (behind the sequence's end, before its window: never written, freed or another sequence's) are
// cleared in shared memory.
#pragma once

#include "mma_utils.cuh"
#include "paged.cuh"
#include "sm100_utils.cuh"

namespace ggr {

constexpr int kPagedSplitMax = 128;  // pieces of one row tile

struct PagedAttnArgs {
    PageView pages;          // fmt also for packed rows: KV_BF16 (one plane), KV_F32 (three bf16 planes)
    PlanView plan;
    int paged;               // 0: keys are rows of packed k / v
    int layer, Hq, G, window;
    const void* q;           // [tokens][Hq * D], f32 or bf16
    void* out;               // the same type
    int64_t q_stride, o_stride;
    const void* pk;          // packed k / v rows as the caller has them, for paged_row_again
    const void* pv;
    int64_t pk_stride, pv_stride;
    int plane_rows;          // packed f32: rows between the planes
    float c;                 // score scale * log2 e
    float* part;             // states of key splits: per (tile, KV head) [rows][D], then [rows] (m, l)
    unsigned* tickets;       // zero between launches
    int* err;
};

__device__ __forceinline__ int paged_first_key(int pos, int window) { return window > 0 ? max(0, pos + 1 - window) : 0; }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// Bounded waits (see mbar_wait) of kernels in which other warps of the CTA may meanwhile compute rows again, which takes as long as
// the row's keys are many: flags[0] is raised by whoever gives up, flags[1] counts paged_row_again's steps, some microseconds each,
// and the limit starts anew as long as it moves. (By the limit alone a CTA would give up its items while a warp has 32 rows of
// 150000 keys, at 0.25 us a row and key.)
__device__ __forceinline__ bool paged_wait(uint32_t bar, uint32_t parity, volatile int* flags) {
    if (tc::mbar_test(bar, parity)) return true;
    int seen = 0;
    for (uint32_t it = 0; it < kTcSpinLimit; ++it) {
        if (tc::mbar_try(bar, parity, 4000u)) return true;
        if ((it & 15u) == 15u) {
            if (flags[0]) return false;
            const int now = flags[1];
            if (now != seen) seen = now, it = 0;
        }
    }
    flags[0] = 1;
    return false;
}
__device__ __forceinline__ bool paged_wait_warp(uint32_t bar, uint32_t parity, volatile int* flags) {
    const bool ok = paged_wait(bar, parity, flags);
    return __all_sync(0xffffffffu, ok);
}

// N consecutive elements of a row of keys or values, from element `at` on, in f32 (codes of 8-bit pages: without their scale).
template <int N, int FMT>
__device__ __forceinline__ void paged_elems(const void* rows, int64_t at, float (&x)[N]) {
    if constexpr (FMT == kKvQ8Head) {
        uint32_t u[(N + 3) / 4];
        const unsigned char* p = static_cast<const unsigned char*>(rows) + at;
        if constexpr (N == 8) {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
            u[0] = w.x, u[1] = w.y;
        } else if constexpr (N == 4) {
            u[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            u[0] = *reinterpret_cast<const uint16_t*>(p);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)(int)(signed char)(u[i >> 2] >> (8 * (i & 3)));
    } else if constexpr (FMT == KV_F32) {
        const float* p = static_cast<const float*>(rows) + at;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 u = *reinterpret_cast<const float2*>(p + i);
            x[i] = u.x, x[i + 1] = u.y;
        }
    } else {
        const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(rows) + at;
        if constexpr (N == 8) {
            unpack8(*reinterpret_cast<const uint4*>(p), x);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const uint32_t u = *reinterpret_cast<const uint32_t*>(p + i);
                x[i] = __uint_as_float(u << 16), x[i + 1] = __uint_as_float(u & 0xffff0000u);
            }
        }
    }
}

// One row again in f32, by a warp: what is not seen is not touched. Only rows whose fast result is not finite, and not known to be
// right as it is (a bf16 row's sum of weights is NaN when one of its scores is, whatever the values are). 32 keys at a time: a lane
// takes q times one of them, then every lane D / 32 elements of their values. A row that has met a NaN score is NaN, and is left
// there; of 8-bit pages the scales tell before anything else is read. Bound by the latency of each 32 keys' loads, 0.25 us a key at
// head_dim 64 and 128, 0.45 at 256 (one key after the other: 1.2, 2.2 and 4.4). `steps`: in shared memory, see paged_wait.
template <int D, int FMT, bool F32>
__device__ __noinline__ void paged_row_again(const PagedAttnArgs& a, const PagedItem& w, int kvh, int r, int lane, int* steps = nullptr) {
    constexpr int E = D / 32;
    const int tok = r / a.G, h = kvh * a.G + r % a.G, pos = w.pos0 + tok, first = paged_first_key(pos, a.window);
    const int64_t qo = (w.tok0 + tok) * a.q_stride + (int64_t)h * D + lane * E;
    constexpr bool q8 = FMT == kKvQ8Head;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] = F32 ? static_cast<const float*>(a.q)[qo + i] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[qo + i]);
        o[i] = 0.0f;
    }
    auto row_of = [&](int j) -> int64_t {
        if (!a.paged) return w.src + j;
        return a.pages.row(a.layer, a.plan.table[w.src + (j >> a.pages.page_log2)], kvh, j & ((1 << a.pages.page_log2) - 1));
    };
    if constexpr (q8) {
        bool odd = false;
        for (int j0 = first; j0 <= pos; j0 += 1024) {
            if (steps && lane == 0) atomicAdd(steps, 1);
#pragma unroll 4
            for (int j = j0 + lane; j <= min(pos, j0 + 1023); j += 32) {
                const int64_t row = row_of(j);
                odd |= isnan(a.pages.ks[row]) | isnan(a.pages.vs[row]);
            }
        }
        if (__any_sync(0xffffffffu, odd)) l = NAN;
    }
    const void* keys = a.paged ? static_cast<const void*>(a.pages.k) : a.pk;
    const void* vals = a.paged ? static_cast<const void*>(a.pages.v) : a.pv;
    const int64_t k_step = a.paged ? D : a.pk_stride, v_step = a.paged ? D : a.pv_stride, head = a.paged ? 0 : (int64_t)kvh * D;
    for (int j0 = first; j0 <= pos && l == l; j0 += 32) {
        if (steps && lane == 0) atomicAdd(steps, 1);
        const int n = min(32, pos + 1 - j0);
        const int64_t row = row_of(j0 + min(lane, n - 1));
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float step = q8 ? a.pages.ks[row] : 1.0f;
#pragma unroll 8
        for (int d = 0; d < D; d += 8) {
            float x[8];
            paged_elems<8, FMT>(keys, row * k_step + head + d, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) part[e & 3] = fmaf(__shfl_sync(0xffffffffu, q[e % E], (d + e) / E), q8 ? x[e] * step : x[e], part[e & 3]);
        }
        float s = ((part[0] + part[1]) + (part[2] + part[3])) * a.c;
        if (lane >= n) s = -INFINITY;
        // (a score of -inf has weight 0, also while there is no larger one to measure it by)
        const float top = fmaxf(m, warp_max(s)), f = m == top ? 1.0f : exp2f(m - top);
        float p = s == -INFINITY ? 0.0f : exp2f(s - top);
        m = top;
        l = l * f + warp_sum(p);
        if constexpr (q8) p *= a.pages.vs[row];
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] *= f;
#pragma unroll 16
        for (int i = 0; i < n; ++i) {
            const float pi = __shfl_sync(0xffffffffu, p, i);
            float x[E];
            paged_elems<E, FMT>(vals, __shfl_sync(0xffffffffu, row, i) * v_step + head + lane * E, x);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(pi, x[e], o[e]);
        }
    }
    const int64_t oo = (w.tok0 + tok) * a.o_stride + (int64_t)h * D + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (F32)
            static_cast<float*>(a.out)[oo + i] = o[i] / l;
        else
            static_cast<__nv_bfloat16*>(a.out)[oo + i] = __float2bfloat16_rn(o[i] / l);
    }
}

// FMT: KV_BF16, kKvQ8Head, or KV_F32 = three bf16 planes. F32: rows in several parts; PACK: the first two of them in one
// fragment of eight rows, the third in another.
template <int D, int FMT, bool F32, bool PACK, bool QSMEM>
struct PagedMma {
    static_assert(F32 || !PACK, "bf16 rows have one part");
    static constexpr bool Q8 = FMT == kKvQ8Head, PLANES = FMT == KV_F32;
    static constexpr int NP = !F32 ? 1 : (Q8 ? 2 : 3) - (PACK ? 1 : 0);  // fragments per product
    static constexpr int PL = PLANES ? 3 : 1;
    static constexpr int ROWS = PACK ? 8 : 16;
    static constexpr int ROW = Q8 ? D : 2 * D;                    // bytes of a cache row
    static constexpr int BOX = ROW < 128 ? ROW : 128;             // bytes of a row in one swizzled block
    static constexpr int NBLK = ROW / BOX;
    static constexpr uint32_t BLK = 16 * BOX;
    static constexpr uint32_t MAT = NBLK * BLK;                   // 16 rows of K or V
    static constexpr uint32_t TILE = 2 * PL * MAT;                // planes of K, planes of V
    static constexpr uint32_t V0 = PL * MAT;
    static constexpr int KS = D / 16, NT = D / 8;
    static constexpr uint32_t QBYTES = QSMEM ? NP * KS * 512 : 0; // q fragments in shared memory, where registers are short

    uint32_t qf[QSMEM ? 1 : NP][QSMEM ? 1 : KS][4];
    uint32_t q_smem;
    float o[NT][4];
    float m0, m1, l0, l1;
    float c0, c1, t0, t1;  // per row: factor of its scores (with the power of two that its q was divided by), lazy threshold
    float q0, q1;          // that power of two
    float u0, u1;          // 8-bit: largest scale of V so far as a power of two; o is in units of u * 2^-13

    // The 16-byte piece `c` of row `r` in a block: 128-byte rows are XORed by row & 7, 64-byte rows (two to a 128-byte line)
    // by (row / 2) & 3.
    static __device__ __forceinline__ uint32_t piece(int r, int c) {
        if constexpr (BOX == 128) return (uint32_t)(c >> 3) * BLK + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        return (uint32_t)r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    }

    __device__ __forceinline__ void start() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.0f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.0f;
        u0 = u1 = 0x1p-100f;
    }

    // Fragments of rows r0 .. r0 + ROWS - 1 (zeros from r1 on). Of 8-bit keys a lane holds four consecutive elements of a row, and
    // the elements of q are taken in that order; the order of the sum does not matter as long as both sides have the same.
    __device__ __forceinline__ void load_q(const PagedAttnArgs& a, const PagedItem& w, int kvh, int r0, int r1, int lane, uint32_t smem) {
        const int gq = lane >> 2, tq = lane & 3;
        q_smem = smem + lane * 16;
        int64_t at[2];
        bool ok[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + gq + 8 * i, tok = r / a.G;
            ok[i] = r < r1 && !(PACK && i);
            at[i] = (w.tok0 + tok) * a.q_stride + (int64_t)(kvh * a.G + r - tok * a.G) * D;
        }
        float by[2] = {1.0f, 1.0f};
        float2 held[Q8 ? KS : 1][2][2];
        if constexpr (Q8) {
            float top[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < (PACK ? 1 : 2); ++i)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        held[ks][i][half] = ok[i] ? load2(a.q, at[i] + ks * 16 + tq * 4 + half * 2) : make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < (PACK ? 1 : 2); ++i) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int half = 0; half < 2; ++half) top[i] = fmaxf(top[i], fmaxf(fabsf(held[ks][i][half].x), fabsf(held[ks][i][half].y)));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
                // (not below 2^-100, zeros included: the threshold in units of a smaller row's scores would be infinite, its maximum
                // would never move from -inf, and the merges would take it for a row that has seen nothing)
                by[i] = __uint_as_float(0x7f000000u - (min(max(__float_as_uint(top[i]), 0x0d800000u), 0x7e800000u) & 0x7f800000u));
            }
        }
        q0 = 1.0f / by[0];
        q1 = 1.0f / by[1];
        c0 = a.c * q0;
        c1 = a.c * q1;
        t0 = (Q8 ? 2.0f : 8.0f) / c0;
        t1 = (Q8 ? 2.0f : 8.0f) / c1;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t f[NP][4] = {};
#pragma unroll
            for (int i = 0; i < (PACK ? 1 : 2); ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int d = ks * 16 + (Q8 ? tq * 4 + half * 2 : tq * 2 + half * 8);
                    if constexpr (!F32 && !Q8) {
                        f[0][i + 2 * half] = ok[i] ? *reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(a.q) + at[i] + d) : 0u;
                    } else {
                        float2 x;
                        if constexpr (Q8)
                            x = held[ks][i][half];
                        else
                            x = ok[i] ? load2(a.q, at[i] + d) : make_float2(0.f, 0.f);
                        put(x.x * by[i], x.y * by[i], f, i, half);
                    }
                }
#pragma unroll
            for (int np = 0; np < NP; ++np) {
                if constexpr (QSMEM) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(q_smem + (np * KS + ks) * 512), "r"(f[np][0]), "r"(f[np][1]),
                                 "r"(f[np][2]), "r"(f[np][3]) : "memory");
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[np][ks][i] = f[np][i];
                }
            }
        }
    }

    static __device__ __forceinline__ float2 load2(const void* p, int64_t at) {
        if constexpr (F32) return *reinterpret_cast<const float2*>(static_cast<const float*>(p) + at);
        const uint32_t x = *reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p) + at);
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }

    // A pair in its parts (bf16, or f16 for 8-bit pages), into the fragments of row i (0: gq, 1: gq + 8) and k half
    static __device__ __forceinline__ void put(float x, float y, uint32_t (&f)[NP][4], int i, int half) {
        if constexpr (Q8) {
            const __half2 h = __floats2half2_rn(x, y);
            f[0][PACK ? 2 * half : i + 2 * half] = *reinterpret_cast<const uint32_t*>(&h);
            if constexpr (F32) {
                const float2 g = __half22float2(h);
                const __half2 l = __floats2half2_rn(x - g.x, y - g.y);
                f[NP - 1][PACK ? 1 + 2 * half : i + 2 * half] = *reinterpret_cast<const uint32_t*>(&l);
            }
            return;
        }
        const uint32_t h = pack_bf16x2(x, y);
        const float x1 = x - __uint_as_float(h << 16), y1 = y - __uint_as_float(h & 0xffff0000u);
        const uint32_t m = pack_bf16x2(x1, y1);
        const uint32_t l = pack_bf16x2(x1 - __uint_as_float(m << 16), y1 - __uint_as_float(m & 0xffff0000u));
        if constexpr (PACK) {
            f[0][2 * half] = h;
            f[0][1 + 2 * half] = m;
            f[NP - 1][2 * half] = l;
        } else if constexpr (F32) {
            f[0][i + 2 * half] = h;
            f[NP > 1 ? 1 : 0][i + 2 * half] = m;
            f[NP - 1][i + 2 * half] = l;
        }
    }

    // Two of four int8, offset to 0 .. 255 by the caller, as an f16 pair, exactly: the selector puts their bytes under the
    // exponent of 1024 .. 1279, and 1024 + 128 is taken off.
    static __device__ __forceinline__ uint32_t codes2(uint32_t w, uint32_t sel) {
        const uint32_t x = __byte_perm(w, 0x64646464u, sel), off = 0xe480e480u;
        const __half2 d = __hadd2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&off));
        return *reinterpret_cast<const uint32_t*>(&d);
    }

    __device__ __forceinline__ void frag(int np, int ks, uint32_t (&f)[4]) const {
        if constexpr (QSMEM) {
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3])
                         : "r"(q_smem + (np * KS + ks) * 512));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = qf[np][ks][i];
        }
    }

    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
        if constexpr (Q8)
            mma_f16_16816(c, x[0], x[1], x[2], x[3], b0, b1);
        else
            mma_bf16_16816(c, x[0], x[1], x[2], x[3], b0, b1);
    }

    // A tile's share of four elements of o. The tensor core adds into its accumulator by truncation, which over hundreds of tiles
    // goes one way (1.4e-6 of o after 37 tiles): in f32 a tile is summed from zero and then added, rounded to nearest.
    struct Sum {
        float c[4];
        __device__ __forceinline__ explicit Sum(const float (&o)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = F32 ? 0.0f : o[i];
        }
        __device__ __forceinline__ void add_to(float (&o)[4]) const {
            if constexpr (F32) {
                tc::unpack_f32x2(tc::add_f32x2(tc::pack_f32x2(o[0], o[1]), tc::pack_f32x2(c[0], c[1])), o[0], o[1]);
                tc::unpack_f32x2(tc::add_f32x2(tc::pack_f32x2(o[2], o[3]), tc::pack_f32x2(c[2], c[3])), o[2], o[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = c[i];
            }
        }
    };

    // Scales of an 8-bit tile for the keys of a lane: keys 2 tq, 2 tq + 1 and those plus 8.
    struct Scales {
        float2 k[2], v[2];
        __device__ __forceinline__ void load(const float* ks, const float* vs, int tq) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                k[j] = *reinterpret_cast<const float2*>(ks + j * 8 + tq * 2);
                v[j] = *reinterpret_cast<const float2*>(vs + j * 8 + tq * 2);
            }
        }
    };

    // The larger of u and the tile's scales of V that the row sees (sc[.][at], sc[.][at + 1]), as a power of two at least as large.
    static __device__ __forceinline__ float top_scale(const float (&sc)[2][4], const float (&sv)[4], int at, float u) {
        float x = 0.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) x = fmaxf(x, sc[j][at + i] == -INFINITY ? 0.0f : sv[2 * j + i]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        return fmaxf(u, __uint_as_float((__float_as_uint(x) + 0x007fffffu) & 0x7f800000u));
    }

    // One tile: K at `kt`, V at `kt + V0`. Rows gq and gq + 8 of the warp see the keys [lo_i, hi_i) of the tile's 16; whole: all rows see all of them.
    __device__ __forceinline__ void step(uint32_t kt, const Scales& scales, bool whole, int lo0, int hi0, int lo1, int hi1, int lane) {
        const int tq = lane & 3;
        // f32: products of low parts have sums of their own, which spares the large ones two thirds of their (truncating) additions
        // (and, where planes give five of them per k-step, two chains)
        float sc[2][4], lo[2][4], lo2[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
            lo[j][0] = lo[j][1] = lo[j][2] = lo[j][3] = 0.0f;
            lo2[j][0] = lo2[j][1] = lo2[j][2] = lo2[j][3] = 0.0f;
        }
        if constexpr (!Q8) {
            const int row = (lane & 7) + ((lane >> 4) & 1) * 8, half = (lane >> 3) & 1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t f[NP][4], b[4];
#pragma unroll
                for (int np = 0; np < NP; ++np) frag(np, ks, f[np]);
#pragma unroll
                for (int pl = 0; pl < PL; ++pl) {
                    ldmatrix_x4(kt + pl * MAT + piece(row, 2 * ks + half), b[0], b[1], b[2], b[3]);
#pragma unroll
                    for (int np = 0; np < NP - pl; ++np) {
                        mma(np + pl == 0 ? sc[0] : (pl == 1 ? lo2[0] : lo[0]), f[np], b[0], b[1]);
                        mma(np + pl == 0 ? sc[1] : (pl == 1 ? lo2[1] : lo[1]), f[np], b[2], b[3]);
                    }
                }
            }
        } else {
            // matrices of a load: keys 0-7 of pieces 2 i and 2 i + 1, keys 8-15 of the same; a piece is one k-step
            const int row = (lane & 7) + ((lane >> 4) & 1) * 8, half = (lane >> 3) & 1;
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) {
                uint32_t r[4];
                ldmatrix_x4(kt + piece(row, 2 * i + half), r[0], r[1], r[2], r[3]);
#pragma unroll
                for (int k = 0; k < 4; ++k) r[k] ^= 0x80808080u;
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
                    const uint32_t x0 = codes2(r[k2], 0x4140), x1 = codes2(r[k2], 0x4342), y0 = codes2(r[2 + k2], 0x4140), y1 = codes2(r[2 + k2], 0x4342);
#pragma unroll
                    for (int np = 0; np < NP; ++np) {
                        uint32_t f[4];
                        frag(np, 2 * i + k2, f);
                        mma(np ? lo[0] : sc[0], f, x0, x1);
                        mma(np ? lo[1] : sc[1], f, y0, y1);
                    }
                }
            }
        }
        if constexpr (NP > 1) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[j][i] += PLANES ? lo[j][i] + lo2[j][i] : lo[j][i];
        }
        if constexpr (PACK) {  // the second parts of the lane's row
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                sc[j][0] += sc[j][2];
                sc[j][1] += sc[j][3];
            }
        }
        float sv[4];  // scales of V for this lane's four keys
        if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 k2 = scales.k[j], v2 = scales.v[j];
                sc[j][0] *= k2.x;
                sc[j][1] *= k2.y;
                sc[j][2] *= k2.x;
                sc[j][3] *= k2.y;
                sv[2 * j] = v2.x;
                sv[2 * j + 1] = v2.y;
            }
        }
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = j * 8 + tq * 2 + i;
                    if (key < lo0 || key >= hi0) sc[j][i] = -INFINITY;
                    if (key < lo1 || key >= hi1) sc[j][2 + i] = -INFINITY;
                }
        }
        float x0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1])), x1 = -INFINITY;
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        if constexpr (!PACK) {
            x1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        }
        // the reference maximum moves only when it grows by more than the threshold: l and o stay exact, they use the same
        const bool need0 = x0 > m0 + t0, need1 = !PACK && x1 > m1 + t1;
        bool rescale = need0 || need1;
        float v0 = u0, v1 = u1;  // the largest scale of V with this tile's
        if constexpr (Q8) {
            v0 = top_scale(sc, sv, 0, u0);
            if constexpr (!PACK) v1 = top_scale(sc, sv, 2, u1);
            rescale |= v0 > u0 || v1 > u1;
        }
        if (__any_sync(0xffffffffu, rescale)) {
            float f0 = need0 ? tc::ex2((m0 - x0) * c0) : 1.0f, f1 = need1 ? tc::ex2((m1 - x1) * c1) : 1.0f;
            if (need0) m0 = x0;
            if (need1) m1 = x1;
            l0 *= f0;
            l1 *= f1;
            if constexpr (Q8) {
                f0 *= u0 / v0;
                f1 *= u1 / v1;
                u0 = v0;
                u1 = v1;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][0] *= f0;
                o[nt][1] *= f0;
                o[nt][2] *= PACK ? f0 : f1;
                o[nt][3] *= PACK ? f0 : f1;
            }
        }
        const float b0 = m0 == -INFINITY ? 0.0f : -m0 * c0, b1 = m1 == -INFINITY ? 0.0f : -m1 * c1;
        const float w0 = __uint_as_float(0x7f000000u + (13u << 23) - __float_as_uint(u0)), w1 = __uint_as_float(0x7f000000u + (13u << 23) - __float_as_uint(u1));
        uint32_t pf[NP][4] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float p[4];
            p[0] = tc::ex2(fmaf(sc[j][0], c0, b0));
            p[1] = tc::ex2(fmaf(sc[j][1], c0, b0));
            l0 += p[0] + p[1];
            if constexpr (!PACK) {
                p[2] = tc::ex2(fmaf(sc[j][2], c1, b1));
                p[3] = tc::ex2(fmaf(sc[j][3], c1, b1));
                l1 += p[2] + p[3];
            }
            if constexpr (Q8) {
#pragma unroll
                for (int i = 0; i < (PACK ? 2 : 4); ++i)  // (a hidden row's scale may be anything)
                    p[i] = p[i] == 0.0f ? 0.0f : p[i] * (sv[2 * j + (i & 1)] * (i < 2 ? w0 : w1));
            }
            if constexpr (!F32 && !Q8) {
                pf[0][2 * j] = pack_bf16x2(p[0], p[1]);
                pf[0][2 * j + 1] = pack_bf16x2(p[2], p[3]);
            } else {
                put(p[0], p[1], pf, 0, j);
                if constexpr (!PACK) put(p[2], p[3], pf, 1, j);
            }
        }
        const uint32_t vt = kt + V0;
        if constexpr (!Q8) {
            const int row = (lane & 7) + ((lane >> 3) & 1) * 8, half = (lane >> 4) & 1;
#pragma unroll
            for (int n2 = 0; n2 < NT / 2; ++n2) {
                uint32_t b[PL][4];
#pragma unroll
                for (int pl = 0; pl < PL; ++pl) ldmatrix_x4_trans(vt + pl * MAT + piece(row, 2 * n2 + half), b[pl][0], b[pl][1], b[pl][2], b[pl][3]);
                Sum s0(o[2 * n2]), s1(o[2 * n2 + 1]);
#pragma unroll
                for (int k = NP * PL - 1; k >= 0; --k) {  // small products first
                    const int np = k % NP, pl = k / NP;
                    if (np + pl >= (NP > PL ? NP : PL)) continue;
                    mma(s0.c, pf[np], b[pl][0], b[pl][1]);
                    mma(s1.c, pf[np], b[pl][2], b[pl][3]);
                }
                s0.add_to(o[2 * n2]);
                s1.add_to(o[2 * n2 + 1]);
            }
        } else {
            // a transposed load of byte pairs: a lane gets elements 2 gq and 2 gq + 1 of a piece for keys 2 tq and 2 tq + 1; the
            // even ones make one n-tile, the odd ones the next, and element() below puts the columns back in order
            const int row = (lane & 7) + ((lane >> 3) & 1) * 8, half = (lane >> 4) & 1;
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) {
                uint32_t r[4];
                ldmatrix_x4_trans(vt + piece(row, 2 * i + half), r[0], r[1], r[2], r[3]);
#pragma unroll
                for (int k = 0; k < 4; ++k) r[k] ^= 0x80808080u;
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
                    const int nt = 2 * (2 * i + k2);
                    const uint32_t e0 = codes2(r[2 * k2], 0x4240), e1 = codes2(r[2 * k2 + 1], 0x4240);
                    const uint32_t d0 = codes2(r[2 * k2], 0x4341), d1 = codes2(r[2 * k2 + 1], 0x4341);
                    Sum s0(o[nt]), s1(o[nt + 1]);
#pragma unroll
                    for (int np = NP - 1; np >= 0; --np) {
                        mma(s0.c, pf[np], e0, e1);
                        mma(s1.c, pf[np], d0, d1);
                    }
                    s0.add_to(o[nt]);
                    s1.add_to(o[nt + 1]);
                }
            }
        }
    }

    // o[nt][0 / 2] and o[nt][1 / 3] are elements element(nt, 0) and element(nt, 1) of rows gq / gq + 8
    static __device__ __forceinline__ int element(int nt, int i, int tq) {
        if constexpr (Q8) return (nt >> 1) * 16 + 4 * tq + 2 * i + (nt & 1);
        return nt * 8 + 2 * tq + i;
    }

    // The rows' state as the merges take it: whole rows of o, maxima in units of q . k
    __device__ __forceinline__ void sum_rows() {
        if constexpr (PACK) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][0] += o[nt][2];
                o[nt][1] += o[nt][3];
            }
        }
        if constexpr (Q8) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][0] *= u0 * 0x1p-13f;
                o[nt][1] *= u0 * 0x1p-13f;
                o[nt][2] *= u1 * 0x1p-13f;
                o[nt][3] *= u1 * 0x1p-13f;
            }
            m0 *= q0;
            m1 *= q1;
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    }

    // Requests the 16 keys from `key` on (a multiple of 16) into `dst`; one lane. Packed keys lie in their rows, paged ones in
    // page `page` of the pool.
    static __device__ __forceinline__ void request(const PagedAttnArgs& a, const CUtensorMap* tk, const CUtensorMap* tv, const PagedItem& w,
                                                   int kvh, int key, int page, uint32_t dst, uint32_t bar) {
        if (a.paged) {
            const int in_page = key & ((1 << a.pages.page_log2) - 1);
            const int z = (a.layer * a.pages.n_pages + page) * a.pages.Hkv + kvh;
#pragma unroll
            for (int b = 0; b < NBLK; ++b) {
                const int x = b * (Q8 ? BOX : BOX / 2);
                tma_load_3d(dst + b * BLK, tk, x, in_page, z, bar);
                tma_load_3d(dst + V0 + b * BLK, tv, x, in_page, z, bar);
            }
        } else {
            const int z = w.src + key;
#pragma unroll
            for (int p = 0; p < PL; ++p)
#pragma unroll
                for (int b = 0; b < NBLK; ++b) {
                    tma_load_3d(dst + p * MAT + b * BLK, tk, b * 64, kvh, z + p * a.plane_rows, bar);
                    tma_load_3d(dst + V0 + p * MAT + b * BLK, tv, b * 64, kvh, z + p * a.plane_rows, bar);
                }
        }
    }

    // Clears the values of a tile's keys outside [lo, hi), by a warp.
    static __device__ __forceinline__ void clear(uint32_t tile, int lo, int hi, int lane) {
        if constexpr (Q8) return;  // codes are finite, and step() drops the scales of what has no weight
        constexpr int per_row = ROW / 16;
        for (int i = lane; i < 16 * per_row * PL; i += 32) {
            const int plane = i / (16 * per_row), r = (i / per_row) & 15, p = i % per_row;
            if (r >= lo && r < hi) continue;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + V0 + plane * MAT + piece(r, p)), "r"(0u) : "memory");
        }
    }
};

template <bool F32>
__device__ __forceinline__ void paged_store4(const PagedAttnArgs& a, int64_t at, float4 x) {
    if constexpr (F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = x;
    } else {
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
    }
}
__device__ __forceinline__ bool finite4(float4 x) { return isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w); }

constexpr int paged_splitk_warps(int D, int fmt, bool f32) {
    return D == 256 ? (fmt == kKvQ8Head ? 8 : 6) : ((D == 64 && fmt == kKvQ8Head) || (f32 && fmt != kKvQ8Head) ? 12 : 8);
}

template <int D, int FMT, bool F32>
struct PagedSplitKShape {
    // Warps and ring stages. bf16 on bf16 streams at nine tenths of the memory's rate with eight warps. Where a tile is more
    // arithmetic, twelve warps hide more of each other's chains (load, multiply, softmax, multiply), if their registers last: 16
    // conversations of 1310 to 20000 keys, eight warps -> twelve: f32 over bf16 pages, 32/4 heads of 128, 54.7 -> 50.1 us; int8,
    // 32/8 heads of 64, 55.3 -> 48.5; int8 at head_dim 128 is even (38.4 and 38.5), and one conversation of 700 keys 9.1 -> 9.8, so
    // that stays at eight.
    static constexpr bool BUSY = F32 || FMT == kKvQ8Head;
    using M = PagedMma<D, FMT, F32, F32, D == 256 || (D == 128 && F32 && FMT == KV_BF16)>;
    static constexpr int R = M::ROWS;
    static constexpr int W = paged_splitk_warps(D, FMT, F32);
    static constexpr int NST = FMT == kKvQ8Head ? (D == 64 ? 6 : (D == 128 ? 4 : 2)) : (D == 64 ? 4 : (BUSY || D == 256 ? 2 : 3));
    static constexpr int LD = D + 8;
    static constexpr uint32_t RING = W * NST * M::TILE;
    static constexpr uint32_t SCALES = FMT == kKvQ8Head ? W * NST * 128 : 0;
    static constexpr uint32_t MERGE = W * R * LD * 4;
    static constexpr uint32_t DATA = RING + SCALES > MERGE ? RING + SCALES : MERGE;  // the merge reuses the rings
    static constexpr uint32_t SMEM = DATA + M::QBYTES + 1024;
};

// An item is 16 packed rows (f32: 8) of one sequence, fewer at its end, and a stretch of keys; blockIdx.x is the KV head.
template <int D, int FMT, bool F32>
__global__ void __launch_bounds__(PagedSplitKShape<D, FMT, F32>::W * 32, 1)
paged_splitk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttnArgs a) {
    using namespace tc;
    using S = PagedSplitKShape<D, FMT, F32>;
    using M = typename S::M;
    constexpr int W = S::W, NST = S::NST, LD = S::LD, R = S::R;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t s_full[W][NST];
    __shared__ float s_m[W][R], s_l[W][R];  // per warp, then weights of the warps
    __shared__ float s_top[R], s_sum[R];
    __shared__ float s_w[R][kPagedSplitMax];
    __shared__ int s_abort, s_last;
    __shared__ unsigned s_bad;  // rows of the tile that have to be computed again

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int gq = lane >> 2, tq = lane & 3, kvh = blockIdx.x;
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    unsigned char* base_p = smem + (base - smem_u32(smem));
    const uint32_t ring = base + warp * NST * M::TILE;
    const uint32_t scales = base + S::RING + warp * NST * 128;
    const float* scales_p = reinterpret_cast<const float*>(base_p + S::RING + warp * NST * 128);
    float* acc = reinterpret_cast<float*>(base_p);  // [W][R][LD] after the rings have drained
    volatile int* abortp = &s_abort;
    // The first item and the number of items are requested together (the list is longer than any grid), and travel while the
    // barriers are set up: what a token step of one conversation takes is a chain of such round trips.
    int item = blockIdx.y;
    PagedItem w = a.plan.items[item];
    const int n_items = a.plan.counts[0];
    if (tid == 0) s_abort = 0;
    if (lane == 0) {
        for (int s = 0; s < NST; ++s) mbar_init(smem_u32(&s_full[warp][s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    // Launches of the library follow one another programmatically (launch_chained). Up to here, and for the pages of the first
    // item, only the plan is read, which no kernel writes.
    bool waited = false;
    if (item >= n_items) {
        grid_wait();
        grid_allow_dependents();
    }
    uint32_t used = 0;  // tiles this warp has been through: ring position and phase
    for (; item < n_items; item += gridDim.y) {
        if (item != (int)blockIdx.y) w = a.plan.items[item];
        const int n_tiles = (w.key1 - w.key0 + 15) >> 4, mine = n_tiles > warp ? (n_tiles - warp + W - 1) / W : 0;
        // keys that some row, and that every row, of the tile sees
        const int tok_lo = w.row0 / a.G, tok_hi = (w.row0 + w.rows - 1) / a.G;
        const int any_lo = paged_first_key(w.pos0 + tok_lo, a.window), any_hi = w.pos0 + tok_hi + 1;
        const int all_lo = paged_first_key(w.pos0 + tok_hi, a.window), all_hi = w.pos0 + tok_lo + 1;
        // Pages of this warp's tiles, 32 at a time: lane i has the one of tile 32 k + i (of the block in use, and of the next)
        auto pages_from = [&](int t) {
            const int key = w.key0 + (warp + (t + lane) * W) * 16;
            return a.paged && t + lane < mine ? a.plan.table[w.src + (key >> a.pages.page_log2)] : 0;
        };
        int pages_now = pages_from(0), pages_next = pages_from(32);
        if (!waited) {
            waited = true;
            grid_wait();
            grid_allow_dependents();
        }
        auto issue = [&](int t) {  // (by the whole warp)
            const uint32_t u = used + t, stage = u % NST;
            const int key = w.key0 + (warp + t * W) * 16;
            const uint32_t bar = smem_u32(&s_full[warp][stage]);
            if (t > 0 && (t & 31) == 0) {
                pages_now = pages_next;
                pages_next = pages_from(t + 32);
            }
            const int page = __shfl_sync(0xffffffffu, pages_now, t & 31);
            if (lane == 0) {
                mbar_expect_tx(bar, M::TILE + (M::Q8 ? 128 : 0));
                M::request(a, &tmK, &tmV, w, kvh, key, page, ring + stage * M::TILE, bar);
                if constexpr (M::Q8) {
                    const int64_t row = a.pages.row(a.layer, page, kvh, key & ((1 << a.pages.page_log2) - 1));
                    bulk_load(scales + stage * 128, a.pages.ks + row, 64, bar);
                    bulk_load(scales + stage * 128 + 64, a.pages.vs + row, 64, bar);
                }
            }
        };
        for (int t = 0; t < NST - 1 && t < mine; ++t) issue(t);
        M x;
        x.start();
        x.load_q(a, w, kvh, w.row0, w.row0 + w.rows, lane, base + S::DATA);
        if constexpr (M::QBYTES > 0) __syncthreads();  // (every warp has written the same fragments)
        const int p0 = w.pos0 + min(w.row0 + gq, w.row0 + w.rows - 1) / a.G, p1 = R == 16 ? w.pos0 + min(w.row0 + gq + 8, w.row0 + w.rows - 1) / a.G : p0;
        const int lo0 = paged_first_key(p0, a.window), lo1 = paged_first_key(p1, a.window);
        for (int t = 0; t < mine; ++t) {
            const uint32_t u = used + t, stage = u % NST;
            if (!mbar_wait_warp(smem_u32(&s_full[warp][stage]), (u / NST) & 1u, abortp)) break;
            const int key = w.key0 + (warp + t * W) * 16;
            const uint32_t kt = ring + stage * M::TILE;
            const bool whole = key >= all_lo && key + 16 <= all_hi;
            if (key < any_lo || key + 16 > any_hi) {
                M::clear(kt, any_lo - key, any_hi - key, lane);
                __syncwarp();
            }
            typename M::Scales sc;
            if constexpr (M::Q8) sc.load(scales_p + stage * 32, scales_p + stage * 32 + 16, tq);
            x.step(kt, sc, whole, lo0 - key, p0 + 1 - key, lo1 - key, p1 + 1 - key, lane);
            __syncwarp();
            if (t + NST - 1 < mine) {
                if (lane == 0) fence_smem_to_async_proxy();
                issue(t + NST - 1);
            }
        }
        used += mine;
        x.sum_rows();
        if (s_abort) {
            for (int i = 0; i < 500; ++i) __nanosleep(1000);  // let copies in flight land
        }
        __syncthreads();  // rings drained
        if (s_abort) break;
#pragma unroll
        for (int nt = 0; nt < M::NT; ++nt) {
            if constexpr (FMT == kKvQ8Head) {
                if (nt & 1) continue;  // an even and an odd n-tile make four consecutive elements
                const int d = M::element(nt, 0, tq);
                *reinterpret_cast<float4*>(&acc[(warp * R + gq) * LD + d]) = make_float4(x.o[nt][0], x.o[nt + 1][0], x.o[nt][1], x.o[nt + 1][1]);
                if constexpr (R == 16)
                    *reinterpret_cast<float4*>(&acc[(warp * R + gq + 8) * LD + d]) = make_float4(x.o[nt][2], x.o[nt + 1][2], x.o[nt][3], x.o[nt + 1][3]);
            } else {
                const int d = M::element(nt, 0, tq);
                *reinterpret_cast<float2*>(&acc[(warp * R + gq) * LD + d]) = make_float2(x.o[nt][0], x.o[nt][1]);
                if constexpr (R == 16) *reinterpret_cast<float2*>(&acc[(warp * R + gq + 8) * LD + d]) = make_float2(x.o[nt][2], x.o[nt][3]);
            }
        }
        if (tq == 0) {
            s_m[warp][gq] = x.m0;
            s_l[warp][gq] = x.l0;
            if constexpr (R == 16) {
                s_m[warp][gq + 8] = x.m1;
                s_l[warp][gq + 8] = x.l1;
            }
        }
        if (tid == 0) s_bad = 0;
        __syncthreads();
        if (tid < R) {
            float top = -INFINITY, sum = 0.0f;
            for (int i = 0; i < W; ++i) top = fmaxf(top, s_m[i][tid]);
            for (int i = 0; i < W; ++i) {
                const float f = s_m[i][tid] == -INFINITY ? 0.0f : ex2((s_m[i][tid] - top) * a.c);
                // (a row that has seen nothing finite so far keeps its NaN, if it has one)
                sum += s_l[i][tid] == 0.0f ? 0.0f : f * s_l[i][tid];
                s_m[i][tid] = f;
            }
            s_top[tid] = top;
            s_sum[tid] = sum;
        }
        __syncthreads();
        const bool split = w.part >= 0;
        constexpr int STATE = R * (D + 2);
        float* state0 = a.part + ((int64_t)(split ? w.part : 0) * a.pages.Hkv + kvh) * STATE;  // of the tile's first piece
        const int64_t state_step = (int64_t)a.pages.Hkv * STATE;
        float* mine_state = state0 + w.split * state_step;
        for (int i = tid; i < w.rows * (D / 4); i += W * 32) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float f = s_m[k][r];
                const float4 y = *reinterpret_cast<const float4*>(&acc[(k * R + r) * LD + d]);
                v.x = fmaf(f, y.x, v.x);
                v.y = fmaf(f, y.y, v.y);
                v.z = fmaf(f, y.z, v.z);
                v.w = fmaf(f, y.w, v.w);
            }
            if (split) {
                __stcg(reinterpret_cast<float4*>(mine_state + r * D + d), v);
            } else {
                const int row = w.row0 + r, tok = row / a.G;
                const float inv = 1.0f / s_sum[r];
                v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                if (!finite4(v) && (F32 || s_sum[r] == s_sum[r])) atomicOr(&s_bad, 1u << r);
                paged_store4<F32>(a, (w.tok0 + tok) * a.o_stride + (int64_t)(kvh * a.G + row - tok * a.G) * D + d, v);
            }
        }
        if (split) {
            if (tid < w.rows) __stcg(reinterpret_cast<float2*>(mine_state + R * D) + tid, make_float2(s_top[tid], s_sum[tid]));
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                // the ticket goes back to zero with the last piece, for the next launch
                s_last = atomicInc(&a.tickets[w.ticket * a.pages.Hkv + kvh], (unsigned)(w.n_split - 1)) == (unsigned)(w.n_split - 1);
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                // weights of the pieces, then the weighted sum in their order: the same bits whichever piece came last
                for (int r = warp; r < w.rows; r += W) {
                    float top = -INFINITY;
                    for (int s = lane; s < w.n_split; s += 32)
                        top = fmaxf(top, __ldcg(reinterpret_cast<const float2*>(state0 + s * state_step + R * D) + r).x);
                    top = warp_max(top);
                    float sum = 0.0f;
                    for (int s = lane; s < w.n_split; s += 32) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(state0 + s * state_step + R * D) + r);
                        const float f = ml.x == -INFINITY ? 0.0f : ex2((ml.x - top) * a.c);
                        s_w[r][s] = f;
                        sum += ml.y == 0.0f ? 0.0f : f * ml.y;
                    }
                    sum = warp_sum(sum);
                    if (lane == 0) s_sum[r] = sum;
                }
                __syncthreads();
                for (int i = tid; i < w.rows * (D / 4); i += W * 32) {
                    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                    for (int s = 0; s < w.n_split; ++s) {
                        const float f = s_w[r][s];
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(state0 + s * state_step + r * D + d));
                        v.x = fmaf(f, y.x, v.x);
                        v.y = fmaf(f, y.y, v.y);
                        v.z = fmaf(f, y.z, v.z);
                        v.w = fmaf(f, y.w, v.w);
                    }
                    const int row = w.row0 + r, tok = row / a.G;
                    const float inv = 1.0f / s_sum[r];
                    v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                    if (!finite4(v) && (F32 || s_sum[r] == s_sum[r])) atomicOr(&s_bad, 1u << r);
                    paged_store4<F32>(a, (w.tok0 + tok) * a.o_stride + (int64_t)(kvh * a.G + row - tok * a.G) * D + d, v);
                }
            }
        }
        __syncthreads();
        if (s_bad) {
            for (int r = warp; r < w.rows; r += W)
                if (s_bad >> r & 1u) paged_row_again<D, FMT, F32>(a, w, kvh, w.row0 + r, lane);
            __syncthreads();
        }
        // the next item's copies go where the generic proxy has just written
        fence_smem_to_async_proxy();
        __syncthreads();
    }
    if (tid == 0 && s_abort && a.err) atomicExch(a.err, 1);
}

template <int D, int FMT, bool F32>
struct PagedRowsShape {
    using M = PagedMma<D, FMT, F32, false, D == 256>;
    static constexpr int W = D == 256 && F32 ? 4 : 8;  // 16 rows each (fragments of q in shared memory: 24 KB a warp there)
    static constexpr int SUB = FMT == KV_F32 && D >= 128 ? 1 : 2;  // tiles of 16 keys in a stage
    static constexpr uint32_t STAGE = SUB * M::TILE;
    static constexpr int NST = STAGE >= 32768 ? 2 : 4;
    static constexpr uint32_t RING = NST * STAGE;
    static constexpr uint32_t SCALES = FMT == kKvQ8Head ? NST * SUB * 128 : 0;
    static constexpr uint32_t SMEM = RING + SCALES + W * M::QBYTES + 1024;
    // consumer warpgroups and a control warpgroup, whose registers go to the others
    static constexpr int THREADS = W * 32 + 128;
};

// An item is up to 128 packed rows (f32 at head_dim 256: 64) of one sequence and all the keys that they see; blockIdx.x is the KV
// head.
template <int D, int FMT, bool F32>
__global__ void __launch_bounds__(PagedRowsShape<D, FMT, F32>::THREADS, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttnArgs a) {
    using namespace tc;
    using S = PagedRowsShape<D, FMT, F32>;
    using M = typename S::M;
    constexpr int NST = S::NST, SUB = S::SUB, KT = 16 * SUB;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t s_full[NST], s_empty[NST], s_raw;
    __shared__ int s_flags[2];  // of paged_wait
    int& s_abort = s_flags[0];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int gq = lane >> 2, tq = lane & 3, kvh = blockIdx.x;
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    unsigned char* base_p = smem + (base - smem_u32(smem));
    volatile int* abortp = s_flags;
    if (tid == 0) {
        s_flags[0] = s_flags[1] = 0;
        for (int s = 0; s < NST; ++s) {
            mbar_init(smem_u32(&s_full[s]), 1);
            mbar_init(smem_u32(&s_empty[s]), S::W);
        }
        mbar_init(smem_u32(&s_raw), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const int n_items = a.plan.counts[0];
    grid_wait();
    grid_allow_dependents();
    uint32_t used = 0;  // stages gone through: ring position and phase
    // keys that some row of an item sees
    auto any_lo_of = [&](const PagedItem& w) { return paged_first_key(w.pos0 + w.row0 / a.G, a.window); };
    auto any_hi_of = [&](const PagedItem& w) { return w.pos0 + (w.row0 + w.rows - 1) / a.G + 1; };
    if (warp >= S::W) {
        // control warpgroup: one producer warp, the others have no role
        if constexpr (S::W == 8) reg_release<56>();
        uint32_t raws = 0;
        bool ok = warp == S::W;
        for (int item = blockIdx.y; ok && item < n_items; item += gridDim.y) {
            const PagedItem w = a.plan.items[item];
            const int n_stages = (w.key1 - w.key0 + KT - 1) / KT, any_lo = any_lo_of(w), any_hi = any_hi_of(w);
            for (int t = 0; t < n_stages; ++t, ++used) {
                const uint32_t stage = used % NST;
                if (!(ok = paged_wait_warp(smem_u32(&s_empty[stage]), ((used / NST) & 1u) ^ 1u, abortp))) break;
                const int key = w.key0 + t * KT;
                const bool edge = key < any_lo || key + KT > any_hi;
                const uint32_t bar = edge ? smem_u32(&s_raw) : smem_u32(&s_full[stage]);
                const uint32_t dst = base + stage * S::STAGE, sc = base + S::RING + stage * SUB * 128;  // (scales: 16 of K, 16 of V per tile)
                if (lane == 0) {
                    // tiles behind the last visible key have no page: they are left out, and step() is not called for them
                    const int subs = min(SUB, (any_hi - key + 15) >> 4);
                    mbar_expect_tx(bar, subs * (M::TILE + (M::Q8 ? 128 : 0)));
                    for (int i = 0; i < subs; ++i) {
                        const int k = key + 16 * i;
                        const int page = a.paged ? a.plan.table[w.src + (k >> a.pages.page_log2)] : 0;
                        M::request(a, &tmK, &tmV, w, kvh, k, page, dst + i * M::TILE, bar);
                        if constexpr (M::Q8) {
                            const int64_t row = a.pages.row(a.layer, page, kvh, k & ((1 << a.pages.page_log2) - 1));
                            bulk_load(sc + i * 128, a.pages.ks + row, 64, bar);
                            bulk_load(sc + i * 128 + 64, a.pages.vs + row, 64, bar);
                        }
                    }
                }
                __syncwarp();
                if (edge) {
                    if (!(ok = paged_wait_warp(bar, raws & 1u, abortp))) break;
                    ++raws;
                    for (int i = 0; i < SUB; ++i) M::clear(dst + i * M::TILE, any_lo - key - 16 * i, any_hi - key - 16 * i, lane);
                    fence_smem_to_async_proxy();  // (this stage's next copy comes after the arrivals below and the readers')
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&s_full[stage]));
                }
            }
        }
    } else {
        if constexpr (S::W == 8) reg_acquire<224>();
        for (int item = blockIdx.y; item < n_items; item += gridDim.y) {
            const PagedItem w = a.plan.items[item];
            const int n_stages = (w.key1 - w.key0 + KT - 1) / KT;
            const int r0 = w.row0 + warp * 16, r1 = w.row0 + w.rows;  // this warp's rows, cut at r1
            const bool mine = r0 < r1;
            M x;
            x.start();
            int p0 = 0, p1 = 0, all_lo = 0, all_hi = 0, see_lo = 0, see_hi = 0;
            if (mine) {
                x.load_q(a, w, kvh, r0, r1, lane, base + S::RING + S::SCALES + warp * M::QBYTES);
                __syncwarp();
                p0 = w.pos0 + min(r0 + gq, r1 - 1) / a.G;
                p1 = w.pos0 + min(r0 + gq + 8, r1 - 1) / a.G;
                const int t0 = w.pos0 + r0 / a.G, t1 = w.pos0 + min(r0 + 15, r1 - 1) / a.G;
                see_lo = paged_first_key(t0, a.window);
                see_hi = t1 + 1;
                all_lo = paged_first_key(t1, a.window);
                all_hi = t0 + 1;
            }
            const int lo0 = paged_first_key(p0, a.window), lo1 = paged_first_key(p1, a.window);
            for (int t = 0; t < n_stages; ++t, ++used) {
                const uint32_t stage = used % NST;
                if (!paged_wait_warp(smem_u32(&s_full[stage]), (used / NST) & 1u, abortp)) break;
#pragma unroll 1
                for (int i = 0; i < SUB; ++i) {
                    const int key = w.key0 + t * KT + 16 * i;
                    if (!mine || key >= see_hi || key + 16 <= see_lo) continue;
                    const bool whole = key >= all_lo && key + 16 <= all_hi;
                    typename M::Scales scales;
                    const float* sc = reinterpret_cast<const float*>(base_p + S::RING + (stage * SUB + i) * 128);
                    if constexpr (M::Q8) scales.load(sc, sc + 16, tq);
                    x.step(base + stage * S::STAGE + i * M::TILE, scales, whole,
                           lo0 - key, p0 + 1 - key, lo1 - key, p1 + 1 - key, lane);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_empty[stage]));
            }
            if (*abortp) break;
            if (!mine) continue;
            x.sum_rows();
            const float i0 = 1.0f / x.l0, i1 = 1.0f / x.l1;
            unsigned again = 0;  // of the warp's 16 rows
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                bool bad = false;
                const int row = r0 + gq + 8 * half, tok = row / a.G;
                const float sum = half ? x.l1 : x.l0;
                const int64_t at = (w.tok0 + tok) * a.o_stride + (int64_t)(kvh * a.G + row - tok * a.G) * D;
                const float inv = half ? i1 : i0;
#pragma unroll
                for (int nt = 0; nt < M::NT; ++nt) {
                    if (row >= r1) break;
                    if constexpr (FMT == kKvQ8Head) {
                        if (nt & 1) continue;
                        const float4 v = make_float4(x.o[nt][2 * half] * inv, x.o[nt + 1][2 * half] * inv, x.o[nt][2 * half + 1] * inv, x.o[nt + 1][2 * half + 1] * inv);
                        bad |= !finite4(v);
                        paged_store4<F32>(a, at + M::element(nt, 0, tq), v);
                    } else {
                        const float v0 = x.o[nt][2 * half] * inv, v1 = x.o[nt][2 * half + 1] * inv;
                        bad |= !isfinite(v0) || !isfinite(v1);
                        const int64_t to = at + M::element(nt, 0, tq);
                        if constexpr (F32)
                            *reinterpret_cast<float2*>(static_cast<float*>(a.out) + to) = make_float2(v0, v1);
                        else
                            *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + to) = pack_bf16x2(v0, v1);
                    }
                }
                const unsigned lanes = __ballot_sync(0xffffffffu, bad && (F32 || sum == sum));  // four to a row
#pragma unroll
                for (int r = 0; r < 8; ++r) again |= (lanes >> (4 * r) & 15u ? 1u : 0u) << (8 * half + r);
            }
            __syncwarp();
            for (int r = 0; again >> r; ++r)
                if (again >> r & 1u) paged_row_again<D, FMT, F32>(a, w, kvh, r0 + r, lane, &s_flags[1]);
        }
    }
    if (s_abort) {
        for (int i = 0; i < 500; ++i) __nanosleep(1000);  // let copies in flight land
    }
    __syncthreads();
    if (tid == 0 && s_abort && a.err) atomicExch(a.err, 1);
}

// f32 rows of k or v as three bf16 planes: x = h + m + l. Rows of `dim` elements, four per thread; `counts` holds the rows in use.
__global__ void __launch_bounds__(256) paged_planes_kernel(const float* k, const float* v, int64_t k_stride, int64_t v_stride, const int* counts, int dim,
                                                           __nv_bfloat16* kp, __nv_bfloat16* vp, int64_t plane) {
    grid_wait();
    grid_allow_dependents();
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= (int64_t)counts[2] * dim) return;
    const int64_t r = i / dim, d = i - r * dim;
    float4 x = *reinterpret_cast<const float4*>((blockIdx.y ? v + r * v_stride : k + r * k_stride) + d);
    __nv_bfloat16* to = (blockIdx.y ? vp : kp) + i;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const uint32_t a = pack_bf16x2(x.x, x.y), b = pack_bf16x2(x.z, x.w);
        *reinterpret_cast<uint2*>(to + p * plane) = make_uint2(a, b);
        x = make_float4(x.x - __uint_as_float(a << 16), x.y - __uint_as_float(a & 0xffff0000u), x.z - __uint_as_float(b << 16), x.w - __uint_as_float(b & 0xffff0000u));
    }
}

}  // namespace ggr
