// Attention over pages (or over packed rows) on the warp-level tensor-core instructions: single tokens, short chunks, and
// everything in 32-bit precision or at head_dim 256. attention_token of the reference (src/engine/runtime/inference.rs:
// 1970-2530) for each new token of a batch, as one online softmax over the visible keys
//     o = sum_j p_j v_j / sum_j p_j,   p_j = 2^((s_j - m) c),   s_j = q . k_j,   c = scale * log2 e.
//
// Two forms of one tile step (16 rows x 16 keys, PagedMma::step):
//  - paged_splitk_kernel: the eight (head_dim 256: four) warps of a CTA share 16 rows and split the keys between them, each
//    with a ring of its own that TMA fills; states are merged in shared memory, and over CTAs by the last one to finish a row
//    tile. Bound by the bytes of the cache: for a few tokens times G heads every cache byte is read once.
//  - paged_rows_kernel: eight warps with 16 rows each walk the same keys through one ring, which a ninth warp fills.
//
// Precision. bf16 rows: q and codes are exact operands, softmax weights (times the scale of an 8-bit row) are rounded once to
// bf16. f32 rows: q and the weights go in as two bf16 parts (the 2^-17 left out is below what the sums lose), f32 keys and
// values as two bf16 planes, products of two low parts left out.
//
// Keys that only some rows of a tile see get weight 0, and 0 times an infinity or NaN in a value would spoil the other rows:
// a row whose result is not finite is computed again, key by key, by paged_row_again. Rows of a tile that nobody sees
// (behind the sequence's end, before its window: never written, freed or another sequence's) are cleared in shared memory.
#pragma once

#include "mma_utils.cuh"
#include "paged.cuh"
#include "sm100_utils.cuh"

namespace ggr {

constexpr int kPagedSplitMax = 128;  // pieces of one row tile

struct PagedAttnArgs {
    PageView pages;          // fmt also for packed rows: KV_BF16 (one plane), KV_F32 (two bf16 planes)
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

// One row again, key by key in f32, by a warp: what is not seen is not touched. Only rows whose fast result is not finite.
template <int D, bool F32>
__device__ __noinline__ void paged_row_again(const PagedAttnArgs& a, const PagedItem& w, int kvh, int r, int lane) {
    constexpr int E = D / 32;
    const int tok = r / a.G, h = kvh * a.G + r % a.G, pos = w.pos0 + tok;
    const int64_t qo = (w.tok0 + tok) * a.q_stride + (int64_t)h * D;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < E; ++i) {
        q[i] = F32 ? static_cast<const float*>(a.q)[qo + lane + 32 * i] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[qo + lane + 32 * i]);
        o[i] = 0.0f;
    }
    auto at = [&](const void* packed, int64_t stride, const unsigned char* pool, const float* scales, int j, int d) -> float {
        if (!a.paged) {
            const int64_t i = (int64_t)(w.src + j) * stride + (int64_t)kvh * D + d;
            return F32 ? static_cast<const float*>(packed)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(packed)[i]);
        }
        const int64_t row = a.pages.row(a.layer, a.plan.table[w.src + (j >> a.pages.page_log2)], kvh, j & ((1 << a.pages.page_log2) - 1));
        if (a.pages.fmt == KV_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(pool)[row * D + d]);
        return (float)reinterpret_cast<const signed char*>(pool)[row * D + d] * scales[row];
    };
    for (int j = paged_first_key(pos, a.window); j <= pos; ++j) {
        float s = 0.0f;
        for (int i = 0; i < E; ++i) s = fmaf(q[i], at(a.pk, a.pk_stride, a.pages.k, a.pages.ks, j, lane + 32 * i), s);
        s = warp_sum(s) * a.c;
        const float top = fmaxf(m, s), f = m == top ? 1.0f : exp2f(m - top), p = exp2f(s - top);
        m = top;
        l = l * f + p;
        for (int i = 0; i < E; ++i) o[i] = o[i] * f + p * at(a.pv, a.pv_stride, a.pages.v, a.pages.vs, j, lane + 32 * i);
    }
    const int64_t oo = (w.tok0 + tok) * a.o_stride + (int64_t)h * D;
    for (int i = 0; i < E; ++i) {
        if (F32)
            static_cast<float*>(a.out)[oo + lane + 32 * i] = o[i] / l;
        else
            static_cast<__nv_bfloat16*>(a.out)[oo + lane + 32 * i] = __float2bfloat16_rn(o[i] / l);
    }
}

// FMT: KV_BF16, kKvQ8Head, or KV_F32 = two bf16 planes. F32: rows in two bf16 parts.
template <int D, int FMT, bool F32>
struct PagedMma {
    static constexpr bool Q8 = FMT == kKvQ8Head, PLANES = FMT == KV_F32;
    static constexpr int NP = F32 ? 2 : 1;
    static constexpr int ROW = Q8 ? D : 2 * D;                    // bytes of a cache row
    static constexpr int BOX = ROW < 128 ? ROW : 128;             // bytes of a row in one swizzled block
    static constexpr int NBLK = ROW / BOX;
    static constexpr uint32_t BLK = 16 * BOX;
    static constexpr uint32_t MAT = NBLK * BLK;                   // 16 rows of K or V
    static constexpr uint32_t TILE = (PLANES ? 4 : 2) * MAT;      // K [K low] V [V low]
    static constexpr uint32_t V0 = (PLANES ? 2 : 1) * MAT;
    static constexpr uint32_t TX = TILE + (Q8 ? 128 : 0);
    static constexpr int KS = D / 16, NT = D / 8;
    static constexpr bool QSMEM = D == 256;                       // q fragments in shared memory: 128 registers of o leave no room
    static constexpr uint32_t QBYTES = QSMEM ? NP * KS * 512 : 0; // of 16 rows

    uint32_t qf[QSMEM ? 1 : NP][QSMEM ? 1 : KS][4];
    uint32_t q_smem;
    float o[NT][4];
    float m0, m1, l0, l1;

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
    }

    // Fragments of rows r0 .. r0 + 15 (zeros from r1 on). Of 8-bit keys a lane holds four consecutive elements of a row, and
    // the elements of q are taken in that order; the order of the sum does not matter as long as both sides have the same.
    __device__ __forceinline__ void load_q(const PagedAttnArgs& a, const PagedItem& w, int kvh, int r0, int r1, int lane, uint32_t smem) {
        const int gq = lane >> 2, tq = lane & 3;
        q_smem = smem + lane * 16;
        int64_t at[2];
        bool ok[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + gq + 8 * i, tok = r / a.G;
            ok[i] = r < r1;
            at[i] = (w.tok0 + tok) * a.q_stride + (int64_t)(kvh * a.G + r - tok * a.G) * D;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t f[NP][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int d = ks * 16 + (Q8 ? tq * 4 + half * 2 : tq * 2 + half * 8);
                    const int reg = i + 2 * half;
                    if constexpr (!F32) {
                        f[0][reg] = ok[i] ? *reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(a.q) + at[i] + d) : 0u;
                    } else {
                        const float2 x = ok[i] ? *reinterpret_cast<const float2*>(static_cast<const float*>(a.q) + at[i] + d) : make_float2(0.f, 0.f);
                        split2(x.x, x.y, f[0][reg], f[NP - 1][reg]);
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

    // x = hi + lo in bf16 pairs
    static __device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
        hi = pack_bf16x2(x, y);
        lo = pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
    }

    // Two of four int8 (selector picks their bytes) as a bf16 pair, exactly: with the sign bit aside a code is 0 .. 127, which
    // the seven mantissa bits of 128 .. 255 hold; 128 (or, for a negative code, 256) is taken off again.
    static __device__ __forceinline__ uint32_t codes2(uint32_t w, uint32_t sel) {
        const uint32_t x = __byte_perm(w, 0x43434343u, sel);
        const uint32_t lo = x & 0xff7fff7fu, hi = x & 0xff80ff80u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&hi));
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
        mma_bf16_16816(c, x[0], x[1], x[2], x[3], b0, b1);
    }

    // One tile: K at `kt`, V at `kt + V0`, the scales of an 8-bit tile at ks16 / ks16 + 16. Rows gq and gq + 8 of the warp see
    // the keys [lo_i, hi_i) of the tile's 16; whole: all rows see all of them.
    __device__ __forceinline__ void step(uint32_t kt, const float* ks16, bool whole, int lo0, int hi0, int lo1, int hi1, float c, int lane) {
        const int tq = lane & 3;
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
        if constexpr (!Q8) {
            const int row = (lane & 7) + ((lane >> 4) & 1) * 8, half = (lane >> 3) & 1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t f[NP][4], b[4];
#pragma unroll
                for (int np = 0; np < NP; ++np) frag(np, ks, f[np]);
                ldmatrix_x4(kt + piece(row, 2 * ks + half), b[0], b[1], b[2], b[3]);
#pragma unroll
                for (int np = 0; np < NP; ++np) {
                    mma(sc[0], f[np], b[0], b[1]);
                    mma(sc[1], f[np], b[2], b[3]);
                }
                if constexpr (PLANES) {
                    ldmatrix_x4(kt + MAT + piece(row, 2 * ks + half), b[0], b[1], b[2], b[3]);
                    mma(sc[0], f[0], b[0], b[1]);
                    mma(sc[1], f[0], b[2], b[3]);
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
                for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
                    for (int np = 0; np < NP; ++np) {
                        uint32_t f[4];
                        frag(np, 2 * i + k2, f);
                        mma(sc[0], f, codes2(r[k2], 0x4140), codes2(r[k2], 0x4342));
                        mma(sc[1], f, codes2(r[2 + k2], 0x4140), codes2(r[2 + k2], 0x4342));
                    }
                }
            }
        }
        float sv[4];  // scales of V for this lane's four keys
        if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 k2 = *reinterpret_cast<const float2*>(ks16 + j * 8 + tq * 2);
                const float2 v2 = *reinterpret_cast<const float2*>(ks16 + 16 + j * 8 + tq * 2);
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
        float x0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
        float x1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        // the reference maximum moves only when it grows by more than a factor of 2^8: l and o stay exact, they use the same
        const float thr = 8.0f / c;
        const bool need0 = x0 > m0 + thr, need1 = x1 > m1 + thr;
        if (__any_sync(0xffffffffu, need0 || need1)) {
            const float f0 = need0 ? tc::ex2((m0 - x0) * c) : 1.0f, f1 = need1 ? tc::ex2((m1 - x1) * c) : 1.0f;
            if (need0) m0 = x0;
            if (need1) m1 = x1;
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][0] *= f0;
                o[nt][1] *= f0;
                o[nt][2] *= f1;
                o[nt][3] *= f1;
            }
        }
        const float b0 = m0 == -INFINITY ? 0.0f : -m0 * c, b1 = m1 == -INFINITY ? 0.0f : -m1 * c;
        uint32_t pf[NP][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float p[4];
            p[0] = tc::ex2(fmaf(sc[j][0], c, b0));
            p[1] = tc::ex2(fmaf(sc[j][1], c, b0));
            p[2] = tc::ex2(fmaf(sc[j][2], c, b1));
            p[3] = tc::ex2(fmaf(sc[j][3], c, b1));
            l0 += p[0] + p[1];
            l1 += p[2] + p[3];
            if constexpr (Q8) {
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = p[i] == 0.0f ? 0.0f : p[i] * sv[2 * j + (i & 1)];  // (a hidden row's scale may be NaN)
            }
            if constexpr (!F32) {
                pf[0][2 * j] = pack_bf16x2(p[0], p[1]);
                pf[0][2 * j + 1] = pack_bf16x2(p[2], p[3]);
            } else {
                split2(p[0], p[1], pf[0][2 * j], pf[NP - 1][2 * j]);
                split2(p[2], p[3], pf[0][2 * j + 1], pf[NP - 1][2 * j + 1]);
            }
        }
        const uint32_t vt = kt + V0;
        if constexpr (!Q8) {
            const int row = (lane & 7) + ((lane >> 3) & 1) * 8, half = (lane >> 4) & 1;
#pragma unroll
            for (int n2 = 0; n2 < NT / 2; ++n2) {
                uint32_t b[4];
                ldmatrix_x4_trans(vt + piece(row, 2 * n2 + half), b[0], b[1], b[2], b[3]);
#pragma unroll
                for (int np = 0; np < NP; ++np) {
                    mma(o[2 * n2], pf[np], b[0], b[1]);
                    mma(o[2 * n2 + 1], pf[np], b[2], b[3]);
                }
                if constexpr (PLANES) {
                    ldmatrix_x4_trans(vt + MAT + piece(row, 2 * n2 + half), b[0], b[1], b[2], b[3]);
                    mma(o[2 * n2], pf[0], b[0], b[1]);
                    mma(o[2 * n2 + 1], pf[0], b[2], b[3]);
                }
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
                for (int k2 = 0; k2 < 2; ++k2) {
                    const int nt = 2 * (2 * i + k2);
                    const uint32_t e0 = codes2(r[2 * k2], 0x4240), e1 = codes2(r[2 * k2 + 1], 0x4240);
                    const uint32_t d0 = codes2(r[2 * k2], 0x4341), d1 = codes2(r[2 * k2 + 1], 0x4341);
#pragma unroll
                    for (int np = 0; np < NP; ++np) {
                        mma(o[nt], pf[np], e0, e1);
                        mma(o[nt + 1], pf[np], d0, d1);
                    }
                }
            }
        }
    }

    // o[nt][0 / 2] and o[nt][1 / 3] are elements element(nt, 0) and element(nt, 1) of rows gq / gq + 8
    static __device__ __forceinline__ int element(int nt, int i, int tq) {
        if constexpr (Q8) return (nt >> 1) * 16 + 4 * tq + 2 * i + (nt & 1);
        return nt * 8 + 2 * tq + i;
    }

    __device__ __forceinline__ void sum_rows() {
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    }

    // Requests the 16 keys from `key` on (a multiple of 16) into `dst`; one lane. Packed keys lie in their rows, paged ones in
    // page `page` of the pool.
    static __device__ __forceinline__ void request(const PagedAttnArgs& a, const CUtensorMap* tk, const CUtensorMap* tv, const PagedItem& w,
                                                   int kvh, int key, int page, uint32_t dst, uint32_t scales, uint32_t bar) {
        if (a.paged) {
            const int in_page = key & ((1 << a.pages.page_log2) - 1);
            const int z = (a.layer * a.pages.n_pages + page) * a.pages.Hkv + kvh;
#pragma unroll
            for (int b = 0; b < NBLK; ++b) {
                const int x = b * (Q8 ? BOX : BOX / 2);
                tma_load_3d(dst + b * BLK, tk, x, in_page, z, bar);
                tma_load_3d(dst + V0 + b * BLK, tv, x, in_page, z, bar);
            }
            if constexpr (Q8) {
                const int64_t row = ((int64_t)z << a.pages.page_log2) + in_page;
                tc::bulk_load(scales, a.pages.ks + row, 64, bar);
                tc::bulk_load(scales + 64, a.pages.vs + row, 64, bar);
            }
        } else {
            const int z = w.src + key;
#pragma unroll
            for (int p = 0; p < (PLANES ? 2 : 1); ++p)
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
        for (int i = lane; i < 16 * per_row * (PLANES ? 2 : 1); i += 32) {
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

template <int D, int FMT, bool F32>
struct PagedSplitKShape {
    using M = PagedMma<D, FMT, F32>;
    static constexpr int W = D == 256 ? 4 : 8;
    static constexpr int NST = FMT == kKvQ8Head ? (D == 64 ? 6 : 4) : (D == 64 ? 4 : 3);
    static constexpr int LD = D + 8;
    static constexpr uint32_t RING = W * NST * M::TILE;
    static constexpr uint32_t SCALES = FMT == kKvQ8Head ? W * NST * 128 : 0;
    static constexpr uint32_t MERGE = W * 16 * LD * 4;
    static constexpr uint32_t DATA = RING + SCALES > MERGE ? RING + SCALES : MERGE;  // the merge reuses the rings
    static constexpr uint32_t SMEM = DATA + M::QBYTES + 1024;
};

// An item is 16 packed rows of one sequence (fewer at its end) and a stretch of keys; blockIdx.y is the KV head.
template <int D, int FMT, bool F32>
__global__ void __launch_bounds__(PagedSplitKShape<D, FMT, F32>::W * 32, 1)
paged_splitk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttnArgs a) {
    using namespace tc;
    using S = PagedSplitKShape<D, FMT, F32>;
    using M = typename S::M;
    constexpr int W = S::W, NST = S::NST, LD = S::LD;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t s_full[W][NST];
    __shared__ float s_m[W][16], s_l[W][16];  // per warp, then weights of the warps
    __shared__ float s_top[16], s_sum[16];
    __shared__ float s_w[16][kPagedSplitMax];
    __shared__ int s_abort, s_last, s_bad;

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int gq = lane >> 2, tq = lane & 3, kvh = blockIdx.y;
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    unsigned char* base_p = smem + (base - smem_u32(smem));
    const uint32_t ring = base + warp * NST * M::TILE;
    const uint32_t scales = base + S::RING + warp * NST * 128;
    const float* scales_p = reinterpret_cast<const float*>(base_p + S::RING + warp * NST * 128);
    float* acc = reinterpret_cast<float*>(base_p);  // [W][16][LD] after the rings have drained
    volatile int* abortp = &s_abort;
    if (tid == 0) s_abort = 0;
    if (lane == 0) {
        for (int s = 0; s < NST; ++s) mbar_init(smem_u32(&s_full[warp][s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    const int n_items = a.plan.counts[0];
    uint32_t used = 0;  // tiles this warp has been through: ring position and phase
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const PagedItem w = a.plan.items[item];
        const int n_tiles = (w.key1 - w.key0 + 15) >> 4, mine = n_tiles > warp ? (n_tiles - warp + W - 1) / W : 0;
        // keys that some row, and that every row, of the tile sees
        const int tok_lo = w.row0 / a.G, tok_hi = (w.row0 + w.rows - 1) / a.G;
        const int any_lo = paged_first_key(w.pos0 + tok_lo, a.window), any_hi = w.pos0 + tok_hi + 1;
        const int all_lo = paged_first_key(w.pos0 + tok_hi, a.window), all_hi = w.pos0 + tok_lo + 1;
        auto issue = [&](int t) {
            const uint32_t u = used + t, stage = u % NST;
            const int key = w.key0 + (warp + t * W) * 16;
            const uint32_t bar = smem_u32(&s_full[warp][stage]);
            const int page = a.paged ? a.plan.table[w.src + (key >> a.pages.page_log2)] : 0;
            mbar_expect_tx(bar, M::TX);
            M::request(a, &tmK, &tmV, w, kvh, key, page, ring + stage * M::TILE, scales + stage * 128, bar);
        };
        if (lane == 0)
            for (int t = 0; t < NST - 1 && t < mine; ++t) issue(t);
        M x;
        x.start();
        x.load_q(a, w, kvh, w.row0, w.row0 + w.rows, lane, base + S::DATA);
        if constexpr (M::QSMEM) __syncthreads();  // (every warp has written the same fragments)
        const int p0 = w.pos0 + min(w.row0 + gq, w.row0 + w.rows - 1) / a.G, p1 = w.pos0 + min(w.row0 + gq + 8, w.row0 + w.rows - 1) / a.G;
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
            x.step(kt, scales_p + stage * 32, whole, lo0 - key, p0 + 1 - key, lo1 - key, p1 + 1 - key, a.c, lane);
            __syncwarp();
            if (lane == 0 && t + NST - 1 < mine) {
                fence_smem_to_async_proxy();
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
                *reinterpret_cast<float4*>(&acc[(warp * 16 + gq) * LD + d]) = make_float4(x.o[nt][0], x.o[nt + 1][0], x.o[nt][1], x.o[nt + 1][1]);
                *reinterpret_cast<float4*>(&acc[(warp * 16 + gq + 8) * LD + d]) = make_float4(x.o[nt][2], x.o[nt + 1][2], x.o[nt][3], x.o[nt + 1][3]);
            } else {
                const int d = M::element(nt, 0, tq);
                *reinterpret_cast<float2*>(&acc[(warp * 16 + gq) * LD + d]) = make_float2(x.o[nt][0], x.o[nt][1]);
                *reinterpret_cast<float2*>(&acc[(warp * 16 + gq + 8) * LD + d]) = make_float2(x.o[nt][2], x.o[nt][3]);
            }
        }
        if (tq == 0) {
            s_m[warp][gq] = x.m0;
            s_m[warp][gq + 8] = x.m1;
            s_l[warp][gq] = x.l0;
            s_l[warp][gq + 8] = x.l1;
        }
        if (tid == 0) s_bad = 0;
        __syncthreads();
        if (tid < 16) {
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
        constexpr int STATE = 16 * (D + 2);
        float* state0 = a.part + ((int64_t)(split ? w.part : 0) * a.pages.Hkv + kvh) * STATE;  // of the tile's first piece
        const int64_t state_step = (int64_t)a.pages.Hkv * STATE;
        float* mine_state = state0 + w.split * state_step;
        for (int i = tid; i < w.rows * (D / 4); i += W * 32) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float f = s_m[k][r];
                const float4 y = *reinterpret_cast<const float4*>(&acc[(k * 16 + r) * LD + d]);
                v.x = fmaf(f, y.x, v.x);
                v.y = fmaf(f, y.y, v.y);
                v.z = fmaf(f, y.z, v.z);
                v.w = fmaf(f, y.w, v.w);
            }
            if (split) {
                __stcg(reinterpret_cast<float4*>(mine_state + r * D + d), v);
            } else {
                const int R = w.row0 + r, tok = R / a.G;
                const float inv = 1.0f / s_sum[r];
                v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                if (!finite4(v)) s_bad = 1;
                paged_store4<F32>(a, (w.tok0 + tok) * a.o_stride + (int64_t)(kvh * a.G + R - tok * a.G) * D + d, v);
            }
        }
        if (split) {
            if (tid < w.rows) __stcg(reinterpret_cast<float2*>(mine_state + 16 * D) + tid, make_float2(s_top[tid], s_sum[tid]));
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
                        top = fmaxf(top, __ldcg(reinterpret_cast<const float2*>(state0 + s * state_step + 16 * D) + r).x);
                    top = warp_max(top);
                    float sum = 0.0f;
                    for (int s = lane; s < w.n_split; s += 32) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(state0 + s * state_step + 16 * D) + r);
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
                    const int R = w.row0 + r, tok = R / a.G;
                    const float inv = 1.0f / s_sum[r];
                    v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                    if (!finite4(v)) s_bad = 1;
                    paged_store4<F32>(a, (w.tok0 + tok) * a.o_stride + (int64_t)(kvh * a.G + R - tok * a.G) * D + d, v);
                }
            }
        }
        __syncthreads();
        if (s_bad) {
            for (int r = warp; r < w.rows; r += W) paged_row_again<D, F32>(a, w, kvh, w.row0 + r, lane);
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
    using M = PagedMma<D, FMT, F32>;
    static constexpr int W = 8;
    static constexpr int SUB = FMT == KV_F32 && D == 256 ? 1 : 2;  // tiles of 16 keys in a stage
    static constexpr uint32_t STAGE = SUB * M::TILE;
    static constexpr int NST = STAGE >= 32768 ? 2 : 4;
    static constexpr uint32_t RING = NST * STAGE;
    static constexpr uint32_t SCALES = FMT == kKvQ8Head ? NST * SUB * 128 : 0;
    static constexpr uint32_t SMEM = RING + SCALES + W * M::QBYTES + 1024;
};

// An item is up to 128 packed rows of one sequence and all the keys that they see; blockIdx.y is the KV head.
template <int D, int FMT, bool F32>
__global__ void __launch_bounds__(288, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttnArgs a) {
    using namespace tc;
    using S = PagedRowsShape<D, FMT, F32>;
    using M = typename S::M;
    constexpr int NST = S::NST, SUB = S::SUB, KT = 16 * SUB;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t s_full[NST], s_empty[NST], s_raw;
    __shared__ int s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int gq = lane >> 2, tq = lane & 3, kvh = blockIdx.y;
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    unsigned char* base_p = smem + (base - smem_u32(smem));
    volatile int* abortp = &s_abort;
    if (tid == 0) {
        s_abort = 0;
        for (int s = 0; s < NST; ++s) {
            mbar_init(smem_u32(&s_full[s]), 1);
            mbar_init(smem_u32(&s_empty[s]), S::W);
        }
        mbar_init(smem_u32(&s_raw), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const int n_items = a.plan.counts[0];
    uint32_t used = 0, raws = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const PagedItem w = a.plan.items[item];
        const int n_stages = (w.key1 - w.key0 + KT - 1) / KT;
        const int tok_lo = w.row0 / a.G, tok_hi = (w.row0 + w.rows - 1) / a.G;
        const int any_lo = paged_first_key(w.pos0 + tok_lo, a.window), any_hi = w.pos0 + tok_hi + 1;
        if (warp == S::W) {
            for (int t = 0; t < n_stages; ++t) {
                const uint32_t u = used + t, stage = u % NST;
                if (!mbar_wait_warp(smem_u32(&s_empty[stage]), ((u / NST) & 1u) ^ 1u, abortp)) break;
                const int key = w.key0 + t * KT;
                const bool edge = key < any_lo || key + KT > any_hi;
                const uint32_t bar = edge ? smem_u32(&s_raw) : smem_u32(&s_full[stage]);
                const uint32_t dst = base + stage * S::STAGE, sc = base + S::RING + stage * SUB * 128;
                if (lane == 0) {
                    // tiles behind the last visible key have no page: they are left out, and step() is not called for them
                    const int subs = min(SUB, (any_hi - key + 15) >> 4);
                    mbar_expect_tx(bar, subs * M::TX);
                    for (int i = 0; i < subs; ++i) {
                        const int k = key + 16 * i;
                        const int page = a.paged ? a.plan.table[w.src + (k >> a.pages.page_log2)] : 0;
                        M::request(a, &tmK, &tmV, w, kvh, k, page, dst + i * M::TILE, sc + i * 128, bar);
                    }
                }
                __syncwarp();
                if (edge) {
                    if (!mbar_wait_warp(bar, raws & 1u, abortp)) break;
                    ++raws;
                    for (int i = 0; i < SUB; ++i) M::clear(dst + i * M::TILE, any_lo - key - 16 * i, any_hi - key - 16 * i, lane);
                    fence_smem_to_async_proxy();  // (this stage's next copy comes after the arrivals below and the readers')
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&s_full[stage]));
                }
            }
            used += n_stages;
        } else {
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
            for (int t = 0; t < n_stages; ++t) {
                const uint32_t u = used + t, stage = u % NST;
                if (!mbar_wait_warp(smem_u32(&s_full[stage]), (u / NST) & 1u, abortp)) break;
#pragma unroll 1
                for (int i = 0; i < SUB; ++i) {
                    const int key = w.key0 + t * KT + 16 * i;
                    if (!mine || key >= see_hi || key + 16 <= see_lo) continue;
                    const bool whole = key >= all_lo && key + 16 <= all_hi;
                    x.step(base + stage * S::STAGE + i * M::TILE, reinterpret_cast<const float*>(base_p + S::RING + (stage * SUB + i) * 128), whole,
                           lo0 - key, p0 + 1 - key, lo1 - key, p1 + 1 - key, a.c, lane);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_empty[stage]));
            }
            used += n_stages;
            if (mine && !*abortp) {
                x.sum_rows();
                const float i0 = 1.0f / x.l0, i1 = 1.0f / x.l1;
                bool bad = false;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int R = r0 + gq + 8 * half, tok = R / a.G;
                    if (R >= r1) continue;
                    const int64_t at = (w.tok0 + tok) * a.o_stride + (int64_t)(kvh * a.G + R - tok * a.G) * D;
                    const float inv = half ? i1 : i0;
#pragma unroll
                    for (int nt = 0; nt < M::NT; ++nt) {
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
                }
                if (__any_sync(0xffffffffu, bad)) {
                    __syncwarp();
                    for (int r = r0; r < min(r0 + 16, r1); ++r) paged_row_again<D, F32>(a, w, kvh, r, lane);
                }
            }
        }
        if (*abortp) break;
    }
    if (s_abort) {
        for (int i = 0; i < 500; ++i) __nanosleep(1000);  // let copies in flight land
    }
    __syncthreads();
    if (tid == 0 && s_abort && a.err) atomicExch(a.err, 1);
}

// f32 rows of k or v as two bf16 planes: x = hi + lo. Rows of `dim` elements, four per thread.
__global__ void __launch_bounds__(256) paged_planes_kernel(const float* k, const float* v, int64_t k_stride, int64_t v_stride, int rows, int dim,
                                                           __nv_bfloat16* kp, __nv_bfloat16* vp, int64_t plane) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= (int64_t)rows * dim) return;
    const int64_t r = i / dim, d = i - r * dim;
    const float4 x = *reinterpret_cast<const float4*>((blockIdx.y ? v + r * v_stride : k + r * k_stride) + d);
    const uint32_t h0 = pack_bf16x2(x.x, x.y), h1 = pack_bf16x2(x.z, x.w);
    const uint32_t l0 = pack_bf16x2(x.x - __uint_as_float(h0 << 16), x.y - __uint_as_float(h0 & 0xffff0000u));
    const uint32_t l1 = pack_bf16x2(x.z - __uint_as_float(h1 << 16), x.w - __uint_as_float(h1 & 0xffff0000u));
    __nv_bfloat16* to = (blockIdx.y ? vp : kp) + i;
    *reinterpret_cast<uint2*>(to) = make_uint2(h0, h1);
    *reinterpret_cast<uint2*>(to + plane) = make_uint2(l0, l1);
}

}  // namespace ggr
