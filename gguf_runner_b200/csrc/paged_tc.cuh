// Attention of chunks and of packed prompts in bf16 on the 5th-generation tensor cores, head_dim 64 and 128.
//
// The pipeline is that of the dense prefill kernel (prefill_tc.cuh): a persistent CTA per SM, a producer warp, one MMA issuer,
// two softmax warpgroups with a 128-row query tile each that take turns on the tensor core, S and O in tensor memory, P
// written over S. What differs is where rows come from:
//  - A query tile holds 128 / G tokens times the G query heads of one KV head (one 3-D copy: element, head, token), so that a
//    key tile is read once for all heads that share it and a chunk of few tokens still fills the tensor core's 128 rows.
//  - A 128-key tile is gathered from its pages, a copy per page (half a page of 256) and 64-column block, issued by the lanes
//    of the producer warp side by side; each lane looks its page up one tile ahead.
//  - Items (two query tiles and a stretch of keys) are cut on the host, longest first, and handed out through a counter. Pieces
//    of a pair of tiles leave un-normalised rows, which paged_tc_merge_kernel weighs in the order of the keys.
//  - 8-bit pages are read into dense f16 rows first (paged_read_kernel, 34 us of 680 for 2048 tokens behind 14336, 40/8 heads
//    of 128), q into f16 beside them: eleven bits leave code * scale 2^-12 off, an eighth of what bf16 weights are (weights: see
//    kPtHalfShift). bf16 rows would add two roundings as large as that of the weights (by their variances 3.2e-3 instead of 2.3e-3
//    from 64 bits), and scales that the softmax warps multiply into scores and weights are two multiplications and half a
//    shared-memory load per score.
// Values that nobody in the item sees (behind the sequence's end, before its window) may be anything, and 0 * NaN is NaN: the
// producer clears them in the first and last tile, before the MMA issuer hears of the tile. Rows that come out not finite are
// computed again by paged_row_again.
#pragma once

#include "paged_mma.cuh"

namespace ggr {

struct PagedTcArgs {
    PagedAttnArgs a;
    int tiles_tokens;  // tokens of a query tile: 128 / G
    int box_rows;      // paged: rows of one copy, min(page_size, 128)
    int linear;        // K and V tiles come from dense rows (packed prompts, or 8-bit pages read into f16 rows)
    const void* q_rows;      // head_dim 256: the 16-bit rows of q that are multiplied (of 8-bit pages the f16 ones)
    int64_t q_rows_stride;
    float out_scale;   // of the merged rows: 1 / kReadVScale for f16 rows
    // Launched programmatically behind the warp-level kernel of the same call, of which it reads nothing: that one lets it in
    // when it has itself waited for all that came before, so that this kernel's CTAs take the SMs as that one's leave them. It
    // waits for it before it ends, which keeps the order for all that follows.
    int behind;
    int* sched;        // [0] items handed out beyond the first wave, [1] CTAs that have left
    float* part;       // states of pieces: [256][D], then [256] (m, l)
};

constexpr int kPtThreads = 384, kPtCtrlRegs = 88, kPtSoftmaxRegs = 208;
static_assert(tc::RegSplitOk<kPtCtrlRegs, kPtSoftmaxRegs>::value, "setmaxnreg split would never complete");
constexpr int kPtExpPolyMask = 0x5;  // groups of four scores of which one pair takes its exponentials from the FMA pipe
template <int D>
constexpr int kPtState = 256 * (D + 2);
template <int D>
constexpr size_t kPtSmem = (size_t)6 * (D / 64) * 128 * 128 + 8 * 4096 + 1024;

// The key tiles of an item that each query tile walks.
struct PtRange {
    int lo0, hi0, lo1, hi1, lo, hi;
    __device__ __forceinline__ int lo_of(int t) const { return t ? lo1 : lo0; }
    __device__ __forceinline__ int hi_of(int t) const { return t ? hi1 : hi0; }
    __device__ __forceinline__ bool active(int t, int j) const { return j >= lo_of(t) && j < hi_of(t); }
};
__device__ __forceinline__ PtRange pt_range(const PagedTcArgs& p, const PagedItem& w) {
    PtRange r;
    int lo_t[2], hi_t[2];
    const int s_lo = w.key0 >> 7, s_hi = (w.key1 + 127) >> 7;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = w.row0 + t * p.tiles_tokens, last = min(first + p.tiles_tokens, w.n_tok) - 1;
        lo_t[t] = hi_t[t] = 0;
        if (first > last) continue;
        lo_t[t] = max(s_lo, paged_first_key(w.pos0 + first, p.a.window) >> 7);
        hi_t[t] = max(lo_t[t], min(s_hi, (w.pos0 + last + 128) >> 7));
    }
    r.lo0 = lo_t[0], r.hi0 = hi_t[0], r.lo1 = lo_t[1], r.hi1 = hi_t[1];
    const bool act0 = r.hi0 > r.lo0, act1 = r.hi1 > r.lo1;
    r.lo = act0 ? r.lo0 : r.lo1;
    r.hi = act0 ? r.hi0 : r.hi1;
    if (act0 && act1) {
        r.lo = min(r.lo0, r.lo1);
        r.hi = max(r.hi0, r.hi1);
    }
    return r;
}

// f16 weights are taken times 2^7, and so is their sum: a weight is at most 2^8 (the lazy reference maximum) and stays in range, and
// what is 2^-21 of the reference (2^-14 without) still has all eleven bits, 2^-31 a value at all. Thousands of keys at 2^-26 of the
// largest weight would else drop out of the result while the sum keeps them.
constexpr float kPtHalfShift = 7.0f;
template <bool HALF>
__device__ __forceinline__ uint32_t pt_pack(float x, float y) {
    if constexpr (!HALF) return pack_bf16x2(x, y);
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// HALF: operands are f16 (of 8-bit pages; V times kReadVScale) instead of bf16.
template <int D, bool HALF>
__global__ void __launch_bounds__(kPtThreads, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ PagedTcArgs p) {
    using namespace tc;
    constexpr int NBLK = D / 64;
    constexpr uint32_t BLK = 128 * 128, TILE = NBLK * BLK, O_COL0 = 256;

    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bars[25];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_flags[2];  // of paged_wait
    int& s_abort = s_flags[0];
    __shared__ __align__(16) PagedItem s_item[2];
    __shared__ int s_live[2];

    const PagedAttnArgs& a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sQ = smem_base, sK = sQ + 2 * TILE, sV = sK + 2 * TILE, sOut = sV + 2 * TILE;

    const uint32_t bar0 = smem_u32(bars);
    const uint32_t q_full = bar0, q_empty = bar0 + 8u, raw = bar0 + 8u * 24;
    auto k_full = [&](int s) { return bar0 + 8u * (2 + s); };
    auto k_empty = [&](int s) { return bar0 + 8u * (4 + s); };
    auto v_full = [&](int s) { return bar0 + 8u * (6 + s); };
    auto v_empty = [&](int s) { return bar0 + 8u * (8 + s); };
    auto s_full = [&](int t) { return bar0 + 8u * (10 + t); };
    auto p_half = [&](int t, int half) { return bar0 + 8u * (12 + 2 * t + half); };
    auto o_final = [&](int t) { return bar0 + 8u * (16 + t); };
    auto o_free = [&](int t) { return bar0 + 8u * (18 + t); };
    auto item_full = [&](int s) { return bar0 + 8u * (20 + s); };
    auto item_empty = [&](int s) { return bar0 + 8u * (22 + s); };

    if (tid == 0) {
        s_flags[0] = s_flags[1] = 0;
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(raw, 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(k_full(s), 1);
            mbar_init(k_empty(s), 1);
            mbar_init(v_full(s), 1);
            mbar_init(v_empty(s), 1);
            mbar_init(s_full(s), 1);
            mbar_init(p_half(s, 0), 128);
            mbar_init(p_half(s, 1), 128);
            mbar_init(o_final(s), 1);
            mbar_init(o_free(s), 128);
            mbar_init(item_full(s), 1);
            mbar_init(item_empty(s), 9);  // lane 0 of the eight softmax warps and of the MMA issuer
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(&s_tmem_base), 512);
        tmem_relinquish();
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = s_tmem_base;
    volatile int* abortp = s_flags;
    volatile int* livep = s_live;
    if (!p.behind) grid_wait();

    if (warp >= 8) {
        reg_release<kPtCtrlRegs>();
        if (warp == 8) {
            // ---------------- scheduler + TMA producer: the whole warp, a lane per copy ----------------
            const int n_items = a.plan.counts[0];
            const int boxes = p.linear ? 1 : 128 / p.box_rows, copies = boxes * NBLK;
            const int box = lane / NBLK, blk = lane % NBLK, box_key = p.linear ? 0 : box * p.box_rows;
            const uint32_t box_at = blk * BLK + box_key * 128, box_bytes = p.linear ? BLK : p.box_rows * 128;
            const uint32_t q_bytes = (uint32_t)p.tiles_tokens * a.G * 128 * NBLK;
            const int page_log2 = a.pages.page_log2;
            int g = 0;  // K / V tiles requested so far (ring position)
            uint32_t raws = 0;
            for (int it = 0;; ++it) {
                const int slot = it & 1;
                if (!paged_wait_warp(item_empty(slot), ((it >> 1) & 1) ^ 1, abortp)) break;
                int r = 0;
                if (lane == 0) r = it == 0 ? (int)blockIdx.x : (int)gridDim.x + atomicAdd(p.sched, 1);
                r = __shfl_sync(0xffffffffu, r, 0);
                const bool live = r < n_items;
                if (live && lane < (int)(sizeof(PagedItem) / 4))
                    reinterpret_cast<int*>(&s_item[slot])[lane] = reinterpret_cast<const int*>(a.plan.items + r)[lane];
                if (lane == 0) s_live[slot] = live;
                __syncwarp();
                if (lane == 0) mbar_arrive(item_full(slot));
                if (!live) break;
                const PagedItem w = s_item[slot];
                const PtRange rg = pt_range(p, w);
                const bool act0 = rg.hi0 > rg.lo0, act1 = rg.hi1 > rg.lo1;
                if (!paged_wait_warp(q_empty, (it & 1) ^ 1, abortp)) break;
                if (lane == 0) {
                    mbar_expect_tx(q_full, ((act0 ? 1 : 0) + (act1 ? 1 : 0)) * q_bytes);
                    for (int t = 0; t < 2; ++t) {
                        if (!(t == 0 ? act0 : act1)) continue;
                        for (int b = 0; b < NBLK; ++b)
                            tma_load_3d(sQ + t * TILE + b * BLK, &tmQ, b * 64, w.kvh * a.G, w.tok0 + w.row0 + t * p.tiles_tokens, q_full);
                    }
                }
                // values outside [any_lo, any_hi) are seen by no row of the item; pages end with the sequence
                const int any_lo = paged_first_key(w.pos0 + w.row0, a.window);
                const int any_hi = w.pos0 + min(w.row0 + 2 * p.tiles_tokens, w.n_tok), kv_end = w.pos0 + w.n_tok;
                auto page_of = [&](int j) {
                    const int key = j * 128 + box_key;
                    return !p.linear && lane < copies && key < kv_end && j < rg.hi ? a.plan.table[w.src + (key >> page_log2)] : 0;
                };
                int page = page_of(rg.lo);
                bool ok = true;
                for (int j = rg.lo; j < rg.hi; ++j, ++g) {
                    const int s = g & 1, key = j * 128 + box_key;
                    const uint32_t ph = ((g >> 1) & 1) ^ 1;
                    const bool mine = lane < copies && (p.linear || key < kv_end);
                    const uint32_t bytes = box_bytes * __popc(__ballot_sync(0xffffffffu, mine));
                    const int y = p.linear ? w.kvh : key & ((1 << page_log2) - 1);
                    const int z = p.linear ? w.lin + key : (a.layer * a.pages.n_pages + page) * a.pages.Hkv + w.kvh;
                    page = page_of(j + 1);
                    if (!(ok = paged_wait_warp(k_empty(s), ph, abortp))) break;
                    if (lane == 0) mbar_expect_tx(k_full(s), bytes);
                    __syncwarp();
                    if (mine) tma_load_3d(sK + s * TILE + box_at, &tmK, blk * 64, y, z, k_full(s));
                    if (!(ok = paged_wait_warp(v_empty(s), ph, abortp))) break;
                    const bool edge = j * 128 < any_lo || (j + 1) * 128 > any_hi;
                    const uint32_t vbar = edge ? raw : v_full(s);
                    if (lane == 0) mbar_expect_tx(vbar, bytes);
                    __syncwarp();
                    if (mine) tma_load_3d(sV + s * TILE + box_at, &tmV, blk * 64, y, z, vbar);
                    if (edge) {
                        if (!(ok = paged_wait_warp(raw, raws & 1u, abortp))) break;
                        ++raws;
                        for (int i = lane; i < 128 * NBLK * 8; i += 32) {
                            const int row = (i >> 3) & 127, k = j * 128 + row;
                            if (k >= any_lo && k < any_hi) continue;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sV + s * TILE + (i >> 10) * BLK + row * 128 + (i & 7) * 16), "r"(0u)
                                         : "memory");
                        }
                        fence_smem_to_async_proxy();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(v_full(s));
                    }
                }
                if (!ok) break;
            }
        } else if (warp == 9) {
            // ---------------- MMA issuer ----------------
            constexpr uint32_t TYPES = (1u << 7) | (1u << 10);  // A and B: bf16, or f16 without
            constexpr uint32_t IDESC_QK = idesc_bf16(128, 0) & ~(HALF ? TYPES : 0u), IDESC_PV = idesc_bf16(D, 1) & ~(HALF ? TYPES : 0u);
            const uint64_t dQ = smem_desc(sQ, 16, 1024), dK = smem_desc(sK, 16, 1024), dV = smem_desc(sV, BLK, 1024);
            const uint32_t tm = __shfl_sync(0xffffffffu, s_tmem_base, 0);
            auto issue_qk = [&](int t, int s) {
                const uint64_t a0 = dQ + (uint64_t)((t * TILE) >> 4), b0 = dK + (uint64_t)((s * TILE) >> 4);
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint32_t off = ((ks >> 2) * BLK + (ks & 3) * 32) >> 4;
                    mma_ss_e(tm + t * 128, a0 + off, b0 + off, IDESC_QK, ks > 0 ? 1u : 0u);
                }
            };
            auto issue_pv_half = [&](int t, int s, int half, bool accumulate) {
                const uint64_t b0 = dV + (uint64_t)((s * TILE) >> 4);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const int ks = half * 4 + kk;
                    mma_ts_e(tm + O_COL0 + t * D, tm + t * 128 + ks * 8, b0 + (uint64_t)((ks * 16 * 128) >> 4), IDESC_PV, (accumulate || ks > 0) ? 1u : 0u);
                }
            };
            int g = 0, c0 = 0, c1 = 0;
            bool ok = true;
            for (int it = 0; ok; ++it) {
                const int slot = it & 1;
                if (!(ok = paged_wait_warp(item_full(slot), (it >> 1) & 1, abortp))) break;
                const int live = __shfl_sync(0xffffffffu, livep[slot], 0);
                PtRange w = pt_range(p, s_item[slot]);
                w.lo0 = __shfl_sync(0xffffffffu, w.lo0, 0);
                w.hi0 = __shfl_sync(0xffffffffu, w.hi0, 0);
                w.lo1 = __shfl_sync(0xffffffffu, w.lo1, 0);
                w.hi1 = __shfl_sync(0xffffffffu, w.hi1, 0);
                w.lo = __shfl_sync(0xffffffffu, w.lo, 0);
                w.hi = __shfl_sync(0xffffffffu, w.hi, 0);
                if (lane == 0) mbar_arrive(item_empty(slot));
                if (!live) break;
                const int lo = w.lo, hi = w.hi;
                // every item moves o_free and o_final of both tiles on by one phase
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (w.hi_of(t) <= w.lo_of(t)) {
                        if (!(ok = paged_wait_warp(o_free(t), (it & 1) ^ 1, abortp))) break;
                        if (lane == 0) mbar_arrive(o_final(t));
                    }
                if (!ok) break;
                if (!(ok = paged_wait_warp(q_full, it & 1, abortp))) break;
                if (hi == lo) {
                    mma_commit_e(q_empty);
                    continue;
                }
                if (!(ok = paged_wait_warp(k_full(g & 1), (g >> 1) & 1, abortp))) break;
                fence_after_sync();
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (w.active(t, lo)) {
                        issue_qk(t, g & 1);
                        mma_commit_e(s_full(t));
                    }
                mma_commit_e(k_empty(g & 1));
                if (hi - lo == 1) mma_commit_e(q_empty);
                for (int j = lo; j < hi; ++j, ++g) {
                    const int s = g & 1;
                    const bool has_next = j + 1 < hi;
                    if (!(ok = paged_wait_warp(v_full(s), (g >> 1) & 1, abortp))) break;
                    bool next_k_ready = false;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int lo_t = w.lo_of(t), hi_t = w.hi_of(t), c_t = t ? c1 : c0;
                        if (j >= lo_t && j < hi_t) {
                            const uint32_t ph = (c_t + j - lo_t) & 1;
                            if (!(ok = paged_wait_warp(p_half(t, 0), ph, abortp))) break;
                            if (j == lo_t && !(ok = paged_wait_warp(o_free(t), (it & 1) ^ 1, abortp))) break;
                            fence_after_sync();
                            issue_pv_half(t, s, 0, j > lo_t);
                            if (!(ok = paged_wait_warp(p_half(t, 1), ph, abortp))) break;
                            fence_after_sync();
                            issue_pv_half(t, s, 1, true);
                            if (j == hi_t - 1) mma_commit_e(o_final(t));
                        }
                        if (has_next && j + 1 >= lo_t && j + 1 < hi_t) {
                            if (!next_k_ready) {
                                if (!(ok = paged_wait_warp(k_full(s ^ 1), ((g + 1) >> 1) & 1, abortp))) break;
                                fence_after_sync();
                                next_k_ready = true;
                            }
                            issue_qk(t, s ^ 1);
                            mma_commit_e(s_full(t));
                        }
                    }
                    if (!ok) break;
                    mma_commit_e(v_empty(s));
                    if (has_next) {
                        mma_commit_e(k_empty(s ^ 1));
                        if (j + 2 == hi) mma_commit_e(q_empty);
                    }
                }
                c0 += w.hi0 - w.lo0;
                c1 += w.hi1 - w.lo1;
            }
        }
    } else {
        // ---------------- softmax warps: one thread per query row ----------------
        reg_acquire<kPtSoftmaxRegs>();
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const int tile_tok = row / a.G, head = row - tile_tok * a.G;  // token of the tile and head of the group
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lane_addr + t * 128, tO = tmem + lane_addr + O_COL0 + t * D;
        const float c = a.c, thr = 8.0f / c;
        bool ok = true;
        int cs = 0;
        for (int it = 0; ok; ++it) {
            const int slot = it & 1;
            if (!(ok = paged_wait(item_full(slot), (it >> 1) & 1, abortp))) break;
            const int live = livep[slot];
            const PagedItem w = s_item[slot];
            __syncwarp();
            if (lane == 0) mbar_arrive(item_empty(slot));
            if (!live) break;
            const PtRange rg = pt_range(p, w);
            const int lo_t = rg.lo_of(t), hi_t = rg.hi_of(t), n_t = hi_t - lo_t;
            const int tok = w.row0 + t * p.tiles_tokens + tile_tok;
            const bool valid = tile_tok < p.tiles_tokens && tok < w.n_tok;
            // Rows that stand for no token (behind the sequence's end; three of 128 where five heads share a KV head) see everything:
            // their results go nowhere, and hidden keys would send their warps through the masks of every tile (40/8 heads, 2048
            // tokens behind 14336: 1186 us instead of 537).
            int vs = 0, ve = 0x7fffffff;
            if (valid) {
                ve = w.pos0 + tok + 1;
                vs = paged_first_key(w.pos0 + tok, a.window);
            }
            float m_used = -INFINITY, l = 0.0f;
            bool odd = false;
            for (int j = lo_t; j < hi_t; ++j) {
                const int k = j - lo_t;
                if (!(ok = paged_wait(s_full(t), (cs + k) & 1, abortp))) break;
                fence_after_sync();
                uint32_t sr[4][32];
#pragma unroll
                for (int cidx = 0; cidx < 4; ++cidx) tmem_ld32(tS + cidx * 32, sr[cidx]);
                tmem_wait_ld();
                const int key0 = j * 128;
                const bool cut = key0 < vs || key0 + 128 > ve, any_cut = __any_sync(0xffffffffu, cut);
                if (cut) {
#pragma unroll
                    for (int cidx = 0; cidx < 4; ++cidx)
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int key = key0 + cidx * 32 + i;
                            if (key < vs || key >= ve) sr[cidx][i] = 0xff800000u;  // -inf
                        }
                }
                float mxa = -INFINITY, mxb = -INFINITY, mxc = -INFINITY, mxd = -INFINITY;
#pragma unroll
                for (int cidx = 0; cidx < 4; ++cidx)
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        mxa = max3_nan(mxa, __uint_as_float(sr[cidx][i]), __uint_as_float(sr[cidx][i + 1]));
                        mxb = max3_nan(mxb, __uint_as_float(sr[cidx][i + 2]), __uint_as_float(sr[cidx][i + 3]));
                        mxc = max3_nan(mxc, __uint_as_float(sr[cidx][i + 4]), __uint_as_float(sr[cidx][i + 5]));
                        mxd = max3_nan(mxd, __uint_as_float(sr[cidx][i + 6]), __uint_as_float(sr[cidx][i + 7]));
                    }
                const float mx = max3_nan(max3_nan(mxa, mxb, mxc), mxd, mxd);
                // (a NaN score: the polynomial, which clamps its argument, would give that key weight 0)
                odd |= mx != mx;
                const bool need = mx > m_used + thr;
                float alpha = 1.0f;
                if (need) {
                    alpha = ex2((m_used - mx) * c);
                    m_used = mx;
                }
                if (k > 0 && __any_sync(0xffffffffu, need)) {
#pragma unroll 1
                    for (int cidx = 0; cidx < D / 32; ++cidx) {
                        uint32_t orow[32];
                        tmem_ld32(tO + cidx * 32, orow);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) orow[i] = __float_as_uint(__uint_as_float(orow[i]) * alpha);
                        tmem_st32(tO + cidx * 32, orow);
                    }
                }
                l *= alpha;
                const float mref = (m_used == -INFINITY) ? 0.0f : m_used;
                const float neg = (HALF ? kPtHalfShift : 0.0f) - mref * c;
                const uint64_t c2 = pack_f32x2(c, c), neg2 = pack_f32x2(neg, neg);
                uint64_t sum_a = 0ull, sum_b = 0ull;
#pragma unroll
                for (int cidx = 0; cidx < 4; ++cidx) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const uint64_t ta = fma_f32x2(pack_f32x2(__uint_as_float(sr[cidx][2 * i]), __uint_as_float(sr[cidx][2 * i + 1])), c2, neg2);
                        const uint64_t tb = fma_f32x2(pack_f32x2(__uint_as_float(sr[cidx][2 * i + 2]), __uint_as_float(sr[cidx][2 * i + 3])), c2, neg2);
                        float x0, x1, p2, p3;
                        unpack_f32x2(ta, x0, x1);
                        const float p0 = ex2(x0), p1 = ex2(x1);
                        if (kPtExpPolyMask & (1 << ((i >> 1) & 3))) {
                            ex2_poly_x2(tb, p2, p3);
                        } else {
                            float x2, x3;
                            unpack_f32x2(tb, x2, x3);
                            p2 = ex2(x2);
                            p3 = ex2(x3);
                        }
                        sum_a = add_f32x2(sum_a, pack_f32x2(p0, p1));
                        sum_b = add_f32x2(sum_b, pack_f32x2(p2, p3));
                        pk[i] = pt_pack<HALF>(p0, p1);
                        pk[i + 1] = pt_pack<HALF>(p2, p3);
                    }
                    if (any_cut) {
                        // the polynomial gives 2^-125 for a hidden key, which a large value there would show: exactly zero instead
                        const int lo = min(max(vs - key0 - cidx * 32, 0), 32), hi = min(max(ve - key0 - cidx * 32, 0), 32);
                        const uint32_t seen = hi > lo ? (0xffffffffu >> (32 - (hi - lo))) << lo : 0u;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            pk[i] &= ((seen >> (2 * i)) & 1u ? 0xffffu : 0u) | ((seen >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
                    }
                    tmem_st16(tS + cidx * 16, pk);
                    if (cidx == 1) {
                        tmem_wait_st();
                        fence_before_sync();
                        mbar_arrive(p_half(t, 0));
                    }
                }
                {
                    float s0, s1;
                    unpack_f32x2(add_f32x2(sum_a, sum_b), s0, s1);
                    l += s0 + s1;
                }
                tmem_wait_st();
                fence_before_sync();
                mbar_arrive(p_half(t, 1));
            }
            if (!ok) break;
            cs += n_t;
            if (!(ok = paged_wait(o_final(t), it & 1, abortp))) break;
            fence_after_sync();
            if (odd || m_used == INFINITY) l = NAN;  // a score of +inf, whose weight the polynomial would also make 0
            const bool split = w.part >= 0;
            if (m_used == -INFINITY && l == l) l = split ? 0.0f : NAN;  // only scores of -inf: no softmax; a piece without weight
            float* state = p.part + (int64_t)(split ? w.part + w.split : 0) * kPtState<D>;
            if (split) __stcg(reinterpret_cast<float2*>(state + 256 * D) + t * 128 + row, make_float2(n_t > 0 ? m_used : -INFINITY, n_t > 0 ? l : 0.0f));
            bool bad = false;
            if (n_t > 0) {
                // rows leave through a per-warp staging area of 32 rows x 128 bytes, 16-byte pieces XORed by the row, and are
                // stored as whole 128-byte lines: 64 bf16 columns at a time, or 32 columns of a piece's f32 state
                const float inv = (HALF ? 1.0f / kReadVScale : 1.0f) / l;
                const uint32_t stage = sOut + (uint32_t)warp * 4096u;
                const int sub_row = lane >> 3, piece = lane & 7;
                const int64_t my_at = valid ? (w.tok0 + tok) * a.o_stride + (int64_t)(w.kvh * a.G + head) * D : -1;
#pragma unroll 1
                for (int cidx = 0; cidx < D / 32; ++cidx) {
                    uint32_t orow[32];
                    tmem_ld32(tO + cidx * 32, orow);
                    tmem_wait_ld();
                    if (split) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128u + (uint32_t)(((i >> 2) ^ (lane & 7)) << 4)),
                                         "r"(orow[i]), "r"(orow[i + 1]), "r"(orow[i + 2]), "r"(orow[i + 3]) : "memory");
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t h[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const float x = __uint_as_float(orow[i + 2 * q]) * inv, y = __uint_as_float(orow[i + 2 * q + 1]) * inv;
                                bad |= !isfinite(x) | !isfinite(y);
                                h[q] = pack_bf16x2(x, y);
                            }
                            const int pc = (cidx & 1) * 4 + (i >> 3);
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128u + (uint32_t)((pc ^ (lane & 7)) << 4)), "r"(h[0]),
                                         "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                        }
                        if (!(cidx & 1)) continue;
                    }
                    __syncwarp();
#pragma unroll
                    for (int k4 = 0; k4 < 8; ++k4) {
                        const int rr = k4 * 4 + sub_row;
                        uint4 x;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                     : "r"(stage + rr * 128u + (uint32_t)((piece ^ (rr & 7)) << 4)));
                        const int64_t at = __shfl_sync(0xffffffffu, my_at, rr);
                        if (at < 0) continue;
                        if (split)
                            __stcg(reinterpret_cast<uint4*>(state + (int64_t)(t * 128 + (warp & 3) * 32 + rr) * D + cidx * 32 + piece * 4), x);
                        else
                            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + at + (cidx >> 1) * 64 + piece * 8) = x;
                    }
                    __syncwarp();
                }
                fence_before_sync();
            }
            mbar_arrive(o_free(t));
            unsigned again = __ballot_sync(0xffffffffu, bad && valid && (HALF || l == l));
            while (again) {
                const int rr = __ffs(again) - 1;
                again &= again - 1;
                const int tk = __shfl_sync(0xffffffffu, tok, rr), hd = __shfl_sync(0xffffffffu, head, rr);
                paged_row_again<D, HALF ? kKvQ8Head : KV_BF16, false>(a, w, w.kvh, tk * a.G + hd, lane, &s_flags[1]);
            }
        }
    }

    // ---------------- common tail ----------------
    if (s_abort) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // let copies in flight land
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == 9) tmem_dealloc(tmem, 512);
    if (tid == 0) {
        if (p.behind) grid_wait();
        if (s_abort && a.err) atomicExch(a.err, 1);
        // the last CTA to leave rewinds the work counter for the next launch
        __threadfence();
        if (atomicAdd(p.sched + 1, 1) == (int)gridDim.x - 1) {
            p.sched[0] = 0;
            p.sched[1] = 0;
            __threadfence();
        }
    }
}

// Weighs the pieces of every cut item, in the order of their keys. L lanes share a row, 16 bytes of each piece apiece (head_dim
// 256: twice), so that a row costs two round trips: the pieces' (m, l), then their rows. The list holds the first piece of each
// item; ROWS: of an item (two query tiles, at head_dim 256 one).
template <int D>
__global__ void __launch_bounds__(256) paged_tc_merge_kernel(const __grid_constant__ PagedTcArgs p) {
    grid_wait();
    const PagedAttnArgs& a = p.a;
    constexpr int ROWS = D == 256 ? 128 : 256, STATE = ROWS * (D + 2);
    constexpr int L = D == 64 ? 16 : 32, V = D / (4 * L), PER = 256 / L;  // lanes of a row, 16-byte pieces of a lane, rows of a CTA
    const int lane = threadIdx.x & 31, sub = threadIdx.x % L;
    const int n = a.plan.counts[0] * ROWS;
    for (int i = blockIdx.x * PER + threadIdx.x / L; i < n; i += gridDim.x * PER) {
        const PagedItem& w = a.plan.items[i / ROWS];
        const int r = i % ROWS, t = r >> 7, tile_tok = (r & 127) / a.G, head = (r & 127) - tile_tok * a.G;
        const int tok = w.row0 + t * p.tiles_tokens + tile_tok;
        const bool valid = tile_tok < p.tiles_tokens && tok < w.n_tok;
        const float* state = p.part + (int64_t)w.part * STATE;
        // pieces in groups of L: a lane holds (m, l) of one, then its weight
        float top = -INFINITY, l = 0.0f;
        float4 o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const int n_split = w.n_split;
        for (int s0 = 0; s0 < n_split; s0 += L) {
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (valid && s0 + sub < n_split) ml = __ldcg(reinterpret_cast<const float2*>(state + (int64_t)(s0 + sub) * STATE + ROWS * D) + r);
            float m = ml.x;
#pragma unroll
            for (int k = L / 2; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
            const float now = fmaxf(top, m), back = top == -INFINITY ? 0.0f : tc::ex2((top - now) * a.c);
            top = now;
            l *= back;
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] = make_float4(o[v].x * back, o[v].y * back, o[v].z * back, o[v].w * back);
            // (nothing seen, and so no rows left: weight 0; a NaN stays one)
            const bool none = ml.x == -INFINITY && ml.y == 0.0f;
            const float f = none ? 0.0f : tc::ex2((ml.x - now) * a.c);
            const int here = min(L, n_split - s0);
#pragma unroll 4
            for (int s = 0; s < here; ++s) {
                const int from = (lane & ~(L - 1)) + s;
                const float fs = __shfl_sync(0xffffffffu, f, from), ls = __shfl_sync(0xffffffffu, ml.y, from);
                const int skip = __shfl_sync(0xffffffffu, none ? 1 : 0, from);  // (by all lanes: head_dim 64 has two rows in a warp)
                if (!valid || skip) continue;
                l = fmaf(fs, ls, l);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float4 x = __ldcg(reinterpret_cast<const float4*>(state + (int64_t)(s0 + s) * STATE + (int64_t)r * D) + v * L + sub);
                    o[v].x = fmaf(fs, x.x, o[v].x);
                    o[v].y = fmaf(fs, x.y, o[v].y);
                    o[v].z = fmaf(fs, x.z, o[v].z);
                    o[v].w = fmaf(fs, x.w, o[v].w);
                }
            }
        }
        const float inv = p.out_scale / l;
        bool bad = false;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            o[v] = make_float4(o[v].x * inv, o[v].y * inv, o[v].z * inv, o[v].w * inv);
            bad |= valid && !finite4(o[v]) && (p.out_scale != 1.0f || l == l);
            if (valid) paged_store4<false>(a, (w.tok0 + tok) * a.o_stride + (int64_t)(w.kvh * a.G + head) * D + (v * L + sub) * 4, o[v]);
        }
        unsigned again = __ballot_sync(0xffffffffu, bad);
        while (again) {
            const int from = __ffs(again) - 1;
            again &= ~((L == 32 ? 0xffffffffu : ((1u << L) - 1)) << (from & ~(L - 1)));
            __syncwarp();
            const int row = __shfl_sync(0xffffffffu, tok * a.G + head, from);
            if (p.out_scale != 1.0f)  // f16 rows: 8-bit pages
                paged_row_again<D, kKvQ8Head, false>(a, w, w.kvh, row, lane);
            else
                paged_row_again<D, KV_BF16, false>(a, w, w.kvh, row, lane);
        }
    }
}

}  // namespace ggr
