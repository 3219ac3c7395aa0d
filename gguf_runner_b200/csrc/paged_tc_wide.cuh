// Attention of chunks and packed prompts in bf16 on the 5th-generation tensor cores at head_dim 256, where the output of one
// 128-row query tile takes half of tensor memory: the pipeline of prefill_tc_wide.cuh (64-key tiles, two score buffers, Q in
// tensor memory as the A operand), with the items, gathered key tiles, cleared values, pieces and row-by-row repair of
// paged_tc.cuh. A CTA takes one item: 128 / G tokens times the G query heads of a KV head, and a stretch of keys. Its start
// (Q into tensor memory) and its end (rows out of it) are not hidden behind another item's tiles; they are what a short
// window leaves as the bound.
#pragma once

#include "paged_tc.cuh"

namespace ggr {

constexpr int kPwThreads = 256, kPwBN = 64, kPwStages = 3, kPwD = 256;
constexpr int kPwState = 128 * (kPwD + 2);
constexpr uint32_t kPwTail = 2048;  // room past the last stage for the row pitch of the staged Q tile
constexpr size_t kPwSmem = (size_t)(kPwD / 64) * (2 * kPwStages * kPwBN * 128) + kPwTail + 1024;

template <bool HALF>
__global__ void __launch_bounds__(kPwThreads, 1)
paged_tc_wide_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedTcArgs p) {
    using namespace tc;
    constexpr int D = kPwD, NBLK = D / 64, NST = kPwStages;
    constexpr uint32_t KBLK = kPwBN * 128, KV_BYTES = NBLK * KBLK, STAGE = 2 * KV_BYTES, O_COL0 = 128, Q_COL0 = O_COL0 + D;

    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bars[24];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;

    const PagedAttnArgs& a = p.a;
    if ((int)blockIdx.x >= a.plan.counts[0]) return;  // (a captured launch has CTAs for the longest plan, and is not chained)
    const PagedItem w = a.plan.items[blockIdx.x];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sK = smem_base, sV = smem_base + KV_BYTES;
    // staged rows are pitched 16 bytes past a multiple of 128: the eight rows of a quarter warp then hit all banks
    constexpr uint32_t Q_PITCH = D * 2 + 16, O_PITCH = D * 4 + 16;
    const uint32_t sQst = smem_base + (NST - 1) * STAGE;
    static_assert(128 * Q_PITCH <= STAGE + kPwTail && 128 * O_PITCH <= NST * STAGE, "staged rows");

    const uint32_t bar0 = smem_u32(bars), q_full = bar0;
    auto k_full = [&](int s) { return bar0 + 8u * (1 + s); };
    auto k_empty = [&](int s) { return bar0 + 8u * (4 + s); };
    auto v_full = [&](int s) { return bar0 + 8u * (7 + s); };
    auto v_empty = [&](int s) { return bar0 + 8u * (10 + s); };
    auto s_full = [&](int b) { return bar0 + 8u * (13 + b); };
    auto p_half = [&](int buf, int half) { return bar0 + 8u * (15 + 2 * buf + half); };
    auto pv_done = [&](int buf) { return bar0 + 8u * (19 + buf); };
    const uint32_t o_final = bar0 + 8u * 21, q_staged = bar0 + 8u * 22, raw = bar0 + 8u * 23;

    const int n_tok = min(p.tiles_tokens, w.n_tok - w.row0), n_rows = n_tok * a.G;
    const int any_lo = paged_first_key(w.pos0 + w.row0, a.window), any_hi = w.pos0 + w.row0 + n_tok;  // seen by some row
    const int lo = max(w.key0, any_lo) / kPwBN, hi = (min(w.key1, any_hi) + kPwBN - 1) / kPwBN;

    if (tid == 0) {
        s_abort = 0;
        mbar_init(q_full, 128);
        for (int s = 0; s < NST; ++s) {
            mbar_init(k_full(s), 1);
            mbar_init(k_empty(s), 1);
            mbar_init(v_full(s), 1);
            mbar_init(v_empty(s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(s_full(s), 1);
            mbar_init(p_half(s, 0), 128);
            mbar_init(p_half(s, 1), 128);
            mbar_init(pv_done(s), 1);
        }
        mbar_init(o_final, 1);
        mbar_init(q_staged, 1);
        mbar_init(raw, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {
        tmem_alloc(smem_u32(&s_tmem_base), 512);
        tmem_relinquish();
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = s_tmem_base;
    volatile int* abortp = &s_abort;
    if (!p.behind) grid_wait();

    if (warp == 4) {
        // ---------------- TMA producer: the whole warp, a lane per copy ----------------
        const int boxes = p.linear ? 1 : kPwBN / p.box_rows, copies = boxes * NBLK;
        const int box = lane / NBLK, blk = lane % NBLK, box_key = p.linear ? 0 : box * p.box_rows;
        const uint32_t box_at = blk * KBLK + box_key * 128, box_bytes = p.linear ? KBLK : p.box_rows * 128;
        const int page_log2 = a.pages.page_log2, kv_end = w.pos0 + w.n_tok;
        auto page_of = [&](int j) {
            const int key = j * kPwBN + box_key;
            return !p.linear && lane < copies && key < kv_end && j < hi ? a.plan.table[w.src + (key >> page_log2)] : 0;
        };
        int page = page_of(lo), s = 0;
        uint32_t ph = 1, raws = 0;
        for (int j = lo; j < hi; ++j) {
            const int key = j * kPwBN + box_key;
            const bool mine = lane < copies && (p.linear || key < kv_end);
            const uint32_t bytes = box_bytes * __popc(__ballot_sync(0xffffffffu, mine));
            const int y = p.linear ? w.kvh : key & ((1 << page_log2) - 1);
            const int z = p.linear ? w.lin + key : (a.layer * a.pages.n_pages + page) * a.pages.Hkv + w.kvh;
            page = page_of(j + 1);
            // the last stage holds the staged Q rows until they are in tensor memory
            if (j - lo == NST - 1 && !mbar_wait_warp(q_full, 0, abortp)) break;
            if (!mbar_wait_warp(k_empty(s), ph, abortp)) break;
            if (lane == 0) mbar_expect_tx(k_full(s), bytes);
            __syncwarp();
            if (mine) tma_load_3d(sK + s * STAGE + box_at, &tmK, blk * 64, y, z, k_full(s));
            if (!mbar_wait_warp(v_empty(s), ph, abortp)) break;
            const bool edge = j * kPwBN < any_lo || (j + 1) * kPwBN > any_hi;
            const uint32_t vbar = edge ? raw : v_full(s);
            if (lane == 0) mbar_expect_tx(vbar, bytes);
            __syncwarp();
            if (mine) tma_load_3d(sV + s * STAGE + box_at, &tmV, blk * 64, y, z, vbar);
            if (edge) {
                if (!mbar_wait_warp(raw, raws & 1u, abortp)) break;
                ++raws;
                for (int i = lane; i < kPwBN * NBLK * 8; i += 32) {
                    const int row = (i >> 3) & (kPwBN - 1), k = j * kPwBN + row;
                    if (k >= any_lo && k < any_hi) continue;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sV + s * STAGE + (i / (kPwBN * 8)) * KBLK + row * 128 + (i & 7) * 16), "r"(0u)
                                 : "memory");
                }
                fence_smem_to_async_proxy();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full(s));
            }
            if (++s == NST) s = 0, ph ^= 1u;
        }
    } else if (warp == 5) {
        // ---------------- MMA issuer ----------------
        if (hi > lo) {
            constexpr uint32_t TYPES = (1u << 7) | (1u << 10);
            constexpr uint32_t IDESC_QK = idesc_bf16(kPwBN, 0) & ~(HALF ? TYPES : 0u), IDESC_PV = idesc_bf16(D, 1) & ~(HALF ? TYPES : 0u);
            const uint64_t dK = smem_desc(sK, 16, 1024), dV = smem_desc(sV, KBLK, 1024);
            const uint32_t tm = __shfl_sync(0xffffffffu, s_tmem_base, 0);
            auto issue_qk = [&](int buf, int s) {
                const uint64_t b0 = dK + (uint64_t)((s * STAGE) >> 4);
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    mma_ts_e(tm + buf * kPwBN, tm + Q_COL0 + ks * 8, b0 + (uint64_t)(((ks >> 2) * KBLK + (ks & 3) * 32) >> 4), IDESC_QK, ks > 0 ? 1u : 0u);
            };
            auto issue_pv_half = [&](int buf, int s, int half, bool accumulate) {
                const uint64_t b0 = dV + (uint64_t)((s * STAGE) >> 4);
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const int ks = half * 2 + kk;
                    mma_ts_e(tm + O_COL0, tm + buf * kPwBN + ks * 8, b0 + (uint64_t)((ks * 16 * 128) >> 4), IDESC_PV, (accumulate || ks > 0) ? 1u : 0u);
                }
            };
            const int tiles = __shfl_sync(0xffffffffu, hi - lo, 0);
            bool ok = mbar_wait_warp(q_full, 0, abortp);
            if (ok) ok = mbar_wait_warp(k_full(0), 0, abortp);
            if (ok) {
                fence_after_sync();
                issue_qk(0, 0);
                mma_commit_e(s_full(0));
                mma_commit_e(k_empty(0));
            }
            int s = 0;
            uint32_t ring_ph = 0;
            for (int n = 0; ok && n < tiles; ++n) {
                const int s1 = s + 1 == NST ? 0 : s + 1;
                const uint32_t ring_ph1 = s + 1 == NST ? ring_ph ^ 1u : ring_ph;
                if (n + 1 < tiles) {
                    if (!(ok = mbar_wait_warp(k_full(s1), ring_ph1, abortp))) break;
                    fence_after_sync();
                    issue_qk((n + 1) & 1, s1);
                    mma_commit_e(s_full((n + 1) & 1));
                    mma_commit_e(k_empty(s1));
                }
                if (!(ok = mbar_wait_warp(v_full(s), ring_ph, abortp))) break;
                if (!(ok = mbar_wait_warp(p_half(n & 1, 0), (n >> 1) & 1, abortp))) break;
                fence_after_sync();
                issue_pv_half(n & 1, s, 0, n > 0);
                if (!(ok = mbar_wait_warp(p_half(n & 1, 1), (n >> 1) & 1, abortp))) break;
                fence_after_sync();
                issue_pv_half(n & 1, s, 1, true);
                mma_commit_e(pv_done(n & 1));
                mma_commit_e(v_empty(s));
                if (n == tiles - 1) mma_commit_e(o_final);
                s = s1;
                ring_ph = ring_ph1;
            }
        }
    } else if (warp < 4) {
        // ---------------- softmax: one thread per query row ----------------
        const int row = warp * 32 + lane, tok = row / a.G, head = row - tok * a.G;
        const bool valid = row < n_rows;
        int vs = 0, ve = 0x7fffffff;  // (rows that stand for no token see everything: see paged_tc.cuh)
        if (valid) {
            ve = w.pos0 + w.row0 + tok + 1;
            vs = paged_first_key(ve - 1, a.window);
        }
        const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
        const uint32_t tO = tmem + lane_addr + O_COL0;
        const float c = a.c, thr = 8.0f / c;
        float m_used = -INFINITY, l = 0.0f;
        bool odd = false;
        bool ok = true;
        const int64_t tok_row = w.tok0 + w.row0 + tok;
        if (hi > lo) {
            // the query row goes to tensor memory as the A operand: it comes in as one bulk copy, the thread reads it back
            if (tid == 0) mbar_expect_tx(q_staged, (uint32_t)n_rows * (uint32_t)(D * 2));
            if (valid)
                bulk_load(sQst + row * Q_PITCH, static_cast<const uint16_t*>(p.q_rows) + tok_row * p.q_rows_stride + (int64_t)(w.kvh * a.G + head) * D, D * 2, q_staged);
            ok = mbar_wait(q_staged, 0, abortp);
#pragma unroll 1
            for (int cidx = 0; ok && cidx < D / 64; ++cidx) {
                uint32_t qr[32];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint4 v4 = make_uint4(0u, 0u, 0u, 0u);
                    if (valid)
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v4.x), "=r"(v4.y), "=r"(v4.z), "=r"(v4.w)
                                     : "r"(sQst + row * Q_PITCH + (uint32_t)(cidx * 8 + i) * 16u));
                    qr[4 * i] = v4.x, qr[4 * i + 1] = v4.y, qr[4 * i + 2] = v4.z, qr[4 * i + 3] = v4.w;
                }
                tmem_st32(tmem + lane_addr + Q_COL0 + cidx * 32, qr);
            }
            tmem_wait_st();
            fence_before_sync();
            if (ok) mbar_arrive(q_full);
        }
        for (int j = lo; ok && j < hi; ++j) {
            const int n = j - lo, buf = n & 1;
            const uint32_t tS = tmem + lane_addr + buf * kPwBN;
            if (!(ok = mbar_wait(s_full(buf), (n >> 1) & 1, abortp))) break;
            fence_after_sync();
            uint32_t sr[2][32];
            tmem_ld32(tS, sr[0]);
            tmem_ld32(tS + 32, sr[1]);
            tmem_wait_ld();
            const int key0 = j * kPwBN;
            const bool cut = key0 < vs || key0 + kPwBN > ve, any_cut = __any_sync(0xffffffffu, cut);
            if (cut) {
#pragma unroll
                for (int cidx = 0; cidx < 2; ++cidx)
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int key = key0 + cidx * 32 + i;
                        if (key < vs || key >= ve) sr[cidx][i] = 0xff800000u;  // -inf
                    }
            }
            float mxa = -INFINITY, mxb = -INFINITY, mxc = -INFINITY, mxd = -INFINITY;
#pragma unroll
            for (int cidx = 0; cidx < 2; ++cidx)
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    mxa = max3_nan(mxa, __uint_as_float(sr[cidx][i]), __uint_as_float(sr[cidx][i + 1]));
                    mxb = max3_nan(mxb, __uint_as_float(sr[cidx][i + 2]), __uint_as_float(sr[cidx][i + 3]));
                    mxc = max3_nan(mxc, __uint_as_float(sr[cidx][i + 4]), __uint_as_float(sr[cidx][i + 5]));
                    mxd = max3_nan(mxd, __uint_as_float(sr[cidx][i + 6]), __uint_as_float(sr[cidx][i + 7]));
                }
            const float mx = max3_nan(max3_nan(mxa, mxb, mxc), mxd, mxd);
            // (a NaN score: see paged_tc.cuh)
            odd |= mx != mx;
            const bool need = mx > m_used + thr;
            float alpha = 1.0f;
            if (need) {
                alpha = ex2((m_used - mx) * c);
                m_used = mx;
            }
            // O must be quiet before it is rescaled: P V of the step before was issued behind this step's Q K^T
            const bool rescale_now = n > 0 && __any_sync(0xffffffffu, need);
            if (rescale_now) {
                if (!(ok = mbar_wait(pv_done((n - 1) & 1), ((n - 1) >> 1) & 1, abortp))) break;
                fence_after_sync();
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
            for (int cidx = 0; cidx < 2; ++cidx) {
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
                if (any_cut) {  // (hidden keys exactly zero: see paged_tc.cuh)
                    const int s_lo = min(max(vs - key0 - cidx * 32, 0), 32), s_hi = min(max(ve - key0 - cidx * 32, 0), 32);
                    const uint32_t seen = s_hi > s_lo ? (0xffffffffu >> (32 - (s_hi - s_lo))) << s_lo : 0u;
#pragma unroll
                    for (int i = 0; i < 16; ++i) pk[i] &= ((seen >> (2 * i)) & 1u ? 0xffffu : 0u) | ((seen >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
                }
                tmem_st16(tS + cidx * 16, pk);
                if (cidx == 0) {
                    tmem_wait_st();
                    fence_before_sync();
                    mbar_arrive(p_half(buf, 0));
                }
            }
            {
                float s0, s1;
                unpack_f32x2(add_f32x2(sum_a, sum_b), s0, s1);
                l += s0 + s1;
            }
            tmem_wait_st();
            fence_before_sync();
            mbar_arrive(p_half(buf, 1));
            if (n > 0 && !rescale_now && !(ok = mbar_wait(pv_done((n - 1) & 1), ((n - 1) >> 1) & 1, abortp))) break;
        }
        if (ok && hi > lo) ok = mbar_wait(o_final, 0, abortp);
        if (odd || m_used == INFINITY) l = NAN;  // (see paged_tc.cuh)
        const bool split = w.part >= 0;
        if (m_used == -INFINITY && l == l) l = split ? 0.0f : NAN;
        float* state = p.part + (int64_t)(split ? w.part + w.split : 0) * kPwState;
        if (ok && split && valid) __stcg(reinterpret_cast<float2*>(state + 128 * D) + row, make_float2(hi > lo ? m_used : -INFINITY, hi > lo ? l : 0.0f));
        bool bad = false;
        if (ok && hi > lo) {
            fence_after_sync();
            // every load into the stages has landed and every MMA that read them has completed: the thread lays its row down
            // there and sends it out as one bulk copy
            const float inv = (HALF ? 1.0f / kReadVScale : 1.0f) / l;
            const uint32_t sOrow = smem_base + row * O_PITCH;
#pragma unroll 1
            for (int cidx = 0; cidx < D / 32; ++cidx) {
                uint32_t orow[32];
                tmem_ld32(tO + cidx * 32, orow);
                tmem_wait_ld();
                if (split) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sOrow + (uint32_t)(cidx * 32 + i) * 4u), "r"(orow[i]), "r"(orow[i + 1]),
                                     "r"(orow[i + 2]), "r"(orow[i + 3]) : "memory");
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
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sOrow + (uint32_t)(cidx * 32 + i) * 2u), "r"(h[0]), "r"(h[1]), "r"(h[2]),
                                     "r"(h[3]) : "memory");
                    }
                }
            }
            if (valid) {
                fence_smem_to_async_proxy();
                if (split)
                    bulk_store(state + row * D, sOrow, D * 4);
                else
                    bulk_store(static_cast<__nv_bfloat16*>(a.out) + tok_row * a.o_stride + (int64_t)(w.kvh * a.G + head) * D, sOrow, D * 2);
                bulk_store_commit_and_wait();
            }
            __syncwarp();
            unsigned again = __ballot_sync(0xffffffffu, bad && valid && (HALF || l == l));
            while (again) {
                const int rr = __ffs(again) - 1;
                again &= again - 1;
                paged_row_again<D, HALF ? kKvQ8Head : KV_BF16, false>(a, w, w.kvh, w.row0 * a.G + warp * 32 + rr, lane);
            }
        }
    }

    if (s_abort) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // let copies in flight land
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == 5) tmem_dealloc(tmem, 512);
    if (tid == 0) {
        if (p.behind) grid_wait();
        if (s_abort && a.err) atomicExch(a.err, 1);
    }
}

}  // namespace ggr
