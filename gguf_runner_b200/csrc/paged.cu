// Paged KV cache, batch plans, and attention over pages and over packed prompts: the host side of
// include/ggr_attn.h's ggr_pages, ggr_batch, ggr_paged_* and ggr_packed_attention.
//
// A plan is made once per step (ggr_batch_set) and used by every layer: the lengths and page tables are cut on the host into
// work items of equal size, which the kernels read from device memory. Captured launches therefore follow the plan: a graph of
// a token step is replayed with the lengths that the last ggr_batch_set gave.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <functional>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../include/ggr_attn.h"
#include "batch_check.h"
#include "paged.cuh"
#include "paged_mma.cuh"
#include "paged_tc.cuh"
#include "paged_tc_wide.cuh"
#include "path_view.h"

using namespace ggr;

static_assert(kKvQ8Head == GGR_KV_Q8_HEAD, "page format");

struct ggr_pages {
    ggr_attn_ctx* ctx;
    int device, n_layers, page_size;
    PageView v{};
    void* owned[4] = {nullptr, nullptr, nullptr, nullptr};
    int users = 0;         // batch plans on the pool, which read it: the last of them gives a destroyed pool's memory back
    bool destroyed = false;
    CUtensorMap tmK16, tmV16;    // 16 rows of a page, one 64- or 128-byte block of columns
    CUtensorMap tmK128, tmV128;  // bf16: min(page_size, 128) rows (head_dim 256: at most 64)
};

namespace {

// Keys of a tile of the tcgen05 kernels, query tiles of an item
constexpr int tc_key_tile(int D) { return D == 256 ? kPwBN : 128; }
constexpr int tc_item_tiles(int D) { return D == 256 ? 1 : 2; }
constexpr int kMaxLists = 4;  // distinct windows of a model's layers
constexpr char kPagesGone[] = "the page pool of the batch plan has been destroyed";
// lists of a plan: items of the three attention kernels, and the pairs of query tiles whose pieces are merged
enum Kind { kSplitK = 0, kRows = 1, kTc = 2, kMerge = 3, kKinds = 4 };

struct Guard {
    int prev = -1;
    explicit Guard(int dev) {
        cudaGetDevice(&prev);
        if (prev != dev) cudaSetDevice(dev);
    }
    ~Guard() {
        int cur = -1;
        cudaGetDevice(&cur);
        if (prev >= 0 && cur != prev) cudaSetDevice(prev);
    }
};

#define PAGED_TRY(c, expr)                                                                              \
    do {                                                                                                \
        cudaError_t e_ = (expr);                                                                        \
        if (e_ != cudaSuccess)                                                                          \
            return path_fail(c, GGR_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_));      \
    } while (0)

int elem_bytes(int dtype) { return dtype == GGR_DTYPE_F32 ? 4 : 2; }

// dims (x: elements, y, z), strides in bytes of y and z; box (bx, by, bz); the block of columns decides the swizzle
bool make_map3(CUtensorMap* map, bool bytes, const void* base, uint64_t dx, uint64_t dy, uint64_t dz, uint64_t sy, uint64_t sz, uint32_t bx, uint32_t by,
               uint32_t bz) {
    PFN_tmapEncodeTiled enc = tmap_encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {dx, dy, dz}, strides[2] = {sy, sz};
    const cuuint32_t box[3] = {bx, by, bz}, estr[3] = {1, 1, 1};
    const uint32_t row = bx * (bytes ? 1 : 2);
    return enc(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

struct ggr_batch {
    ggr_attn_ctx* ctx;
    ggr_pages* pages;  // null: packed prompts
    int device, dtype, max_seqs, max_tokens, max_pages;
    int Hq, Hkv, D, G, sm_count, smem_optin, n_layers;
    std::vector<int> list_of;   // layer -> list
    std::vector<int> windows;   // list -> window
    size_t item_cap[kKinds] = {};
    size_t part_tiles = 0;      // partial states (of 16 rows, per KV head) that the scratch holds
    bool tc = false;            // the tcgen05 kernel takes this shape and dtype
    int tc_tokens = 0;          // tokens of one of its query tiles
    size_t tc_parts = 0;        // its partial states
    float* d_tc_part = nullptr;
    int* d_sched = nullptr;
    // 8-bit pages on their way to the tcgen05 kernel: dense f16 rows and which pages go there, q in f16
    __half* d_dense = nullptr;
    __half* d_q16 = nullptr;
    size_t dense_rows = 0;
    CUtensorMap tmKd, tmVd;
    size_t at_dense_entries = 0, at_dense_table = 0;
    int n_dense = 0;
    unsigned captured = 0;       // kinds of kernels that captured launches of this plan hold
    // device image of the plan: fixed places, so that captured launches keep their pointers
    unsigned char* d_plan = nullptr;
    unsigned char* h_plan[2] = {nullptr, nullptr};
    cudaEvent_t up[2] = {nullptr, nullptr};
    bool up_used[2] = {false, false};
    int turn = 0;
    size_t at_counts = 0, at_pos = 0, at_slot = 0, at_entries = 0, at_table = 0, at_items[kMaxLists][kKinds] = {}, bytes = 0;
    double* d_freqs = nullptr;  // RoPE frequencies in 64 bits: of ordinary layers, of window layers
    float* d_part = nullptr;
    unsigned* d_tickets = nullptr;
    __nv_bfloat16* d_planes = nullptr;  // packed f32 rows: [k, v][3 planes][max_tokens][Hkv * D]
    // the plan in force
    bool set = false;
    int n_seqs = 0, n_tokens = 0, n_entries = 0, n_rows = 0;
    int n_items[kMaxLists][kKinds] = {};
    std::vector<PagedItem> scratch;
    int rows_step = 128;

    const int* counts(int list, int kind) const { return reinterpret_cast<const int*>(d_plan + at_counts) + (list * kKinds + kind) * 4; }
    const int* dense_counts() const { return reinterpret_cast<const int*>(d_plan + at_counts) + windows.size() * kKinds * 4; }
    const int* table() const { return reinterpret_cast<const int*>(d_plan + at_table); }
    const PagedItem* items(int list, int kind) const { return reinterpret_cast<const PagedItem*>(d_plan + at_items[list][kind]); }
};

namespace {

// ---- planning --------------------------------------------------------------------------------------

struct Tile {
    int seq, row0, rows, key0, key1;
};

// Size of the pieces that row tiles are cut into along their keys, in 16-key tiles. One CTA per SM streams a piece at its
// share of the memory's rate and spends some microseconds on its start and its merge whatever its size, so pieces are made as
// large as still gives every SM one, or (ragged batches) several. Modelled for a handful of counts per SM, smallest time taken.
int choose_piece(const std::vector<Tile>& tiles, int Hkv, int slots, double tile_bytes, double sm_rate, int min_tiles, size_t max_pieces, int* longest_out) {
    int64_t total = 0;
    int longest = 1;
    for (const Tile& t : tiles) {
        const int n = (t.key1 - t.key0 + 15) / 16;
        total += n;
        longest = std::max(longest, n);
    }
    *longest_out = longest;
    int best = longest;
    double best_cost = -1.0;
    auto consider = [&](int piece) {
        piece = std::max(piece, std::max(min_tiles, (longest + kPagedSplitMax - 1) / kPagedSplitMax));
        piece = std::min(piece, longest);
        int64_t pieces = 0, cut = 0;
        for (const Tile& t : tiles) {
            const int n = (t.key1 - t.key0 + 15) / 16, k = (n + piece - 1) / piece;
            pieces += k;
            if (k > 1) cut += k;
        }
        if ((size_t)cut > max_pieces) return;
        const double ctas = (double)pieces * Hkv;
        const double rate = std::min(sm_rate, 6.6e12 / std::min(ctas, (double)slots));
        const double t0 = 3e-6, one = t0 + piece * tile_bytes / rate;
        double cost = ctas <= slots ? one : (total * Hkv * tile_bytes / rate + ctas * t0) / slots + 0.5 * one;
        if (cut) cost += 2.5e-6;
        if (best_cost < 0.0 || cost < best_cost) {
            best_cost = cost;
            best = piece;
        }
    };
    consider(longest);
    for (int w = 1; w <= 12; ++w) {
        // the smallest piece that gives at most w CTAs per SM
        int lo = 1, hi = longest;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            int64_t pieces = 0;
            for (const Tile& t : tiles) pieces += ((t.key1 - t.key0 + 15) / 16 + mid - 1) / mid;
            if (pieces * Hkv <= (int64_t)w * slots)
                hi = mid;
            else
                lo = mid + 1;
        }
        consider(lo);
        if (lo <= min_tiles) break;
    }
    return best;
}

// The same for the tcgen05 kernel. `tiles`: 128-key tiles of every pair of query tiles, longest first, of which each stands for Hkv
// items. Items are taken longest first by whichever SM is free, so that only the longest and the last ones matter: those
// above some length or after some whole wave are cut, so far that the SMs end together. A step over a tile takes 2.1 us, an item 3 us besides (its start, its
// epilogue; at head_dim 256 0.75 per 64-key tile and 6), a piece's rows one more, and the merge 4 and 0.03 per piece. Returns how many pairs stay whole; *piece: the size of the others' pieces.
int choose_tc_cut(const std::vector<int>& tiles, int Hkv, int sm_count, size_t max_pieces, bool wide, int* piece, double* cost_us) {
    const double t = wide ? 0.75 : 2.1, t0 = wide ? 6.0 : 3.0;
    const int n = (int)tiles.size();
    int best_whole = n;
    double best_cost = -1.0;
    std::vector<double> ends;
    std::vector<std::pair<int, int>> sizes;  // tiles of a piece, how many such (negative: cut)
    auto consider = [&](int whole, int size) {
        size_t cut = 0;
        for (int i = whole; i < n; ++i) cut += tiles[i] > size ? (size_t)(tiles[i] + size - 1) / size * Hkv : 0;
        if (cut > max_pieces) return;
        // pieces in the order they are taken in, onto a heap of the times at which the SMs are free
        sizes.clear();
        for (int i = 0; i < n; ++i) {
            const int k = i < whole ? 1 : (tiles[i] + size - 1) / size;
            sizes.emplace_back((tiles[i] + k - 1) / k, k * Hkv * (k > 1 ? -1 : 1));
        }
        std::stable_sort(sizes.begin(), sizes.end(), [](const auto& x, const auto& y) { return x.first > y.first; });
        ends.assign(sm_count, 0.0);
        double last = 0.0;
        for (const auto& s : sizes) {
            const double d = t0 + (s.second < 0 ? 1.0 : 0.0) + s.first * t;
            for (int k = std::abs(s.second); k > 0; --k) {
                std::pop_heap(ends.begin(), ends.end(), std::greater<double>());
                last = std::max(last, ends.back() += d);
                std::push_heap(ends.begin(), ends.end(), std::greater<double>());
            }
        }
        const double cost = last + (cut ? 4.0 + 0.03 * cut : 0.0);
        if (best_cost < 0.0 || cost < best_cost) {
            best_cost = cost;
            best_whole = whole;
            *piece = size;
        }
    };
    *piece = 1;
    *cost_us = 0.0;
    if (!n) return n;
    if ((int64_t)n * Hkv > 8 * sm_count) {  // many items: they even out by themselves
        double sum = 0.0;
        for (int x : tiles) sum += (t0 + x * t) * Hkv;
        *cost_us = sum / sm_count + 0.5 * (t0 + tiles[0] * t);
        return n;
    }
    consider(n, 1);
    // the longest ones, wherever they stand (ragged lengths)
    for (double f : {0.85, 0.7, 0.5, 0.34, 0.25, 0.17, 0.11, 0.07})
        if (tiles[0] * f >= 2.0) consider(0, (int)std::ceil(tiles[0] * f));
    // and the last wave of equal ones
    const int waves = (int)((int64_t)n * Hkv / sm_count);
    for (int w = waves; w >= std::max(1, waves - 1); --w) {
        const int whole = (int)((int64_t)w * sm_count / Hkv);
        if (whole >= n) continue;
        for (int k : {2, 3, 4, 6, 8, 12})
            if (tiles[whole] / k >= 2) consider(whole, (tiles[whole] + k - 1) / k);
    }
    *cost_us = best_cost;
    return best_whole;
}

int first_key(int pos, int window) { return window > 0 ? std::max(0, pos + 1 - window) : 0; }

// Which sequences leave the split-K kernel: those with more packed rows (new tokens times query heads of a KV head) than the
// result. It streams the keys once per 16 (f32: 8) rows, the others once per 128 or 256 but with fewer CTAs and a longer start,
// so the border depends on how many sequences there are and how long they are. Estimated for a few borders, smallest taken.
// Measured, us of the split-K kernel / the other one, 32/8 heads of 128, bf16, by rows: 1 sequence of 1000 keys, 256 rows: 11 / 18;
// 1 of 8000, 32: 15 / 30, 128: 32 / 30, 256: 49 / 33; 8 of 2000, 32: 17 / 32, 64: 33 / 32, 128: 64 / 34; 32 of 1000, 16: 30 / 43, 32: 54 /
// 43, 64: 94 / 43. f32: 1 of 8000, 256: 167 / 609; 8 of 2000, 64: 92 / 124, 128: 160 / 158; 32 of 1000, 16: 69 / 128, 64: 235 / 129.
// 8/4 heads of 256, bf16: 1 of 8000, 4: 18 / 23, 16: 36 / 24; 8 of 2000, 4: 18 / 16.
struct BatchShape {
    int D, G, Hkv, sm_count;
    bool tc, q8;
    int split_rows, rows_step, item_tokens, key_tile;  // rows of a tile of the warp-level kernels, tokens of an item and keys of a tile of tcgen05
    size_t max_pieces;
    double split_step_us;  // a 16-key tile of the split-K kernel, per SM
};
struct Work {
    int rows, keys;  // of a sequence: packed rows, keys that they walk
};
int choose_border(const std::vector<Work>& seqs, const BatchShape& s) {
    int borders[9], n_borders = 0;
    // whoever has at most one tile's rows stays, unless head_dim 256 has the tcgen05 kernel; long prompts go
    const int lo = s.tc && s.D == 256 ? 0 : (s.tc ? 16 : 8), hi = s.tc ? 256 : 4096;
    bool open = false;
    for (const Work& w : seqs) open |= w.rows > lo && w.rows <= hi;
    if (!open) return lo;
    borders[n_borders++] = lo;
    for (int b = lo ? 2 * lo : 8; b <= hi && n_borders < 8; b *= s.tc ? 2 : 3) borders[n_borders++] = b;
    borders[n_borders++] = hi;
    int best = lo;
    double best_cost = -1.0;
    std::vector<int> tiles;
    for (int k = 0; k < n_borders; ++k) {
        const int border = borders[k];
        double steps = 0.0, ctas = 0.0, items = 0.0, sum = 0.0, longest = 0.0, rows = 0.0, most = 0.0;
        tiles.clear();
        for (const Work& w : seqs) {
            if (w.rows == 0) continue;
            if (w.rows <= border) {
                const int n = (w.rows + s.split_rows - 1) / s.split_rows;
                steps += (double)n * ((w.keys + 15) / 16) * s.Hkv;
                ctas += (double)n * s.Hkv;
                most = std::max(most, std::min(16.0, (double)w.rows));
            } else if (s.tc) {
                const int per = s.item_tokens * s.G;
                for (int r = 0; r < w.rows; r += per) tiles.push_back((w.keys + s.key_tile - 1) / s.key_tile);
                rows += w.keys;
            } else {
                const int n = (w.rows + s.rows_step - 1) / s.rows_step;
                const double one = (double)((w.keys + 15) / 16) * (w.rows > s.rows_step / 2 ? 1.2 : 0.95) * s.D / 128;
                items += (double)n * s.Hkv;
                sum += n * one * s.Hkv;
                longest = std::max(longest, one);
            }
        }
        double cost = 0.0;
        if (ctas > 0.0) cost += 5.0 + (steps * s.split_step_us + std::max(ctas, (double)s.sm_count) * 4.5) / s.sm_count + (s.D == 256 ? 0.8 * most : 0.0);
        if (items > 0.0) cost += 8.0 + (items <= s.sm_count ? longest : sum / s.sm_count + 0.5 * longest);
        if (!tiles.empty()) {
            std::sort(tiles.begin(), tiles.end(), std::greater<int>());
            int piece;
            double tc;
            choose_tc_cut(tiles, s.Hkv, s.sm_count, s.max_pieces, s.D == 256, &piece, &tc);
            cost += tc + (s.D == 256 ? 0.0 : 4.0) + (s.q8 ? 5.0 + rows * s.Hkv * s.D * 1e-6 : 0.0);
        }
        if (best_cost < 0.0 || cost < best_cost) {
            best_cost = cost;
            best = border;
        }
    }
    return best;
}

}  // namespace

static int pages_create(ggr_attn_ctx* c, int32_t n_pages, int32_t page_size, int32_t kv_format, void* k, void* v, float* k_scale, float* v_scale,
                                ggr_pages** out) {
    if (!c) return GGR_ERR_INVALID;
    if (!out) return path_fail(c, GGR_ERR_INVALID, "null argument");
    *out = nullptr;
    const PathView p = path_view(c);
    if (n_pages <= 0) return path_fail(c, GGR_ERR_INVALID, "a page pool needs at least one page");
    if (page_size < kPageRowsMin || page_size > 256 || (page_size & (page_size - 1)))
        return path_fail(c, GGR_ERR_INVALID, "page_size must be 16, 32, 64, 128 or 256");
    if (kv_format != GGR_KV_BF16 && kv_format != GGR_KV_Q8_HEAD)
        return path_fail(c, GGR_ERR_UNSUPPORTED, "pages are built in GGR_KV_BF16 and GGR_KV_Q8_HEAD");
    if (p.D != 64 && p.D != 128 && p.D != 256) return path_fail(c, GGR_ERR_UNSUPPORTED, "pages are built for head_dim 64, 128 and 256");
    if (p.sharded) return path_fail(c, GGR_ERR_UNSUPPORTED, "a context that holds a shard of the positions has no pages");
    if ((int64_t)n_pages * page_size >= ((int64_t)1 << 31) || (int64_t)p.n_layers * n_pages * p.Hkv >= ((int64_t)1 << 31))
        return path_fail(c, GGR_ERR_RANGE, "the page pool has more rows than a 32-bit index names");
    const bool q8 = kv_format == GGR_KV_Q8_HEAD, given = k || v || k_scale || v_scale;
    if (given && (!k || !v || (q8 && (!k_scale || !v_scale)) || (!q8 && (k_scale || v_scale))))
        return path_fail(c, GGR_ERR_INVALID, "give all arrays of the page pool or none");
    for (const void* x : {(const void*)k, (const void*)v, (const void*)k_scale, (const void*)v_scale})
        if ((uintptr_t)x % 128) return path_fail(c, GGR_ERR_INVALID, "the arrays of a page pool must start on a 128-byte boundary");
    Guard guard(p.device);
    std::unique_ptr<ggr_pages> pg(new (std::nothrow) ggr_pages());
    if (!pg) return path_fail(c, GGR_ERR_ALLOC, "out of host memory");
    pg->ctx = c;
    pg->device = p.device;
    pg->n_layers = p.n_layers;
    pg->page_size = page_size;
    PageView& view = pg->v;
    view.fmt = kv_format;
    view.D = p.D;
    view.Hkv = p.Hkv;
    view.n_pages = n_pages;
    while ((1 << view.page_log2) < page_size) ++view.page_log2;
    const size_t rows = (size_t)p.n_layers * n_pages * p.Hkv * page_size, bytes = rows * p.D * (q8 ? 1 : 2);
    if (given) {
        view.k = static_cast<unsigned char*>(k);
        view.v = static_cast<unsigned char*>(v);
        view.ks = k_scale;
        view.vs = v_scale;
    } else {
        for (int i = 0; i < (q8 ? 4 : 2); ++i) {
            const size_t n = i < 2 ? bytes : rows * sizeof(float);
            if (cudaMalloc(&pg->owned[i], n) != cudaSuccess || cudaMemsetAsync(pg->owned[i], 0, n, p.stream) != cudaSuccess) {
                cudaGetLastError();
                for (void* x : pg->owned) cudaFree(x);
                return path_fail(c, GGR_ERR_ALLOC, "unable to allocate the page pool (" + std::to_string(2 * bytes) + " bytes)");
            }
        }
        view.k = static_cast<unsigned char*>(pg->owned[0]);
        view.v = static_cast<unsigned char*>(pg->owned[1]);
        view.ks = static_cast<float*>(pg->owned[2]);
        view.vs = static_cast<float*>(pg->owned[3]);
    }
    const uint64_t row_bytes = (uint64_t)p.D * (q8 ? 1 : 2), groups = (uint64_t)p.n_layers * n_pages * p.Hkv;
    const uint32_t box = (uint32_t)(row_bytes < 128 ? row_bytes : 128) / (q8 ? 1 : 2);
    for (int i = 0; i < 2; ++i)
        if (!make_map3(i ? &pg->tmV16 : &pg->tmK16, q8, i ? view.v : view.k, p.D, page_size, groups, row_bytes, row_bytes * page_size, box, 16, 1)) {
            for (void* x : pg->owned) cudaFree(x);
            return path_fail(c, GGR_ERR_CUDA, "cuTensorMapEncodeTiled failed for the page pool");
        }
    if (!q8)
        for (int i = 0; i < 2; ++i)
            if (!make_map3(i ? &pg->tmV128 : &pg->tmK128, false, i ? view.v : view.k, p.D, page_size, groups, row_bytes, row_bytes * page_size, 64,
                           std::min(page_size, tc_key_tile(p.D)), 1)) {
                for (void* x : pg->owned) cudaFree(x);
                return path_fail(c, GGR_ERR_CUDA, "cuTensorMapEncodeTiled failed for the page pool");
            }
    *out = pg.release();
    return GGR_OK;
}

static void pages_free(ggr_pages* pages) {
    Guard guard(pages->device);
    for (void* x : pages->owned) cudaFree(x);  // (cudaFree waits for the work that uses it)
    delete pages;
}

extern "C" void ggr_pages_destroy(ggr_pages* pages) {
    if (!pages || pages->destroyed) return;
    pages->destroyed = true;
    if (!pages->users) pages_free(pages);
}

extern "C" int ggr_pages_device_ptrs(const ggr_pages* pages, void** k, void** v, float** k_scale, float** v_scale, uint64_t* array_bytes) {
    if (!pages) return GGR_ERR_INVALID;
    if (k) *k = pages->v.k;
    if (v) *v = pages->v.v;
    if (k_scale) *k_scale = pages->v.ks;
    if (v_scale) *v_scale = pages->v.vs;
    if (array_bytes)
        *array_bytes = (uint64_t)pages->n_layers * pages->v.n_pages * pages->v.Hkv * pages->page_size * pages->v.D * (pages->v.fmt == GGR_KV_Q8_HEAD ? 1 : 2);
    return GGR_OK;
}

extern "C" void ggr_batch_destroy(ggr_batch* b) {
    if (!b) return;
    Guard guard(b->device);
    for (int i = 0; i < 2; ++i) {
        if (b->up_used[i]) cudaEventSynchronize(b->up[i]);
        if (b->up[i]) cudaEventDestroy(b->up[i]);
        if (b->h_plan[i]) cudaFreeHost(b->h_plan[i]);
    }
    cudaFree(b->d_plan);
    cudaFree(b->d_freqs);
    cudaFree(b->d_part);
    cudaFree(b->d_tickets);
    cudaFree(b->d_planes);
    cudaFree(b->d_tc_part);
    cudaFree(b->d_sched);
    cudaFree(b->d_dense);
    cudaFree(b->d_q16);
    if (b->pages && --b->pages->users == 0 && b->pages->destroyed) pages_free(b->pages);
    delete b;
}

static int batch_create(ggr_attn_ctx* c, ggr_pages* pages, int32_t dtype, int32_t max_seqs, int32_t max_tokens, int32_t max_pages, ggr_batch** out) {
    if (!c) return GGR_ERR_INVALID;
    if (!out) return path_fail(c, GGR_ERR_INVALID, "null argument");
    *out = nullptr;
    const PathView p = path_view(c);
    if (pages && pages->ctx != c) return path_fail(c, GGR_ERR_INVALID, "the pages belong to another context");
    if (pages && pages->destroyed) return path_fail(c, GGR_ERR_INVALID, kPagesGone);
    if (dtype != GGR_DTYPE_F32 && dtype != GGR_DTYPE_BF16) return path_fail(c, GGR_ERR_INVALID, "unknown dtype");
    if (max_seqs <= 0 || max_tokens <= 0 || max_pages < (pages ? 1 : 0)) return path_fail(c, GGR_ERR_INVALID, "a batch plan needs room for a sequence, a token and a page");
    if (p.D != 64 && p.D != 128 && p.D != 256) return path_fail(c, GGR_ERR_UNSUPPORTED, "batch plans are built for head_dim 64, 128 and 256");
    if (p.sharded) return path_fail(c, GGR_ERR_UNSUPPORTED, "a context that holds a shard of the positions has no batch plans");
    if ((int64_t)max_tokens * p.G >= ((int64_t)1 << 31)) return path_fail(c, GGR_ERR_RANGE, "max_tokens is out of range");
    Guard guard(p.device);
    std::unique_ptr<ggr_batch, void (*)(ggr_batch*)> b(new (std::nothrow) ggr_batch(), ggr_batch_destroy);
    if (!b) return path_fail(c, GGR_ERR_ALLOC, "out of host memory");
    b->ctx = c;
    b->pages = pages;
    if (pages) ++pages->users;
    b->device = p.device;
    b->dtype = dtype;
    b->max_seqs = max_seqs;
    b->max_tokens = max_tokens;
    b->max_pages = max_pages;
    b->Hq = p.Hq;
    b->Hkv = p.Hkv;
    b->D = p.D;
    b->G = p.G;
    b->sm_count = p.sm_count;
    b->smem_optin = p.smem_optin;
    b->n_layers = p.n_layers;
    for (int l = 0; l < p.n_layers; ++l) {
        const int w = p.windows->empty() ? 0 : (*p.windows)[l];
        size_t i = 0;
        while (i < b->windows.size() && b->windows[i] != w) ++i;
        if (i == b->windows.size()) b->windows.push_back(w);
        b->list_of.push_back((int)i);
    }
    if (b->windows.size() > kMaxLists) return path_fail(c, GGR_ERR_UNSUPPORTED, "more than four distinct windows");
    // items: row tiles of the longest plan, and the pieces that cutting them may add
    const size_t rows = (size_t)max_tokens * p.G, lists = b->windows.size();
    b->part_tiles = (size_t)(8 * p.sm_count + p.Hkv - 1) / p.Hkv + 16;
    const size_t step = dtype == GGR_DTYPE_F32 ? 8 : 16;
    b->rows_step = dtype == GGR_DTYPE_F32 && p.D == 256 ? 64 : 128;
    b->item_cap[kSplitK] = (rows + step - 1) / step + max_seqs + b->part_tiles;
    b->item_cap[kRows] = (rows + b->rows_step - 1) / b->rows_step + max_seqs;
    b->tc = dtype == GGR_DTYPE_BF16 && p.G <= 128;
    if (b->tc) {
        b->tc_tokens = 128 / p.G;
        const size_t item_tokens = tc_item_tiles(p.D) * b->tc_tokens, pairs = (((size_t)max_tokens + item_tokens - 1) / item_tokens + max_seqs) * p.Hkv;
        b->tc_parts = 2 * (size_t)p.sm_count;
        b->item_cap[kTc] = pairs + b->tc_parts;
        b->item_cap[kMerge] = b->tc_parts;
    }
    size_t at = 0;
    auto place = [&](size_t n) {
        const size_t here = at;
        at = (at + n + 255) / 256 * 256;
        return here;
    };
    b->at_counts = place((lists * kKinds + 1) * 4 * sizeof(int));
    b->at_pos = place((size_t)max_tokens * sizeof(int));
    b->at_slot = place((size_t)max_tokens * sizeof(int));
    b->at_entries = place((size_t)max_pages * sizeof(int2));
    b->at_table = place((size_t)max_pages * sizeof(int));
    if (b->tc && pages && pages->v.fmt == GGR_KV_Q8_HEAD) {
        b->at_dense_entries = place((size_t)max_pages * sizeof(int2));
        b->at_dense_table = place((size_t)max_pages * sizeof(int));
    }
    for (size_t l = 0; l < lists; ++l)
        for (int k = 0; k < kKinds; ++k) b->at_items[l][k] = place(b->item_cap[k] * sizeof(PagedItem));
    b->bytes = at;
    const size_t state = 16 * (size_t)(p.D + 2) * sizeof(float) * p.Hkv;
    bool ok = cudaMalloc((void**)&b->d_plan, b->bytes) == cudaSuccess && cudaMalloc((void**)&b->d_part, b->part_tiles * state) == cudaSuccess &&
              cudaMalloc((void**)&b->d_tickets, b->part_tiles * p.Hkv * sizeof(unsigned)) == cudaSuccess;
    if (ok && !pages && dtype == GGR_DTYPE_F32)
        ok = cudaMalloc((void**)&b->d_planes, (size_t)6 * max_tokens * p.Hkv * p.D * sizeof(__nv_bfloat16)) == cudaSuccess;
    if (ok && b->tc) ok = cudaMalloc((void**)&b->d_sched, 2 * sizeof(int)) == cudaSuccess;
    if (ok && b->tc && pages && pages->v.fmt == GGR_KV_Q8_HEAD)
        ok = cudaMalloc((void**)&b->d_q16, (size_t)max_tokens * p.Hq * p.D * sizeof(__half)) == cudaSuccess;
    for (int i = 0; ok && i < 2; ++i)
        ok = cudaHostAlloc((void**)&b->h_plan[i], b->bytes, cudaHostAllocDefault) == cudaSuccess &&
             cudaEventCreateWithFlags(&b->up[i], cudaEventDisableTiming) == cudaSuccess;
    if (!ok) {
        cudaGetLastError();
        return path_fail(c, GGR_ERR_ALLOC, "unable to allocate the batch plan");
    }
    if (cudaMemsetAsync(b->d_plan, 0, b->bytes, p.stream) != cudaSuccess ||
        cudaMemsetAsync(b->d_tickets, 0, b->part_tiles * p.Hkv * sizeof(unsigned), p.stream) != cudaSuccess ||
        (b->tc && cudaMemsetAsync(b->d_sched, 0, 2 * sizeof(int), p.stream) != cudaSuccess))
        return path_fail(c, GGR_ERR_CUDA, "unable to clear the batch plan");
    if (pages) {
        const int half = p.rope_dim / 2;
        std::vector<double> freqs(2 * half);
        for (int k = 0; k < 2; ++k)
            for (int i = 0; i < half; ++i) freqs[k * half + i] = std::pow((double)path_rope_theta(c, k != 0), -(double)(2 * i) / p.rope_dim);
        if (cudaMalloc((void**)&b->d_freqs, freqs.size() * sizeof(double)) != cudaSuccess) {
            cudaGetLastError();
            return path_fail(c, GGR_ERR_ALLOC, "unable to allocate the batch plan");
        }
        PAGED_TRY(c, cudaMemcpyAsync(b->d_freqs, freqs.data(), freqs.size() * sizeof(double), cudaMemcpyHostToDevice, p.stream));
        PAGED_TRY(c, cudaStreamSynchronize(p.stream));
    }
    *out = b.release();
    return GGR_OK;
}

static int batch_set(ggr_batch* b, int32_t n_seqs, const int32_t* q_len, const int32_t* kv_len, const int32_t* page_table, int32_t table_stride) {
    if (!b) return GGR_ERR_INVALID;
    // a step that is refused is not the one before: the caller's rows are no longer that step's
    b->set = false;
    ggr_attn_ctx* c = b->ctx;
    const PathView p = path_view(c);
    if (b->pages && b->pages->destroyed) return path_fail(c, GGR_ERR_INVALID, kPagesGone);
    if (n_seqs > b->max_seqs) return path_fail(c, GGR_ERR_RANGE, "more sequences than the batch plan holds");
    const int ps = b->pages ? b->pages->page_size : 0;
    BatchTotals totals;
    const char* why;
    if (const int rc = batch_check(ps, b->pages ? b->pages->v.n_pages : 0, n_seqs, q_len, kv_len, page_table, table_stride, b->max_tokens, b->max_pages, &totals, &why))
        return path_fail(c, rc, why);
    const int64_t tokens = totals.tokens, entries = totals.entries, rows = totals.rows;
    Guard guard(b->device);
    if (path_capturing(c)) return path_fail(c, GGR_ERR_INVALID, "a batch plan cannot be set while its stream is captured");
    const int turn = b->turn;
    unsigned char* h = b->h_plan[turn];
    if (b->up_used[turn]) PAGED_TRY(c, cudaEventSynchronize(b->up[turn]));
    int* tok_pos = reinterpret_cast<int*>(h + b->at_pos);
    int* tok_slot = reinterpret_cast<int*>(h + b->at_slot);
    int2* entry = reinterpret_cast<int2*>(h + b->at_entries);
    int* table = reinterpret_cast<int*>(h + b->at_table);
    struct Seq {
        int tok0, src;
    };
    std::vector<Seq> seqs(n_seqs);
    {
        int tok = 0, e = 0, dense = 0;
        for (int i = 0; i < n_seqs; ++i) {
            seqs[i] = {tok, b->pages ? e : tok};
            const int first = kv_len[i] - q_len[i];
            const int32_t* row = b->pages ? page_table + (int64_t)i * table_stride : nullptr;
            for (int t = 0; t < q_len[i]; ++t, ++tok) {
                tok_pos[tok] = first + t;
                tok_slot[tok] = row ? row[(first + t) / ps] * ps + (first + t) % ps : 0;
            }
            if (row)
                for (int j = 0; j * (int64_t)ps < kv_len[i]; ++j, ++e) {
                    table[e] = row[j];
                    entry[e] = make_int2(dense + j * ps, std::min(ps, kv_len[i] - j * ps));
                }
            dense += kv_len[i];
        }
    }
    const bool f32 = b->dtype == GGR_DTYPE_F32, q8 = b->pages && b->pages->v.fmt == GGR_KV_Q8_HEAD;
    // kernel of every sequence; captured launches hold certain kernels, and a plan that has any keeps to those
    std::vector<int> kind(n_seqs, kSplitK), lin(n_seqs, 0);
    auto allowed = [&](int k) { return !b->captured || (b->captured >> k & 1); };
    int64_t dense = 0;
    int border = 0;
    if (b->pages || !f32) {
        const int widest = *std::min_element(b->windows.begin(), b->windows.end()) == 0 ? 0 : *std::max_element(b->windows.begin(), b->windows.end());
        std::vector<Work> work(n_seqs);
        for (int i = 0; i < n_seqs; ++i)
            work[i] = {(int)std::min<int64_t>((int64_t)q_len[i] * b->G, 1 << 30), kv_len[i] - first_key(kv_len[i] - q_len[i], widest)};
        BatchShape s{};
        s.D = b->D, s.G = b->G, s.Hkv = b->Hkv, s.sm_count = b->sm_count;
        s.tc = b->tc, s.q8 = q8;
        s.split_rows = f32 ? 8 : 16, s.rows_step = b->rows_step;
        s.item_tokens = b->tc ? tc_item_tiles(b->D) * b->tc_tokens : 0, s.key_tile = tc_key_tile(b->D);
        s.max_pieces = b->tc_parts;
        s.split_step_us = (f32 ? 0.19 : (q8 ? 0.13 : 0.1)) * (b->D == 256 ? (f32 ? 2.0 : 4.0) : b->D / 128.0);
        border = choose_border(work, s);
    }
    for (int i = 0; i < n_seqs; ++i) {
        const int64_t n_rows = (int64_t)q_len[i] * b->G;
        int k = n_rows <= border ? kSplitK : (b->tc ? kTc : kRows);
        if (!allowed(k)) k = allowed(kRows) ? kRows : (allowed(kSplitK) ? kSplitK : kTc);
        kind[i] = k;
        if (k == kTc && q8 && q_len[i] > 0) {
            lin[i] = (int)dense;
            dense += ((int64_t)kv_len[i] + ps - 1) / ps * ps;
        } else if (k == kTc && !b->pages) {
            lin[i] = seqs[i].tok0;
        }
    }
    // (39 MB that a plan of token steps never needs)
    if (!b->d_tc_part && std::find(kind.begin(), kind.end(), (int)kTc) != kind.end() &&
        cudaMalloc((void**)&b->d_tc_part, b->tc_parts * 128 * tc_item_tiles(b->D) * (b->D + 2) * sizeof(float)) != cudaSuccess) {
        cudaGetLastError();
        return path_fail(c, GGR_ERR_ALLOC, "unable to allocate the partial states of a batch plan");
    }
    if (dense > (int64_t)b->dense_rows) {
        if (!b->captured || !b->d_dense) {
            const size_t row = (size_t)b->Hkv * b->D;
            if (b->d_dense) {
                PAGED_TRY(c, cudaStreamSynchronize(p.stream));
                cudaFree(b->d_dense);
            }
            b->d_dense = nullptr;
            // twice what it was, so that a prompt that comes in chunks makes room a few times and not at every step; the plan's pages
            // are the most that can be asked for
            size_t want = std::min(std::max<size_t>(2 * b->dense_rows, 4096), (size_t)b->max_pages * ps);
            want = std::max(std::min(want, ((size_t)1 << 31) - 1), (size_t)dense);
            b->dense_rows = 0;
            auto make = [&] { return want < ((size_t)1 << 31) && cudaMalloc((void**)&b->d_dense, 2 * want * row * sizeof(__half)) == cudaSuccess; };
            bool made = make();
            if (!made && want > (size_t)dense) {
                cudaGetLastError();
                want = (size_t)dense;
                made = make();
            }
            if (made) {
                if (!make_map3(&b->tmKd, false, b->d_dense, b->D, b->Hkv, want, (uint64_t)b->D * 2, row * 2, 64, 1, tc_key_tile(b->D)) ||
                    !make_map3(&b->tmVd, false, b->d_dense + want * row, b->D, b->Hkv, want, (uint64_t)b->D * 2, row * 2, 64, 1, tc_key_tile(b->D)))
                    return path_fail(c, GGR_ERR_CUDA, "cuTensorMapEncodeTiled failed for the dequantised rows");
                b->dense_rows = want;
            } else {
                cudaGetLastError();
                b->d_dense = nullptr;
            }
        }
        // where the rows do not fit (no memory, or captured launches hold the smaller buffer) the warp-level kernel reads the pages
        if (dense > (int64_t)b->dense_rows)
            for (int i = 0; i < n_seqs; ++i)
                if (kind[i] == kTc) {
                    if (!allowed(kRows) && !allowed(kSplitK)) return path_fail(c, GGR_ERR_RANGE, "the captured launches of this plan hold less room for dequantised pages");
                    kind[i] = allowed(kRows) ? kRows : kSplitK;
                }
    }
    int n_dense = 0;
    if (q8 && b->tc) {
        int2* de = reinterpret_cast<int2*>(h + b->at_dense_entries);
        int* dt = reinterpret_cast<int*>(h + b->at_dense_table);
        const int widest = *std::min_element(b->windows.begin(), b->windows.end()) == 0 ? 0 : *std::max_element(b->windows.begin(), b->windows.end());
        for (int i = 0; i < n_seqs; ++i) {
            if (kind[i] != kTc || q_len[i] == 0) continue;
            for (int j = first_key(kv_len[i] - q_len[i], widest) / ps; j * (int64_t)ps < kv_len[i]; ++j, ++n_dense) {
                dt[n_dense] = table[seqs[i].src + j];
                de[n_dense] = make_int2(lin[i] + j * ps, std::min(ps, kv_len[i] - j * ps));
            }
        }
        int* counts = reinterpret_cast<int*>(h + b->at_counts) + b->windows.size() * kKinds * 4;
        counts[1] = n_dense;
        counts[2] = (int)tokens;
    }
    const double tile_bytes = 16.0 * 2 * b->D * (q8 ? 1 : 2);
    for (size_t l = 0; l < b->windows.size(); ++l) {
        const int window = b->windows[l];
        std::vector<Tile> tiles[kKinds];
        std::vector<int> pair_tiles;
        const int kt = tc_key_tile(b->D);
        for (int i = 0; i < n_seqs; ++i) {
            const int first = kv_len[i] - q_len[i], n_rows = q_len[i] * b->G;
            if (kind[i] == kTc) {
                const int step = tc_item_tiles(b->D) * b->tc_tokens;
                for (int t = 0; t < q_len[i]; t += step) {
                    const int lo = first_key(first + t, window) & ~(kt - 1), hi = std::min(first + t + step, kv_len[i]);
                    tiles[kTc].push_back({i, t, 0, lo, hi});
                }
                continue;
            }
            const int step = kind[i] == kRows ? b->rows_step : (f32 ? 8 : 16);  // rows of a tile of the kernel
            for (int r = 0; r < n_rows; r += step) {
                const int m = std::min(step, n_rows - r);
                const int lo = first_key(first + r / b->G, window), hi = first + (r + m - 1) / b->G + 1;
                tiles[kind[i]].push_back({i, r, m, lo & ~15, hi});
            }
        }
        int* counts = reinterpret_cast<int*>(h + b->at_counts) + l * kKinds * 4;
        for (int k = 0; k < kTc; ++k) {
            PagedItem* items = reinterpret_cast<PagedItem*>(h + b->at_items[l][k]);
            int n = 0, part = 0, ticket = 0, longest = 1;
            const int piece = k == kSplitK && !tiles[k].empty()
                                  ? choose_piece(tiles[k], b->Hkv, b->sm_count, tile_bytes, q8 || f32 ? 40e9 : 65e9, paged_splitk_warps(b->D, q8 ? kKvQ8Head : KV_BF16, f32), b->part_tiles, &longest)
                                  : 1 << 27;
            std::stable_sort(tiles[k].begin(), tiles[k].end(), [](const Tile& x, const Tile& y) { return x.key1 - x.key0 > y.key1 - y.key0; });
            for (const Tile& t : tiles[k]) {
                const int n16 = (t.key1 - t.key0 + 15) / 16, cuts = std::max(1, (n16 + piece - 1) / piece), each = (n16 + cuts - 1) / cuts;
                PagedItem it{};
                it.tok0 = seqs[t.seq].tok0;
                it.pos0 = kv_len[t.seq] - q_len[t.seq];
                it.n_tok = q_len[t.seq];
                it.row0 = t.row0;
                it.rows = t.rows;
                it.src = seqs[t.seq].src;
                it.part = -1;
                it.n_split = (n16 + each - 1) / each;
                if (it.n_split > 1) {
                    it.part = part;
                    it.ticket = ticket++;
                    part += it.n_split;
                }
                for (int s = 0; s < it.n_split; ++s) {
                    it.split = s;
                    it.key0 = t.key0 + s * each * 16;
                    it.key1 = (int)std::min<int64_t>(t.key1, it.key0 + (int64_t)each * 16);
                    items[n++] = it;
                }
            }
            counts[k * 4] = n;
            b->n_items[l][k] = n;
        }
        {
            PagedItem* merge = reinterpret_cast<PagedItem*>(h + b->at_items[l][kMerge]);
            auto n_tiles = [kt](const Tile& t) { return (t.key1 - t.key0 + kt - 1) / kt; };
            std::stable_sort(tiles[kTc].begin(), tiles[kTc].end(), [&](const Tile& x, const Tile& y) { return n_tiles(x) > n_tiles(y); });
            for (const Tile& t : tiles[kTc]) pair_tiles.push_back(n_tiles(t));
            int n = 0, n_merge = 0, part = 0, piece = 1;
            double cost_us;
            const int whole = choose_tc_cut(pair_tiles, b->Hkv, b->sm_count, b->tc_parts, b->D == 256, &piece, &cost_us);
            b->scratch.clear();
            for (const Tile& t : tiles[kTc]) {
                const bool cut = &t - tiles[kTc].data() >= whole;
                const int nt = n_tiles(t), cuts = cut ? (nt + piece - 1) / piece : 1, each = (nt + cuts - 1) / cuts;
                PagedItem it{};
                it.tok0 = seqs[t.seq].tok0;
                it.pos0 = kv_len[t.seq] - q_len[t.seq];
                it.n_tok = q_len[t.seq];
                it.row0 = t.row0;
                it.src = seqs[t.seq].src;
                it.lin = lin[t.seq];
                it.n_split = (nt + each - 1) / each;
                for (it.kvh = 0; it.kvh < b->Hkv; ++it.kvh) {
                    it.part = -1;
                    if (it.n_split > 1) {
                        it.part = part;
                        part += it.n_split;
                    }
                    for (int s = 0; s < it.n_split; ++s) {
                        it.split = s;
                        it.key0 = t.key0 + s * each * kt;
                        it.key1 = (int)std::min<int64_t>(t.key1, it.key0 + (int64_t)each * kt);
                        b->scratch.push_back(it);
                        if (s == 0 && it.n_split > 1) merge[n_merge++] = it;
                    }
                }
            }
            std::stable_sort(b->scratch.begin(), b->scratch.end(), [](const PagedItem& x, const PagedItem& y) { return x.key1 - x.key0 > y.key1 - y.key0; });
            n = (int)b->scratch.size();
            if (n) memcpy(h + b->at_items[l][kTc], b->scratch.data(), n * sizeof(PagedItem));
            counts[kTc * 4] = b->n_items[l][kTc] = n;
            counts[kMerge * 4] = b->n_items[l][kMerge] = n_merge;
        }
        for (int k = 0; k < kKinds; ++k) {
            counts[k * 4 + 1] = (int)entries;
            counts[k * 4 + 2] = (int)tokens;
        }
    }
    auto copy = [&](size_t at, size_t n) -> cudaError_t {
        return n ? cudaMemcpyAsync(b->d_plan + at, h + at, n, cudaMemcpyHostToDevice, p.stream) : cudaSuccess;
    };
    PAGED_TRY(c, copy(b->at_counts, (b->windows.size() * kKinds + 1) * 4 * sizeof(int)));
    PAGED_TRY(c, copy(b->at_dense_entries, n_dense * sizeof(int2)));
    PAGED_TRY(c, copy(b->at_dense_table, n_dense * sizeof(int)));
    PAGED_TRY(c, copy(b->at_pos, tokens * sizeof(int)));
    PAGED_TRY(c, copy(b->at_slot, tokens * sizeof(int)));
    PAGED_TRY(c, copy(b->at_entries, entries * sizeof(int2)));
    PAGED_TRY(c, copy(b->at_table, entries * sizeof(int)));
    for (size_t l = 0; l < b->windows.size(); ++l)
        for (int k = 0; k < kKinds; ++k) PAGED_TRY(c, copy(b->at_items[l][k], b->n_items[l][k] * sizeof(PagedItem)));
    // (all zero already, unless a launch that ran into a time limit left before its merges)
    PAGED_TRY(c, cudaMemsetAsync(b->d_tickets, 0, b->part_tiles * b->Hkv * sizeof(unsigned), p.stream));
    PAGED_TRY(c, cudaEventRecord(b->up[turn], p.stream));
    b->up_used[turn] = true;
    b->turn = turn ^ 1;
    b->n_seqs = n_seqs;
    b->n_tokens = (int)tokens;
    b->n_entries = (int)entries;
    b->n_rows = (int)rows;
    b->n_dense = n_dense;
    b->set = true;
    return GGR_OK;
}

namespace {

int check_call(ggr_attn_ctx* c, ggr_batch* b, int layer, bool wants_pages) {
    if (!b || b->ctx != c) return path_fail(c, GGR_ERR_INVALID, "the batch plan belongs to another context");
    if (b->pages && b->pages->destroyed) return path_fail(c, GGR_ERR_INVALID, kPagesGone);
    if (!b->set) return path_fail(c, GGR_ERR_INVALID, "the batch plan has not been set");
    if (layer < 0 || layer >= b->n_layers) return path_fail(c, GGR_ERR_RANGE, "layer outside the cache");
    if (wants_pages && !b->pages) return path_fail(c, GGR_ERR_INVALID, "the batch plan has no pages");
    if (!wants_pages && b->pages) return path_fail(c, GGR_ERR_INVALID, "packed prompts need a batch plan without pages");
    return GGR_OK;
}

// rows of `dim` elements at `stride`: vector loads and tensor maps need whole 16-byte pieces
int check_rows(ggr_attn_ctx* c, const char* name, const void* x, int64_t* stride, int dim, int es) {
    if (!x) return path_fail(c, GGR_ERR_INVALID, std::string("null ") + name);
    if (*stride == 0) *stride = dim;
    if (*stride < dim) return path_fail(c, GGR_ERR_INVALID, std::string(name) + ": rows overlap");
    if ((uintptr_t)x % 16 || (*stride * es) % 16) return path_fail(c, GGR_ERR_INVALID, std::string(name) + ": rows must start on 16-byte boundaries");
    if (*stride * es >= ((int64_t)1 << 39)) return path_fail(c, GGR_ERR_RANGE, std::string(name) + ": row stride out of range");
    return GGR_OK;
}

// Tensor maps of a launch: 16-row tiles for the warp-level kernels, 128-row tiles and query tiles for the tcgen05 kernel.
struct Maps {
    const CUtensorMap *k16, *v16, *k128, *v128;
};

template <int FMT, int D>
cudaError_t launch_read(const ReadArgs& a, bool bf16, bool chained, int grid, cudaStream_t stream) {
    return launch_chained(chained, bf16 ? paged_read_kernel<FMT, D, kReadBf16> : paged_read_kernel<FMT, D, kReadF32>, dim3(grid), 256, 0, stream, a);
}

// Launches are programmatic (launch_chained) except in a capture, whose edges are full ones, and between event pairs.
bool chain(const ggr_attn_ctx* c, bool capturing) { return !capturing && !path_timing(c); }

int read_grid(const ggr_batch* b, int64_t entries) {
    const int64_t blocks = entries * (b->pages->page_size / 16) * b->Hkv;
    return (int)std::min<int64_t>((blocks + 1) / 2, (int64_t)16 * b->sm_count);
}

// 8-bit pages and q as the f16 rows that the tcgen05 kernels multiply
template <int D>
int launch_dense_rows(ggr_attn_ctx* c, const PathView& p, ggr_batch* b, const PagedAttnArgs& args, bool capturing) {
    {
        ReadArgs r{};
        r.pages = b->pages->v;
        r.counts = b->dense_counts();
        r.table = reinterpret_cast<const int*>(b->d_plan + b->at_dense_table);
        r.entries = reinterpret_cast<const int2*>(b->d_plan + b->at_dense_entries);
        r.layer = args.layer;
        r.k_out = b->d_dense;
        r.v_out = b->d_dense + b->dense_rows * b->Hkv * b->D;
        r.k_stride = r.v_stride = (int64_t)b->Hkv * b->D;
        r.q = static_cast<const __nv_bfloat16*>(args.q);
        r.q_stride = args.q_stride;
        r.q_out = b->d_q16;
        r.q_dim = b->Hq * D;
        {
            PathTimer t(c, 1);
            PAGED_TRY(c, launch_chained(chain(c, capturing), paged_read_kernel<kKvQ8Head, D, kReadHalf>, dim3(read_grid(b, capturing ? b->max_pages : b->n_dense)), 256, 0,
                                        p.stream, r));
        }
        path_launched(c);
    }
    return GGR_OK;
}

// `behind`: right behind a warp-level kernel of the same call that lets it in
template <int D, int FMT>
int launch_tc(ggr_attn_ctx* c, const PathView& p, ggr_batch* b, int list, const Maps& m, const PagedAttnArgs& args, int rows, bool capturing, bool behind) {
    constexpr bool q8 = FMT == kKvQ8Head;
    PagedTcArgs t{};
    t.behind = behind;
    t.a = args;
    t.a.plan.counts = b->counts(list, kTc);
    t.a.plan.items = b->items(list, kTc);
    t.tiles_tokens = b->tc_tokens;
    t.box_rows = b->pages ? std::min(b->pages->page_size, tc_key_tile(D)) : tc_key_tile(D);
    t.linear = !b->pages || q8;
    t.out_scale = q8 ? 1.0f / kReadVScale : 1.0f;
    t.sched = b->d_sched;
    t.part = b->d_tc_part;
    // (tensor maps move 16-bit elements as they are: bf16 stands for f16 too)
    const CUtensorMap &tk = q8 ? b->tmKd : *m.k128, &tv = q8 ? b->tmVd : *m.v128;
    const int n = b->n_items[list][kTc];
    if constexpr (D == 256) {
        static KernelSmemSetup setup;
        PAGED_TRY(c, setup.ensure(paged_tc_wide_kernel<q8>, p.device, p.smem_optin, (int)kPwSmem));
        t.q_rows = q8 ? static_cast<const void*>(b->d_q16) : args.q;
        t.q_rows_stride = q8 ? b->Hq * D : args.q_stride;
        PathTimer timer(c, 0);
        PAGED_TRY(c, launch_chained(chain(c, capturing), paged_tc_wide_kernel<q8>, dim3(capturing ? (int)b->item_cap[kTc] : n), kPwThreads, kPwSmem, p.stream, tk, tv, t));
    } else {
        const void* q_rows = q8 ? static_cast<const void*>(b->d_q16) : args.q;
        CUtensorMap tq;
        if (!make_map3(&tq, false, q_rows, D, b->Hq, rows, (uint64_t)D * 2, (uint64_t)(q8 ? b->Hq * D : args.q_stride) * 2, 64, b->G, b->tc_tokens))
            return path_fail(c, GGR_ERR_CUDA, "cuTensorMapEncodeTiled failed for the query rows");
        static KernelSmemSetup setup;
        PAGED_TRY(c, setup.ensure(paged_tc_kernel<D, q8>, p.device, p.smem_optin, (int)kPtSmem<D>));
        PathTimer timer(c, 0);
        PAGED_TRY(c, launch_chained(chain(c, capturing), paged_tc_kernel<D, q8>, dim3(capturing ? b->sm_count : std::min(b->sm_count, n)), kPtThreads, kPtSmem<D>, p.stream, tq, tk, tv, t));
    }
    PAGED_TRY(c, cudaGetLastError());
    path_launched(c);
    if (!capturing && !b->n_items[list][kMerge]) return GGR_OK;
    t.a.plan.counts = b->counts(list, kMerge);
    t.a.plan.items = b->items(list, kMerge);
    const int cut = capturing ? (int)b->tc_parts / 2 : b->n_items[list][kMerge];
    {
        PathTimer timer(c, 2);
        const int grid = std::min(cut * (D == 256 ? 16 : D / 4), 16 * b->sm_count);
        PAGED_TRY(c, launch_chained(chain(c, capturing), paged_tc_merge_kernel<D>, dim3(grid), 256, 0, p.stream, t));
    }
    path_launched(c);
    return GGR_OK;
}

template <int D, int FMT, bool F32>
int launch_attention(ggr_attn_ctx* c, const PathView& p, ggr_batch* b, int list, const Maps& m, PagedAttnArgs a, int rows, bool capturing) {
    if (capturing && !b->n_tokens) return path_fail(c, GGR_ERR_INVALID, "a captured launch needs a plan with tokens: it holds the kernels of that plan");
    // a captured launch has to serve whatever plan its replays find: enough CTAs for any, items dealt in turn
    const int most = (2 * b->sm_count + b->Hkv - 1) / b->Hkv;
    const bool tc = b->n_items[list][kTc] > 0;
    if constexpr (!F32 && FMT == kKvQ8Head) {
        if (tc) {
            const int rc = launch_dense_rows<D>(c, p, b, a, capturing);
            if (rc) return rc;
        }
    }
    bool behind = false;
    for (int k = 0; k < kTc; ++k) {
        const int n = b->n_items[list][k];
        if (!n) continue;
        behind = chain(c, capturing);
        a.plan.counts = b->counts(list, k);
        a.plan.items = b->items(list, k);
        const dim3 grid(b->Hkv, capturing ? most : std::min(n, 65535));
        if (k == kSplitK) {
            if constexpr (FMT == KV_F32) continue;
            else {
                using S = PagedSplitKShape<D, FMT, F32>;
                static KernelSmemSetup setup;
                PAGED_TRY(c, setup.ensure(paged_splitk_kernel<D, FMT, F32>, p.device, p.smem_optin, (int)S::SMEM));
                PathTimer t(c, 0);
                PAGED_TRY(c, launch_chained(chain(c, capturing), paged_splitk_kernel<D, FMT, F32>, grid, S::W * 32, S::SMEM, p.stream, *m.k16, *m.v16, a));
            }
        } else {
            using S = PagedRowsShape<D, FMT, F32>;
            static KernelSmemSetup setup;
            PAGED_TRY(c, setup.ensure(paged_rows_kernel<D, FMT, F32>, p.device, p.smem_optin, (int)S::SMEM));
            PathTimer t(c, 0);
            PAGED_TRY(c, launch_chained(chain(c, capturing), paged_rows_kernel<D, FMT, F32>, grid, S::THREADS, S::SMEM, p.stream, *m.k16, *m.v16, a));
        }
        PAGED_TRY(c, cudaGetLastError());
        path_launched(c);
        if (capturing) b->captured |= 1u << k;
    }
    if constexpr (!F32) {
        if (tc) {
            const int rc = launch_tc<D, FMT>(c, p, b, list, m, a, rows, capturing, behind);
            if (rc) return rc;
            if (capturing) b->captured |= 1u << kTc;
        }
    }
    return GGR_OK;
}

template <int FMT, bool F32>
int launch_by_dim(ggr_attn_ctx* c, const PathView& p, ggr_batch* b, int list, const Maps& m, const PagedAttnArgs& a, int rows, bool cap) {
    switch (b->D) {
        case 64: return launch_attention<64, FMT, F32>(c, p, b, list, m, a, rows, cap);
        case 128: return launch_attention<128, FMT, F32>(c, p, b, list, m, a, rows, cap);
        default: return launch_attention<256, FMT, F32>(c, p, b, list, m, a, rows, cap);
    }
}

PagedAttnArgs attention_args(const PathView& p, const ggr_batch* b, int layer) {
    PagedAttnArgs a{};
    a.plan.table = b->table();
    a.layer = layer;
    a.Hq = b->Hq;
    a.G = b->G;
    a.window = b->windows[b->list_of[layer]];
    a.c = p.score_scale * kLog2e;
    a.part = b->d_part;
    a.tickets = b->d_tickets;
    a.err = p.d_err;
    a.pages.Hkv = b->Hkv;
    a.pages.D = b->D;
    return a;
}

}  // namespace

static int paged_append(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, int32_t rotate, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                const void* v, int64_t v_stride, void* q_out) {
    if (!c) return GGR_ERR_INVALID;
    int rc = check_call(c, b, layer, true);
    if (rc) return rc;
    const PathView p = path_view(c);
    const int es = elem_bytes(b->dtype), q_dim = b->Hq * b->D, kv_dim = b->Hkv * b->D;
    if (!rotate && (q || q_out)) return path_fail(c, GGR_ERR_INVALID, "q is taken only to be rotated");
    Guard guard(p.device);
    const bool capturing = path_capturing(c);
    if (!b->n_tokens && !capturing) return GGR_OK;  // (rows of an empty tensor may have no address)
    if ((rc = check_rows(c, "k", k, &k_stride, kv_dim, es)) || (rc = check_rows(c, "v", v, &v_stride, kv_dim, es))) return rc;
    int64_t qo_stride = q_dim;
    if (rotate) {
        if ((rc = check_rows(c, "q", q, &q_stride, q_dim, es)) || (rc = check_rows(c, "q_out", q_out, &qo_stride, q_dim, es))) return rc;
        if (p.position_plan) return path_fail(c, GGR_ERR_UNSUPPORTED, "a position plan belongs to one generation: batches rotate by cache position");
        if (q == q_out && (p.rope_dim != b->D || q_stride != qo_stride))
            return path_fail(c, GGR_ERR_INVALID, "q_out may be q itself only for dense rows whose heads are rotated as a whole");
    }
    int in_bf16 = b->dtype == GGR_DTYPE_BF16;
    if (rotate && path_has_fixups(c, layer)) {
        if (q_stride != q_dim || k_stride != kv_dim || v_stride != kv_dim) return path_fail(c, GGR_ERR_UNSUPPORTED, "bias and QK-norm need dense rows");
        if (capturing) return path_fail(c, GGR_ERR_UNSUPPORTED, "bias and QK-norm of a batch are not captured: their scratch follows the batch");
        if ((rc = path_fixups(c, layer, b->n_tokens, &q, &k, &v, &in_bf16))) return rc;
    }
    AppendArgs a{};
    a.pages = b->pages->v;
    a.rope = path_rope(c, layer);
    a.freqs = b->d_freqs + (path_rope_window_kind(c, layer) ? p.rope_dim / 2 : 0);
    a.counts = b->counts(0, 0);
    a.tok_pos = reinterpret_cast<const int*>(b->d_plan + b->at_pos);
    a.tok_slot = reinterpret_cast<const int*>(b->d_plan + b->at_slot);
    a.layer = layer;
    a.rotate = rotate != 0;
    a.write_q = rotate != 0;
    a.in_bf16 = in_bf16;
    a.q_bf16 = b->dtype == GGR_DTYPE_BF16;
    a.Hq = b->Hq;
    a.heads = (rotate ? b->Hq : 0) + 2 * b->Hkv;
    a.heads_inv = (unsigned)(((1ull << 32) + a.heads - 1) / a.heads);
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.qo_stride = qo_stride;
    const int n = capturing ? b->max_tokens : b->n_tokens;
    // (two tasks of 16 bytes per thread, once there are CTAs enough)
    const int tasks = a.heads * b->D / (in_bf16 ? 16 : 8);
    a.tokens_per_cta = n < 8 * b->sm_count ? 1 : std::max(1, 512 / tasks);
    const int grid = (n + a.tokens_per_cta - 1) / a.tokens_per_cta;
    const size_t smem = rotate ? (size_t)2 * a.tokens_per_cta * a.rope.rope_half * sizeof(float) : 0;
    {
        PathTimer t(c, 1);
        PAGED_TRY(c, launch_chained(chain(c, capturing), in_bf16 ? paged_append_kernel<true> : paged_append_kernel<false>, dim3(grid), 256, smem, p.stream, a));
    }
    path_launched(c);
    return GGR_OK;
}

static int paged_read(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, int32_t out_dtype, void* k_out, int64_t k_stride, void* v_out, int64_t v_stride) {
    if (!c) return GGR_ERR_INVALID;
    int rc = check_call(c, b, layer, true);
    if (rc) return rc;
    if (out_dtype != GGR_DTYPE_F32 && out_dtype != GGR_DTYPE_BF16) return path_fail(c, GGR_ERR_INVALID, "unknown dtype");
    const int kv_dim = b->Hkv * b->D, es = elem_bytes(out_dtype);
    const PathView p = path_view(c);
    Guard guard(p.device);
    const bool capturing = path_capturing(c);
    if (!b->n_entries && !capturing) return GGR_OK;
    if ((rc = check_rows(c, "k_out", k_out, &k_stride, kv_dim, es)) || (rc = check_rows(c, "v_out", v_out, &v_stride, kv_dim, es))) return rc;
    ReadArgs a{};
    a.pages = b->pages->v;
    a.counts = b->counts(0, 0);
    a.table = b->table();
    a.entries = reinterpret_cast<const int2*>(b->d_plan + b->at_entries);
    a.layer = layer;
    a.k_out = k_out;
    a.v_out = v_out;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    const int grid = read_grid(b, capturing ? b->max_pages : b->n_entries);
    const bool bf16 = out_dtype == GGR_DTYPE_BF16;
    {
        PathTimer t(c, 1);
        const bool chained = chain(c, capturing), q8 = b->pages->v.fmt == GGR_KV_Q8_HEAD;
        switch (b->D) {
            case 64: PAGED_TRY(c, (q8 ? launch_read<kKvQ8Head, 64> : launch_read<KV_BF16, 64>)(a, bf16, chained, grid, p.stream)); break;
            case 128: PAGED_TRY(c, (q8 ? launch_read<kKvQ8Head, 128> : launch_read<KV_BF16, 128>)(a, bf16, chained, grid, p.stream)); break;
            default: PAGED_TRY(c, (q8 ? launch_read<kKvQ8Head, 256> : launch_read<KV_BF16, 256>)(a, bf16, chained, grid, p.stream));
        }
    }
    path_launched(c);
    return GGR_OK;
}

static int paged_attention(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, const void* q, int64_t q_stride, void* out, int64_t out_stride) {
    if (!c) return GGR_ERR_INVALID;
    int rc = check_call(c, b, layer, true);
    if (rc) return rc;
    const PathView p = path_view(c);
    const int es = elem_bytes(b->dtype), q_dim = b->Hq * b->D;
    if (p.image_blocks) return path_fail(c, GGR_ERR_UNSUPPORTED, "bidirectional blocks belong to one generation: batches attend causally");
    Guard guard(p.device);
    const bool capturing = path_capturing(c);
    if (!b->n_tokens && !capturing) return GGR_OK;
    if ((rc = check_rows(c, "q", q, &q_stride, q_dim, es)) || (rc = check_rows(c, "out", out, &out_stride, q_dim, es))) return rc;
    PagedAttnArgs a = attention_args(p, b, layer);
    a.paged = 1;
    a.pages = b->pages->v;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.o_stride = out_stride;
    const int list = b->list_of[layer];
    const Maps m{&b->pages->tmK16, &b->pages->tmV16, &b->pages->tmK128, &b->pages->tmV128};
    const bool f32 = b->dtype == GGR_DTYPE_F32;
    const int rows = capturing ? b->max_tokens : b->n_tokens;
    if (b->pages->v.fmt == GGR_KV_BF16)
        return f32 ? launch_by_dim<KV_BF16, true>(c, p, b, list, m, a, rows, capturing) : launch_by_dim<KV_BF16, false>(c, p, b, list, m, a, rows, capturing);
    return f32 ? launch_by_dim<kKvQ8Head, true>(c, p, b, list, m, a, rows, capturing) : launch_by_dim<kKvQ8Head, false>(c, p, b, list, m, a, rows, capturing);
}

static int packed_attention(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                    int64_t v_stride, void* out, int64_t out_stride) {
    if (!c) return GGR_ERR_INVALID;
    int rc = check_call(c, b, layer, false);
    if (rc) return rc;
    const PathView p = path_view(c);
    const int es = elem_bytes(b->dtype), q_dim = b->Hq * b->D, kv_dim = b->Hkv * b->D;
    if (p.image_blocks) return path_fail(c, GGR_ERR_UNSUPPORTED, "bidirectional blocks belong to one generation: batches attend causally");
    Guard guard(p.device);
    const bool capturing = path_capturing(c);
    if (!b->n_tokens && !capturing) return GGR_OK;
    if ((rc = check_rows(c, "q", q, &q_stride, q_dim, es)) || (rc = check_rows(c, "k", k, &k_stride, kv_dim, es)) ||
        (rc = check_rows(c, "v", v, &v_stride, kv_dim, es)) || (rc = check_rows(c, "out", out, &out_stride, q_dim, es)))
        return rc;
    const int rows = capturing ? b->max_tokens : b->n_tokens;
    const bool f32 = b->dtype == GGR_DTYPE_F32;
    PagedAttnArgs a = attention_args(p, b, layer);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.o_stride = out_stride;
    a.pk = k;
    a.pv = v;
    a.pk_stride = k_stride;
    a.pv_stride = v_stride;
    CUtensorMap tk, tv, tk128, tv128;
    const Maps m{&tk, &tv, &tk128, &tv128};
    const int list = b->list_of[layer];
    if (f32) {
        const int64_t plane = (int64_t)b->max_tokens * kv_dim;
        __nv_bfloat16 *kp = b->d_planes, *vp = b->d_planes + 3 * plane;
        a.plane_rows = b->max_tokens;
        const uint64_t sy = (uint64_t)b->D * 2, sz = (uint64_t)kv_dim * 2;
        if (!make_map3(&tk, false, kp, b->D, b->Hkv, (uint64_t)3 * b->max_tokens, sy, sz, 64, 1, 16) ||
            !make_map3(&tv, false, vp, b->D, b->Hkv, (uint64_t)3 * b->max_tokens, sy, sz, 64, 1, 16))
            return path_fail(c, GGR_ERR_CUDA, "cuTensorMapEncodeTiled failed for the packed rows");
        {
            PathTimer t(c, 1);
            PAGED_TRY(c, launch_chained(chain(c, capturing), paged_planes_kernel, dim3((unsigned)(((int64_t)rows * kv_dim / 4 + 255) / 256), 2), 256, 0, p.stream,
                                        static_cast<const float*>(k), static_cast<const float*>(v), k_stride, v_stride, b->counts(0, 0), kv_dim, kp, vp, plane));
        }
        path_launched(c);
        return launch_by_dim<KV_F32, true>(c, p, b, list, m, a, rows, capturing);
    }
    const uint64_t sy = (uint64_t)b->D * 2;
    if (!make_map3(&tk, false, k, b->D, b->Hkv, rows, sy, (uint64_t)k_stride * 2, 64, 1, 16) ||
        !make_map3(&tv, false, v, b->D, b->Hkv, rows, sy, (uint64_t)v_stride * 2, 64, 1, 16) ||
        !make_map3(&tk128, false, k, b->D, b->Hkv, rows, sy, (uint64_t)k_stride * 2, 64, 1, tc_key_tile(b->D)) ||
        !make_map3(&tv128, false, v, b->D, b->Hkv, rows, sy, (uint64_t)v_stride * 2, 64, 1, tc_key_tile(b->D)))
        return path_fail(c, GGR_ERR_CUDA, "cuTensorMapEncodeTiled failed for the packed rows");
    return launch_by_dim<KV_BF16, false>(c, p, b, list, m, a, rows, capturing);
}

// ---- C entries: nothing that the standard library throws leaves them -------------------------------

template <typename F>
static int guarded(F&& f) {
    try {
        return f();
    } catch (...) {
        return GGR_ERR_ALLOC;  // (only allocations of the host throw here)
    }
}

extern "C" int ggr_pages_create(ggr_attn_ctx* c, int32_t n_pages, int32_t page_size, int32_t kv_format, void* k, void* v, float* k_scale, float* v_scale, ggr_pages** out) {
    return guarded([&] { return pages_create(c, n_pages, page_size, kv_format, k, v, k_scale, v_scale, out); });
}

extern "C" int ggr_batch_create(ggr_attn_ctx* c, ggr_pages* pages, int32_t dtype, int32_t max_seqs, int32_t max_tokens, int32_t max_pages, ggr_batch** out) {
    return guarded([&] { return batch_create(c, pages, dtype, max_seqs, max_tokens, max_pages, out); });
}

extern "C" int ggr_batch_set(ggr_batch* b, int32_t n_seqs, const int32_t* q_len, const int32_t* kv_len, const int32_t* page_table, int32_t table_stride) {
    return guarded([&] { return batch_set(b, n_seqs, q_len, kv_len, page_table, table_stride); });
}

extern "C" int ggr_paged_append(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, int32_t rotate, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out) {
    return guarded([&] { return paged_append(c, b, layer, rotate, q, q_stride, k, k_stride, v, v_stride, q_out); });
}

extern "C" int ggr_paged_read(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, int32_t out_dtype, void* k_out, int64_t k_stride, void* v_out, int64_t v_stride) {
    return guarded([&] { return paged_read(c, b, layer, out_dtype, k_out, k_stride, v_out, v_stride); });
}

extern "C" int ggr_paged_attention(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, const void* q, int64_t q_stride, void* out, int64_t out_stride) {
    return guarded([&] { return paged_attention(c, b, layer, q, q_stride, out, out_stride); });
}

extern "C" int ggr_packed_attention(ggr_attn_ctx* c, ggr_batch* b, int32_t layer, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* out, int64_t out_stride) {
    return guarded([&] { return packed_attention(c, b, layer, q, q_stride, k, k_stride, v, v_stride, out, out_stride); });
}
