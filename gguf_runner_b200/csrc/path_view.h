// What the translation units beside ggr_attn.cu see of a context: its shape, stream and RoPE parameters, and the calls that
// record an error, a launch or a device time in it. Defined in ggr_attn.cu.
#pragma once

#include <cuda_runtime.h>

#include <string>
#include <vector>

#include "../../include/ggr_attn.h"
#include "common.cuh"

namespace ggr {

struct PathView {
    int device, n_layers, Hq, Hkv, D, G;
    int rope_dim;
    int sm_count, smem_optin;
    cudaStream_t stream;
    float score_scale;    // multiplies q . k: 1 / sqrt(D), or 1 where q is pre-scaled
    bool position_plan;   // logical positions are set (one generation's, not a batch's)
    bool image_blocks;    // bidirectional blocks are set
    bool sharded;         // the context holds a shard of the positions
    int* d_err;           // error word that kernels raise when a bounded wait runs out
    const std::vector<int32_t>* windows;  // per layer, or empty
};

PathView path_view(const ggr_attn_ctx* c);
RopeParams path_rope(const ggr_attn_ctx* c, int layer);
// theta of a layer's frequencies, and of the other kind of layer
float path_rope_theta(const ggr_attn_ctx* c, bool window_kind);
bool path_rope_window_kind(const ggr_attn_ctx* c, int layer);
int path_fail(ggr_attn_ctx* c, int status, const std::string& msg);
void path_create_error(const std::string& msg);
bool path_capturing(ggr_attn_ctx* c);
bool path_timing(const ggr_attn_ctx* c);
void path_launched(ggr_attn_ctx* c);
// event pair around one launch when kernel timing is on: kind as in ggr_attn_kernel_time
cudaEvent_t path_timer_start(ggr_attn_ctx* c, int kind);
void path_timer_stop(ggr_attn_ctx* c, cudaEvent_t stop);
// bias / QK-norm fixups of the layer on n dense rows: redirects the pointers to f32 scratch rows where there are any
bool path_has_fixups(const ggr_attn_ctx* c, int layer);
int path_fixups(ggr_attn_ctx* c, int layer, int n, const void** q, const void** k, const void** v, int* in_bf16);

struct PathTimer {
    ggr_attn_ctx* c;
    cudaEvent_t stop;
    PathTimer(ggr_attn_ctx* ctx, int kind) : c(ctx), stop(path_timer_start(ctx, kind)) {}
    ~PathTimer() { path_timer_stop(c, stop); }
};

}  // namespace ggr
