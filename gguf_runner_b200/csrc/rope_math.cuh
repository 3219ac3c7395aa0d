// Element arithmetic of RoPE and of the cache rows, shared by the kernels that rotate and append: input loads, one rotated
// element, the 8-bit code, and 8-element vectors in and out of registers.
#pragma once

#include "common.cuh"

namespace ggr {

__device__ __forceinline__ float load_in(const void* p, int64_t idx, int in_bf16) {
    if (in_bf16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[idx]);
    return reinterpret_cast<const float*>(p)[idx];
}

// One rotated element of a head (NeoX split-half or adjacent pairs).
__device__ __forceinline__ float rope_elem(const void* x, int64_t base, int i, int D, const RopeParams& rp,
                                           const float* cs, const float* sn, int in_bf16) {
    if (rp.style == 0) {
        const int half = rp.rope_half;
        if (i < half) {
            float v0 = load_in(x, base + i, in_bf16), v1 = load_in(x, base + i + half, in_bf16);
            return __fsub_rn(__fmul_rn(v0, cs[i]), __fmul_rn(v1, sn[i]));
        } else if (i < rp.rope_dim) {
            int j = i - half;
            float v0 = load_in(x, base + j, in_bf16), v1 = load_in(x, base + i, in_bf16);
            return __fadd_rn(__fmul_rn(v0, sn[j]), __fmul_rn(v1, cs[j]));
        }
        return load_in(x, base + i, in_bf16);
    } else {
        int j = i >> 1;
        if ((i & 1) == 0) {
            float v0 = load_in(x, base + i, in_bf16), v1 = load_in(x, base + i + 1, in_bf16);
            return __fsub_rn(__fmul_rn(v0, cs[j]), __fmul_rn(v1, sn[j]));
        }
        float v0 = load_in(x, base + i - 1, in_bf16), v1 = load_in(x, base + i, in_bf16);
        return __fadd_rn(__fmul_rn(v0, sn[j]), __fmul_rn(v1, cs[j]));
    }
}

__device__ __forceinline__ int8_t q8_code(float x, float inv) {
    // src/engine/runtime/inference.rs:264-266: round half away from zero, clamp to +-127
    float r = roundf(__fmul_rn(x, inv));
    r = fminf(127.0f, fmaxf(-127.0f, r));
    return (int8_t)r;
}

__device__ __forceinline__ void unpack8(const uint4& u, float f[8]) {
    f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
    f[4] = __uint_as_float(u.z << 16); f[5] = __uint_as_float(u.z & 0xffff0000u);
    f[6] = __uint_as_float(u.w << 16); f[7] = __uint_as_float(u.w & 0xffff0000u);
}
__device__ __forceinline__ uint4 pack8(const float f[8]) {
    __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    __nv_bfloat162 c = __floats2bfloat162_rn(f[4], f[5]), d = __floats2bfloat162_rn(f[6], f[7]);
    uint4 u;
    u.x = *reinterpret_cast<uint32_t*>(&a);
    u.y = *reinterpret_cast<uint32_t*>(&b);
    u.z = *reinterpret_cast<uint32_t*>(&c);
    u.w = *reinterpret_cast<uint32_t*>(&d);
    return u;
}

template <typename TIn>
__device__ __forceinline__ void load8_in(const TIn* p, float x[8]);
template <>
__device__ __forceinline__ void load8_in<float>(const float* p, float x[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8_in<__nv_bfloat16>(const __nv_bfloat16* p, float x[8]) {
    unpack8(*reinterpret_cast<const uint4*>(p), x);
}
__device__ __forceinline__ void store8_f32(float* p, const float x[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

}  // namespace ggr
