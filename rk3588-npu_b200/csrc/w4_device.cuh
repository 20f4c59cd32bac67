// w4_device.cuh -- device parts of the 4-bit projections: unpacking codes,
// copies, splitting an fp32 x, the epilogues.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "device_common.cuh"
#include "projection.cuh"
#include "w4_internal.h"

namespace kvattn {

// ------------------------------------------------------------------ unpacking
// The zero point z as the constants of unpack().
template <int BF>
__device__ __forceinline__ uint2 zero_consts(uint32_t z) {
    if (BF) return make_uint2((0x4300u | z) * 0x10001u, 0u);
    return make_uint2((0x6400u | z) * 0x10001u, (0xD400u | z << 4) * 0x10001u);  // 1024 + z, -(64 + z)
}

// (a & b) | c in one instruction (only one of b and c may be an immediate).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// Eight codes minus their zero point as four pairs of fp16 / bf16 values, in
// input order.  The way of setting integers under a fixed exponent is that of
// Kim, Henry, Fahim and Hassan Awadalla, "Who Says Elephants Can't Run" (2022).
template <int BF>
__device__ __forceinline__ void unpack(uint32_t w, uint2 zc, uint32_t (&p)[4]) {
    if (BF) {
        const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&zc.x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = and_or(w >> (4 * i), 0x000F000Fu, 0x43004300u);
            const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), z);
            p[i] = *reinterpret_cast<const uint32_t*>(&r);
        }
    } else {
        const __half2 z = *reinterpret_cast<const __half2*>(&zc.x), z16 = *reinterpret_cast<const __half2*>(&zc.y);
        const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t u = w >> (8 * i);
            const uint32_t lo = and_or(u, 0x000F000Fu, 0x64006400u), hi = and_or(u, 0x00F000F0u, 0x64006400u);
            const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), z);
            const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, z16);
            p[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
            p[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
        }
    }
}

// ------------------------------------------------------------------- staging
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The three bf16 parts of an fp32 value, each with the next 8 significant
// bits (the third rounded; exact for any value whose third part is normal).
// Infinity and NaN stay in the first part alone.
__device__ __forceinline__ void split3(float x, uint16_t& a, uint16_t& b, uint16_t& c) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7F800000u) == 0x7F800000u) {
        a = (u & 0x007FFFFFu) ? 0x7FFFu : (uint16_t)(u >> 16);
        b = c = 0;
        return;
    }
    a = (uint16_t)(u >> 16);
    const float r = x - __uint_as_float(u & 0xFFFF0000u);  // exact
    const uint32_t v = __float_as_uint(r);
    b = (uint16_t)(v >> 16);
    const __nv_bfloat16 t = __float2bfloat16_rn(r - __uint_as_float(v & 0xFFFF0000u));
    c = *reinterpret_cast<const uint16_t*>(&t);
}

// ------------------------------------------------------------------ epilogue
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
// f(a value of the element type).
template <class F>
__device__ __forceinline__ void with_type(int dtype, F f) {
    if (dtype == STEP_F32) f(0.f);
    else if (dtype == STEP_F16) f(__half());
    else f(__nv_bfloat16());
}

__device__ __forceinline__ float load_as(const void* p, size_t i, int dtype) {
    float v = 0.f;
    with_type(dtype, [&](auto one) { v = to_float(static_cast<const decltype(one)*>(p)[i]); });
    return v;
}
__device__ __forceinline__ void store_as(void* p, size_t i, int dtype, float v) {
    with_type(dtype, [&](auto one) { static_cast<decltype(one)*>(p)[i] = from_float<decltype(one)>(v); });
}

// silu(g) u
__device__ __forceinline__ float gated(float g, float u) { return __fdiv_rn(g, 1.0f + expf(-g)) * u; }

__device__ __forceinline__ void w4_epilogue(const W4Args& a, int row, int n, float y, float y2) {
    switch (a.mode) {
        case W4_QKV: gemv_epilogue<0>(a.g, row, n, y, y2); break;
        case W4_RESID: gemv_epilogue<1>(a.g, row, n, y, y2); break;
        case W4_GATE_UP: gemv_epilogue<2>(a.g, row, n, y, y2); break;
        case W4_LOGITS: gemv_epilogue<3>(a.g, row, n, y, y2); break;
        case W4_LINEAR:
            if (a.bias) y += __ldg(a.bias + n);
            if (a.residual) y += load_as(a.residual, (size_t)row * a.ldr + n, a.out_dtype);
            store_as(a.out, (size_t)row * a.ldo + n, a.out_dtype, y);
            break;
        default:
            store_as(a.out, (size_t)row * a.ldo + n, a.out_dtype, gated(y, y2));
    }
}

}  // namespace kvattn
