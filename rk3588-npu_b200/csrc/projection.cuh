// projection.cuh -- what the fp16 and the 4-bit projections of the Qwen2
// forward share: the reference's fp16 rounding, the RMSNorm sum and the call
// sites' epilogues.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "device_common.cuh"
#include "kvattn_internal.h"

namespace kvattn {

// fp16 -> fp32 exactly as worker/include/core/half.h:34-43 (its exponent-0
// branch included).
__device__ __forceinline__ float dec_f16_ref(uint32_t h) {
    const uint32_t sign = (h & 0x8000u) << 16, e = (h >> 10) & 0x1Fu, mant = h & 0x3FFu;
    uint32_t x;
    if (e == 0) x = sign | (mant << 13);
    else if (e == 31) x = sign | 0x7F800000u | (mant << 13);
    else x = sign | ((e + 112u) << 23) | (mant << 13);
    return __uint_as_float(x);
}

// Round an fp32 value through the reference's fp16 (f16_to_f32(f32_to_f16(x))).
__device__ __forceinline__ float f16_round(float x) { return dec_f16_ref(enc_f16_trunc(x)); }

// One fp32 chunk's rounded squares added to s, in order (op_rmsnorm.cpp:12-15).
__device__ __forceinline__ float sum_sq4(float s, const float4& v) {
    s = __fadd_rn(s, __fmul_rn(v.x, v.x));
    s = __fadd_rn(s, __fmul_rn(v.y, v.y));
    s = __fadd_rn(s, __fmul_rn(v.z, v.z));
    return __fadd_rn(s, __fmul_rn(v.w, v.w));
}

// The call site's fp32 epilogue of output n of input row `row`, from the fp32
// sums of its weight row (acc) and, for gate/up, of its up row (acc2).
template <int MODE>
__device__ __forceinline__ void gemv_epilogue(const GemvArgs& a, int row, int n, float acc, float acc2) {
    const float r = f16_round(acc);
    if (MODE == 0) {
        const float v = __fadd_rn(r, a.bias[n]);  // op_vec_add_bias (op_elementwise.cpp:8-11)
        if (n < a.n0) a.out0[(size_t)row * a.n0 + n] = v;
        else if (n < a.n0 + a.n1) a.out1[(size_t)row * a.n1 + (n - a.n0)] = v;
        else a.out2[(size_t)row * (a.N - a.n0 - a.n1) + (n - a.n0 - a.n1)] = v;
    } else if (MODE == 1) {
        float* h = a.resid + (size_t)row * a.N + n;  // op_vec_add (op_elementwise.cpp:3-5)
        *h = __fadd_rn(*h, r);
    } else if (MODE == 2) {
        // op_silu (op_silu.cpp:4-7), then gate *= up, then f32_to_f16
        const float u = f16_round(acc2);
        const float sg = __fdiv_rn(r, __fadd_rn(1.0f, expf(-r)));
        a.out16[(size_t)row * a.N + n] = enc_f16_trunc(__fmul_rn(sg, u));
    } else {
        a.logits[(size_t)row * a.N + n] = r;
    }
}

}  // namespace kvattn
