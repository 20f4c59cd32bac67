// w4_internal.h -- the 4-bit projections' arguments and launch plan, shared by
// the kernels, the C ABI (step_ops.cu) and the model (qwen2_engine.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kvattn_internal.h"
#include "step_ops.h"

namespace kvattn {

// What x is: 16-bit codes of the operand type; fp32 kept whole (three bf16
// parts); the model's fp32 rows rounded through the reference's fp16, plain or
// after an RMSNorm.
enum { W4_X_16 = 0, W4_X_F32 = 1, W4_X_ROUND = 2, W4_X_NORM = 3 };
// Epilogues: the model's call sites (GemvArgs) and the public operators.
enum { W4_QKV = 0, W4_RESID = 1, W4_GATE_UP = 2, W4_LOGITS = 3, W4_LINEAR = 4, W4_GATED = 5 };

struct W4Args {
    const uint32_t* codes[2] = {};
    const __half* scales[2] = {};
    const uint8_t* zeros[2] = {};
    int N = 0, K = 0, M = 0;
    int T = 0, S = 0, Q = 0;  // tiles of 16 rows, spans of 128 inputs, groups per row
    const void* x = nullptr;
    long long ldx = 0;
    int in = W4_X_16, mode = W4_LINEAR;
    int pieces = 1;           // operand rows per x row (3 for W4_X_F32)
    void* work = nullptr;     // room for w4_split_bytes, or NULL
    int out_dtype = STEP_F32;
    const float* bias = nullptr;
    const void* residual = nullptr;
    long long ldr = 0;
    void* out = nullptr;
    long long ldo = 0;
    GemvArgs g;               // the model's epilogues and norm
    // the launch plan
    int rows = 0;             // x rows per pass
    int ks = 1, cs = 1;       // a tile's spans over ks warps and cs CTAs
    int chunk = 0;            // spans of x staged at a time
    int last_groups = 0;      // groups of a row's last span
    bool tma = false;         // (tcgen05 form) x comes by TMA
    bool early = false;       // the weights may be read before the previous kernel of the stream ends

    void set_matrix(int i, const w4_matrix& w) {
        codes[i] = static_cast<const uint32_t*>(w.codes);
        scales[i] = static_cast<const __half*>(w.scales);
        zeros[i] = static_cast<const uint8_t*>(w.zeros);
        N = w.n;
        K = w.k;
        T = (w.n + 15) / 16;
        S = (w.k + 127) / 128;
        Q = (w.k + w.group - 1) / w.group;
    }
};

constexpr int kSms = 148;
constexpr int kW4MaxSmem = 227 * 1024;
// Spans that a warp copies at a time (two such batches in shared memory).
constexpr int w4_batch(int nw, int nt) { return nw == 2 || nt >= 4 ? 2 : 4; }
// Floats of a warp's partial tile: 20 per column (16 rows, padded against bank
// conflicts), 4 more so that the warps' tiles start in different banks.
constexpr int w4_red_floats(int nw, int nt) { return nw * nt * 8 * 20 + 4; }

struct W4Plan {
    int nt, rows, passes, ks, cs, chunk, gx, smem;
};

inline W4Plan w4_plan(int M, int T, int S, int pieces, int nw, int sms) {
    W4Plan p{};
    const int nt_max = nw == 2 ? 4 : 8;
    const int most = nt_max * 8 / pieces;
    p.passes = (M + most - 1) / most;
    p.rows = (M + p.passes - 1) / p.passes;
    const int vr = p.rows * pieces;
    p.nt = vr <= 8 ? 1 : vr <= 16 ? 2 : vr <= 32 ? 4 : 8;
    // warps that share a tile's spans: as many as keep every warp of two
    // CTAs per SM busy, no more than there are spans
    const int share = std::max(1, std::min(S, sms * 16 / std::max(1, T * p.passes)));
    p.ks = share >= 8 ? 8 : share >= 4 ? 4 : share >= 2 ? 2 : 1;
    p.cs = share >= 64 ? 8 : share >= 32 ? 4 : share >= 16 ? 2 : 1;
    const int fixed = 8 * (2 * w4_batch(nw, p.nt) * nw * 1216 + w4_red_floats(nw, p.nt) * 4);
    const int spans = (S + p.cs - 1) / p.cs;
    // staged spans: all of the CTA's, or as many batches of its warps as fit
    const int fit = ((kW4MaxSmem - fixed) / (vr * 2) - 32) / 128;
    const int unit = w4_batch(nw, p.nt);
    while (p.ks > 1 && p.ks * unit > fit) p.ks /= 2;
    p.chunk = spans <= fit ? spans : fit / (p.ks * unit) * (p.ks * unit);
    p.smem = fixed + vr * (p.chunk * 128 + 32) * 2;
    const int groups = (T + 8 / p.ks - 1) / (8 / p.ks);
    const int per_sm = p.smem <= 113 * 1024 && p.nt * nw <= 2 ? 2 : 1;
    p.gx = std::min(groups, std::max(1, sms * per_sm / (p.passes * p.cs)));
    return p;
}

// The tcgen05 form's plan: tiles of 128 weight rows (64 of each matrix of a
// gated block) x nb operand rows of x.
struct W4TcPlan {
    int nb, rows, cs, gx, gy;
};

inline W4TcPlan w4_tc_plan(int M, int T, int S, int pieces, int nw) {
    W4TcPlan p{};
    p.nb = M * pieces <= 64 ? 64 : M * pieces <= 128 ? 128 : 256;
    p.rows = p.nb / pieces;
    p.gy = (M + p.rows - 1) / p.rows;
    const int per = nw == 2 ? 4 : 8;
    p.gx = (T + per - 1) / per;
    // CTAs that share a tile's inputs: as many as fit the SMs in clusters (which
    // do not cross a GPC: 16 of 8, 34 of 4, 72 of 2), with four spans or more each
    p.cs = 1;
    const int tiles = p.gx * p.gy;
    for (int c = 2, fit = 72; c <= 8; c *= 2, fit = c == 4 ? 34 : 16)
        if (tiles <= fit && S / c >= 4) p.cs = c;
    return p;
}

// Rows from which the tcgen05 form is the faster one: its tiles cost the same
// for one row as for 64, so it depends on how many of them there are.  Measured, us
// (w4_kernels.cu / tcgen05): 1536 x 8960, 16 rows 18 / 12, 12 rows 12.3 / 12.3;
// 8960 x 1536 gated, 24 rows 15.9 / 14, 16 rows 11.4 / 14; 151936 x 1536, 48 rows
// 158 / 138, 32 rows 103 / 137.
inline bool w4_use_tc(int M, int T, int pieces, int nw) {
    const int tiles = (T + 7) / 8 * nw, rows = M * pieces;
    return rows > (tiles <= kSms / 2 ? 14 : tiles <= kSms ? 20 : 40);
}

cudaError_t launch_w4(W4Args a, int group, bool bf, int nw, cudaStream_t st);
// The three bf16 parts of fp32 rows, for the tcgen05 form: [3 M][K rounded up to 8].
inline size_t w4_split_bytes(int M, int K) { return (size_t)3 * M * ((K + 7) / 8 * 8) * 2; }
cudaError_t launch_split_rows(const float* x, long long ldx, int M, int K, void* parts, cudaStream_t st);
cudaError_t launch_w4_tc(W4Args a, int group, bool bf, int nw, cudaStream_t st);
// The status of the waits in launch_w4_tc's kernels on the current device
// (0, or KV_ERR_TIMEOUT), cleared by reading it.
cudaError_t step_status(int* status);
cudaError_t launch_w4_quantize(const w4_matrix& m, const void* w, int dtype, long long ldw, cudaStream_t st);
cudaError_t launch_w4_dequantize(const w4_matrix& m, float* out, long long ldo, cudaStream_t st);
cudaError_t launch_logits(const logits_call& c, cudaStream_t st);

}  // namespace kvattn
