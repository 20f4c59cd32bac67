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

// Spans that a warp copies at a time, and how many such batches it has
// room for.  Measured, us with 4 x 2 / 2 x 4: 151936 x 1536, one row 29.5 / 33.2 (fewer, larger
// batches pay for less pointer arithmetic); two matrices with 2 x 2 / 1 x 4: 8960 x 1536 in
// groups of 32, 8 rows 9.9 / 8.9.
constexpr int w4_batch(int nw) { return nw == 2 ? 1 : 4; }
constexpr int w4_ring(int nw) { return nw == 2 ? 4 : 2; }
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
    void* work = nullptr;     // room for w4_rows_bytes, or NULL
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
    int batches = 2;    // of codes per warp in shared memory
    int last_groups = 0;      // groups of a row's last span
    int* status = nullptr;    // where a wait of the tcgen05 form that runs out is noted: a pool's status words, or NULL, the public calls'
    long long wait_limit = 0; // SM clocks; 0: what is not ready has run out
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

// The part that the plans below are made for.  On fewer SMs their grids run in
// more turns than planned: slower, and nothing else, as a CTA waits for none but its cluster's.
constexpr int kSms = 148;
constexpr long long kW4WaitLimit = 2000000000LL;  // SM clocks: about a second
constexpr int kW4MaxSmem = 227 * 1024;
// Floats of a warp's partial tile: 20 per column (16 rows, padded against bank
// conflicts), 4 more so that the warps' tiles start in different banks.
constexpr int w4_red_floats(int nw, int nt) { return nw * nt * 8 * 20 + 4; }

struct W4Plan {
    int nt, rows, passes, ks, cs, chunk, batches, gx, smem;
};

// How a product is laid out: x rows per pass; the warps that share a tile's
// spans (ks), by the least
//   tiles in turn * (a warp's spans + 2 for joining the parts),
// where a last turn that fills part of the SMs counts half of itself at least; and
// the CTAs that share them (cs) where tiles are few, as long as all run at once.
// Measured, us at ks = 1 / 2 / 4 / 8: 2048 x 1536, one row 5.9 / 4.7 / 3.9 / 3.6; gated 8960 x
// 1536, one row 9.7 / 8.9 / 6.5 / 8.1, 16 rows 13.7 / 10.8 / 11.6 / 12.9; 20000 x 4096, one row
// 18.1 / 15.3 / 14.5 / 16.3; 151936 x 1536, one row 29.5 / 36 / 44 / 67.  Clusters in several
// waves lost: 1536 x 8960, one row 6.1 us without, 9.0 in threes, 21 in sixes.
inline W4Plan w4_plan(int M, int T, int S, int pieces, int nw, int sms) {
    W4Plan best{};
    const int most = 32 / pieces;
    const int passes = (M + most - 1) / most, rows = (M + passes - 1) / passes, vr = rows * pieces;
    const int nt = vr <= 8 ? 1 : vr <= 16 ? 2 : 4;
    const int unit = w4_batch(nw), batch = unit * nw * 1216, red = 8 * w4_red_floats(nw, nt) * 4;
    const int fit = ((kW4MaxSmem - red - 8 * w4_ring(nw) * batch) / (vr * 2) - 32) / 128;  // spans of x that fit at once
    double least = 0;
    for (int ks = 1; ks <= 8 && ks <= S; ks *= 2) {
        W4Plan p{nt, rows, passes, ks, 1};
        const int groups = (T + 8 / ks - 1) / (8 / ks);
        if (ks == 8)
            while (p.cs < 8 && groups * passes * p.cs * 2 <= sms && S >= 8 * p.cs * 2 * 2) p.cs *= 2;
        const int spans = (S + p.cs - 1) / p.cs, per_warp = (spans + ks - 1) / ks;
        if (fit < ks * unit && fit < spans) continue;
        // all of the CTA's spans, or as many batches of its warps as fit
        p.chunk = spans <= fit ? spans : fit / (ks * unit) * (ks * unit);
        const int fixed = red + vr * (p.chunk * 128 + 32) * 2;
        const int own = (per_warp + unit - 1) / unit;  // a tile's batches: no more room than that where there is one tile
        double turns = 0;
        for (p.batches = std::min(own, w4_ring(nw));; p.batches = w4_ring(nw)) {
            p.smem = fixed + 8 * p.batches * batch;
            const int per_sm = p.smem <= 113 * 1024 && nt * nw <= 2 ? 2 : 1;
            const int slots = std::max(1, sms * per_sm / (passes * p.cs));
            p.gx = std::min(groups, slots);
            turns = (double)groups / slots;
            if (turns <= 1 || p.batches == w4_ring(nw)) break;
        }
        const double whole = (double)(long long)turns, part = turns - whole;
        const double cost = std::max(1.0, whole + (part > 0 ? 0.5 + 0.5 * part : 0)) * (per_warp + 2);
        if (least == 0 || cost < least) least = cost, best = p;
    }
    return best;
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
// for one row as for 64, somewhat more with small groups (each is scaled by
// itself), and the other form suffers from long rows, of which it keeps every
// staged x.  Measured, us (w4_kernels.cu / tcgen05): 1536 x 8960, 16 rows 18 / 12,
// 8 rows 7.8 / 12; 2048 x 1536, 48 rows 11.1 / 10.5, 32 rows 6.3 / 9.7; 8960 x 1536
// gated, 24 rows 15.9 / 13.4, 16 rows 10.6 / 13.3; the same in groups of 32, 48 rows
// 30.5 / 19.5, 32 rows 18.9 / 19.3; 151936 x 1536, 48 rows 158 / 127, 32 rows 96 / 125.
// The parts of an fp32 x take a launch of their own first, so they need five rows
// (15 of parts): 4 and 5 rows of fp32, 1536 x 8960 16.6 / 13.5 and 25.1 / 13.5, 4096 x 4096
// 10.2 / 12.3 and 14.0 / 12.4, gated 13.6 / 20.0 and 16.8 / 20.0, 1536 x 8960 gated in groups of
// 32 22.3 / 28.7 and 31.2 / 28.7.
inline bool w4_use_tc(int M, int T, int S, int pieces, int nw, int group) {
    const int tiles = (T + 7) / 8 * nw, rows = M * pieces;
    if (tiles <= kSms && S >= 32) return rows > (pieces == 3 ? 14 : group == 32 ? 10 : 8);
    if (tiles <= kSms && nw == 2) return rows > (group == 32 ? 32 : 20);
    return rows > 40;
}
// Rows of 16-bit values that a tensor map can describe.
inline bool w4_tma_rows(const void* x, long long ldx) {
    return reinterpret_cast<size_t>(x) % 16 == 0 && ldx % 8 == 0 && ldx < 1ll << 38;
}

cudaError_t launch_w4(W4Args a, int group, bool bf, int nw, cudaStream_t st);
// Rows of x made for the tcgen05 form: an fp32 row's three bf16 parts, or a 16-bit row
// as it is, K rounded up to 8 elements each.
inline size_t w4_rows_bytes(int M, int K, int pieces) { return (size_t)pieces * M * ((K + 7) / 8 * 8) * 2; }
cudaError_t launch_rows(bool f32, const void* x, long long ldx, int M, int K, void* to, cudaStream_t st);
cudaError_t launch_w4_tc(W4Args a, int group, bool bf, int nw, cudaStream_t st);
// The limit of the waits in launch_w4_tc's kernels from now on (< 0: kW4WaitLimit).
void set_wait_limit(long long clocks);
// The status of those waits in the public calls' launches on the current
// device (0, or KV_ERR_TIMEOUT), cleared by reading it.
cudaError_t step_status(int* status);
cudaError_t launch_w4_quantize(const w4_matrix& m, const void* w, int dtype, long long ldw, cudaStream_t st);
cudaError_t launch_w4_dequantize(const w4_matrix& m, float* out, long long ldo, cudaStream_t st);
cudaError_t launch_logits(const logits_call& c, cudaStream_t st);

}  // namespace kvattn
