// w4_kernels.cu -- projections with 4-bit weights (w4_matrix of step_ops.h):
// the product, the gated feed-forward block on two of them, and the kernels
// that bring a matrix to 4 bits and back.
//
// Product: y^T = W x^T as mma.sync m16n8k16 tiles, W the A operand (16 weight
// rows x 16 inputs), up to 32 rows of x the B operand.  With
//   y[m][n] = sum_g s[n][g] * (sum_{k in g} (q[n][k] - z[n][g]) x[m][k])
// the integers q - z are exact in fp16 and in bf16, so the tensor core sums
// exact products in fp32 within a group, and the group's scale multiplies
// the fp32 sum: no weight is ever rounded.  What x is, is the only choice of
// the operand type: fp16 as fp16, bf16 as bf16, and an fp32 row as three
// bf16 rows (its first, second and third 8 significant bits) whose products
// are added at the end, so one fp32 row costs no more than three of the 8
// columns that a tile has anyway.
//
// A nibble becomes an operand without a conversion: or-ed under the exponent
// of 1024 (fp16; 128 for bf16) it is 1024 + q, from which 1024 + z is
// subtracted exactly; the nibble above it is 1024 + 16 q, brought back by one
// fused multiply-add.  Two weights per instruction.
//
// Bound: the codes' bytes for few rows.  Each lane copies the 32 bytes of
// codes that it will unpack itself to its own slots of a ring in shared memory
// (cp.async, batches of spans ahead, across tiles), so loads never wait for the
// math and need no barrier; a warp's 16 rows x 128 inputs are one contiguous
// KiB in memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_common.cuh"
#include "kvattn.h"
#include "kvattn_internal.h"
#include "projection.cuh"
#include "step_ops.h"
#include "w4_device.cuh"
#include "w4_internal.h"

namespace kvattn {

namespace {

constexpr int kWarps = 8;
constexpr int kSlot = 1024 + 128 + 64;  // a span of one tile: codes, up to 4 groups' scales and zero points
constexpr int kRedLd = 20;              // floats per column of a reduced tile: 16 rows, padded against bank conflicts

// ------------------------------------------------------------------ products
// mma16816 into fresh sums.
template <int BF>
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// The x rows of a pass, inputs [k0, k0 + len) (len a multiple of 128; zeros
// from K on), staged into xs as operand codes by the whole CTA: row m at m *
// pieces * ld halves, an fp32 row as its three parts `ld` apart.  8 / mrows
// warps share a row; a warp's loads of a batch are all issued before any is
// used, and 16-bit rows go by cp.async (the caller waits).  `wide`: rows of x
// are 16-byte aligned.
__device__ __forceinline__ void stage_rows(const W4Args& a, int m0, int mrows, int k0, int len, uint16_t* xs, int ld,
                                           bool wide) {
    constexpr int kU = 4;  // 16-byte loads in flight per lane
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = a.K;
    const int wpr = mrows > 4 ? 1 : mrows > 2 ? 2 : mrows > 1 ? 4 : 8;
    const int first = (warp % wpr) * 32 + lane, step = wpr * 32;
    for (int m = warp / wpr; m < mrows; m += kWarps / wpr) {
        if (a.in == W4_X_16) {
            const uint16_t* src = static_cast<const uint16_t*>(a.x) + (size_t)(m0 + m) * a.ldx + k0;
            uint16_t* dst = xs + (size_t)m * ld;
            for (int i = first * 8; i < len; i += step * 8) {
                if (wide && k0 + i + 8 <= K) {
                    cp16(smem_u32(dst + i), src + i);
                } else {
                    uint32_t h[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = k0 + i + j < K ? (uint32_t)__ldg(src + i + j) : 0u;
                    *reinterpret_cast<uint4*>(dst + i) =
                        make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                }
            }
            continue;
        }
        const float* xr = static_cast<const float*>(a.x) + (size_t)(m0 + m) * a.ldx;
        uint16_t* dst = xs + (size_t)m * a.pieces * ld;
        float inv = 1.f;
        if (a.in == W4_X_NORM) {
            // 1 / rms of the whole row (op_rmsnorm.cpp:12-15), by each of its warps
            float s = 0.f;
            for (int i = lane * 4; i < K; i += 128 * 6) {
                float4 v[6];
#pragma unroll
                for (int u = 0; u < 6; ++u)
                    if (i + u * 128 < K) v[u] = __ldg(reinterpret_cast<const float4*>(xr + i + u * 128));
#pragma unroll
                for (int u = 0; u < 6; ++u)
                    if (i + u * 128 < K) s = sum_sq4(s, v[u]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(s, (float)K), a.g.eps)));
        }
        for (int i0 = first * 4; i0 < len; i0 += step * 4 * kU) {
            float4 f[kU], nw[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int i = i0 + u * step * 4;
                f[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < len) {
                    const int k = k0 + i;
                    if (wide && k + 4 <= K) {
                        f[u] = __ldg(reinterpret_cast<const float4*>(xr + k));
                        if (a.in == W4_X_NORM) nw[u] = __ldg(reinterpret_cast<const float4*>(a.g.norm_w + k));
                    } else {  // the model's rows are always wide and whole
                        if (k < K) f[u].x = __ldg(xr + k);
                        if (k + 1 < K) f[u].y = __ldg(xr + k + 1);
                        if (k + 2 < K) f[u].z = __ldg(xr + k + 2);
                        if (k + 3 < K) f[u].w = __ldg(xr + k + 3);
                        nw[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int i = i0 + u * step * 4;
                if (i >= len) break;
                float v[4] = {f[u].x, f[u].y, f[u].z, f[u].w};
                if (a.in == W4_X_F32) {
                    uint16_t p[3][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split3(v[j], p[0][j], p[1][j], p[2][j]);
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        *reinterpret_cast<uint2*>(dst + q * ld + i) =
                            make_uint2(p[q][0] | (uint32_t)p[q][1] << 16, p[q][2] | (uint32_t)p[q][3] << 16);
                } else {
                    // the reference's fp16 (f32_to_f16 before every projection),
                    // after the norm (op_rmsnorm.cpp:17-18) where there is one
                    if (a.in == W4_X_NORM) {
                        const float w[4] = {nw[u].x, nw[u].y, nw[u].z, nw[u].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] = __fmul_rn(__fmul_rn(v[j], inv), w[j]);
                    }
                    *reinterpret_cast<uint2*>(dst + i) =
                        make_uint2(enc_f16_trunc(v[0]) | (uint32_t)enc_f16_trunc(v[1]) << 16,
                                   enc_f16_trunc(v[2]) | (uint32_t)enc_f16_trunc(v[3]) << 16);
                }
            }
        }
    }
}

// BF: bf16 operands (else fp16).  NT: n8 tiles of x rows per pass.  NW: 2 for
// the gated block.  GP: groups per span (1, 2 or 4).
//
// Work: CTA b of gx (cluster rank r of cs, pass blockIdx.y) takes the tiles
// (i kWarps / ks + w / ks) gx + b, i = 0, 1, .., of its warps w, and of those
// the spans [S r / cs, S (r + 1) / cs), warp w every ks-th from w % ks on.  So
// what does not divide evenly is spread over different SMs.  The partial
// tiles of ks warps and cs CTAs are added in a fixed order (shared memory,
// other CTAs' by DSMEM): results do not depend on timing.  With ks = cs = 1
// warps never wait for one another.
template <int BF, int NT, int NW, int GP>
__global__ void __launch_bounds__(kWarps * 32, NT * NW <= 2 ? 2 : 1)
    w4_kernel(const __grid_constant__ W4Args a) {
    constexpr int kRing = w4_ring(NW);
    constexpr int kU = w4_batch(NW);         // spans per batch
    constexpr int kBatch = kU * NW * kSlot;  // bytes; kRing batches per warp, one in use, the others in flight
    constexpr int kCols = NT * 8;
    constexpr int kRedWarp = w4_red_floats(NW, NT);
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int ks = a.ks, tpc = kWarps / ks, sub = warp / ks, part = warp % ks;
    const int cs = a.cs, rank = (int)blockIdx.x % cs;
    const int bx = (int)blockIdx.x / cs, gx = (int)gridDim.x / cs;
    const int m0 = blockIdx.y * a.rows, mrows = min(a.rows, a.M - m0), vr = mrows * a.pieces;
    const int ldx = a.chunk * 128 + 32;  // halves per staged row: an odd number of 64-byte units
    uint16_t* xs = reinterpret_cast<uint16_t*>(smem);
    uint8_t* ring = smem + (size_t)a.rows * a.pieces * ldx * 2 + (size_t)warp * (a.batches * kBatch);
    float* red = reinterpret_cast<float*>(smem + (size_t)a.rows * a.pieces * ldx * 2 + (size_t)kWarps * a.batches * kBatch);

    const int s0 = (int)((long long)a.S * rank / cs), s1 = (int)((long long)a.S * (rank + 1) / cs);
    const int rounds = (a.T + tpc * gx - 1) / (tpc * gx);
    const int nmax = (s1 - s0 + ks - 1) / ks;                               // spans per warp, at most
    const int nmine = s0 + part < s1 ? (s1 - s0 - part + ks - 1) / ks : 0;  // this warp's
    const int tile0 = sub * gx + bx, tstep = tpc * gx;

    // The warp's (tile, span) sequence, kRing - 1 batches ahead of the math: pointers that
    // advance by constants; a batch ends with its tile.
    int ptiles = nmine > 0 && tile0 < a.T ? (a.T - tile0 + tstep - 1) / tstep : 0, pleft = nmine;
    int pgroup = (s0 + part) * GP;  // the next span's first group
    const uint8_t *pc[NW], *ps[NW], *pz[NW];
#pragma unroll
    for (int q = 0; q < NW; ++q) {
        pc[q] = reinterpret_cast<const uint8_t*>(a.codes[q]) + ((size_t)tile0 * a.S + s0 + part) * 1024 + lane * 16;
        ps[q] = reinterpret_cast<const uint8_t*>(a.scales[q]) + ((size_t)tile0 * a.Q + pgroup) * 32 + lane * 4;
        pz[q] = a.zeros[q] ? a.zeros[q] + ((size_t)tile0 * a.Q + pgroup) * 16 + lane * 4 : nullptr;
    }
    const size_t cjump = ((size_t)tstep * a.S - (size_t)nmine * ks) * 1024;
    const long long gjump = (long long)tstep * a.Q - (long long)nmine * ks * GP;
    const uint32_t ring_s = smem_u32(ring);
    uint32_t poff = 0;
    auto issue = [&]() {
        if (ptiles > 0) {
            const int n = min(kU, pleft);
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (u >= n) break;
#pragma unroll
                for (int q = 0; q < NW; ++q) {
                    const uint32_t dst = ring_s + poff + (u * NW + q) * kSlot;
                    cp16(dst + lane * 16, pc[q]);
                    cp16(dst + 512 + lane * 16, pc[q] + 512);
                    // 32 bytes of scales and 16 of zero points per group; a row's last span may have fewer groups
                    if (lane < GP * 8 && (GP == 1 || pgroup + (lane >> 3) < a.Q)) cp4(dst + 1024 + lane * 4, ps[q]);
                    if (pz[q] && lane < GP * 4 && (GP == 1 || pgroup + (lane >> 2) < a.Q)) cp4(dst + 1152 + lane * 4, pz[q]);
                    pc[q] += ks * 1024;
                    ps[q] += ks * GP * 32;
                    if (pz[q]) pz[q] += ks * GP * 16;
                }
                pgroup += ks * GP;
            }
            pleft -= n;
            if (pleft == 0) {
                pleft = nmine;
                --ptiles;
                pgroup -= nmine * ks * GP;
#pragma unroll
                for (int q = 0; q < NW; ++q) {
                    pc[q] += cjump;
                    ps[q] += gjump * 32;
                    if (pz[q]) pz[q] += gjump * 16;
                }
            }
        }
        cp_commit();
        poff = poff == (kRing - 1) * kBatch ? 0 : poff + kBatch;
    };

    // In the model's chain (a.early) the weights, which no kernel of the chain
    // writes, are fetched before the wait for the previous kernel.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!a.early) asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) issue();
    if (a.early) asm volatile("griddepcontrol.wait;" ::: "memory");

    const bool wide = (reinterpret_cast<size_t>(a.x) & 15) == 0 && (a.ldx * (a.in == W4_X_16 ? 2 : 4)) % 16 == 0;
    const int chunks = (s1 - s0 + a.chunk - 1) / a.chunk;
    auto stage_chunk = [&](int ch) {
        const int b = s0 + ch * a.chunk, e = min(b + a.chunk, s1);
        stage_rows(a, m0, mrows, b * 128, (e - b) * 128, xs, ldx, wide);
        cp_commit();
        cp_wait<0>();
    };
    const int per_chunk = a.chunk / ks;  // a warp's spans per staged chunk (whole batches, or chunk holds every span)
    if (chunks == 1) {
        stage_chunk(0);
        __syncthreads();
    }

    uint32_t slot = 0;
    uint2 zl[NW], zh[NW];  // zero points of rows g and g + 8
#pragma unroll
    for (int q = 0; q < NW; ++q) zl[q] = zh[q] = zero_consts<BF>(8u);
    int xrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xrow[t] = min(t * 8 + g, vr - 1) * ldx;
#pragma unroll 1
    for (int rd = 0; rd < rounds; ++rd) {
        const int tile = tile0 + rd * tstep;
        const bool live = tile < a.T;
        float acc[NW][NT][4];
#pragma unroll
        for (int q = 0; q < NW; ++q)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[q][t][0] = acc[q][t][1] = acc[q][t][2] = acc[q][t][3] = 0.f;
        const uint16_t* xp = xs + part * 128 + 8 * c;
        int left = s1 - s0 - part;  // spans from this one to the range's end
#pragma unroll 1
        for (int it = 0; it < nmax; it += kU) {
            if (chunks > 1 && it % per_chunk == 0) {
                __syncthreads();
                stage_chunk(it / per_chunk);
                __syncthreads();
                xp = xs + part * 128 + 8 * c;
            }
            if (it >= nmine || !live) continue;
            cp_wait<kRing - 2>();
            __syncwarp();  // scales came by other lanes; the batch refilled next was read by all of them
            issue();
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (it + u >= nmine) break;
                const uint8_t* const sl0 = ring + slot + u * NW * kSlot;
                uint32_t lo[NW][4], hi[NW][4];  // codes of rows g and g + 8, 8 inputs a word
#pragma unroll
                for (int q = 0; q < NW; ++q) {
                    const uint8_t* sl = sl0 + q * kSlot + lane * 16;
                    const uint4 a4 = *reinterpret_cast<const uint4*>(sl), b4 = *reinterpret_cast<const uint4*>(sl + 512);
                    lo[q][0] = a4.x, lo[q][1] = a4.y, lo[q][2] = a4.z, lo[q][3] = a4.w;
                    hi[q][0] = b4.x, hi[q][1] = b4.y, hi[q][2] = b4.z, hi[q][3] = b4.w;
                }
                float d[NW][NT][4];  // this group's sums
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t p[NW][4], r[NW][4];
#pragma unroll
                    for (int q = 0; q < NW; ++q) {
                        if (j % (4 / GP) == 0 && a.zeros[q]) {
                            const uint32_t z = *reinterpret_cast<const uint16_t*>(sl0 + q * kSlot + 1152 + j / (4 / GP) * 16 + g * 2);
                            zl[q] = zero_consts<BF>(z & 15u);
                            zh[q] = zero_consts<BF>((z >> 8) & 15u);
                        }
                        unpack<BF>(lo[q][j], zl[q], p[q]);
                        unpack<BF>(hi[q][j], zh[q], r[q]);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        // columns from vr on hold some row's values and are not read
                        const uint4 b = *reinterpret_cast<const uint4*>(xp + xrow[t] + 32 * j);
#pragma unroll
                        for (int q = 0; q < NW; ++q) {
                            if (j % (4 / GP) == 0) mma16816_first<BF>(d[q][t], p[q][0], r[q][0], p[q][1], r[q][1], b.x, b.y);
                            else mma16816<BF>(d[q][t], p[q][0], r[q][0], p[q][1], r[q][1], b.x, b.y);
                            mma16816<BF>(d[q][t], p[q][2], r[q][2], p[q][3], r[q][3], b.z, b.w);
                        }
                    }
                    if ((j + 1) % (4 / GP) == 0) {
                        const int gq = j / (4 / GP);
                        // a group that the row does not have: its x is zero, its slot's old bytes may be anything
                        const bool none = GP > 1 && gq > 0 && left == 1 && s1 == a.S && gq >= a.last_groups;
#pragma unroll
                        for (int q = 0; q < NW; ++q) {
                            float2 sc = __half22float2(*reinterpret_cast<const __half2*>(sl0 + q * kSlot + 1024 + gq * 32 + g * 4));
                            if (none) sc = make_float2(0.f, 0.f);
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                acc[q][t][0] = fmaf(sc.x, d[q][t][0], acc[q][t][0]);
                                acc[q][t][1] = fmaf(sc.x, d[q][t][1], acc[q][t][1]);
                                acc[q][t][2] = fmaf(sc.y, d[q][t][2], acc[q][t][2]);
                                acc[q][t][3] = fmaf(sc.y, d[q][t][3], acc[q][t][3]);
                            }
                        }
                    }
                }
                xp += ks * 128;
                left -= ks;
            }
            slot = slot == (kRing - 1) * kBatch ? 0 : slot + kBatch;
        }
        // partial tiles of this warp: [matrix][column][row]
        if (live) {
#pragma unroll
            for (int q = 0; q < NW; ++q)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        red[warp * kRedWarp + (q * kCols + t * 8 + 2 * c + (i & 1)) * kRedLd + g + (i >> 1) * 8] = acc[q][t][i];
        }
        if (ks == 1 && cs == 1) {
            __syncwarp();
            if (live) {
                for (int e = lane; e < 16 * mrows; e += 32) {
                    const int n = tile * 16 + (e & 15), m = e >> 4;
                    if (n >= a.N) continue;
                    float y[2] = {0.f, 0.f};
#pragma unroll
                    for (int q = 0; q < NW; ++q) {
                        const float* at = red + warp * kRedWarp + (q * kCols + m * a.pieces) * kRedLd + (e & 15);
                        for (int p = a.pieces - 1; p >= 0; --p) y[q] += at[p * kRedLd];  // the smallest parts first
                    }
                    w4_epilogue(a, m0 + m, n, y[0], y[1]);
                }
            }
            __syncwarp();
            continue;
        }
        if (cs > 1) cluster_sync();
        else __syncthreads();
        const int lone = tpc * mrows * 16 * ks <= kWarps * 32 ? ks : 1;  // lanes that share an output: its parts, where that fits
        const int per = lone > 1 ? 1 : ks;                               // parts per lane
        const int lu = threadIdx.x % lone, e0 = threadIdx.x / lone, n16 = e0 & 15, mstep = lone > 1 ? mrows * tpc : kWarps * 2;
        for (int i = (e0 >> 4) + rank * mstep; i - (e0 >> 4) < mrows * tpc; i += cs * mstep) {
            const int ts = mrows == 1 ? i : i / mrows, m = i - ts * mrows;
            const bool some = ts < tpc;
            float y[2] = {0.f, 0.f};
            if (some) {
                for (int p = a.pieces - 1; p >= 0; --p)  // the smallest parts first
#pragma unroll
                    for (int q = 0; q < NW; ++q) {
                        const float* at = red + (ts * ks + lu) * kRedWarp + (q * kCols + m * a.pieces + p) * kRedLd + n16;
                        for (int r = 0; r < cs; ++r) {
                            const uint32_t far = cs > 1 ? cluster_map(smem_u32(at), r) : 0u;
                            float v[kWarps];
#pragma unroll
                            for (int u = 0; u < kWarps; ++u)
                                v[u] = u >= per ? 0.f : cs > 1 ? ld_cluster_f32(far + u * kRedWarp * 4) : at[u * kRedWarp];
#pragma unroll
                            for (int u = 0; u < kWarps; ++u) y[q] += v[u];
                        }
                    }
            }
            for (int o = 1; o < lone; o <<= 1)
#pragma unroll
                for (int q = 0; q < NW; ++q) y[q] += __shfl_xor_sync(0xffffffffu, y[q], o);
            const int n = (bx + (ts + rd * tpc) * gx) * 16 + n16;
            if (some && lu == 0 && n < a.N) w4_epilogue(a, m0 + m, n, y[0], y[1]);
        }
        if (cs > 1) cluster_sync();  // red is written again, or this CTA ends, only when nobody reads it
        else __syncthreads();
    }
    cp_wait<0>();
}

// ------------------------------------------------------- to 4 bits and back
// One warp per (tile, span), row by row: lane l holds inputs 4 l .. 4 l + 3, so
// a row's 128 inputs are one contiguous access and half a code word is a
// lane's own.  The 16 rows' loads are issued together, in units of W bytes,
// the widest that the addresses allow.  Group statistics are maxima, exact in
// any order.  Bound: the bytes of the 16- or 32-bit side.
template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <int W>
struct Unit;
template <>
struct Unit<16> { using type = uint4; };
template <>
struct Unit<8> { using type = uint2; };
template <>
struct Unit<4> { using type = uint32_t; };
template <>
struct Unit<2> { using type = uint16_t; };

// rint(v / s), v and s of at most 11 significant bits, inv = 1 / s correctly
// rounded: one correction by the exact residual leaves the quotient within an
// ulp, and exact where fp32 holds it (ties among those); no other quotient of
// such values is nearer than 2^-13 to a half.  Adding 1.5 * 2^23 rounds it
// to a whole number, ties to even, in the low bits.
__device__ __forceinline__ int round_quotient(float v, float s, float inv) {
    const float q = v * inv;
    const float r = fmaf(fmaf(-q, s, v), inv, q);
    return __float_as_int(__fadd_rn(r, 12582912.f)) - 0x4B400000;
}

template <class T, int W, int GL /* lanes per group */, bool ZP>
__global__ void __launch_bounds__(256)
    w4_quantize_kernel(const T* __restrict__ w, long long ldw, int N, int K, int S, int Q,
                       uint32_t* __restrict__ codes, __half* __restrict__ scales, uint8_t* __restrict__ zeros) {
    using U = typename Unit<W>::type;
    constexpr int kE = W / 2;  // elements per unit
    const int lane = threadIdx.x & 31;
    const int s = blockIdx.x * 8 + (threadIdx.x >> 5), t = blockIdx.y;
    if (s >= S) return;
    const int k0 = s * 128 + lane * 4;
    union Four {
        U u[4 / kE];
        T e[4];
        uint2 bits;
    };
    Four v[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const T* row = w + (size_t)min(t * 16 + r, N - 1) * ldw + k0;
        v[r].bits = make_uint2(0u, 0u);
#pragma unroll
        for (int i = 0; i < 4; i += kE) {
            if (k0 + i + kE <= K) {
                v[r].u[i / kE] = __ldg(reinterpret_cast<const U*>(row + i));
            } else {
#pragma unroll
                for (int ii = 0; ii < kE; ++ii)
                    if (k0 + i + ii < K) v[r].e[i + ii] = row[i + ii];
            }
        }
    }
    const int gi = s * (32 / GL) + lane / GL;
    // The 16 rows' extremes over the GL lanes of a group together: at each step a
    // lane hands half of its rows to its partner and takes the partner's other
    // half, so each lane ends with kRows rows' (16 / GL, or one) and makes their
    // scales, which come back by shuffles: no lane repeats another's division.
    constexpr int kRows = GL >= 16 ? 1 : 16 / GL;
    const int li = lane % GL;
    auto reduce = [&](float (&x)[16]) {
#pragma unroll
        for (int o = 1, n = 8; o < GL; o <<= 1, n >>= 1) {
            if (n >= 1) {
                const bool up = li & o;
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < n) {
                        const float mine = up ? x[r + n] : x[r], other = up ? x[r] : x[r + n];
                        x[r] = fmaxf(mine, __shfl_xor_sync(0xffffffffu, other, o));
                    }
            } else {
                x[0] = fmaxf(x[0], __shfl_xor_sync(0xffffffffu, x[0], o));
            }
        }
    };
    float top[16], neg[16];  // max w (max |w| without zero points), max -w
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float f0 = to_f(v[r].e[0]), f1 = to_f(v[r].e[1]), f2 = to_f(v[r].e[2]), f3 = to_f(v[r].e[3]);
        if (ZP) {
            top[r] = fmaxf(fmaxf(fmaxf(f0, f1), fmaxf(f2, f3)), 0.f);
            neg[r] = fmaxf(-fminf(fminf(f0, f1), fminf(f2, f3)), 0.f);
        } else {
            top[r] = fmaxf(fmaxf(fabsf(f0), fabsf(f1)), fmaxf(fabsf(f2), fabsf(f3)));
        }
    }
    reduce(top);
    if (ZP) reduce(neg);
    // this lane's rows: bit i of li decided bit 3 - i of the row
    const int row0 = (li & 1) << 3 | (li & 2) << 1 | (GL > 4 ? (li & 4) >> 1 : 0) | (GL > 8 ? (li & 8) >> 3 : 0);
    float sc[kRows], inv[kRows];
    int zi[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const __half sh = __float2half_rn(ZP ? __fdiv_rn(__fadd_rn(top[r], neg[r]), 15.0f) : __fdiv_rn(top[r], 7.0f));
        sc[r] = __half2float(sh);
        zi[r] = ZP && sc[r] > 0.f ? (int)fminf(fmaxf(rintf(__fdiv_rn(neg[r], sc[r])), 0.f), 15.f) : 8;
        inv[r] = sc[r] > 0.f ? __frcp_rn(sc[r]) : 0.f;  // no scale: every code is the zero point
        const int row = row0 + r, h = row >> 3, g = row & 7;
        if (gi < Q && li < 16) {
            const size_t at = ((size_t)t * Q + gi) * 16 + g * 2 + h;
            scales[at] = sh;
            if (ZP) zeros[at] = (uint8_t)zi[r];
        }
    }
    uint32_t* word = codes + ((size_t)t * S + s) * 256 + ((lane >> 1) & 3) * 4 + (lane >> 3);  // + [h][4 g][.]
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int h = r >> 3, g = r & 7;
        // the lane of the group that has row r
        const int from = lane - li + ((r >> 3 & 1) | (r >> 2 & 1) << 1 | (GL > 4 ? (r >> 1 & 1) << 2 : 0) | (GL > 8 ? (r & 1) << 3 : 0));
        const float s_r = __shfl_sync(0xffffffffu, sc[r % kRows], from), i_r = __shfl_sync(0xffffffffu, inv[r % kRows], from);
        const int z_r = ZP ? __shfl_sync(0xffffffffu, zi[r % kRows], from) : 8;
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = i_r > 0.f ? to_f(v[r].e[i]) : 0.f;
            q[i] = (uint32_t)min(max(round_quotient(f, s_r, i_r) + z_r, 0), 15);
        }
        // inputs 0..3 of a word stand at 0, 4, 1, 5 (times four bits), 4..7 at 2, 6, 3, 7
        uint32_t part = q[0] | q[1] << 16 | q[2] << 4 | q[3] << 20;
        part = (lane & 1) ? part << 8 : part;
        part |= __shfl_xor_sync(0xffffffffu, part, 1);
        if (!(lane & 1)) word[h * 128 + g * 16] = part;
    }
}

// Lane l writes inputs (W / 4) l .. of each block of 8 W inputs.
template <int W>
__global__ void __launch_bounds__(256)
    w4_dequantize_kernel(const uint32_t* __restrict__ codes, const __half* __restrict__ scales,
                         const uint8_t* __restrict__ zeros, int N, int K, int S, int Q, int lg /* log2 group */,
                         float* __restrict__ out, long long ldo) {
    using U = typename Unit<W>::type;
    constexpr int kE = W / 4, kB = 4 / kE;  // values per unit, units per lane and row
    const int lane = threadIdx.x & 31;
    const int s = blockIdx.x * 8 + (threadIdx.x >> 5), t = blockIdx.y;
    if (s >= S) return;
    const uint32_t* span = codes + ((size_t)t * S + s) * 256;
#pragma unroll
    for (int b = 0; b < kB; ++b) {
        const int kk = b * 32 * kE + lane * kE, k = s * 128 + kk;  // inside the span, inside the row
        if (k >= K) continue;
        // the group's scales and zero points of all 16 rows
        const size_t at = ((size_t)t * Q + (k >> lg)) * 16;
        union {
            uint4 u[2];
            __half h[16];
        } sc;
        sc.u[0] = __ldg(reinterpret_cast<const uint4*>(scales + at));
        sc.u[1] = __ldg(reinterpret_cast<const uint4*>(scales + at) + 1);
        union {
            uint4 u;
            uint8_t b[16];
        } z;
        z.u = make_uint4(0x08080808u, 0x08080808u, 0x08080808u, 0x08080808u);
        if (zeros) z.u = __ldg(reinterpret_cast<const uint4*>(zeros + at));
        const uint32_t* word = span + ((kk >> 3) & 3) * 4 + (kk >> 5);
        float* to = out + (size_t)t * 16 * ldo + k;
        uint32_t all[16];  // every row's word before any is used
#pragma unroll
        for (int r = 0; r < 16; ++r) all[r] = __ldg(word + (r >> 3) * 128 + (r & 7) * 16);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (t * 16 + r >= N) break;
            const int h = r >> 3, g = r & 7;
            const uint32_t w = all[r];
            const float s_r = __half2float(sc.h[g * 2 + h]), z_r = 8388608.f + (float)(z.b[g * 2 + h] & 15);
            union {
                U u;
                float f[kE];
            } v;
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                const int ii = (kk & 7) + i;
                // 2^23 + code, exactly, then the code less its zero point
                v.f[i] = (__uint_as_float((w >> (4 * ((ii >> 1) + 4 * (ii & 1)))) & 15u | 0x4B000000u) - z_r) * s_r;
            }
            if (k + kE <= K) {
                *reinterpret_cast<U*>(to + (size_t)r * ldo) = v.u;
            } else {
#pragma unroll
                for (int i = 0; i < kE; ++i)
                    if (k + i < K) to[(size_t)r * ldo + i] = v.f[i];
            }
        }
    }
}

// ------------------------------------------------------------------ launching
template <int BF, int NT, int NW, int GP>
cudaError_t launch_inst(const W4Args& a, int gx, int passes, int smem, cudaStream_t st) {
    auto fn = w4_kernel<BF, NT, NW, GP>;
    static SmemGrant grant;
    cudaError_t e = grant.raise(reinterpret_cast<const void*>(fn), kW4MaxSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(gx * a.cs), (unsigned)passes);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (a.cs > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = (unsigned)a.cs;
        attr[na].val.clusterDim.y = 1;
        attr[na].val.clusterDim.z = 1;
        ++na;
    }
    // may start while the previous kernel of the stream ends: it waits for
    // that kernel before it reads anything (a.early: but weights)
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
    cfg.attrs = attr;
    cfg.numAttrs = na;
    return counted(cudaLaunchKernelEx(&cfg, fn, a));
}

template <int BF, int NT, int NW>
cudaError_t launch_gp(const W4Args& a, int group, int gx, int passes, int smem, cudaStream_t st) {
    if (group == 128) return launch_inst<BF, NT, NW, 1>(a, gx, passes, smem, st);
    if (group == 64) return launch_inst<BF, NT, NW, 2>(a, gx, passes, smem, st);
    return launch_inst<BF, NT, NW, 4>(a, gx, passes, smem, st);
}

template <int BF>
cudaError_t launch_nt(const W4Args& a, int nt, int nw, int group, int gx, int passes, int smem, cudaStream_t st) {
    if (nw == 2) {
        if (nt == 1) return launch_gp<BF, 1, 2>(a, group, gx, passes, smem, st);
        if (nt == 2) return launch_gp<BF, 2, 2>(a, group, gx, passes, smem, st);
        return launch_gp<BF, 4, 2>(a, group, gx, passes, smem, st);
    }
    if (nt == 1) return launch_gp<BF, 1, 1>(a, group, gx, passes, smem, st);
    if (nt == 2) return launch_gp<BF, 2, 1>(a, group, gx, passes, smem, st);
    return launch_gp<BF, 4, 1>(a, group, gx, passes, smem, st);
}

}  // namespace

cudaError_t launch_w4(W4Args a, int group, bool bf, int nw, cudaStream_t st) {
    if (w4_use_tc(a.M, a.T, a.S, a.pieces, nw, group)) {
        if (a.in == W4_X_16 && w4_tma_rows(a.x, a.ldx)) return launch_w4_tc(a, group, bf, nw, st);
        if ((a.in == W4_X_16 || a.in == W4_X_F32) && a.work) {
            const cudaError_t e = launch_rows(a.in == W4_X_F32, a.x, a.ldx, a.M, a.K, a.work, st);
            if (e != cudaSuccess) return e;
            a.x = a.work;
            a.ldx = (a.K + 7) / 8 * 8;
            a.in = W4_X_16;
            return launch_w4_tc(a, group, bf, nw, st);
        }
    }
    const W4Plan p = w4_plan(a.M, a.T, a.S, a.pieces, nw, kSms);
    a.batches = p.batches;
    a.rows = p.rows;
    a.ks = p.ks;
    a.cs = p.cs;
    a.chunk = p.chunk;
    a.last_groups = a.Q - (a.S - 1) * (128 / group);
    return bf ? launch_nt<1>(a, p.nt, nw, group, p.gx, p.passes, p.smem, st)
              : launch_nt<0>(a, p.nt, nw, group, p.gx, p.passes, p.smem, st);
}

namespace {

// The widest power of two up to `most` bytes that an address and a row stride share.
int unit_bytes(const void* p, long long ld_bytes, int most) {
    int w = most;
    while (reinterpret_cast<size_t>(p) % w || ld_bytes % w) w /= 2;
    return w;
}

template <class T, int W, int GL>
void quantize_zp(const w4_matrix& m, const void* w, long long ldw, dim3 grid, int S, int Q, int tile0, cudaStream_t st) {
    const T* src = static_cast<const T*>(w) + (size_t)tile0 * 16 * ldw;
    uint32_t* codes = static_cast<uint32_t*>(m.codes) + (size_t)tile0 * S * 256;
    __half* scales = static_cast<__half*>(m.scales) + (size_t)tile0 * Q * 16;
    uint8_t* zeros = static_cast<uint8_t*>(m.zeros);
    const int N = m.n - tile0 * 16;
    if (zeros)
        w4_quantize_kernel<T, W, GL, true><<<grid, 256, 0, st>>>(src, ldw, N, m.k, S, Q, codes, scales, zeros + (size_t)tile0 * Q * 16);
    else
        w4_quantize_kernel<T, W, GL, false><<<grid, 256, 0, st>>>(src, ldw, N, m.k, S, Q, codes, scales, nullptr);
}

template <class T, int W>
void quantize_group(const w4_matrix& m, const void* w, long long ldw, dim3 grid, int S, int Q, int tile0, cudaStream_t st) {
    if (m.group == 128) quantize_zp<T, W, 32>(m, w, ldw, grid, S, Q, tile0, st);
    else if (m.group == 64) quantize_zp<T, W, 16>(m, w, ldw, grid, S, Q, tile0, st);
    else quantize_zp<T, W, 8>(m, w, ldw, grid, S, Q, tile0, st);
}

template <class T>
void quantize_w(const w4_matrix& m, const void* w, long long ldw, dim3 grid, int S, int Q, int tile0, cudaStream_t st) {
    const int u = unit_bytes(w, ldw * 2, 8);
    if (u == 8) quantize_group<T, 8>(m, w, ldw, grid, S, Q, tile0, st);
    else if (u >= 4) quantize_group<T, 4>(m, w, ldw, grid, S, Q, tile0, st);
    else quantize_group<T, 2>(m, w, ldw, grid, S, Q, tile0, st);
}

constexpr int kMaxGridY = 65535;  // tiles per launch

}  // namespace

cudaError_t launch_w4_quantize(const w4_matrix& m, const void* w, int dtype, long long ldw, cudaStream_t st) {
    const int T = (m.n + 15) / 16, S = (m.k + 127) / 128, Q = (m.k + m.group - 1) / m.group;
    for (int t0 = 0; t0 < T; t0 += kMaxGridY) {
        const dim3 grid((unsigned)((S + 7) / 8), (unsigned)(T - t0 < kMaxGridY ? T - t0 : kMaxGridY));
        if (dtype == STEP_F16) quantize_w<__half>(m, w, ldw, grid, S, Q, t0, st);
        else quantize_w<__nv_bfloat16>(m, w, ldw, grid, S, Q, t0, st);
        const cudaError_t e = counted(cudaGetLastError());
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_w4_dequantize(const w4_matrix& m, float* out, long long ldo, cudaStream_t st) {
    const int T = (m.n + 15) / 16, S = (m.k + 127) / 128, Q = (m.k + m.group - 1) / m.group;
    const int lg = m.group == 128 ? 7 : m.group == 64 ? 6 : 5;
    const int u = unit_bytes(out, ldo * 4, 16);
    auto fn = u == 16 ? w4_dequantize_kernel<16> : u == 8 ? w4_dequantize_kernel<8> : w4_dequantize_kernel<4>;
    for (int t0 = 0; t0 < T; t0 += kMaxGridY) {
        const dim3 grid((unsigned)((S + 7) / 8), (unsigned)(T - t0 < kMaxGridY ? T - t0 : kMaxGridY));
        const uint8_t* zeros = static_cast<const uint8_t*>(m.zeros);
        fn<<<grid, 256, 0, st>>>(static_cast<const uint32_t*>(m.codes) + (size_t)t0 * S * 256,
                                 static_cast<const __half*>(m.scales) + (size_t)t0 * Q * 16,
                                 zeros ? zeros + (size_t)t0 * Q * 16 : nullptr, m.n - t0 * 16, m.k, S, Q, lg,
                                 out + (size_t)t0 * 16 * ldo, ldo);
        const cudaError_t e = counted(cudaGetLastError());
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace kvattn
